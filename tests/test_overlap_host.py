"""Whether two matrices share a byte, against sets of addresses; and what the serving operators refuse of it."""
import ctypes as C

import pytest

from conftest import compile_and_run
from test_serving_refusals_host import A, append, attend, read, refused, rules, struct

CHECK = r"""
#include "overlap.h"
#include <cstdio>
#include <random>
#include <set>
using namespace tb;

int main() {
    std::mt19937 rng(3);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    const char* base = reinterpret_cast<const char*>(1 << 20);
    int both[2] = {0, 0};
    for (int t = 0; t < 200000; ++t) {
        RowSpan s[2];
        std::set<long long> bytes[2];
        for (int i = 0; i < 2; ++i) {
            s[i].bytes = pick(1, 9); s[i].rows = pick(0, 5);
            s[i].pitch = t % 2 && i ? s[0].pitch : s[i].bytes + pick(0, 14);
            s[i].at = base + pick(0, 60);
            if (s[i].pitch < s[i].bytes) s[i].bytes = s[i].pitch;
            for (long long r = 0; r < s[i].rows; ++r)
                for (long long x = 0; x < s[i].bytes; ++x) bytes[i].insert((long long)((const char*)s[i].at - base) + r * s[i].pitch + x);
        }
        bool want = false;
        for (long long x : bytes[0]) want |= bytes[1].count(x) > 0;
        if (spans_overlap(s[0], s[1]) != want || spans_overlap(s[1], s[0]) != want) { printf("case %d\n", t); return 1; }
        ++both[want];
    }
    for (int t = 0; t < 50000; ++t) {
        const int rows = pick(1, 4), heads = pick(1, 4), bytes = pick(1, 4);
        long long hp, rp;
        if (t % 2) { hp = bytes + pick(0, 5); rp = (heads - 1) * hp + bytes + pick(0, 20); }
        else { rp = bytes + pick(0, 5); hp = (rows - 1) * rp + bytes + pick(0, 20); }
        const char* at[2] = {base + pick(0, 50), base + pick(0, 50)};
        std::set<long long> all[2];
        for (int i = 0; i < 2; ++i)
            for (int r = 0; r < rows; ++r) for (int h = 0; h < heads; ++h) for (int x = 0; x < bytes; ++x) all[i].insert((at[i] - base) + r * rp + h * hp + x);
        bool want = false;
        for (long long x : all[0]) want |= all[1].count(x) > 0;
        if (heads_overlap(at[0], at[1], rows, rp, heads, hp, bytes) != want) { printf("heads %d\n", t); return 1; }
        ++both[want];
    }
    if (both[0] < 1000 || both[1] < 1000) return 1;
    puts("ok");
    return 0;
}
"""

W = 4 * 64                   # query heads * head_dim of the calls below


def test_overlaps_are_those_of_sets_of_addresses(tmp_path):
    assert compile_and_run(tmp_path, CHECK).strip() == "ok"


@pytest.mark.parametrize("over", [dict(q=3 * A + 16), dict(q=3 * A + 512 * 4 * 3 + 2032), dict(q=3 * A - 16), dict(q=A + 64), dict(qkv=A + 4096),
                                  dict(q=A - 4 * W * 2 + 16)])
def test_append_refuses_rows_that_meet(over):
    """In the middle of the rows, at their end, in front of them, in the pool."""
    args = dict(qkv=3 * A, q=2 * A)
    args.update(over)
    refused("lie over", *append(struct(), **args))


@pytest.mark.parametrize("over", [dict(att=3 * A + 256), dict(att=3 * A - 3 * W * 2), dict(att=A + 1024), dict(lse=3 * A + 4), dict(lse=2 * A + 1000),
                                  dict(lse=A + 40), dict(ws=3 * A + 16, n=4096), dict(ws=2 * A, n=64), dict(ws=A, n=64)])
def test_attention_refuses_rows_that_meet(over):
    args = dict(q=3 * A, att=2 * A)
    args.update(over)
    refused("lie over", *attend(struct(), **args))


@pytest.mark.parametrize("over", [dict(v=2 * A + 64), dict(v=2 * A + 3 * 256), dict(k=A + 64), dict(v=A + 10 * 16 * 2 * 64 * 2 - 16)])
def test_read_refuses_outputs_that_meet(over):
    args = dict(k=2 * A, v=3 * A)
    args.update(over)
    refused("lie over", *read(struct(), **args))


def test_rows_side_by_side_do_not_meet():
    """(what is accepted here goes on to ask for a device, and there is none)"""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses would be followed")
    from turkce_llm_b200 import lib
    c = struct(K=16 * A, V=32 * A)
    calls = [append(c, qkv=3 * A, ld=768, q=3 * A + 512 * 4, ld_q=1536), append(c, qkv=3 * A, bf16=1, ld=768, q=3 * A + 1024, ld_q=768),
             attend(c, q=3 * A, ld_q=2 * W, att=3 * A + 2 * W, ld_att=2 * W), read(c, k=2 * A, v=2 * A + 256, ld_row=256),
             ("tb_logits_adjust", C.byref(rules()), A, 200, A + 400, 200, 4, 100, None)]
    for name, *args in calls:
        with pytest.raises(lib.TbError) as e:
            lib.check(getattr(lib.load(), name)(*args))
        assert "over" not in str(e.value), (name, str(e.value))
