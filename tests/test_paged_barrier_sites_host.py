"""The model of the chunk kernel's barriers against the kernel's source, and the waits that the first model leaves out.

Every place of the kernel that sets up a barrier, waits on one or arrives at one is listed here with the role that it belongs to: a change of
their order, of a parity or of a count fails until this list, and the model with it, follow.  The model adds the waits at a tile's start (the
query rows, and their way to tensor memory) and those of bf16 blocks that not all rows see, whose values are looked through before they are
released.  Not modelled: what happens behind a wait that has run out (every role ends, and the barriers by name are passed with a no)."""
import os
import re

import pytest

from conftest import CSRC
from test_paged_barriers_host import RING, Run, programs, stages


def kernel():
    with open(os.path.join(CSRC, "attention_paged.cu")) as f:
        text = f.read()
    at = text.index("\npaged_chunk_kernel(")
    return text, text[at:text.index("\ntemplate <", at)]


def sites(body):
    """(what, barrier, phase or count) in the order of the source, without casts."""
    body = re.sub(r"//[^\n]*", "", body)
    body = body.replace("(uint32_t)", "").replace("1u", "1").replace("Sh::", "")
    found = []
    for m in re.finditer(r"\b(mbar_init|mbar_wait|mbar_arrive|mbar_expect_tx|umma_commit|all_of)\(|bar\.sync (\d+), (\d+)", body):
        if m.group(2):
            found.append(("sync", m.group(2), m.group(3)))
            continue
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(body[i], 0)
            i += 1
        args, level, inside = [], 0, body[m.end():i - 1]
        piece = ""
        for c in inside:
            level += {"(": 1, "[": 1, ")": -1, "]": -1}.get(c, 0)
            if c == "," and level == 0:
                args.append(piece.strip())
                piece = ""
            else:
                piece += c
        args.append(piece.strip())
        what = m.group(1).replace("mbar_", "").replace("umma_", "")
        if what == "wait":
            args = args[:-1]                                    # (the flag of a wait that has run out)
        if what == "expect_tx":
            args = args[:1]                                     # (the bytes)
        found.append((what, *[a.lstrip("&") for a in args]))
    return found


SETUP = [("init", "q_full", "1"), ("init", "q_ready", "4"), ("init", "v_land", "1"), ("init", "s_full[i]", "1"), ("init", "s_free[i]", "4"),
         ("init", "p_full[i]", "4"), ("init", "o_full[i]", "1"), ("init", "raw_full[i]", "1"), ("init", "raw_empty[i]", "4"), ("init", "k_full[i]", "1"),
         ("init", "k_empty[i]", "1"), ("init", "v_full[i]", "E4M3 ? 4 : 1"), ("init", "v_empty[i]", "1"), ("init", "ks_full[i]", "4")]
PRODUCER = [("expect_tx", "q_full")]
PRODUCER_8 = [("wait", "k_empty[st]", "((j / KST) & 1) ^ 1"), ("expect_tx", "k_full[st]"), ("wait", "raw_empty[rs]", "((j / RST) & 1) ^ 1"),
              ("expect_tx", "raw_full[rs]")]
PRODUCER_16 = [("wait", "k_empty[st]", "((j / KST) & 1) ^ 1"), ("expect_tx", "k_full[st]"), ("wait", "v_empty[vst]", "((j / VST) & 1) ^ 1"),
               ("expect_tx", "bar"), ("wait", "v_land", "(landed & 1)"), ("arrive", "v_full[vst]")]
ISSUER = [("wait", "TS ? q_ready : q_full", "0"), ("wait", "k_full[st]", "((j / KST) & 1)"), ("wait", "s_free[b]", "((i >> 1) & 1) ^ 1"), ("commit", "s_full[b]"),
          ("commit", "k_empty[st]"), ("wait", "p_full[b]", "(j & 1)"), ("wait", "v_full[vst]", "((j / VST) & 1)"), ("commit", "o_full[b]"),
          ("commit", "v_empty[vst]")]
GROUP = [("wait", "q_full", "0"), ("arrive", "q_ready"), ("wait", "q_ready", "0"), ("wait", "ks_full[j & 7]", "((j >> 3) & 1)"), ("wait", "s_full[b]", "(j & 1)"),
         ("arrive", "s_free[b]"), ("wait", "o_full[b]", "((j - 1) & 1)"), ("arrive", "p_full[b]"), ("wait", "o_full[0]", "((nkv - 1) & 1)"),
         ("wait", "o_full[1]", "((nkv - 1) & 1)"), ("wait", "v_full[(nkv - 1) % VST]", "(((nkv - 1) / VST) & 1)"), ("sync", "1", "256"),
         ("all_of", "ok", "1", "256"), ("sync", "1", "256"), ("all_of", "ok", "1", "256")]
CONVERTER = [("wait", "q_full", "0"), ("arrive", "q_ready"), ("all_of", "ok", "2", "128"), ("arrive", "ks_full[j & 7]"),
             ("wait", "raw_full[rs]", "((j / RST) & 1)"), ("wait", "v_empty[vst]", "((j / VST) & 1) ^ 1"), ("all_of", "false", "2", "128"),
             ("arrive", "v_full[vst]"), ("arrive", "raw_empty[rs]")]


def test_the_kernel_has_the_barriers_that_the_model_knows():
    found = sites(kernel()[1])
    want = SETUP + PRODUCER + PRODUCER_8 + PRODUCER_16 + ISSUER + GROUP + CONVERTER
    for i, (a, b) in enumerate(zip(found, want)):
        assert a == b, (i, a, b)
    assert len(found) == len(want), (found[len(want):], want[len(found):])


def test_the_ring_of_scales_is_as_long_as_the_model_says():
    text, body = kernel()
    assert "[%d][128] key scales" % RING in text and "for (int i = 0; i < %d; ++i) mbar_init(&ks_full[i], 4);" % RING in body
    assert len(re.findall(r"\(j & %d\) \* PT_KEYS|\(j & %d\) \* \(PT_KEYS / 4\)" % (RING - 1, RING - 1), body)) == 2


def whole(n, nh, e4m3, edge):
    """The first model's programs with what they leave out; blocks from `edge` on are not seen by all rows."""
    kst, vst, rst = stages(nh, e4m3)
    prog = programs(n, kst, vst, rst, e4m3)
    prog[0] = [("arrive", "q_full")] + prog[0]
    if not e4m3:
        landed, out, j = 0, [], 0
        for op in prog[0]:
            if op[0] == "arrive" and op[1].startswith("v_full"):
                if j >= edge:
                    out += [("arrive", "v_land"), ("wait", "v_land", landed)]
                    landed += 1
                j += 1
            out.append(op)
        prog[0] = out
    in_tensor_memory = nh == 2 or e4m3
    prog[1] = [("wait", "q_ready" if in_tensor_memory else "q_full", 0)] + prog[1]
    if e4m3:
        prog[4] = [("wait", "q_full", 0), ("arrive", "q_ready")] + prog[4]
        for b in (0, 1):
            prog[2 + b] = [("wait", "q_ready", 0)] + prog[2 + b]
    elif in_tensor_memory:
        prog[2] = [("wait", "q_full", 0), ("arrive", "q_ready")] + prog[2]
    return prog


def stem(name):
    return re.sub(r"[\[\d].*", "", name)


@pytest.mark.parametrize("nh,e4m3", [(1, False), (2, False), (1, True), (2, True)])
def test_the_model_has_every_wait_and_arrival_of_the_kernel(nh, e4m3):
    """(copies and products arrive as well: expect_tx and commit)"""
    prog = whole(6, nh, e4m3, 2)
    in_tensor_memory = nh == 2 or e4m3

    def listed(entries):
        out = set()
        for e in entries:
            if e[0] in ("wait", "arrive", "commit", "expect_tx"):
                for name in ["v_land", "v_full"] if e[1] == "bar" else [("q_ready" if in_tensor_memory else "q_full")] if "?" in e[1] else [e[1]]:
                    out.add(("wait" if e[0] == "wait" else "arrive", stem(name)))
        return out

    def modelled(ops):
        return {("wait" if op[0] == "wait" else "arrive", stem(op[1])) for op in ops if op[0] in ("wait", "arrive", "tensor")}

    assert modelled(prog[0]) == listed(PRODUCER + (PRODUCER_8 if e4m3 else PRODUCER_16))
    assert modelled(prog[1]) == listed(ISSUER)
    group = listed(GROUP)
    if not e4m3:
        group -= {("wait", "ks_full"), ("wait", "q_ready")}
    if e4m3 or not in_tensor_memory:
        group -= {("wait", "q_full"), ("arrive", "q_ready")}
    assert modelled(prog[2]) | modelled(prog[3]) == group
    if e4m3:
        assert modelled(prog[4]) == listed(CONVERTER)


@pytest.mark.parametrize("nh,e4m3", [(1, False), (2, False), (1, True), (2, True)])
def test_every_wait_means_the_phase_it_names(nh, e4m3):
    for n in (1, 2, 3, 7):
        for edge in sorted({0, n - 1, n}):
            prog = whole(n, nh, e4m3, edge)
            roles = list(range(-1, len(prog)))
            for order in (roles, roles[::-1]):
                run = Run(prog)
                run.finish(order)
                assert run.at == [len(p) for p in prog] and not run.queue
            for r in range(len(prog)):
                for place in range(len(prog[r])):
                    run = Run(prog)
                    first = [r] + [x for x in roles if x != r]
                    run.finish(first, until=(r, place))
                    run.finish([x for x in roles if x != r], frozen=r)
                    run.finish(first)
                    assert run.at == [len(p) for p in prog]


@pytest.mark.parametrize("change", [("((j / VST) & 1) ^ 1u, abort_flag", "((j / VST) & 1), abort_flag"), ("mbar_init(&s_free[i], 4)", "mbar_init(&s_free[i], 8)"),
                                    ("umma_commit(&k_empty[st]);", ";"), ("if (lane == 0) mbar_arrive(&p_full[b]);", "mbar_arrive(&p_full[b]), mbar_arrive(&p_full[b]);")])
def test_a_change_of_the_kernel_is_found(change):
    body = kernel()[1]
    assert change[0] in body
    assert sites(body.replace(change[0], change[1])) != sites(body)
