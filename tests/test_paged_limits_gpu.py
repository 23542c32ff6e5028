"""Attention over a paged cache at the limits of what its cache may hold, against the formula in 64 bits."""
import numpy as np
import pytest
import torch

import paged_plain as plain
from test_paged_gpu import Batch, attend

pytestmark = pytest.mark.gpu


def upload(b):
    for name in ("k", "v"):
        if b.e4m3:
            b.dev[name].copy_(torch.from_numpy(b.host[name]).cuda().view(torch.float8_e4m3fn))
            b.dev[name + "_scale"].copy_(torch.from_numpy(b.host[name + "_scale"]))
        else:
            b.dev[name].copy_(b.host[name])


def at(b, s, t):
    """Where key t of sequence s (a number or an array of them) lies: page, place in it."""
    return b.table[s, t // b.page], t % b.page


# ---------------------------------------------------------------------------------------------- scales of values

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 8])
@pytest.mark.parametrize("kv", [9, 33, 600, 5000])
@pytest.mark.parametrize("ends", [(-126, 56), (-126, 118), (-70, 118), (-126, -126), (118, 118)])
def test_value_scales_at_the_ends_of_their_range(tb, dim, new, kv, ends):
    """Single tokens and few of them: every key counts in the sum, however small its value's scale is beside others."""
    b = Batch(True, [new], [kv], 1, dim, 16, seed=kv)
    rng = np.random.default_rng(dim + new)
    t = np.arange(kv)
    exponent = rng.choice(ends, kv)
    exponent[-1 - new // 2] = ends[1]
    page, slot = at(b, 0, t)
    b.host["v_scale"][page, 0, slot] = np.ldexp(1 + rng.random(kv), exponent).astype(np.float32)
    upload(b)
    q, got, lse = attend(b, 2, seed=21)
    k, v = b.sequence("k", 0), b.sequence("v", 0)
    positions = np.arange(kv - new, kv)
    want, want_lse, spread, size = plain.attention(q, k, v, positions, dim ** -0.5)
    # Scores: sums of dim float32 products of rows that are exact but for 2^-24 of their largest element.  Exponents of scales are added to
    # them, numbers below 2^8 in float32: half a unit in the last place is 2^-17, of a score, of the reference and of their difference, twice
    # (a probability and their sum): 2^-15 in all with log 2.  Probabilities are f16, 2^13 for the row's largest product of probability and
    # scale (a scale of less than 2^-80 of the largest counts as that much there): off by 2^-25 where they are small, 2^-38 of that
    # product, times a code of 448.  The smallest bf16 is 2^-133.
    scales = b.host["v_scale"][page, 0, slot].astype(np.float64)
    score = (dim + 4) * 2.0 ** -24 * size + 2.0 ** -24 * np.abs(q).max(axis=2) * np.abs(k[:, 0]).sum(axis=1).max() * dim ** -0.5
    lost = np.zeros_like(want_lse)
    for r in range(new):
        n = positions[r] + 1
        for h in range(2):
            p = np.exp(k[:n, 0] @ q[r, h].astype(np.float64) * dim ** -0.5 - want_lse[r, h])
            lost[r, h] = 2.0 ** -29 * n * (p * np.maximum(scales[:n], 2.0 ** -80 * scales[:n].max())).max()
    bound = 2.0 ** -8 * np.abs(want) + (2.0 ** -11 * 1.01 + 2 * score[..., None] + 2.0 ** -15) * spread + lost[..., None] + 2.0 ** -133
    assert (np.abs(got - want) <= bound).all(), np.nanmax(np.abs(got - want) / bound)
    assert (np.abs(lse - want_lse) <= score + 2.0 ** -15 + 2.0 ** -20 * (1 + np.abs(want_lse))).all()


@pytest.mark.parametrize("new", [1, 4, 40])
@pytest.mark.parametrize("size", [1e17, 1e30])
def test_a_row_of_zeros_halves_the_value_beside_it(tb, new, size):
    """All scores alike: the result is the mean of the values, whatever their scales are."""
    b = Batch(True, [new], [new + 63], 1, 64, 16, seed=1)
    for name, codes in (("k", 0), ("v", 0)):
        b.host[name][:] = codes
    b.host["k_scale"][:] = 1.0
    b.host["v_scale"][:] = 2.0 ** -126
    t = np.arange(0, new + 63, 2)                               # every other key has codes of 256 (0x78)
    page, slot = at(b, 0, t)
    b.host["v"][page, 0, slot] = 0x78
    b.host["v_scale"][page, 0, slot] = np.float32(size / 256)
    upload(b)
    q, got, lse = attend(b, 2, seed=22)
    n = np.arange(64, 64 + new)
    want = np.float32(size / 256) * 256.0 * ((n + 1) // 2) / n
    # (equal probabilities: f16 holds them, exponents are whole numbers; bf16 at the end)
    assert (np.abs(got / want[:, None, None] - 1) <= 2.0 ** -8 + 2.0 ** -15).all()
    assert (np.abs(lse - np.log(n)[:, None]) <= 2.0 ** -15).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("before", [0, 30, 200, 4000])
@pytest.mark.parametrize("new", [6, 40, 200])
@pytest.mark.parametrize("up", [3, 23, 40, 100])
def test_scales_of_later_tokens_do_not_reach_earlier_rows(tb, dim, before, new, up):
    """The values of some tokens of a chunk are 2^up times the others: rows in front of them have the same bits as without them, those that
    see them are right."""
    kv = before + new
    b = Batch(True, [new, 1], [kv, 50], 1, dim, 16, seed=new)
    clean = attend(b, 2, seed=23)
    large = [before + (2 * new) // 3, kv - 1]
    for t in large:
        page, slot = at(b, 0, np.array(t))
        b.host["v_scale"][page, 0, slot] *= np.float32(2.0 ** up)
    upload(b)
    q, got, lse = attend(b, 2, seed=23)
    unseen = large[0] - before
    others = np.r_[:unseen, new:b.rows]
    assert (got[others] == clean[1][others]).all() and (lse[others] == clean[2][others]).all()
    k, v = b.sequence("k", 0), b.sequence("v", 0)
    positions = np.arange(before, kv)
    want, want_lse, spread, size = plain.attention(q[:new], k, v, positions, dim ** -0.5)
    # f16 probabilities (2^7 and more for a row's largest: off by 2^-25 of that where they are small, times a code of 448 and the largest scale
    # that the row sees, twice a power of two) and f16 values (off by 2^-31 of that scale); single tokens: less
    score = (dim + 4) * 2.0 ** -24 * size + 2.0 ** -21 * np.abs(q[:new]).max(axis=2) * np.abs(k[:, 0]).sum(axis=1).max() * dim ** -0.5
    scales = b.host["v_scale"][at(b, 0, np.arange(kv))[0], 0, np.arange(kv) % 16].astype(np.float64)
    most = np.maximum.accumulate(scales)[positions][:, None, None]
    lost = positions[:, None, None] * (2.0 ** -32 * 448 * 2 + 2.0 ** -31) * most
    bound = 2.0 ** -8 * np.abs(want) + (2 * 2.0 ** -11 * 1.01 + 2 * score[..., None] + 2.0 ** -15) * spread + lost + 1e-30
    assert (np.abs(got[:new] - want) <= bound).all(), np.nanmax(np.abs(got[:new] - want) / bound)
    assert (np.abs(lse[:new] - want_lse) <= score + 2.0 ** -15 + 2.0 ** -20 * (1 + np.abs(want_lse))).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_scales_that_grow_along_a_chunk(tb, dim):
    """Every token's value is 2^3 times the one before it, over a range of 2^120: each row is about its own last keys, and right."""
    b = Batch(True, [40], [40], 1, dim, 16, seed=3)
    page, slot = at(b, 0, np.arange(40))
    b.host["v_scale"][page, 0, slot] = np.ldexp(np.float32(1.5), 3 * np.arange(40) - 80)
    upload(b)
    q, got, _ = attend(b, 2, seed=24)
    k, v = b.sequence("k", 0), b.sequence("v", 0)
    want, _, spread, size = plain.attention(q, k, v, np.arange(40), dim ** -0.5)
    score = (dim + 4) * 2.0 ** -24 * size + 2.0 ** -21 * np.abs(q).max(axis=2) * np.abs(k[:, 0]).sum(axis=1).max() * dim ** -0.5
    # (as above, with the row's own scale as the largest it sees)
    lost = np.arange(1, 41)[:, None, None] * (2.0 ** -32 * 448 * 2 + 2.0 ** -31) * (1.5 * 2.0 ** (3 * np.arange(40) - 80))[:, None, None]
    bound = 2.0 ** -8 * np.abs(want) + (2 * 2.0 ** -11 * 1.01 + 2 * score[..., None] + 2.0 ** -15) * spread + lost
    assert (np.abs(got - want) <= bound).all(), np.nanmax(np.abs(got - want) / bound)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("exponent", [-126, -60, 118])
def test_chunks_of_values_at_the_ends_of_their_range(tb, dim, exponent):
    b = Batch(True, [40], [240], 1, dim, 16, seed=4)
    page, slot = at(b, 0, np.arange(240))
    b.host["v_scale"][page, 0, slot] = np.ldexp((1 + np.random.default_rng(5).random(240)).astype(np.float32), exponent)
    upload(b)
    q, got, lse = attend(b, 2, seed=27)
    k, v = b.sequence("k", 0), b.sequence("v", 0)
    want, want_lse, spread, size = plain.attention(q, k, v, np.arange(200, 240), dim ** -0.5)
    score = (dim + 4) * 2.0 ** -24 * size + 2.0 ** -21 * np.abs(q).max(axis=2) * np.abs(k[:, 0]).sum(axis=1).max() * dim ** -0.5
    # (as above; the smallest bf16 is 2^-133)
    lost = 240 * (2.0 ** -32 * 448 * 2 + 2.0 ** -31) * 2.0 ** (exponent + 1)
    bound = 2.0 ** -8 * np.abs(want) + (2 * 2.0 ** -11 * 1.01 + 2 * score[..., None] + 2.0 ** -15) * spread + lost + 2.0 ** -133
    assert (np.abs(got - want) <= bound).all(), np.nanmax(np.abs(got - want) / bound)
    assert (np.abs(lse - want_lse) <= score + 2.0 ** -15 + 2.0 ** -20 * (1 + np.abs(want_lse))).all()


def test_a_value_above_float32_counts_once(tb):
    """A code times a scale of 2^121 is more than float32 has, its product with a small probability is not; beside a code that is none in another
    column (such codes are added by themselves)."""
    b = Batch(True, [40], [240], 1, 64, 16, seed=7)
    page, slot = at(b, 0, np.arange(240))
    b.host["k"][page, 0, slot] = 0
    b.host["k_scale"][page, 0, slot] = 1.0
    b.host["k"][page[210], 0, slot[210], 0] = 0xfe              # -448
    b.host["k_scale"][page[210], 0, slot[210]] = np.float32(20 * np.log(2) / 448 * 8)
    b.host["v"][page[210], 0, slot[210]] = 0x7e                 # 448
    b.host["v_scale"][page[210], 0, slot[210]] = 2.0 ** 121
    b.host["v"][page[205], 0, slot[205], 7] = 0x7f
    upload(b)
    q = torch.zeros(43, 64, dtype=torch.bfloat16)
    q[:, 0] = 1.0
    _, got, _ = attend(b, 1, seed=28, q=q)
    seen = np.arange(210, 240)                                  # rows that see it: 2^-20 of its value over the other keys' number
    want = 448.0 * 2.0 ** 121 * 2.0 ** -20 / (seen + 2.0 ** -20)
    got = got[10:, 0]
    assert np.isnan(got[:, 7]).all()
    # (the score 2^-17 of itself off by float32 and the scale's rounding, f16 twice, bf16)
    assert (np.abs(np.delete(got, 7, axis=1) / want[:, None] - 1) <= 2.0 ** -8 + 2 * 2.0 ** -11 + 2.0 ** -14).all()


# ---------------------------------------------------------------------------------------------- pages outside the pool

@pytest.mark.parametrize("bad", [-1, 1 << 20, 0x7fffffff])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,page", [(48, 16), (64, 64), (128, 16)])
@pytest.mark.parametrize("new,kv", [(1, 200), (3, 5000), (40, 200), (40, 40), (200, 3000)])
def test_rows_that_see_a_page_outside_the_pool_are_nan(tb, e4m3, dim, page, new, kv, bad):
    """Nothing takes the page's place: a result that looked right would hold some other sequence's values.  Rows in front of the page, and other
    sequences, have the same bits as without it."""
    b = Batch(e4m3, [2, new, 1], [70, kv, 30], 2, dim, page, seed=dim + new)
    clean = attend(b, 4, seed=25)
    for piece in {(kv - 1) // page, (kv - 1) // page // 2}:
        b.table_dev.copy_(torch.from_numpy(b.table.astype(np.int32)))
        b.table_dev[1, piece] = bad
        q, got, lse = attend(b, 4, seed=25, check=False)
        with pytest.raises(tb.TbError, match="code 75"):
            tb.sync_check()
        sees = np.zeros(b.rows, bool)
        sees[2:2 + new] = kv - new + np.arange(new) >= piece * page
        assert np.isnan(got[sees]).all() and np.isnan(lse[sees]).all()
        assert (got[~sees] == clean[1][~sees]).all() and (lse[~sees] == clean[2][~sees]).all()
    b.table_dev.copy_(torch.from_numpy(b.table.astype(np.int32)))
    again = attend(b, 4, seed=25)                               # (and nothing of it stays)
    assert (again[1] == clean[1]).all() and (again[2] == clean[2]).all()


def test_a_bad_page_is_told_by_the_check_alone_and_once(tb):
    """Calls that check their own work on the host neither fail for it nor take it away; a batch's bad length on one stream leaves the tickets of
    a head on another alone (its choice is the same before and after)."""
    b = Batch(False, [1, 1], [40, 50], 2, 64, 16, seed=2)
    b.table_dev[1, 2] = -3
    x = torch.randn(4, 128, device="cuda").to(torch.bfloat16)
    e = torch.randn(1000, 128, device="cuda").to(torch.bfloat16)
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    tb.lmhead_argmax_bf16(x, e, tok)
    before = tok.clone()
    attend(b, 2, seed=8, check=False)
    torch.cuda.synchronize()
    A, B, C = np.ones((64, 32), np.float32), np.ones((32, 48), np.float32), np.zeros((64, 48), np.float32)
    tb.matmul_host(A, B, C, 64, 32, 48)
    assert (C == 32).all()
    other = torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(other):
            tb.lmhead_argmax_bf16(x, e, tok)
        attend(b, 2, seed=8, check=False)
        with pytest.raises(tb.TbError, match="code 75"):
            tb.sync_check()
        tb.sync_check()
    torch.cuda.synchronize()
    assert torch.equal(tok, before)


# ---------------------------------------------------------------------------------------------- scores of minus infinity

@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("kv", [300, 4000])
def test_keys_of_minus_infinity_have_no_weight(tb, e4m3, dim, new, kv):
    """The first keys, whole blocks of them, score minus infinity: the result is that of the others alone."""
    cut = kv - 90
    b = Batch(e4m3, [new], [kv], 1, dim, 16, seed=kv)
    page, slot = at(b, 0, np.arange(cut))
    if e4m3:
        b.host["k"][page, 0, slot] = 0
        b.host["k"][page, 0, slot, 0] = 0xb8                    # -1 times an infinite scale
        b.host["k_scale"][page, 0, slot] = np.inf
    else:
        b.host["k"][page, 0, slot, 0] = -float("inf")
    upload(b)
    q = torch.randn(new + 3, 2 * dim).to(torch.bfloat16)
    q[:, ::dim] = q[:, ::dim].abs() + 1
    rows, got, lse = attend(b, 2, seed=26, q=q)
    k, v = b.sequence("k", 0)[cut:], b.sequence("v", 0)[cut:]
    want, want_lse, spread, size = plain.attention(rows, k, v, np.arange(90 - new, 90), dim ** -0.5)
    assert plain.within(got, want, spread, size, dim) <= 1.0
    assert (np.abs(lse - want_lse) <= (dim + 4) * 2.0 ** -24 * size + 2.0 ** -20 * (1 + np.abs(want_lse))).all()


# ---------------------------------------------------------------------------------------------- many rows

def test_more_tiles_than_65535(tb):
    """128 heads over one key head: a tile is one token.  A prompt of 65,600 of them, a row here and there against the formula."""
    new, H, dim = 65600, 128, 16
    b = Batch(False, [new], [new], 1, dim, 256, seed=6)
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(new, H * dim, device="cuda", generator=g).to(torch.bfloat16)
    att, lse = torch.empty_like(q), torch.empty(new, H, device="cuda")
    b.cache.attend(q, att, b.q_start, b.kv_len, new, new, lse=lse, workspace=b.cache.workspace(H, new, new, new))
    tb.sync_check()
    k, v = b.sequence("k", 0), b.sequence("v", 0)
    for r in (0, 1, 127, 40000, new - 1):
        rows = q[r].double().cpu().numpy().reshape(1, H, dim)
        want, want_lse, spread, size = plain.attention(rows, k, v, np.array([r]), dim ** -0.5)
        assert plain.within(att[r].double().cpu().numpy().reshape(1, H, dim), want, spread, size, dim) <= 1.0
        assert (np.abs(lse[r].cpu().numpy() - want_lse[0]) <= (dim + 4) * 2.0 ** -24 * size[0] + 2.0 ** -20 * (1 + np.abs(want_lse[0]))).all()


def test_profile_claims_no_work_that_only_the_device_knows(tb):
    """Both kernels of a call claimed all rows times the largest number of keys."""
    b = Batch(False, [40, 1], [300, 200], 2, 64, 16, seed=1)
    tb.profile_begin()
    attend(b, 2, seed=1, max_kv=16 * b.table.shape[1])
    seen = tb.profile_end()
    assert {"paged_rows", "paged_chunk"} <= set(seen)
    assert all(seen[n]["flops"] == 0 and seen[n]["bytes"] == 0 for n in seen if n.startswith("paged"))


# ---------------------------------------------------------------------------------------------- 8-bit codes

@pytest.mark.parametrize("exponent", [-126, -123, -118, -112, -104, -100, -99, -40, 100, 118])
def test_codes_of_rows_of_any_size_are_the_nearest(tb, exponent):
    """Elements next to the middles of two codes, in rows whose scale is anywhere in the range: bit for bit."""
    rng = np.random.default_rng(exponent + 200)
    rows, dim = 400, 64
    b = Batch(True, [rows], [rows], 1, dim, 16, seed=0)
    scale = np.ldexp((1 + rng.random(rows)).astype(np.float32), exponent)
    big = np.minimum(scale.astype(np.float64) * 448, np.finfo(np.float32).max).astype(np.float32)
    scale = np.maximum((big.astype(np.float64) / 448).astype(np.float32), np.float32(2.0 ** -126))
    middles = (plain.E4M3[1:] + plain.E4M3[:-1]) / 2
    x = (rng.choice(middles, (rows, dim)) * scale[:, None].astype(np.float64)).astype(np.float32)
    x = (x.view(np.int32) + rng.integers(-1, 2, x.shape).astype(np.int32)).view(np.float32) * rng.choice([-1, 1], x.shape).astype(np.float32)
    x[:, 5] = big
    qkv = torch.zeros(rows, 3 * dim)
    qkv[:, 2 * dim:] = torch.from_numpy(x)
    q = torch.empty(rows, dim, dtype=torch.bfloat16, device="cuda")
    b.cache.append(qkv.cuda(), q, b.q_start, b.kv_len)
    tb.sync_check()
    page, slot = at(b, 0, np.arange(rows))
    assert (b.dev["v_scale"].cpu().numpy()[page, 0, slot] == scale).all()
    codes = b.dev["v"].view(torch.uint8).cpu().numpy()[page, 0, slot]
    assert (codes == plain.e4m3_codes(x, scale[:, None])).all(), (codes != plain.e4m3_codes(x, scale[:, None])).sum()


@pytest.mark.parametrize("new", [1, 8, 40])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** 126, 1.5 * 2.0 ** 127])
def test_the_largest_queries_of_8_bit_rows(tb, dim, new, size):
    """A query element as large as bf16 has: the scores are numbers, and one key has all of the weight."""
    b = Batch(True, [new], [200 + new], 1, dim, 16, seed=8)
    page, slot = at(b, 0, np.arange(200 + new))
    b.host["k_scale"][page, 0, slot] = 2.0 ** -12
    b.host["k"][page, 0, slot, 3] = np.random.default_rng(2).permutation(200 + new) % 100   # (the largest of them: 99, twice at most)
    b.host["k"][page[150], 0, slot[150], 3] = 0x7e
    upload(b)
    q = torch.randn(new + 3, 2 * dim).to(torch.bfloat16)
    q[:, 3] = q[:, dim + 3] = size
    _, got, lse = attend(b, 2, seed=29, q=q)
    want = b.sequence("v", 0)[150, 0]
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want)).all()
    score = float(torch.tensor(size).to(torch.bfloat16)) * 448 * 2.0 ** -12 * dim ** -0.5
    assert (np.abs(lse / score - 1) <= 2.0 ** -18).all()
