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
