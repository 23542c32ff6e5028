"""Operators over a paged cache (tb_kv_append, tb_kv_read, tb_attention_paged) against their plain forms in 64 bits."""
import numpy as np
import pytest
import torch

import paged_plain as plain

pytestmark = pytest.mark.gpu

GARBAGE = 0x7ffffff0          # in table entries behind a sequence's last page


class Batch:
    """A cache of random contents with pages in no order: every row that belongs to no sequence is NaN (in 8 bits: code and scale)."""

    def __init__(self, e4m3, new, kv, G, dim, page, seed, extra_pages=2, width=None):
        from turkce_llm_b200.paged import PagedCache
        rng = np.random.default_rng(seed)
        self.new, self.kv, self.G, self.dim, self.page, self.e4m3 = list(new), list(kv), G, dim, page, e4m3
        need = [-(-n // page) for n in kv]
        width = width or max(1, max(need) + 1)
        pages = sum(need) + extra_pages
        order = rng.permutation(pages)[:sum(need)]
        table = np.full((len(kv), width), GARBAGE, np.int64)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        self.table = table
        shape = (pages, G, page, dim)
        self.host = {}
        used = np.zeros((pages, page), bool)
        for s, n in enumerate(kv):
            for t in range(n):
                used[table[s, t // page], t % page] = True
        self.used = used
        for name in ("k", "v"):
            x = rng.standard_normal(shape).astype(np.float32)
            if e4m3:
                codes = rng.integers(0, 127, shape).astype(np.uint8) | (rng.integers(0, 2, shape) << 7).astype(np.uint8)
                scale = (0.002 + 0.008 * rng.random(shape[:3])).astype(np.float32)
                codes.transpose(0, 2, 1, 3)[~used] = 0x7f
                scale.transpose(0, 2, 1)[~used] = np.nan
                self.host[name], self.host[name + "_scale"] = codes, scale
            else:
                t = torch.from_numpy(x).to(torch.bfloat16)
                t.permute(0, 2, 1, 3)[torch.from_numpy(~used)] = float("nan")
                self.host[name] = t
        dev = {}
        for name in ("k", "v"):
            if e4m3:
                dev[name] = torch.from_numpy(self.host[name]).cuda().view(torch.float8_e4m3fn)
                dev[name + "_scale"] = torch.from_numpy(self.host[name + "_scale"]).cuda()
            else:
                dev[name], dev[name + "_scale"] = self.host[name].cuda(), None
        self.dev = dev
        self.table_dev = torch.from_numpy(table.astype(np.int32)).cuda()
        self.cache = PagedCache(dev["k"], dev["v"], self.table_dev, k_scale=dev["k_scale"], v_scale=dev["v_scale"])
        starts = np.concatenate(([0], np.cumsum(new)))
        self.starts, self.rows = starts, int(starts[-1])
        self.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.kv_len = torch.tensor(kv, dtype=torch.int32, device="cuda")

    def sequence(self, name, s, n=None):
        """Rows of a sequence as float64 [kv, G, dim]."""
        t = np.arange(self.kv[s] if n is None else n)
        at = self.table[s, t // self.page], slice(None), t % self.page
        if self.e4m3:
            return plain.e4m3_values(self.host[name][at]) * self.host[name + "_scale"][at][..., None].astype(np.float64)
        return self.host[name][at[0], :, at[2]].double().numpy()


def attend(b, H, seed, max_q=None, max_kv=None, stride=0, check=True, scale=None, q=None):
    rng = np.random.default_rng(seed)
    width = H * b.dim
    if q is None:
        q = torch.from_numpy(rng.standard_normal((b.rows + 3, width)).astype(np.float32)).to(torch.bfloat16)
    qd = torch.empty(b.rows + 3, width + stride, dtype=torch.bfloat16, device="cuda")[:, :width]
    qd.copy_(q)
    att = torch.full((b.rows + 3, width + stride), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((b.rows + 3, H), 5.0, device="cuda")
    max_q, max_kv = max_q or max(1, max(b.new)), max(b.kv) if max_kv is None else max_kv
    ws = b.cache.workspace(H, b.rows + 3, max_q, max_kv)
    b.cache.attend(qd, att[:, :width], b.q_start, b.kv_len, max_q, max_kv, scale=scale, lse=lse, workspace=ws)
    if check:
        from turkce_llm_b200 import lib
        lib.sync_check()
    got, got_lse = att.float().cpu().numpy(), lse.cpu().numpy()
    assert (got[b.rows:] == 7.0).all() and (got[:, width:] == 7.0).all() and (got_lse[b.rows:] == 5.0).all()
    return q.float().numpy()[:b.rows].reshape(b.rows, H, b.dim), got[:b.rows, :width].reshape(b.rows, H, b.dim), got_lse[:b.rows]


def compare(b, H, q, got, lse, skip=(), scale=None):
    scale = b.dim ** -0.5 if scale is None else scale
    for s in range(len(b.new)):
        if s in skip or b.new[s] == 0:
            continue
        rows = slice(b.starts[s], b.starts[s + 1])
        positions = np.arange(b.kv[s] - b.new[s], b.kv[s])
        want, want_lse, spread, size = plain.attention(q[rows], b.sequence("k", s), b.sequence("v", s), positions, scale)
        worst = plain.within(got[rows], want, spread, size, b.dim)
        assert worst <= 1.0, (s, b.new[s], b.kv[s], worst)
        none = np.isinf(want_lse)
        assert (lse[rows][none] == want_lse[none]).all() and (got[rows][none] == 0).all()
        # a sum of dim products per score, a logarithm of float32
        off = np.abs(lse[rows][~none] - want_lse[~none])
        assert (off <= (b.dim + 4) * 2.0 ** -24 * size[~none] + 2.0 ** -20 * (1 + np.abs(want_lse[~none]))).all(), (s, off.max())


EDGES = [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 200, 333]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,page", [(8, 16), (16, 32), (24, 64), (48, 128), (64, 16), (64, 256), (80, 32), (96, 16), (128, 64)])
def test_single_tokens(tb, e4m3, dim, page):
    if e4m3 and dim % 16:
        pytest.skip("8-bit rows are multiples of 16 elements")
    b = Batch(e4m3, [1] * len(EDGES), EDGES, 3, dim, page, seed=dim + page)
    for H in (3, 6):
        compare(b, H, *attend(b, H, seed=1))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("G,H", [(1, 1), (1, 5), (2, 14), (1, 16), (1, 24), (2, 80)])
def test_shared_heads(tb, e4m3, G, H):
    new = [1, 1, 2, 3, 0, 1, 7]
    kv = [1, 40, 17, 130, 5, 0, 90]                            # (a sequence with a row and no key: zeros)
    b = Batch(e4m3, new, kv, G, 64, 16, seed=H)
    compare(b, H, *attend(b, H, seed=2, stride=8))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,page,G,H", [(64, 16, 6, 6), (64, 64, 2, 6), (32, 32, 1, 3), (128, 16, 2, 4), (96, 256, 1, 2), (16, 128, 2, 16)])
def test_chunks(tb, e4m3, dim, page, G, H):
    new = [5, 1, 64, 130, 17, 0, 33]
    kv = [5, 300, 64, 131, 200, 44, 20]                        # (the last: 13 rows before the first key)
    b = Batch(e4m3, new, kv, G, dim, page, seed=dim)
    compare(b, H, *attend(b, H, seed=3))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,kv", [([1], [5000]), ([3], [2100]), ([40], [3001]), ([1, 1], [1, 4097]), ([300, 1], [700, 2500])])
def test_long_caches_in_pieces(tb, e4m3, new, kv):
    b = Batch(e4m3, new, kv, 2, 64, 16, seed=kv[0])
    for bound in (max(kv), 3 * max(kv)):                        # (room for longer sequences: other pieces)
        if bound > b.table.shape[1] * 16:
            b = Batch(e4m3, new, kv, 2, 64, 16, seed=kv[0], width=-(-bound // 16))
        compare(b, 4, *attend(b, 4, seed=4, max_kv=bound))


def test_scale_and_large_scores(tb):
    """Scores of some hundred: the running maximum moves, one or a few keys take all of the weight."""
    b = Batch(False, [4, 1, 20], [4, 600, 300], 1, 64, 32, seed=9)
    for scale in (3.0, 0.01):
        compare(b, 2, *attend(b, 2, seed=5, scale=scale), scale=scale)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [1, 5, 40, 200])
def test_what_a_row_does_not_see_does_not_reach_it(tb, e4m3, new):
    """Keys and values behind a row's position are NaN and infinity: in the rest of a page, and in later rows of the chunk."""
    b = Batch(e4m3, [new, 1], [150 + new, 30], 2, 64, 16, seed=new)
    bad = 150 + new // 2 + 1                                    # this row of the chunk and its successors see something bad
    rng = np.random.default_rng(3)
    for t in range(bad, 150 + new):
        page, slot = b.table[0, t // 16], t % 16
        for name in ("k", "v"):
            if e4m3:
                b.host[name + "_scale"][page, :, slot] = np.nan
            else:
                b.host[name][page, :, slot] = torch.from_numpy(rng.choice([np.nan, np.inf, -np.inf, 1.0], (2, 64))).to(torch.bfloat16)
    for name in ("k", "v"):
        if e4m3:
            b.dev[name + "_scale"].copy_(torch.from_numpy(b.host[name + "_scale"]))
        else:
            b.dev[name].copy_(b.host[name])
    q, got, lse = attend(b, 4, seed=6)
    good = min(new, bad - 150)
    positions = np.arange(150, 150 + good)
    want, want_lse, spread, size = plain.attention(q[:good], b.sequence("k", 0, bad), b.sequence("v", 0, bad), positions, 0.125)
    assert plain.within(got[:good], want, spread, size, 64) <= 1.0
    assert np.isfinite(lse[:good]).all()
    if good < new:
        assert not np.isfinite(got[new - 1]).all()
    want, _, spread, size = plain.attention(q[new:], b.sequence("k", 1), b.sequence("v", 1), np.arange(29, 30), 0.125)
    assert plain.within(got[new:], want, spread, size, 64) <= 1.0


def test_infinite_value_reaches_the_rows_that_see_it(tb):
    b = Batch(False, [100], [100], 1, 64, 16, seed=1)
    page = b.table[0, 37 // 16]
    b.dev["v"][page, 0, 37 % 16, 5] = float("inf")
    b.dev["v"][page, 0, 37 % 16, 60] = float("nan")
    _, got, _ = attend(b, 1, seed=7)
    assert np.isfinite(got[:37]).all()
    assert np.isinf(got[37:, 0, 5]).all() and np.isnan(got[37:, 0, 60]).all()
    assert np.isfinite(np.delete(got, [5, 60], axis=2)).all()


def test_bad_pages_and_lengths_are_left_out_and_reported(tb):
    b = Batch(False, [1, 1, 1, 20], [40, 50, 60, 70], 2, 64, 16, seed=2)
    b.table_dev[1, 2] = -3
    q, got, lse = attend(b, 2, seed=8, check=False)
    with pytest.raises(tb.TbError, match="code 75"):
        tb.sync_check()
    compare(b, 2, q, got, lse, skip=(1,))
    b = Batch(False, [1, 1, 1, 20], [40, 50, 60, 70], 2, 64, 16, seed=2)
    b.kv_len[2] = 1 << 30
    q, got, lse = attend(b, 2, seed=8, check=False)
    with pytest.raises(tb.TbError, match="code 76"):
        tb.sync_check()
    compare(b, 2, q, got, lse, skip=(2,))
    assert (got[2] == 7.0).all()
    tb.sync_check()                                             # (said once)


def test_replayed_graph_follows_the_lengths_and_the_table(tb):
    """One capture, replayed after other tokens have come: lengths, table, queries and contents change in place."""
    H, bound = 4, 400
    a = Batch(False, [1, 3, 2], [30, 200, 90], 2, 64, 16, seed=1, extra_pages=60, width=bound // 16)
    b = Batch(False, [2, 1, 3], [400, 17, 64], 2, 64, 16, seed=2, extra_pages=60, width=bound // 16)
    pages = max(a.dev["k"].shape[0], b.dev["k"].shape[0])
    from turkce_llm_b200.paged import PagedCache
    pools = {n: torch.zeros(pages, 2, 16, 64, dtype=torch.bfloat16, device="cuda") for n in ("k", "v")}
    table = torch.zeros_like(a.table_dev)
    cache = PagedCache(pools["k"], pools["v"], table)
    q = torch.zeros(6, H * 64, dtype=torch.bfloat16, device="cuda")
    att, lse = torch.zeros_like(q), torch.zeros(6, H, device="cuda")
    q_start, kv_len = torch.zeros_like(a.q_start), torch.zeros_like(a.kv_len)
    ws = cache.workspace(H, 6, 4, bound)

    def load(x):
        for n in ("k", "v"):
            pools[n][:x.dev[n].shape[0]].copy_(x.dev[n])
        table.copy_(x.table_dev)
        q_start.copy_(x.q_start)
        kv_len.copy_(x.kv_len)
        q.copy_(torch.from_numpy(np.random.default_rng(x.kv[0]).standard_normal((6, H * 64)).astype(np.float32)))

    load(a)
    cache.attend(q, att, q_start, kv_len, 4, bound, lse=lse, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(q, att, q_start, kv_len, 4, bound, lse=lse, workspace=ws)
    for x in (b, a):
        load(x)
        att.zero_()
        graph.replay()
        torch.cuda.synchronize()
        compare(x, H, q.float().cpu().numpy()[:x.rows].reshape(x.rows, H, 64), att.float().cpu().numpy()[:x.rows].reshape(x.rows, H, 64),
                lse.cpu().numpy()[:x.rows])
    tb.sync_check()


def test_two_calls_side_by_side(tb):
    """Two streams, a workspace each: the same results as one after the other, bit for bit."""
    H = 2
    bs = [Batch(e, [1, 2], [3000, 2500], 2, 64, 16, seed=i) for i, e in enumerate((False, True))]
    qs = [torch.randn(3, H * 64, device="cuda").to(torch.bfloat16) for _ in bs]
    ws = [b.cache.workspace(H, 3, 2, 3000) for b in bs]
    alone = []
    for b, q, w in zip(bs, qs, ws):
        out = torch.zeros_like(q)
        b.cache.attend(q, out, b.q_start, b.kv_len, 2, 3000, workspace=w)
        alone.append(out)
    tb.sync_check()
    streams = [torch.cuda.Stream() for _ in bs]
    outs = [torch.zeros_like(q) for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for b, q, w, o, st in zip(bs, qs, ws, outs, streams):
            with torch.cuda.stream(st):
                b.cache.attend(q, o, b.q_start, b.kv_len, 2, 3000, workspace=w)
    torch.cuda.synchronize()
    for o, a in zip(outs, alone):
        assert torch.equal(o, a)
    tb.sync_check()


def test_one_workspace_for_calls_of_all_sizes_and_types(tb):
    """Single tokens of many and of few CTAs, whole items, chunks in pieces and tiles that are not cut, one after the other."""
    cases = [(False, [1, 1, 1], [5000, 4000, 3000], 64), (True, [1], [9000], 64), (False, [60, 1], [900, 40], 64), (False, [1, 1], [30, 500], 64),
             (True, [1, 1, 1], [5000, 4000, 3000], 128), (False, [200], [3000], 128), (True, [1, 1], [2100, 700], 64), (True, [90, 1], [2000, 1500], 64)]
    bs = [Batch(e, new, kv, 2, dim, 16, seed=i) for i, (e, new, kv, dim) in enumerate(cases)]
    ws = max((b.cache.workspace(4, b.rows, max(b.new), max(b.kv)) for b in bs), key=lambda w: 0 if w is None else w.nbytes)
    for _ in range(2):
        for b in bs:
            q = torch.randn(b.rows, 4 * b.dim, device="cuda").to(torch.bfloat16)
            att, lse = torch.zeros_like(q), torch.zeros(b.rows, 4, device="cuda")
            b.cache.attend(q, att, b.q_start, b.kv_len, max(b.new), max(b.kv), lse=lse, workspace=ws)
            compare(b, 4, q.float().cpu().numpy().reshape(b.rows, 4, b.dim), att.float().cpu().numpy().reshape(b.rows, 4, b.dim), lse.cpu().numpy())
    tb.sync_check()


@pytest.mark.parametrize("e4m3,dim", [(False, 64), (True, 64), (False, 128), (True, 128)])
def test_many_sequences_of_all_kinds(tb, e4m3, dim):
    """More sequences than a warp has lanes and than one look of the single tokens' kernel takes; chunks among them, empty ones too."""
    rng = np.random.default_rng(dim + e4m3)
    new = [int(rng.choice([0, 1, 1, 1, 1, 2, 9])) for _ in range(300)]
    new[17], new[200], new[299] = 150, 40, 33
    kv = [n + int(rng.integers(0, 200)) for n in new]
    kv[0], kv[150], kv[17], kv[31] = new[0] + 2500, new[150] + 3000, 1200, new[31]
    b = Batch(e4m3, new, kv, 2, dim, 32, seed=dim)
    compare(b, 4, *attend(b, 4, seed=10))


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_chunk_among_hundreds_of_single_tokens(tb, e4m3):
    new = [1] * 700
    new[333] = 100
    kv = [n + s % 40 for s, n in enumerate(new)]
    b = Batch(e4m3, new, kv, 16, 64, 16, seed=21)
    compare(b, 16, *attend(b, 16, seed=16))


@pytest.mark.parametrize("e4m3,dim,G", [(False, 64, 16), (True, 64, 8), (True, 128, 8), (False, 128, 8)])
def test_more_tiles_than_the_chip_holds_at_once(tb, e4m3, dim, G):
    new = [130] * 19 + [3]
    kv = [130 + 7 * s for s in range(19)] + [1]
    b = Batch(e4m3, new, kv, G, dim, 64, seed=G)
    compare(b, G, *attend(b, G, seed=11))


def test_replayed_chunks_follow_the_lengths(tb):
    """Two graphs of one workspace, replayed in turn: other chunks, other tiles, other pieces than those of the capture."""
    H, G, rows, bound = 4, 2, 260, 2048
    for e4m3 in (False, True):
        a = Batch(e4m3, [200, 1, 2], [1900, 700, 60], G, 64, 32, seed=1, width=bound // 32)
        b = Batch(e4m3, [17, 1, 240], [30, 2000, 1000], G, 64, 32, seed=2, width=bound // 32)
        ws = a.cache.workspace(H, rows, rows, bound)
        held = []
        for x in (a, b):
            q = torch.randn(rows, H * 64, device="cuda").to(torch.bfloat16)
            att, lse = torch.zeros_like(q), torch.zeros(rows, H, device="cuda")
            lens, starts = torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
            graph = torch.cuda.CUDAGraph()
            x.cache.attend(q, att, starts, lens, rows, bound, lse=lse, workspace=ws)
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                x.cache.attend(q, att, starts, lens, rows, bound, lse=lse, workspace=ws)
            lens.copy_(x.kv_len)
            starts.copy_(x.q_start)
            held.append((x, graph, q, att, lse, lens, starts))
        for _ in range(3):
            for x, graph, q, att, lse, _, _ in held:
                att.zero_()
                graph.replay()
                torch.cuda.synchronize()
                compare(x, H, *(t[:x.rows].float().cpu().numpy().reshape(x.rows, H, -1) for t in (q, att)), lse[:x.rows].cpu().numpy())
                assert (att[x.rows:] == 0).all()
    tb.sync_check()


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("dim", [64, 128])
def test_8_bit_rows_of_very_different_sizes(tb, new, dim):
    """Scales of values over 2^90, of keys over 2^20; queries with one element that is 2^9 times the others."""
    b = Batch(True, [new, 1], [500 + new, 300], 1, dim, 16, seed=dim)
    rng = np.random.default_rng(4)
    b.host["v_scale"][:] = np.ldexp(b.host["v_scale"], rng.integers(-60, 30, b.host["v_scale"].shape))
    b.host["k_scale"][:] = np.ldexp(b.host["k_scale"], rng.integers(-20, 1, b.host["k_scale"].shape))
    b.host["v_scale"][b.table[0, 3], 0, 2] = 0.0
    for n in ("k", "v"):
        b.dev[n + "_scale"].copy_(torch.from_numpy(b.host[n + "_scale"]))
    q = torch.randn(b.rows + 3, 2 * dim).to(torch.bfloat16)
    q[:, 5] *= 512
    q[:, dim + 9] *= 512
    rows, got, lse = attend(b, 2, seed=12, q=q)
    # Beside the bound of other batches: rows go to the tensor cores exact but for 2^-21 of their largest element, against every key.
    # Probabilities are f16.  In chunks, at least 2^7 for a row's largest: off by 2^-25 at most where they are small, which is 2^-32 of the
    # largest, times every value; and values are f16 against the largest scale s, 64 s and more, off by 2^-25 of that 64th: 2^-31 s.  For
    # single tokens, at least 2^13 for the largest product p s: off by 2^-38 of it per key, times a code of 448 at most (2^-29).
    # The logarithm: exponents of up to 2^7 are added to scores of single tokens in float32, half a unit in the last place is 2^-18.
    for s in range(2):
        at = slice(b.starts[s], b.starts[s + 1])
        k, v = b.sequence("k", s), b.sequence("v", s)
        want, want_lse, spread, size = plain.attention(rows[at], k, v, np.arange(b.kv[s] - b.new[s], b.kv[s]), dim ** -0.5)
        more = 2.0 ** -21 * np.abs(rows[at]).max(axis=2) * np.abs(k[:, 0]).sum(axis=1).max() * dim ** -0.5
        score = (dim + 4) * 2.0 ** -24 * size + more
        scales = np.stack([b.host["v_scale"][b.table[s, t // 16], 0, t % 16] for t in range(b.kv[s])]).astype(np.float64)
        if b.new[s] > 16 // 2:
            lost = 2.0 ** -32 * np.abs(v[:, 0]).sum(axis=0)[None, None] + 2.0 ** -31 * scales.max()
        else:
            p = np.exp(np.einsum("td,rhd->rht", k[:, 0], rows[at].astype(np.float64)) * dim ** -0.5 - want_lse[..., None])
            lost = 2.0 ** -29 * b.kv[s] * (p * scales).max(axis=2)[..., None]
        bound = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 * 1.01 + 2 * score[..., None] + 2.0 ** -17) * spread + lost + 1e-30
        assert (np.abs(got[at] - want) <= bound).all(), np.nanmax(np.abs(got[at] - want) / bound)
        assert (np.abs(lse[at] - want_lse) <= score + 2.0 ** -18 + 2.0 ** -20 * (1 + np.abs(want_lse))).all()


@pytest.mark.parametrize("new", [1, 40])
def test_8_bit_values_of_zeros(tb, new):
    """Rows of zeros have the smallest scale there is: many of them, alone, in front of and behind others."""
    for zeros in (slice(0, 400), slice(0, 150), slice(100, 400)):
        b = Batch(True, [new], [300 + new], 1, 64, 16, seed=6)
        for t in range(*zeros.indices(300 + new)):
            b.host["v"][b.table[0, t // 16], 0, t % 16] = 0
            b.host["v_scale"][b.table[0, t // 16], 0, t % 16] = 2.0 ** -126
        b.dev["v"].copy_(torch.from_numpy(b.host["v"]).cuda().view(torch.float8_e4m3fn))
        b.dev["v_scale"].copy_(torch.from_numpy(b.host["v_scale"]))
        compare(b, 2, *attend(b, 2, seed=15))


@pytest.mark.parametrize("new", [1, 40])
def test_codes_that_are_no_numbers(tb, new):
    """A NaN code in a key takes its rows along, one in a value its column, and neither reaches a row that does not see it."""
    for name in ("k", "v"):
        b = Batch(True, [new, 1], [200 + new, 100], 2, 64, 16, seed=3)
        t = 200 + new // 2                                      # rows new // 2 and later see it
        b.host[name][b.table[0, t // 16], 1, t % 16, 7] = 0xff
        b.dev[name].copy_(torch.from_numpy(b.host[name]).cuda().view(torch.float8_e4m3fn))
        q, got, lse = attend(b, 4, seed=13)
        sees = np.zeros((b.rows, 4), bool)
        sees[new // 2:new, 2:] = True                           # query heads 2, 3 read key head 1
        if name == "k":
            assert np.isnan(got[sees]).all() and np.isnan(lse[sees]).all()
        else:
            assert np.isnan(got[sees][:, 7]).all() and np.isfinite(np.delete(got[sees], 7, axis=1)).all() and np.isfinite(lse).all()
        assert np.isfinite(got[~sees]).all() and np.isfinite(lse[~sees]).all()
        clean = Batch(True, [new, 1], [200 + new, 100], 2, 64, 16, seed=3)
        _, other, _ = attend(clean, 4, seed=13)
        assert (got[~sees] == other[~sees]).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("e4m3", [False, True])
def test_a_query_that_is_not_finite_spoils_its_own_row_alone(tb, e4m3, bad):
    b = Batch(e4m3, [40, 1], [100, 60], 1, 64, 16, seed=5)
    q = torch.randn(b.rows + 3, 2 * 64).to(torch.bfloat16)
    clean = attend(b, 2, seed=14, q=q)[1]
    q[7, 64 + 3] = bad
    q[40, 5] = bad
    got = attend(b, 2, seed=14, q=q)[1]
    spoilt = np.zeros((b.rows, 2), bool)
    spoilt[7, 1] = spoilt[40, 0] = True
    assert np.isnan(got[spoilt]).all() and (got[~spoilt] == clean[~spoilt]).all()


# ---------------------------------------------------------------------------------------------- writing and reading

def tables(positions, half, seed=0):
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(half) / max(half, 1))
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("bf16_in", [False, True])
@pytest.mark.parametrize("dim,page,G,H,rot,form", [(64, 16, 6, 6, 64, 0), (64, 32, 2, 6, 64, 1), (64, 16, 1, 4, 20, 1), (16, 64, 3, 3, 16, 0),
                                                   (48, 128, 1, 5, 6, 0), (128, 256, 2, 2, 128, 1), (96, 16, 2, 4, 0, 0), (80, 32, 1, 1, 80, 1),
                                                   (8, 16, 2, 2, 8, 1), (24, 16, 1, 3, 24, 1)])
def test_append_writes_what_the_formula_says_and_nothing_else(tb, e4m3, bf16_in, dim, page, G, H, rot, form):
    if e4m3 and dim % 16:
        pytest.skip("8-bit rows are multiples of 16 elements")
    new, kv = [1, 40, 0, 7, 33, 1], [1, 45, 12, 300, 33, 129]
    b = Batch(e4m3, new, kv, G, dim, page, seed=dim + rot)
    rng = np.random.default_rng(dim + H)
    width = (H + 2 * G) * dim
    x = torch.from_numpy((rng.standard_normal((b.rows + 2, width)) * 10.0 ** rng.uniform(-3, 3, (b.rows + 2, 1))).astype(np.float32))
    x = x.to(torch.bfloat16) if bf16_in else x
    x[3, H * dim:(H + G) * dim] = 0                             # a row of zeros
    pad = 8
    xd = torch.empty(b.rows + 2, width + pad, dtype=x.dtype, device="cuda")[:, :width]
    xd.copy_(x)
    q = torch.full((b.rows + 2, H * dim + pad), 3.0, dtype=torch.bfloat16, device="cuda")
    cos, sin = tables(301, rot // 2)
    args = (torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()) if rot else ()
    b.cache.append(xd, q[:, :H * dim], b.q_start, b.kv_len, *args, form=form)
    tb.sync_check()
    got_q = q.float().cpu().numpy()
    assert (got_q[b.rows:] == 3.0).all() and (got_q[:, H * dim:] == 3.0).all()
    want = {n: (t.copy() if isinstance(t, np.ndarray) else t.clone()) for n, t in b.host.items()}
    x = x.float().numpy()
    for s in range(len(new)):
        for i in range(new[s]):
            r, t = b.starts[s] + i, kv[s] - new[s] + i
            heads = x[r].reshape(H + 2 * G, dim)
            turned = np.concatenate((plain.rotate32(heads[:H + G], cos[t], sin[t], form), heads[H + G:]))
            wq = torch.from_numpy(turned[:H].reshape(-1)).to(torch.bfloat16).float().numpy()
            assert (got_q[r, :H * dim] == wq).all(), (s, i)
            at = b.table[s, t // page], slice(None), t % page
            for name, rows in (("k", turned[H:H + G]), ("v", turned[H + G:])):
                if e4m3:
                    scale = np.maximum((np.abs(rows).max(-1).astype(np.float64) / 448).astype(np.float32), np.float32(2.0 ** -126))
                    want[name][at], want[name + "_scale"][at] = plain.e4m3_codes(rows, scale[:, None]), scale
                else:
                    want[name][at] = torch.from_numpy(rows).to(torch.bfloat16)
    for name in ("k", "v"):
        if e4m3:
            assert (b.dev[name].view(torch.uint8).cpu().numpy() == want[name]).all()
            assert np.array_equal(b.dev[name + "_scale"].cpu().numpy(), want[name + "_scale"], equal_nan=True)
        else:
            assert torch.equal(b.dev[name].cpu().view(torch.int16), want[name].view(torch.int16))


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("at", [1, 2, 3])
def test_append_with_tables_that_begin_anywhere(tb, form, at):
    """Rows of 32 angles are whole 16-byte pieces, the table's first byte need not be: the same result as from an aligned one."""
    b = Batch(False, [1, 70, 30], [9, 100, 30], 2, 64, 16, seed=8)
    x = torch.randn(b.rows, (4 + 4) * 64, device="cuda")
    cos, sin = (torch.from_numpy(t).cuda() for t in tables(128, 32))
    results = []
    for shift in (0, at):
        held = [torch.zeros(128 * 32 + 8, device="cuda") for _ in range(2)]
        views = [h[shift:shift + 128 * 32].view(128, 32) for h in held]
        views[0].copy_(cos)
        views[1].copy_(sin)
        q = torch.zeros(b.rows, 4 * 64, dtype=torch.bfloat16, device="cuda")
        b.dev["k"].zero_()
        b.cache.append(x, q, b.q_start, b.kv_len, *views, form=form)
        tb.sync_check()
        results.append((q, b.dev["k"].clone()))
    for got, want in zip(results[1], results[0]):
        assert torch.equal(got, want)


def test_append_rotates_as_the_projection_epilogue_does(tb):
    """Pairs, whole head: the same angles and pairs as tb_gemm_qkv_rope_bf16 (there on the unrounded float32 product)."""
    T, H, dim = 64, 6, 64
    D = H * dim
    x = torch.randn(T, D, device="cuda").to(torch.bfloat16)
    w = (torch.randn(D, 3 * D, device="cuda") * 0.05).to(torch.bfloat16)
    cos, sin = (torch.from_numpy(t).cuda() for t in tables(T, dim // 2))
    bias = torch.zeros(3 * D, device="cuda")
    fused = torch.empty(3, 1, H, T, dim, dtype=torch.bfloat16, device="cuda")
    tb.gemm_qkv_rope_bf16(x, w, bias, cos, sin, 1, T, H, dim, fused)
    qkv = torch.empty(T, 3 * D, device="cuda")
    tb.gemm_bf16(tb.NN, x, w, T, 3 * D, D, D, 3 * D, C32=qkv, ldc32=3 * D)
    b = Batch(False, [T], [T], H, dim, 64, seed=0)
    q = torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    b.cache.append(qkv, q, b.q_start, b.kv_len, cos, sin)
    k, v = torch.empty_like(q), torch.empty_like(q)
    b.cache.read(b.q_start, k, v)
    tb.sync_check()
    for got, want in zip((q, k, v), fused[:, 0]):
        want = want.permute(1, 0, 2).reshape(T, D)
        # one rounding to bf16 each of sums that differ in their last bits: a step (2^-7) where one falls on the other side
        assert ((got.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 1e-6).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_row_that_is_not_finite_reads_back_as_nan(tb, bad):
    b = Batch(True, [3], [40], 2, 64, 16, seed=4)
    x = torch.randn(3, 6 * 64, device="cuda")
    x[1, 4 * 64 + 5] = bad                                      # value head 0 of row 1, position 38
    q = torch.empty(3, 64 * 2, dtype=torch.bfloat16, device="cuda")
    b.cache.append(x, q, b.q_start, b.kv_len)
    k, v = (torch.empty(40, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    b.cache.read(torch.tensor([0, 40], dtype=torch.int32, device="cuda"), k, v)
    tb.sync_check()
    nan = torch.isnan(torch.cat((k, v), 1)).view(40, 4, 64)
    assert torch.nonzero(nan.any(-1)).tolist() == [[38, 2]] and nan[38, 2].all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,page,G", [(64, 16, 6), (16, 64, 1), (48, 32, 5), (128, 256, 2), (96, 16, 3)])
def test_read_back(tb, e4m3, dim, page, G):
    kv, first, count = [1, 300, 70, 64, 33], [0, 17, 69, 0, 5], [1, 200, 1, 64, 0]
    b = Batch(e4m3, [0] * 5, kv, G, dim, page, seed=dim)
    start = np.concatenate(([0], np.cumsum(count)))
    rows = int(start[-1])
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v, only = (torch.full((rows + 2, G * dim), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    b.cache.read(dev(start), k, v, first=dev(first))
    b.cache.read(dev(start), None, only, first=dev(first))
    tb.sync_check()
    assert torch.equal(only, v)
    for name, got in (("k", k), ("v", v)):
        want = np.concatenate([b.sequence(name, s)[first[s]:first[s] + count[s]].reshape(-1, G * dim) for s in range(5)])
        # code * scale is one float32 product, then bf16
        want = torch.from_numpy(want.astype(np.float32)).to(torch.bfloat16)
        assert torch.equal(got[:rows].cpu(), want)
        assert (got[rows:] == 9.0).all()


def test_bad_pages_and_positions_are_not_written(tb):
    b = Batch(False, [1, 1, 1], [40, 50, 60], 2, 64, 16, seed=2)
    before = b.dev["k"].clone()
    x = torch.randn(3, 6 * 64, device="cuda")
    q = torch.full((3, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    b.table_dev[0, 2] = b.dev["k"].shape[0]
    b.cache.append(x, q, b.q_start, b.kv_len)
    with pytest.raises(tb.TbError, match="code 71"):
        tb.sync_check()
    b.kv_len[1] = 16 * b.table.shape[1] + 1
    b.kv_len[0] = 0
    b.cache.append(x, q, b.q_start, b.kv_len)
    with pytest.raises(tb.TbError, match="code 72"):
        tb.sync_check()
    changed = (b.dev["k"].view(torch.int16) != before.view(torch.int16)).any(-1).any(1).nonzero().tolist()
    want = [[int(b.table[1, 3]), 49 % 16], [int(b.table[2, 3]), 59 % 16]]
    assert sorted(changed) == sorted(want)
    k = torch.full((3, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    b.cache.read(b.q_start, k, None, first=torch.tensor([-1, 1 << 30, 2], dtype=torch.int32, device="cuda"))
    with pytest.raises(tb.TbError, match="code 72"):
        tb.sync_check()
    assert (k[:2] == 9.0).all() and not (k[2] == 9.0).any()


# ---------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("G", [6, 2])
def test_a_text_in_chunks_attends_as_the_whole(tb, e4m3, G):
    """Two texts go through the cache in chunks of different sizes, token by token at the end, rows of both in one call; the
    result is the attention over what was appended, and in bf16 that of tb_attention_fwd over the whole text."""
    H, dim, page = 6, 64, 16
    T = [97, 203]
    chunks = [(64, 100), (1, 100), (30, 0), (1, 1), (1, 2)]
    width = (H + 2 * G) * dim
    b = Batch(e4m3, [0, 0], T, G, dim, page, seed=1)
    cos, sin = (torch.from_numpy(t).cuda() for t in tables(256, dim // 2))
    qkv = [torch.randn(t, width, device="cuda") for t in T]
    done, result, rotated = [0, 0], [[], []], [[], []]
    ws = b.cache.workspace(H, 200, 100, 256)
    for n in chunks:
        rows = torch.cat([qkv[s][done[s]:done[s] + n[s]] for s in (0, 1)])
        done = [done[s] + n[s] for s in (0, 1)]
        q_start = torch.tensor([0, n[0], sum(n)], dtype=torch.int32, device="cuda")
        kv_len = torch.tensor(done, dtype=torch.int32, device="cuda")
        q, att = (torch.empty(sum(n), H * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        b.cache.append(rows, q, q_start, kv_len, cos, sin)
        b.cache.attend(q, att, q_start, kv_len, 100, 256, workspace=ws)
        for s in (0, 1):
            part = slice(0, n[0]) if s == 0 else slice(n[0], sum(n))
            result[s].append(att[part])
            rotated[s].append(q[part])
    tb.sync_check()
    assert done == T
    for s in (0, 1):
        got, q = torch.cat(result[s]), torch.cat(rotated[s])
        k, v = (torch.empty(sum(T), G * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        b.cache.read(torch.tensor([0, T[0], sum(T)], dtype=torch.int32, device="cuda"), k, v)
        part = slice(0, T[0]) if s == 0 else slice(T[0], sum(T))
        if e4m3:
            host = {n: b.dev[n].view(torch.uint8).cpu().numpy() for n in ("k", "v")}
            host.update({n + "_scale": b.dev[n + "_scale"].cpu().numpy() for n in ("k", "v")})
            b.host = host
            keys, values = b.sequence("k", s), b.sequence("v", s)
            # what was written is the projection to within half a step of 8 bits (2^-4)
            wide = qkv[s][:, (H + G) * dim:].double().cpu().numpy().reshape(T[s], G, dim)
            most = np.abs(wide).max(-1, keepdims=True)
            assert (np.abs(values - wide) <= 2.0 ** -4 * np.abs(wide) + 2.0 ** -10 * most / 448 * 1.01).all()
        else:
            keys, values = (x[part].double().cpu().numpy().reshape(T[s], G, dim) for x in (k, v))
        qn = q.double().cpu().numpy().reshape(T[s], H, dim)
        want, _, spread, size = plain.attention(qn, keys, values, np.arange(T[s]), dim ** -0.5)
        assert plain.within(got.double().cpu().numpy().reshape(T[s], H, dim), want, spread, size, dim) <= 1.0
        if not e4m3:
            each = lambda x, heads: x.view(T[s], heads, dim).repeat_interleave(H // heads, 1).permute(1, 0, 2).contiguous()  # noqa: E731
            Q, K, V = each(q, H), each(k[part], G), each(v[part], G)
            att, lse = torch.empty(T[s], H * dim, dtype=torch.bfloat16, device="cuda"), torch.empty(H, T[s], device="cuda")
            tb.attention_fwd(Q, K, V, att, lse, 1, H, T[s], dim, dim ** -0.5)
            tb.sync_check()
            assert plain.within(att.double().cpu().numpy().reshape(T[s], H, dim), want, spread, size, dim) <= 1.0
