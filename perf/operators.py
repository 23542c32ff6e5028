"""What the serving operators are measured on: a paged cache of keys and values that is written (with the position
rotation, in bf16 or in 8 bits), attended to and read back, and the rules that change logits before a token is chosen.

A server that decodes many sequences of different lengths appends the keys and values of a chunk of new tokens to the
cache, lets the chunk attend to all that is cached, and bends the logits of the last rows (penalties for repeated tokens,
biases, grammar masks).  Every case here is one such call.  With `own` false the operators are computed in their plain
form: elementary operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

ROPE_BASE = 10000.0
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -126


def listed():
    return [
        # one user, the next token: nothing but latency.  The model of this repository: 6 heads of 64
        {"name": "append_one_token", "op": "append", "type": "bf16", "input": "f32", "seqs": 1, "new": 1, "context": 300, "ragged": False,
         "singles": 0, "heads": 6, "kv_heads": 6, "dim": 64, "rot": 64, "form": "pairs", "page": 16},
        # prompts of different lengths go into an 8-bit cache; keys shared by three heads each, half of the head rotated
        {"name": "append_prompts_e4m3", "op": "append", "type": "e4m3", "input": "bf16", "seqs": 48, "new": 512, "context": 200, "ragged": True,
         "singles": 0, "heads": 12, "kv_heads": 4, "dim": 64, "rot": 32, "form": "halves", "page": 32},
        # a cached prefix of one conversation is taken out
        {"name": "read_prefix", "op": "read", "type": "bf16", "seqs": 1, "keys": 500, "ragged": False, "kv_heads": 6, "dim": 64, "page": 16},
        # 64 sequences leave an 8-bit cache
        {"name": "read_sequences_e4m3", "op": "read", "type": "e4m3", "seqs": 64, "keys": 1024, "ragged": True, "kv_heads": 6, "dim": 64, "page": 64},
        # one user, the next token, a short conversation
        {"name": "attend_one_token", "op": "attend", "type": "bf16", "seqs": 1, "new": 1, "context": 299, "ragged": False, "singles": 0,
         "heads": 6, "kv_heads": 6, "dim": 64, "page": 16},
        # the benchmark's 64 sequences, each at another place of a longer text
        {"name": "attend_tokens_64", "op": "attend", "type": "bf16", "seqs": 64, "new": 1, "context": 4095, "ragged": True, "singles": 0,
         "heads": 6, "kv_heads": 6, "dim": 64, "page": 16},
        # many users, shared keys in 8 bits
        {"name": "attend_tokens_shared_e4m3", "op": "attend", "type": "e4m3", "seqs": 128, "new": 1, "context": 8191, "ragged": True, "singles": 0,
         "heads": 12, "kv_heads": 2, "dim": 64, "page": 64},
        # 16 prompts of the training context, nothing cached before
        {"name": "attend_prompts", "op": "attend", "type": "bf16", "seqs": 16, "new": 1024, "context": 0, "ragged": False, "singles": 0,
         "heads": 6, "kv_heads": 6, "dim": 64, "page": 64},
        # one chunk of a long prompt, wide heads, 8 bits
        {"name": "attend_chunk_long_e4m3", "op": "attend", "type": "e4m3", "seqs": 2, "new": 512, "context": 16000, "ragged": True, "singles": 0,
         "heads": 8, "kv_heads": 2, "dim": 128, "page": 32},
        # a server's step: the chunk of one prompt beside 32 sequences that decode
        {"name": "attend_mixed", "op": "attend", "type": "bf16", "seqs": 33, "new": 250, "context": 2000, "ragged": True, "singles": 32,
         "heads": 6, "kv_heads": 6, "dim": 64, "page": 16},
        # one user's logits
        {"name": "adjust_one_row", "op": "adjust", "rows": 1, "vocab": 31769, "prompt": 120, "output": 40, "bias": 8, "masks": 0},
        # a server's batch: penalties, biases and a grammar for most rows
        {"name": "adjust_256_rows", "op": "adjust", "rows": 256, "vocab": 31769, "prompt": 1000, "output": 500, "bias": 300, "masks": 40},
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "attend", "adjust"])
    if op == "adjust":
        vocab = _log_int(rng, 300, 150000)
        return {"op": op, "rows": _log_int(rng, 1, max(1, min(256, 8000000 // vocab))), "vocab": vocab, "prompt": _log_int(rng, 1, 2000) - 1,
                "output": _log_int(rng, 1, 1000) - 1, "bias": rng.choice([0, 1, 17, 300]), "masks": rng.choice([0, 1, 40])}
    kv_heads = rng.choice([1, 2, 3, 4, 6])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    dim = rng.choice([16, 32, 48, 64, 64, 64, 96, 128])
    case = {"op": op, "type": rng.choice(["bf16", "e4m3"]), "ragged": rng.random() < 0.7, "kv_heads": kv_heads, "dim": dim,
            "page": rng.choice([16, 16, 32, 64, 128])}
    if op == "read":
        seqs = _log_int(rng, 1, 64)
        case.update(seqs=seqs, keys=_log_int(rng, 1, max(1, min(4096, 13000000 // (seqs * kv_heads * dim)))))
        return case
    seqs = _log_int(rng, 1, 128)
    case.update(seqs=seqs, heads=heads)
    if op == "append":
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, min(1024, 24000 * 12 * 64 // (seqs * heads * dim))))
        case.update(input=rng.choice(["f32", "bf16"]), new=new, context=_log_int(rng, 1, 400) - 1, singles=0,
                    rot=rng.choice([dim, dim, dim // 2, 0]), form=rng.choice(["pairs", "halves"]))
        return case
    if rng.random() < 0.5:
        context = _log_int(rng, 1, max(1, min(16000, 128 * 4000 * 128 // (seqs * kv_heads * dim))))
        case.update(new=rng.choice([1, 1, 1, 2, 4]), context=context - 1, singles=0)
    else:
        # no more pairs of a query and a key than in the largest listed cases
        new = _log_int(rng, 5, 1024)
        seqs = max(1, min(seqs, 16 * 1024 // new))
        context = _log_int(rng, 1, max(1, min(16000, 2000000000 // (seqs * new * heads * dim))))
        case.update(seqs=seqs, new=new, context=context - 1, singles=rng.choice([0, 0, seqs // 2]))
    return case


# ---------------------------------------------------------------------------------------------- the shape of a batch

def _lengths(count, most, ragged, turn):
    """Whole numbers up to `most`: all equal, or spread over the range with the first the largest."""
    if not ragged:
        return [most] * count
    return [most] + [max(1, int(most * ((i * 0.6180339887 + turn) % 1.0))) if most else 0 for i in range(1, count)]


def _batch(case):
    """(new tokens, cached keys with them) of every sequence."""
    if case["op"] == "read":
        keys = _lengths(case["seqs"], case["keys"], case["ragged"], 0.1)
        return keys, keys
    new = _lengths(case["seqs"], case["new"], case["ragged"], 0.1)
    if case["singles"]:
        new[-case["singles"]:] = [1] * case["singles"]
    before = _lengths(case["seqs"], case["context"], case["ragged"], 0.4)
    return new, [n + b for n, b in zip(new, before)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _zipf(gen, shape, vocab):
    """Token ids, Zipf(1.1) over the vocabulary."""
    cdf = torch.cumsum(torch.arange(1, vocab + 1, device="cuda", dtype=torch.float64) ** -1.1, 0)
    u = torch.rand(shape, device="cuda", dtype=torch.float64, generator=gen) * cdf[-1]
    return torch.searchsorted(cdf, u).clamp_(max=vocab - 1).to(torch.int32)


def prepare(case, seed):
    gen = _generator(seed)
    s = {"op": case["op"], "case": case}
    if case["op"] == "adjust":
        _prepare_adjust(s, case, gen)
        return s
    new, kv = _batch(case)
    page, dim, kv_heads = case["page"], case["dim"], case["kv_heads"]
    width = max(1, max(-(-n // page) for n in kv))
    used = sum(-(-n // page) for n in kv)
    pages = used + 3
    # pages in no order; behind a sequence's last page the table holds whatever was there
    order = torch.randperm(pages, device="cuda", generator=gen)[:used].to(torch.int32)
    table = torch.zeros(case["seqs"], width, device="cuda", dtype=torch.int32)
    filled = torch.arange(width, device="cuda")[None] < _ints([-(-n // page) for n in kv])[:, None]
    table[filled] = order
    s.update(table=table, kv_len=_ints(kv), q_start=_ints(_starts(new)), rows=sum(new), max_q=max(new), max_kv=max(kv), page=page)
    shape = (pages, kv_heads, page, dim)
    if case["type"] == "e4m3":
        # scales as rows of keys and values have them: the largest of a row's numbers over the largest of the format
        for name in ("k", "v"):
            x = _normal(gen, *shape)
            scale = (x.abs().amax(-1) / E4M3_MAX).clamp_(min=SMALLEST_SCALE)
            s[name], s[name + "_scale"] = (x / scale[..., None]).to(torch.float8_e4m3fn), scale
    else:
        for name in ("k", "v"):
            s[name], s[name + "_scale"] = _normal(gen, *shape).to(torch.bfloat16), None
    if case["op"] == "append":
        heads = case["heads"]
        qkv = _normal(gen, s["rows"], (heads + 2 * kv_heads) * dim)
        s["qkv"] = qkv if case["input"] == "f32" else qkv.to(torch.bfloat16)
        s["q"] = torch.empty(s["rows"], heads * dim, device="cuda", dtype=torch.bfloat16)
        half = case["rot"] // 2
        if half:
            angle = torch.arange(s["max_kv"], device="cuda", dtype=torch.float64)[:, None] * \
                ROPE_BASE ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
            s.update(cos=angle.cos().float(), sin=angle.sin().float())
        else:
            s.update(cos=None, sin=None)
    elif case["op"] == "attend":
        s["q"] = _normal(gen, s["rows"], case["heads"] * dim).to(torch.bfloat16)
        s["att"] = torch.empty(s["rows"], case["heads"] * dim, device="cuda", dtype=torch.bfloat16)
        s["lse"] = torch.empty(s["rows"], case["heads"], device="cuda")
    else:
        s["out"] = [torch.empty(s["rows"], kv_heads * dim, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    if own:
        from turkce_llm_b200 import lib
        from turkce_llm_b200.paged import PagedCache
        lib.init(0)
        s["cache"] = PagedCache(s["k"], s["v"], table, k_scale=s["k_scale"], v_scale=s["v_scale"])
        s["form"] = {"pairs": lib.ROPE_PAIRS, "halves": lib.ROPE_HALVES}[case.get("form", "pairs")]
        if case["op"] == "attend":
            s["workspace"] = s["cache"].workspace(case["heads"], s["rows"], s["max_q"], s["max_kv"])
    return s


def _prepare_adjust(s, case, gen):
    rows, vocab = case["rows"], case["vocab"]
    s["logits"] = _normal(gen, rows, vocab) * 3
    s["out"] = torch.empty_like(s["logits"])
    for name, turn in (("prompt", 0.2), ("output", 0.7)):
        lens = _lengths(rows, case[name], True, turn)
        s[name] = _zipf(gen, (rows, max(1, case[name])), vocab)
        s[name + "_len"] = _ints(lens)
    # some rows without a penalty, as in a batch of different users
    s["repetition"] = 1.0 + 0.5 * torch.rand(rows, device="cuda", generator=gen) * (torch.arange(rows, device="cuda") % 4 != 3)
    s["frequency"] = 0.5 * torch.rand(rows, device="cuda", generator=gen)
    s["presence"] = torch.rand(rows, device="cuda", generator=gen) - 0.3
    s["bias_start"] = s["bias_id"] = s["bias_value"] = s["mask"] = s["mask_row"] = None
    if case["bias"]:
        counts = _lengths(rows, case["bias"], True, 0.5)
        s["bias_start"] = _ints(_starts(counts))
        s["bias_id"] = torch.randint(vocab, (sum(counts),), device="cuda", generator=gen).to(torch.int32)
        s["bias_value"] = _normal(gen, sum(counts)) * 2
    if case["masks"]:
        # a grammar's states: some allow a handful of tokens, some half of the vocabulary
        words = -(-vocab // 32)
        share = torch.rand(case["masks"], 1, 1, device="cuda", generator=gen) ** 3
        bits = (torch.rand(case["masks"], words, 32, device="cuda", generator=gen) < share).to(torch.int64)
        s["mask"] = (bits << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)
        row = torch.randint(case["masks"], (rows,), device="cuda", generator=gen).to(torch.int32)
        s["mask_row"] = torch.where(torch.arange(rows, device="cuda") % 5 == 4, torch.full_like(row, -1), row)
    if own:
        from turkce_llm_b200 import lib
        from turkce_llm_b200.logit_rules import LogitRules
        lib.init(0)
        names = ("prompt", "prompt_len", "output", "output_len", "repetition", "frequency", "presence", "bias_start", "bias_id",
                 "bias_value", "mask", "mask_row")
        s["rules"] = LogitRules(rows, vocab, **{n: s[n] for n in names})


# ---------------------------------------------------------------------------------------------- one pass

def run(s):
    if s["op"] == "append":
        if own:
            s["cache"].append(s["qkv"], s["q"], s["q_start"], s["kv_len"], s["cos"], s["sin"], form=s["form"])
        else:
            _plain_append(s)
        out = {"q": s["q"], "k": s["k"], "v": s["v"]}
        return out if s["k_scale"] is None else {**out, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if s["op"] == "attend":
        if own:
            s["cache"].attend(s["q"], s["att"], s["q_start"], s["kv_len"], s["max_q"], s["max_kv"], lse=s["lse"], workspace=s["workspace"])
            return {"att": s["att"], "lse": s["lse"]}
        return _plain_attend(s)
    if s["op"] == "read":
        if own:
            s["cache"].read(s["q_start"], s["out"][0], s["out"][1])
            return {"k": s["out"][0], "v": s["out"][1]}
        return _plain_read(s)
    if own:
        s["rules"].apply(s["logits"], s["out"])
        return s["out"]
    return _plain_adjust(s)


# ---------------------------------------------------------------------------------------------- plain forms

def _rows_of(s):
    """Sequence of every row and its position in the sequence's text."""
    row = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["q_start"], row, right=True) - 1
    end = s["q_start"].long()[seq + 1]
    return seq, s["kv_len"].long()[seq] - end + row


def _rotate(x, cos, sin, form):
    """x [rows, heads, dim]; cos, sin [rows, 1, half]: pairs of neighbours, or of the two halves of the rotated part."""
    if cos is None:
        return x
    half = cos.shape[-1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if form == "pairs" else (turned[..., :half], turned[..., half:])
    c, d = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((c, d), -1).flatten(-2) if form == "pairs" else torch.cat((c, d), -1)
    return torch.cat((turned, rest), -1)


def _plain_append(s):
    case, page = s["case"], s["page"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    seq, pos = _rows_of(s)
    x = s["qkv"].float().view(-1, H + 2 * G, D)
    cos, sin = (None, None) if s["cos"] is None else (s["cos"][pos][:, None], s["sin"][pos][:, None])
    s["q"].copy_(_rotate(x[:, :H], cos, sin, case["form"]).reshape(s["rows"], H * D))
    at = s["table"].long()[seq, pos // page], slice(None), pos % page
    _write(s, "k", at, _rotate(x[:, H:H + G], cos, sin, case["form"]))
    _write(s, "v", at, x[:, H + G:])


def _write(s, name, at, x):
    """x [rows, heads, dim] in the cache's type: in 8 bits with one scale for every row of a head."""
    if s[name + "_scale"] is None:
        s[name][at] = x.to(torch.bfloat16)
        return
    scale = (x.abs().amax(-1).double() / E4M3_MAX).float().clamp_(min=SMALLEST_SCALE)
    s[name + "_scale"][at] = scale
    # The nearest code, halves to the even one.  In 64 bits: many quotients of bf16 rows lie next to the middle of two codes
    q = x.double() / scale.double()[..., None]
    codes = torch.arange(127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    middle = (codes[1:] + codes[:-1]) / 2
    code = torch.bucketize(q.abs(), middle)
    code += (code % 2 == 1) & (q.abs() == middle[code.clamp(max=125)])
    s[name].view(torch.uint8)[at] = code.to(torch.uint8) | (q.signbit().to(torch.uint8) << 7)


def _cached(s, name, most):
    """[sequences, most, heads, dim] in 32 bits, and where they are keys of the sequence."""
    j = torch.arange(most, device="cuda")
    page = s["table"].long()[:, j // s["page"]]
    at = page, slice(None), (j % s["page"])[None].expand_as(page)
    x = s[name][at].float()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][at][..., None]
    return x, j[None] < s["kv_len"][:, None]


def _plain_read(s):
    k, there = _cached(s, "k", s["max_kv"])
    v, _ = _cached(s, "v", s["max_kv"])
    return {"k": k[there].flatten(1).to(torch.bfloat16), "v": v[there].flatten(1).to(torch.bfloat16)}


def _plain_attend(s):
    case = s["case"]
    B, H, G, D, most_q, most_kv = case["seqs"], case["heads"], case["kv_heads"], case["dim"], s["max_q"], s["max_kv"]
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    new = start[1:] - start[:-1]
    i = torch.arange(most_q, device="cuda")
    rows = (start[:-1, None] + i).clamp(max=s["rows"] - 1)
    # [B, G, heads of a group x new tokens, D]
    q = s["q"][rows].float().view(B, most_q, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * most_q, D)
    k, there = _cached(s, "k", most_kv)
    z = (q @ k.permute(0, 2, 3, 1)).view(B, G, H // G, most_q, most_kv).mul_(1.0 / math.sqrt(D))
    del k
    pos = (kv_len - new)[:, None] + i
    seen = (torch.arange(most_kv, device="cuda") <= pos[..., None]) & there[:, None]
    z.masked_fill_(~seen[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = z.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v, _ = _cached(s, "v", most_kv)
    o = (p.view(B, G, H // G * most_q, most_kv) @ v.permute(0, 2, 1, 3)).view(B, G, H // G, most_q, D) / total
    lse = (total.log() + top).squeeze(-1)
    valid = i[None] < new[:, None]
    return {"att": o.permute(0, 3, 1, 2, 4)[valid].reshape(s["rows"], H * D).to(torch.bfloat16),
            "lse": lse.permute(0, 3, 1, 2)[valid].reshape(s["rows"], H)}


def _seen(s, name):
    """How often every token of the vocabulary is among the first `len` ids of each row."""
    ids, vocab = s[name].long(), s["case"]["vocab"]
    there = (torch.arange(ids.shape[1], device="cuda") < s[name + "_len"][:, None]) & (ids < vocab)
    return torch.zeros(ids.shape[0], vocab, device="cuda", dtype=torch.int32).scatter_add_(1, ids.clamp(max=vocab - 1), there.int())


def _plain_adjust(s):
    z = s["logits"]
    often, before = _seen(s, "output"), _seen(s, "prompt")
    r = s["repetition"][:, None]
    z = torch.where((often > 0) | (before > 0), torch.where(z > 0, z / r, z * r), z)
    z = z - s["frequency"][:, None] * often
    z = z - s["presence"][:, None] * (often > 0)
    if s["bias_id"] is not None:
        at = torch.arange(s["bias_id"].numel(), device="cuda", dtype=torch.int32)
        row = torch.searchsorted(s["bias_start"], at, right=True) - 1
        z = z + torch.zeros_like(z).index_put_((row, s["bias_id"].long()), s["bias_value"], accumulate=True)
    if s["mask"] is not None:
        bits = (s["mask"][..., None] >> torch.arange(32, device="cuda")) & 1
        allowed = bits.bool().flatten(1)[:, :z.shape[1]][s["mask_row"].long().clamp(min=0)] | (s["mask_row"] < 0)[:, None]
        z = z.masked_fill(~allowed, -math.inf)
    return z


# ---------------------------------------------------------------------------------------------- what a pass cannot do without

def _row_bytes(case):
    """One key or value of one head in the cache."""
    return case["dim"] * 2 if case["type"] == "bf16" else case["dim"] + 4


def work(case):
    if case["op"] == "adjust":
        S, V = case["rows"], case["vocab"]
        ids = sum(sum(_lengths(S, case[n], True, t)) for n, t in (("prompt", 0.2), ("output", 0.7)))
        bias = sum(_lengths(S, case["bias"], True, 0.5)) if case["bias"] else 0
        return {"bytes": 8 * S * V + 4 * ids + 8 * bias + min(S, case["masks"]) * 4 * -(-V // 32), "flops": 4.0 * S * V}
    new, kv = _batch(case)
    rows, D, G = sum(new), case["dim"], case["kv_heads"]
    tables = 4 * sum(-(-n // case["page"]) for n in kv) + 8 * case["seqs"]
    if case["op"] == "read":
        return {"bytes": 2 * rows * G * (_row_bytes(case) + 2 * D) + tables, "flops": 2.0 * rows * G * D}
    H = case["heads"]
    if case["op"] == "append":
        size = 4 if case["input"] == "f32" else 2
        move = rows * (H + 2 * G) * D * size + rows * H * D * 2 + 2 * rows * G * _row_bytes(case) + rows * case["rot"] * 4
        return {"bytes": move + 4 * rows + 8 * case["seqs"], "flops": 3.0 * rows * (H + G) * case["rot"]}
    pairs = sum(n * (k - n) + n * (n + 1) / 2 for n, k in zip(new, kv))
    return {"bytes": 4 * rows * H * D + 4 * rows * H + 2 * sum(kv) * G * _row_bytes(case) + tables, "flops": 4.0 * pairs * H * D}


# ---------------------------------------------------------------------------------------------- the definitions, in 64 bits

def _to_e4m3(x):
    """The nearest number with four bits of significand and exponents from -6, halves to even; beyond the largest: the largest."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -40)))
    exponent = torch.where(x.abs() >= torch.exp2(exponent + 1), exponent + 1, exponent)
    exponent = torch.where(x.abs() < torch.exp2(exponent), exponent - 1, exponent).clamp(min=-6)
    step = torch.exp2(exponent - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adjust":
        return _exact_adjust(s, case)
    new, kv = _batch(case)
    page, D, G = case["page"], case["dim"], case["kv_heads"]
    table = s["table"].long()
    wide = {n: s[n].double() for n in ("k", "v")}

    def gathered(name, b):
        j = torch.arange(kv[b], device="cuda")
        x = s[name][table[b, j // page], :, j % page].double()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][table[b, j // page], :, j % page].double()[..., None]
        return x                                                     # [keys, heads, dim]

    if case["op"] == "read":
        return {n: torch.cat([gathered(n, b).reshape(-1, G * D) for b in range(case["seqs"])]) for n in ("k", "v")}
    H = case["heads"]
    if case["op"] == "attend":
        att, lse, first = [], [], 0
        for b in range(case["seqs"]):
            k, v = gathered("k", b), gathered("v", b)
            q = s["q"][first:first + new[b]].double().view(new[b], H, D)
            first += new[b]
            hidden = torch.arange(kv[b], device="cuda")[None] > torch.arange(new[b], device="cuda")[:, None] + kv[b] - new[b]
            o, l = [], []
            for h in range(H):
                z = (q[:, h] @ k[:, h * G // H].T / D ** 0.5).masked_fill_(hidden, -math.inf)
                l.append(torch.logsumexp(z, -1))
                o.append(torch.softmax(z, -1) @ v[:, h * G // H])
            att.append(torch.stack(o, 1).flatten(1))
            lse.append(torch.stack(l, 1))
        return {"att": torch.cat(att), "lse": torch.cat(lse)}
    out = {"q": [], "k": wide["k"], "v": wide["v"]}
    if case["type"] == "e4m3":
        out.update(k_scale=s["k_scale"].double(), v_scale=s["v_scale"].double())
    half, first = case["rot"] // 2, 0
    for b in range(case["seqs"]):
        pos = torch.arange(kv[b] - new[b], kv[b], device="cuda")
        x = s["qkv"][first:first + new[b]].double().view(new[b], H + 2 * G, D)
        first += new[b]
        if half:
            turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
            e = torch.arange(half, device="cuda")
            i, j = (2 * e, 2 * e + 1) if case["form"] == "pairs" else (e, half + e)
            y = torch.complex(x[:, :H + G, i], x[:, :H + G, j]) * turn
            x[:, :H + G, i], x[:, :H + G, j] = y.real, y.imag
        out["q"].append(x[:, :H].flatten(1))
        for name, rows in (("k", x[:, H:H + G]), ("v", x[:, H + G:])):
            at = table[b, pos // page], slice(None), pos % page
            if case["type"] == "e4m3":
                # (a scale is what the cache holds: a number of 32 bits)
                scale = (rows.abs().amax(-1) / E4M3_MAX).clamp(min=SMALLEST_SCALE).float().double()
                out[name + "_scale"][at] = scale
                rows = _to_e4m3(rows / scale[..., None])
            out[name][at] = rows
    out["q"] = torch.cat(out["q"])
    return out


def _exact_adjust(s, case):
    z = s["logits"].double()
    for b in range(case["rows"]):
        said = s["output"][b, :s["output_len"][b]].long()
        known = torch.unique(torch.cat((said, s["prompt"][b, :s["prompt_len"][b]].long())))
        r = float(s["repetition"][b])
        z[b, known] = torch.where(z[b, known] > 0, z[b, known] / r, z[b, known] * r)
        token, count = torch.unique(said, return_counts=True)
        z[b, token] -= float(s["frequency"][b]) * count + float(s["presence"][b])
        if case["bias"]:
            a, e = int(s["bias_start"][b]), int(s["bias_start"][b + 1])
            z[b].index_put_((s["bias_id"][a:e].long(),), s["bias_value"][a:e].double(), accumulate=True)
        if case["masks"] and int(s["mask_row"][b]) >= 0:
            word = s["mask"][int(s["mask_row"][b])].long() & 0xffffffff
            v = torch.arange(case["vocab"], device="cuda")
            z[b, ((word[v // 32] >> (v % 32)) & 1) == 0] = -math.inf
    return z
