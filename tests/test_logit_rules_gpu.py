"""Penalties, biases and masks on logits (tb_logits_adjust) against the formula in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def formula(z, rules):
    """z float64 [rows, vocab]; rules: lists per row."""
    z = z.astype(np.float64).copy()
    size = np.abs(z)                                             # the largest magnitude on the way, for the error bound
    rows, vocab = z.shape
    for s in range(rows):
        said = [t for t in rules["output"][s] if t < vocab]
        known = sorted(set(said) | {t for t in rules["prompt"][s] if t < vocab})
        r = float(rules["repetition"][s])
        for t in known:
            z[s, t] = z[s, t] / r if z[s, t] > 0 else z[s, t] * r
        size[s] = np.maximum(size[s], np.abs(z[s]))
        for t in set(said):
            c = said.count(t)
            z[s, t] -= float(rules["frequency"][s]) * c
            size[s, t] += abs(float(rules["frequency"][s])) * c
            z[s, t] -= float(rules["presence"][s])
            size[s, t] += abs(float(rules["presence"][s]))
        for t, v in rules["bias"][s]:
            if t < vocab:
                z[s, t] += float(v)
                size[s, t] += abs(float(v))
        if rules["allowed"][s] is not None:
            z[s, ~rules["allowed"][s]] = -np.inf
    return z, size


def make(rows, vocab, seed, prompt=20, output=30, bias=6, masks=3):
    rng = np.random.default_rng(seed)
    pad = vocab + 5                                              # an id that is none
    r = {"repetition": (1 + 0.6 * rng.random(rows)).astype(np.float32), "frequency": (rng.random(rows) - 0.3).astype(np.float32),
         "presence": (rng.random(rows) - 0.3).astype(np.float32)}
    r["repetition"][::3] = 1.0
    arrays = {}
    few = max(1, vocab // 3)
    for name, most in (("prompt", prompt), ("output", output)):
        lens = rng.integers(0, most + 1, rows)
        lens[0] = most
        ids = rng.integers(0, few, (rows, most)) * 3 % vocab
        ids[rng.random(ids.shape) < 0.1] = pad
        r[name] = [list(ids[s, :lens[s]]) for s in range(rows)]
        arrays[name], arrays[name + "_len"] = ids.astype(np.int32), lens.astype(np.int32)
    counts = rng.integers(0, bias + 1, rows) if bias else np.zeros(rows, int)
    r["bias"] = [[(int(rng.integers(0, min(vocab, 7 if s % 2 else vocab))), np.float32(rng.standard_normal())) for _ in range(counts[s])]
                 for s in range(rows)]
    flat = [e for row in r["bias"] for e in row]
    arrays["bias_start"] = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    arrays["bias_id"] = np.array([t for t, _ in flat], np.int32)
    arrays["bias_value"] = np.array([v for _, v in flat], np.float32)
    if not flat:
        arrays["bias_start"] = arrays["bias_id"] = arrays["bias_value"] = None
    r["allowed"] = [None] * rows
    if masks:
        bits = rng.random((masks, vocab)) < rng.random((masks, 1))
        bits[0] = False                                          # a mask that allows nothing
        words = np.zeros((masks, -(-vocab // 32)), np.uint32)
        for v in range(vocab):
            words[:, v // 32] |= bits[:, v].astype(np.uint32) << np.uint32(v % 32)
        row = rng.integers(-1, masks, rows)
        row[-1] = 0
        r["allowed"] = [bits[m] if m >= 0 else None for m in row]
        arrays["mask"], arrays["mask_row"] = words.view(np.int32), row.astype(np.int32)
    arrays.update({n: r[n] for n in ("repetition", "frequency", "presence")})
    return r, {n: torch.from_numpy(a).cuda() for n, a in arrays.items() if a is not None}


def check(got, z, rules):
    want, size = formula(z, rules)
    assert np.array_equal(np.isinf(got), np.isinf(want))
    fine = np.isfinite(want)
    # five roundings of numbers no larger than `size`, and up to 6 additions of biases
    assert (np.abs(got[fine] - want[fine]) <= 12 * 2.0 ** -24 * size[fine]).all()


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31769), (3, 31), (2, 33), (5, 4097), (64, 500), (7, 12289), (2, 150001), (300, 100)])
def test_rules_follow_the_formula(tb, rows, vocab):
    from turkce_llm_b200.logit_rules import LogitRules
    rules, arrays = make(rows, vocab, seed=rows + vocab)
    for ld in (vocab, (vocab + 3) // 4 * 4, vocab + 1):
        z = torch.randn(rows, ld, device="cuda") * 4
        out = torch.full((rows, ld), 9.0, device="cuda")
        r = LogitRules(rows, vocab, **arrays)
        before = z.clone()
        r.apply(z[:, :vocab], out[:, :vocab])
        tb.sync_check()
        assert torch.equal(z, before) and (out[:, vocab:] == 9.0).all()
        check(out[:, :vocab].cpu().numpy(), z[:, :vocab].cpu().numpy(), rules)
        r.apply(z[:, :vocab])                                    # in place: the same bits
        tb.sync_check()
        assert torch.equal(z[:, :vocab], out[:, :vocab]) and torch.equal(z[:, vocab:], before[:, vocab:])


@pytest.mark.parametrize("left_out", [("prompt", "prompt_len"), ("output", "output_len"), ("repetition",), ("frequency", "presence"),
                                      ("bias_start", "bias_id", "bias_value"), ("mask", "mask_row")])
def test_every_rule_may_be_left_out(tb, left_out):
    from turkce_llm_b200.logit_rules import LogitRules
    rows, vocab = 6, 1000
    rules, arrays = make(rows, vocab, seed=3)
    neutral = {"prompt": [[]] * rows, "output": [[]] * rows, "repetition": np.ones(rows), "frequency": np.zeros(rows),
               "presence": np.zeros(rows), "bias_id": None, "mask": None}
    for n in left_out:
        del arrays[n]
        if n == "bias_id":
            rules["bias"] = [[]] * rows
        elif n == "mask":
            rules["allowed"] = [None] * rows
        elif n in neutral:
            rules[n] = neutral[n]
    z = torch.randn(rows, vocab, device="cuda")
    out = torch.empty_like(z)
    LogitRules(rows, vocab, **arrays).apply(z, out)
    tb.sync_check()
    check(out.cpu().numpy(), z.cpu().numpy(), rules)


def test_no_rule_is_a_copy_and_special_values_pass(tb):
    from turkce_llm_b200.logit_rules import LogitRules
    z = torch.tensor([[float("nan"), float("inf"), -float("inf"), -0.0, 1e-42, 3.0]], device="cuda")
    out = torch.empty_like(z)
    LogitRules(1, 6).apply(z, out)
    tb.sync_check()
    assert torch.equal(out.view(torch.int32), z.view(torch.int32))
    # NaN under a mask is gone, a seen NaN stays one
    mask = torch.tensor([[0b111110]], dtype=torch.int32, device="cuda")
    ids = torch.tensor([[1, 2, 5]], dtype=torch.int32, device="cuda")
    n = torch.tensor([3], dtype=torch.int32, device="cuda")
    LogitRules(1, 6, prompt=ids, prompt_len=n, repetition=torch.tensor([2.0], device="cuda"), mask=mask).apply(z, out)
    tb.sync_check()
    assert out[0, 0] == -float("inf") and out[0, 1] == float("inf") and out[0, 2] == -float("inf") and out[0, 5] == 1.5


def test_the_same_token_many_times(tb):
    """A count of thousands, and biases for one token that are added in the order of their list."""
    from turkce_llm_b200.logit_rules import LogitRules
    vocab, n = 700, 5000
    ids = torch.full((1, n), 123, dtype=torch.int32, device="cuda")
    values = torch.tensor([1e8, 1.0, -1e8, 0.5], device="cuda")
    z = torch.zeros(1, vocab, device="cuda")
    dev = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    LogitRules(1, vocab, output=ids, output_len=dev(n), frequency=torch.tensor([0.25], device="cuda"), bias_start=dev(0, 4),
               bias_id=dev(7, 7, 7, 7), bias_value=values).apply(z)
    tb.sync_check()
    want = np.zeros(vocab, np.float32)
    want[123], want[7] = -0.25 * n, 0.5                           # (1e8 + 1 is 1e8 in float32)
    assert (z[0].cpu().numpy() == want).all()


def test_what_lies_outside_its_array_is_left_out_and_reported(tb):
    from turkce_llm_b200.logit_rules import LogitRules
    rows, vocab = 3, 64
    dev = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    z = torch.ones(rows, vocab, device="cuda")
    ids = torch.full((rows, 4), 5, dtype=torch.int32, device="cuda")
    freq = torch.ones(rows, device="cuda")
    mask = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    cases = [dict(output=ids, output_len=dev(4, 100, 1), frequency=freq), dict(mask=mask, mask_row=dev(0, 2, -1)),
             dict(bias_start=dev(0, 1, 9, 2), bias_id=dev(3, 3), bias_value=torch.ones(2, device="cuda"))]
    for case in cases:
        out = torch.full_like(z, 9.0)
        LogitRules(rows, vocab, **case).apply(z, out)
        with pytest.raises(tb.TbError, match="code 81"):
            tb.sync_check()
        out = out.cpu().numpy()
        want = np.ones((rows, vocab), np.float32)
        if "output" in case:
            want[:, 5] = [-3, -3, 0]
        elif "mask" in case:
            want[0] = -np.inf
        else:
            want[0, 3] = 2
        assert (out == want).all()


def test_adjusted_head_and_choice(tb):
    """The LM head's logits with a repeated winner and a mask: the choice moves to where the rules send it."""
    from turkce_llm_b200.logit_rules import LogitRules
    S, V, K = 5, 1000, 128
    x = torch.randn(S, K, device="cuda").to(torch.bfloat16)
    e = torch.randn(V, K, device="cuda").to(torch.bfloat16)
    tok, logits = torch.zeros(S, dtype=torch.int32, device="cuda"), torch.empty(S, V, device="cuda")
    tb.lmhead_argmax_bf16(x, e, tok, logits=logits, ld_logits=V)
    mask = torch.full((1, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")
    mask[0, :16] = 0                                              # tokens from 512 on
    out = torch.empty_like(logits)
    rules = LogitRules(S, V, output=tok[:, None].contiguous(), output_len=torch.ones(S, dtype=torch.int32, device="cuda"),
                       presence=torch.full((S,), 1e6, device="cuda"), mask=mask,
                       mask_row=torch.tensor([0, -1, 0, -1, 0], dtype=torch.int32, device="cuda"))
    rules.apply(logits, out)
    tb.sync_check()
    z = logits.clone()
    z[torch.arange(S), tok.long()] -= 1e6
    z[::2, :512] = -float("inf")
    assert torch.equal(out.argmax(1), z.argmax(1)) and (out.argmax(1) != tok).all()
