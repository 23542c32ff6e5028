"""Rules on logits at the limits of what they are given (tb_logits_adjust)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def dev(*a, dtype=torch.int32):
    return torch.tensor(a, dtype=dtype, device="cuda")


@pytest.mark.parametrize("vocab", [100, 1003])
def test_logits_and_result_side_by_side_in_one_matrix(tb, vocab):
    from turkce_llm_b200.logit_rules import LogitRules
    both = torch.randn(5, 2 * vocab, device="cuda")
    before = both.clone()
    ids = torch.randint(0, vocab, (5, 8), dtype=torch.int32, device="cuda")
    rules = LogitRules(5, vocab, output=ids, output_len=dev(8, 8, 0, 3, 8), presence=torch.full((5,), 2.0, device="cuda"))
    rules.apply(both[:, :vocab], both[:, vocab:])
    tb.sync_check()
    assert torch.equal(both[:, :vocab], before[:, :vocab])
    want = before[:, :vocab].clone()
    for s, n in enumerate((8, 8, 0, 3, 8)):
        t = ids[s, :n].long().unique()
        want[s, t] -= 2.0
    assert torch.equal(both[:, vocab:], want)
    with pytest.raises(tb.TbError, match="overlaps"):
        rules.apply(both[:, :vocab], both[:, vocab - 1:2 * vocab - 1])


@pytest.mark.parametrize("repetition", [2.0 ** -32, 1e-6, 0.7, 1.3, 3.0, 1e6, 2.0 ** 32])
def test_quotients_of_any_size(tb, repetition):
    """Logits from the smallest number to the largest: what float32 division and multiplication give."""
    from turkce_llm_b200.logit_rules import LogitRules
    rng = np.random.default_rng(1)
    vocab = 4000
    z = np.ldexp(1 + rng.random(vocab), rng.integers(-149, 127, vocab)).astype(np.float32) * rng.choice([-1, 1], vocab).astype(np.float32)
    z[:8] = [0.0, -0.0, np.inf, -np.inf, np.finfo(np.float32).max, -np.finfo(np.float32).max, 1e-45, -1e-45]
    ids = torch.arange(vocab, dtype=torch.int32, device="cuda")[None].contiguous()
    out = torch.empty(1, vocab, device="cuda")
    r = np.float32(repetition)
    LogitRules(1, vocab, prompt=ids, prompt_len=dev(vocab), repetition=torch.tensor([float(r)], device="cuda")).apply(torch.from_numpy(z)[None].cuda(), out)
    tb.sync_check()
    with np.errstate(all="ignore"):
        want = np.where(z > 0, z / r, z * r).astype(np.float32)
    got = out[0].cpu().numpy()
    # A quotient by the nearest inverse (half a unit, and half a unit of its own: within two) is corrected by its remainder.  That is exact where it
    # is a multiple of 2^-149, from numbers of 2^-103 on: the nearest number.  Below, what is added is off by its own size at most: within two
    # units.  Above 2^96 the first quotient may be infinite where the nearest one is within two units of it.
    ordinary = (z <= 0) | (np.abs(z) > 2.0 ** -64) & (np.abs(z) < 2.0 ** 64)
    assert np.array_equal(got[ordinary], want[ordinary])
    unit = np.maximum(np.abs(want).astype(np.float64) * 2.0 ** -23, 2.0 ** -149)
    finite = np.isfinite(want) & np.isfinite(got)
    assert (np.abs(got[finite].astype(np.float64) - want[finite]) <= 2 * unit[finite]).all()
    assert (got[~finite] == want[~finite]).all() or (np.abs(want[~finite]) >= np.finfo(np.float32).max * (1 - 2.0 ** -21)).all()


@pytest.mark.parametrize("repetition", [0.0, -1.0, 1e-45, 2.0 ** -33, 1e10, 3.4e38, float("inf"), float("nan")])
def test_a_penalty_outside_its_range_is_left_out_and_reported(tb, repetition):
    """1e-45 and the like made infinities of logits of any size; zero and negative ones mean nothing."""
    from turkce_llm_b200.logit_rules import LogitRules
    z = torch.tensor([[1.5, -2.0, 0.25, 1e-38]], device="cuda").repeat(2, 1)
    ids = torch.tensor([[0, 1, 3, 3]], dtype=torch.int32, device="cuda").repeat(2, 1)
    rules = LogitRules(2, 4, output=ids, output_len=dev(4, 4), repetition=torch.tensor([repetition, 2.0], device="cuda"), presence=torch.tensor([1.0, 0.0], device="cuda"))
    rules.apply(z)
    with pytest.raises(tb.TbError, match="code 81"):
        tb.sync_check()
    assert z[0].tolist() == [0.5, -3.0, 0.25, -1.0] and z[1].tolist() == [0.75, -4.0, 0.25, float(np.float32(1e-38) / np.float32(2))]


def test_empty_arrays_are_no_way_around_a_rule(tb):
    """A mask without words or rows is refused, starts that speak of entries where there are none are reported."""
    from turkce_llm_b200.logit_rules import LogitRules
    for shape in ((0, 4), (3, 0), (2, 4), (3, 3)):
        with pytest.raises(tb.TbError, match="masks have to have"):
            LogitRules(3, 100, mask=torch.zeros(shape, dtype=torch.int32, device="cuda"))
    for shape in ((0, 4), (1, 0)):
        with pytest.raises(tb.TbError, match="masks have to have"):
            LogitRules(3, 100, mask=torch.zeros(shape, dtype=torch.int32, device="cuda"), mask_row=dev(0, 0, 0))
    z = torch.randn(2, 100, device="cuda")
    before = z.clone()
    none = dict(bias_id=torch.zeros(0, dtype=torch.int32, device="cuda"), bias_value=torch.zeros(0, device="cuda"))
    LogitRules(2, 100, bias_start=dev(0, 0, 0), **none).apply(z)
    tb.sync_check()
    LogitRules(2, 100, bias_start=dev(0, 2, 2), **none).apply(z)
    with pytest.raises(tb.TbError, match="code 81"):
        tb.sync_check()
    assert torch.equal(z, before)
