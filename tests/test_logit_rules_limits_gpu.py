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
