"""Rules for the next token on CPU: the plain form and its refusals."""

import pytest
import torch
from logit_rule_cases import check, exact, make

from easydel_b200.ops import serving


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", [dict(), dict(penalties=False), dict(biases=0), dict(masked=False), dict(penalties=False, biases=0, masked=False)])
def test_plain_form(dtype, what):
    c = make(6, 77, dtype, "cpu", **what)
    got = serving.adjust_logits(c["logits"], **c["kw"])
    assert got.dtype == torch.float32
    check(got, *exact(c))
    z = c["logits"].clone()
    want, mag = exact(c)
    assert serving.adjust_logits(z, out=z, **c["kw"]) is z
    check(z, want, mag)


def test_forbidden_tokens_and_masks_cover_what_is_not_finite():
    z = torch.tensor([[float("nan"), float("inf"), 1.0, 2.0]])
    bias = (torch.tensor([0, 2], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), torch.tensor([-float("inf")] * 2))
    got = serving.adjust_logits(z, bias=bias)
    assert got.tolist() == [[-float("inf"), -float("inf"), 1.0, 2.0]]
    got = serving.adjust_logits(z, mask=(torch.tensor([[0b1000]], dtype=torch.int32), None))
    assert got.tolist() == [[-float("inf")] * 3 + [2.0]]


@pytest.mark.parametrize("kw", [
    dict(presence=torch.zeros(3)), dict(presence=torch.zeros(2, dtype=torch.float64)), dict(count_rows=torch.zeros(2, dtype=torch.int32)),
    dict(counts=torch.zeros(2, 9, dtype=torch.int32)), dict(counts=torch.zeros(1, 10, dtype=torch.int32)), dict(counts=torch.zeros(2, 10)),
    dict(bias=(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1))),
    dict(bias=(torch.zeros(3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2))),
    dict(bias=(torch.zeros(3, dtype=torch.int32), torch.zeros(1, dtype=torch.int64), torch.zeros(1))),
    dict(bias=(torch.zeros(3, dtype=torch.int32), None, None)),
    dict(mask=(torch.zeros(1, 1, dtype=torch.int32), None)), dict(mask=(torch.zeros(2, 0, dtype=torch.int32), None)),
    dict(mask=(torch.zeros(2, 1, dtype=torch.int64), None)), dict(mask=(torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2))),
    dict(out=torch.zeros(2, 9)), dict(out=torch.zeros(2, 10, dtype=torch.float64)),
])
def test_refusals(kw):
    with pytest.raises(ValueError):
        serving.adjust_logits(torch.zeros(2, 10), **kw)
    with pytest.raises(ValueError):
        serving.adjust_logits(torch.zeros(2, 10, dtype=torch.float16))
