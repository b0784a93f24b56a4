"""What a call of the adapters keeps by its sizes and strides: calls that write to different places never share it."""

import pytest
import torch
from adapter_cases import make

from easydel_b200.ops import adapters


@pytest.mark.parametrize("order", [(False, True), (True, False)])
def test_new_results_and_results_in_place_have_plans_of_their_own(order, monkeypatch):
    monkeypatch.setattr(adapters, "_plans", {})
    c = make(6, 16, (32,), 4, 2, torch.bfloat16, "cpu")
    y = torch.zeros(6, 64, dtype=torch.bfloat16)[:, :32]
    other = torch.zeros(6, 48, dtype=torch.bfloat16)[:, :32]
    plan = lambda out: adapters._plan_of(y, c["x"], c["a"], c["b"], c["index"], c["scale"], None, out)  # noqa: E731
    for _ in range(2):
        for in_place in order:
            p = plan(y if in_place else None)
            assert p.shape.ldo == (64 if in_place else 32) and p.shape.ldy == 64
        assert plan(other).shape.ldo == 48


def test_refuses_more_rows_than_a_launch_counts():
    x, y = torch.zeros(1, 1, dtype=torch.bfloat16).expand(2 ** 31, 1), torch.zeros(1, 2, dtype=torch.bfloat16).expand(2 ** 31, 2)
    a, b = torch.zeros(1, 1, 1, dtype=torch.bfloat16), torch.zeros(1, 2, 1, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="rows"):
        adapters._plan_of(y, x, a, b, None, 1.0, None, None)
    assert adapters._plan_of(y[1:], x[1:], a, b, None, 1.0, None, None).T == 2 ** 31 - 1
