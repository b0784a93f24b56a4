"""Calls of the adapters one after the other, and rows of one block in every order, against the formulas in 64 bits."""

import pytest
import torch
from adapter_cases import check, exact, make

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _call(c, **kw):
    from easydel_b200.ops import adapters

    return adapters.lora_add(c["y"], c["x"], c["a"], c["b"], c["index"], c["scale"], parts=c["parts"], **kw)


@pytest.mark.parametrize("T", [6, 300, 700])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("order", [("new", "in place", "grad"), ("in place", "new", "grad"), ("in place", "grad", "new")])
def test_new_results_and_results_in_place_of_one_strided_y(order, dtype, T, monkeypatch):
    from easydel_b200.ops import adapters

    monkeypatch.setattr(adapters, "_plans", {})
    c = make(T, 64, (32,), 8, 3, dtype, "cuda")
    want, mag = exact(c)
    wide = torch.full((T, 64), 7.0, dtype=dtype, device="cuda")
    plain = c["y"]
    for how in order:
        wide[:, :32] = plain
        c["y"] = wide[:, :32]
        if how == "in place":
            assert _call(c, out=c["y"]) is c["y"]
            check(wide[:, :32], want, mag, 64, how)
        elif how == "new":
            got = _call(c)
            assert got.stride() == (32, 1)
            check(got, want, mag, 64, how)
        else:
            got = _call(dict(c, x=c["x"].detach().requires_grad_()))
            check(got.detach(), want, mag, 64, how)
        assert (wide[:, 32:] == 7.0).all(), how
