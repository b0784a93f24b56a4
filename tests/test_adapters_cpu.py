"""Adapters of many requests on CPU: the plain form, its gradients, refusals."""

import pytest
import torch
from adapter_cases import check, exact, make

from easydel_b200.ops import adapters


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("parts,r", [((24,), 4), ((16, 8, 8), 3)])
@pytest.mark.parametrize("index", ["none", "mixed", "bare"])
def test_plain_form_and_gradients(dtype, parts, r, index):
    c = make(13, 20, parts, r, 1 if index == "none" else 3, dtype, "cpu", index)
    x, y, a, b = (c[k].requires_grad_() for k in ("x", "y", "a", "b"))
    out = adapters.lora_add(y, x, a, b, c["index"], c["scale"], parts=parts)
    out.backward(c["dy"])
    val, mag = exact({k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in c.items()}, grads=True)
    for name, got, length in (("out", out.detach(), 20), ("dx", x.grad, 32), ("da", a.grad, 13), ("db", b.grad, 13)):
        check(got, val[name], mag[name], length, name)
    assert torch.equal(y.grad, c["dy"])


def test_gradients_against_differences():
    c = make(6, 5, (4, 3), 2, 2, torch.float64, "cpu")
    leaves = [c[k].requires_grad_() for k in ("y", "x", "a", "b")]
    f = lambda y, x, a, b: adapters.lora_add_reference(y, x, a, b, c["index"], c["scale"], parts=c["parts"])  # noqa: E731
    assert torch.autograd.gradcheck(f, leaves)


def test_leading_dimensions_out_and_empty():
    c = make(6, 8, (8,), 2, 2, torch.float32, "cpu")
    flat = adapters.lora_add(c["y"], c["x"], c["a"], c["b"], c["index"], c["scale"])
    cube = adapters.lora_add(c["y"].view(2, 3, 8), c["x"].view(2, 3, 8), c["a"], c["b"], c["index"], c["scale"])
    assert torch.equal(cube.view(6, 8), flat)
    y = c["y"].clone()
    assert adapters.lora_add(y, c["x"], c["a"], c["b"], c["index"], c["scale"], out=y) is y and torch.equal(y, flat)
    none = adapters.lora_add(c["y"][:0], c["x"][:0], c["a"], c["b"], c["index"][:0], c["scale"])
    assert none.shape == (0, 8)


@pytest.mark.parametrize("change,error", [
    (dict(a=lambda c: c["a"][0]), ValueError),
    (dict(a=lambda c: c["a"][:, :1]), ValueError),
    (dict(a=lambda c: c["a"][:, :, :4]), ValueError),
    (dict(b=lambda c: c["b"][:1]), ValueError),
    (dict(y=lambda c: c["y"][:, :7]), ValueError),
    (dict(y=lambda c: c["y"].half()), TypeError),
    (dict(x=lambda c: c["x"].half()), TypeError),
    (dict(a=lambda c: c["a"].bfloat16()), TypeError),
    (dict(index=lambda c: c["index"].long()), ValueError),
    (dict(index=lambda c: c["index"][:-1]), ValueError),
    (dict(index=lambda c: None), ValueError),
    (dict(scale=lambda c: c["scale"].double()), ValueError),
    (dict(scale=lambda c: c["scale"][:1]), ValueError),
    (dict(scale=lambda c: c["scale"].clone().requires_grad_()), NotImplementedError),
    (dict(parts=lambda c: (8, 8)), ValueError),
    (dict(parts=lambda c: (8, 0)), ValueError),
    (dict(out=lambda c: torch.zeros(6, 8, dtype=torch.bfloat16)), ValueError),
])
def test_refusals(change, error):
    c = make(6, 8, (8,), 2, 2, torch.float32, "cpu")
    kw = {k: c[k] for k in ("y", "x", "a", "b", "index", "scale")}
    kw.update({k: f(c) for k, f in change.items()})
    with pytest.raises(error):
        adapters.lora_add(**kw)


def test_refuses_too_many_ranks_and_out_with_gradients():
    c = make(2, 8, (8,), 513, 1, torch.float32, "cpu")
    with pytest.raises(ValueError, match="512"):
        adapters.lora_add(c["y"], c["x"], c["a"], c["b"], c["index"])
    c = make(2, 8, (8,), 2, 1, torch.float32, "cpu")
    with pytest.raises(ValueError, match="inference"):
        adapters.lora_add(c["y"], c["x"].requires_grad_(), c["a"], c["b"], c["index"], out=c["y"])
