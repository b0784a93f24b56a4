"""Adapters of float32 rows keep all bits of their operands: results against 64 bits, within a bound that a lost part breaks."""

import pytest
import torch
from adapter_bits import bound, make
from adapter_cases import exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 8, 300, 700])
@pytest.mark.parametrize("K,widths,r", [(64, (64,), 16), (512, (96, 32), 8), (1024, (256,), 32), (33, (7,), 5), (4096, (48,), 64)])
def test_float32_keeps_its_bits(T, K, widths, r):
    from easydel_b200.ops import adapters

    c = make(T, K, widths, r, 2, "cuda")
    leaf = {k: c[k].detach().requires_grad_() for k in ("x", "a", "b")}
    out = adapters.lora_add(c["y"], leaf["x"], leaf["a"], leaf["b"], c["index"], c["scale"], parts=c["parts"])
    out.backward(c["dy"])
    val, _ = exact(c, grads=True)
    N = sum(widths)
    for name, got, top in (("out", out.detach(), bound(K, None, r)), ("dx", leaf["x"].grad, bound(N, None, len(widths) * r)),
                           ("da", leaf["a"].grad, bound(N, T, r)), ("db", leaf["b"].grad, bound(K, T, r))):
        off = (got.double().cpu() - val[name]).abs()
        assert (off <= top * val[name]).all(), (name, float((off / val[name].clamp(min=1e-300)).max() / top))


def test_float32_values_near_the_largest():
    from easydel_b200.ops import adapters

    c = make(9, 64, (32,), 8, 2, "cuda")
    c["x"][3, 5] = torch.finfo(torch.float32).max            # rounds to infinity in bf16
    c["a"] *= 2.0 ** -80
    c["b"] *= 2.0 ** -30
    want, _ = exact(c)
    got = adapters.lora_add(c["y"], c["x"], c["a"], c["b"], c["index"], c["scale"])
    assert ((got.double().cpu() - want).abs() <= bound(64, None, 8) * want).all()
    c["x"][4, 6], c["x"][5, 7] = float("inf"), float("nan")
    got = adapters.lora_add(c["y"], c["x"], c["a"], c["b"], c["index"], c["scale"])
    rows = torch.ones(9, dtype=torch.bool)
    rows[4:6] = False
    assert not torch.isfinite(got[4:6]).any() and ((got.double().cpu() - want).abs() <= bound(64, None, 8) * want)[rows].all()


@pytest.mark.parametrize("T", [4, 600])
def test_two_parts_of_the_inner_value_are_rounded(T):
    """bf16 rows: u is (1 + 2^-7 - 2^-17, 1 + 2^-7) and out their difference. Rounded to nearest, the first part is 1 + 2^-7 and the second
    holds what is left; cut off, the first is 1 and the second would need sixteen bits."""
    from easydel_b200.ops import adapters

    zeros = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    x, a, b, y = zeros(T, 64), zeros(1, 8, 64), zeros(1, 32, 8), zeros(T, 32)
    x[:, 0], x[:, 1], x[:, 2] = 1.0, 2.0 ** -7, -2.0 ** -17
    a[0, 0, :3], a[0, 1, :2] = 1.0, 1.0
    b[0, :, 0], b[0, :, 1] = 1.0, -1.0
    assert (adapters.lora_add(y, x, a, b) == -2.0 ** -17).all()
