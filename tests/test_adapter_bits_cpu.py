"""The bound of `adapter_bits` tells three parts of an operand from two: shown on 64-bit results with and without the third."""

import pytest
import torch
from adapter_bits import bound, make, parts, values
from adapter_cases import exact


def test_three_parts_are_the_value():
    for v in (values(1000), torch.randn(100000), torch.randn(100000) * 2.0 ** 100, torch.randn(100000) * 2.0 ** -90):
        assert torch.equal(sum(p.double() for p in parts(v)), v.double())
    v = values(1000)
    off = (v.double() - sum(p.double() for p in parts(v, 2))) / v.double()
    assert (off > 0.9 * 2.0 ** -17).all()


@pytest.mark.parametrize("T,K,widths,r", [(8, 64, (64,), 16), (300, 512, (96, 32), 8), (40, 33, (7,), 5)])
@pytest.mark.parametrize("short", ["x", "a", "b", "dy"])
def test_a_lost_part_is_outside_the_bound(T, K, widths, r, short):
    c = make(T, K, widths, r, 2)
    val, _ = exact(c, grads=True)
    cut, _ = exact(dict(c, **{short: sum(p.double() for p in parts(c[short], 2))}), grads=True)
    N = sum(widths)
    tops = dict(out=bound(K, None, r), dx=bound(N, None, len(widths) * r), da=bound(N, T, r), db=bound(K, T, r))
    for name, uses in (("out", "xab"), ("dx", ("dy", "a", "b")), ("da", ("dy", "b", "x")), ("db", ("x", "a", "dy"))):
        if short in uses:
            off = (cut[name] - val[name]).abs() / val[name]
            assert (off > tops[name]).all(), name
