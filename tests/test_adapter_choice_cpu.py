"""Which adapters in training run on the kernels: those that two library products would not do faster."""

import pytest
import torch

from easydel_b200.layers import linears
from easydel_b200.layers.linears import ColumnParallelLinear, eLoRA
from easydel_b200.ops.adapters import pays

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,rows,inner,outer,rank,on", [
    (BF, 8192, 64, 64, 64, True), (BF, 8192, 64, 64, 68, False), (BF, 1, 64, 64, 512, False), (BF, 8192, 64, 64, 14, False), (BF, 512, 64, 64, 14, True),
    (BF, 513, 64, 60, 16, False), (BF, 512, 33, 64, 16, True), (BF, 512, 33, 64, 20, False),
    (F32, 8192, 64, 64, 16, True), (F32, 8192, 64, 64, 20, False), (F32, 512, 64, 64, 32, True), (F32, 512, 64, 64, 36, False),
    (F32, 8192, 33, 64, 5, True), (F32, 8192, 33, 64, 3, False), (F32, 8192, 33, 64, 17, False),
])
def test_the_rule(dtype, rows, inner, outer, rank, on):
    assert pays(torch.empty(rows, inner, dtype=dtype), torch.empty(outer, rank, dtype=dtype)) is on
    assert pays(torch.empty(1, rows, inner, dtype=dtype), torch.empty(outer, rank, dtype=dtype)) is on


@pytest.mark.parametrize("rank,on", [(16, True), (96, False)])
def test_the_layer_goes_by_it(rank, on, monkeypatch):
    called = []
    monkeypatch.setattr(linears._lib, "use_kernels", lambda x: True)
    monkeypatch.setattr(linears.F, "linear", lambda x, w, bias=None, name=None: torch.nn.functional.linear(x, w, bias))
    monkeypatch.setattr(linears, "lora_add", lambda y, *a: called.append(1) or y)
    layer = eLoRA(ColumnParallelLinear(32, 64, dtype=BF), rank)
    with torch.no_grad():
        layer.lora_b.normal_()
    x = torch.randn(3, 32).to(BF)
    out = layer(x)
    assert bool(called) is on
    if not on:
        want = torch.nn.functional.linear(x, layer.base.weight) + \
            torch.nn.functional.linear(torch.nn.functional.linear(x, layer.lora_a), layer.lora_b) * layer.scaling
        assert torch.equal(out, want)
