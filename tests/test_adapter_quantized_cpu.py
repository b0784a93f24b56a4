"""Adapters beside quantised projections."""

import pytest
import torch
from adapter_cases import check, exact

from easydel_b200.layers.adapters import AdapterSet
from easydel_b200.layers.quantization import QuantizedLinear
from easydel_b200.modules.llama import LlamaConfig, LlamaForCausalLM


def quantized(fmt, dtype, device="cpu", param_dtype=None):
    cfg = LlamaConfig(vocab_size=64, hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2,
                      max_position_embeddings=512)
    torch.manual_seed(0)
    return LlamaForCausalLM(cfg, dtype=dtype, param_dtype=param_dtype or dtype).eval().to(device).quantize(fmt)


def loaded(model, count=2, rank=8, device="cpu"):
    aset = AdapterSet(model, count, rank)
    g = torch.Generator().manual_seed(3)
    for i in range(count):
        aset.load(f"a{i}", {f"{name}.lora_{k}": (torch.randn(*s, generator=g) * s[1] ** -0.5).to(device) for name, bank in aset.banks.items()
                            for k, s in (("a", (rank - i, bank.a.shape[2])), ("b", (sum(bank.parts), rank - i)))}, 0.5 + i)
    return aset


def run_projections(model, aset, T, dtype, device="cpu"):
    index = (torch.arange(T) % 3 - 1).to(torch.int32).to(device)
    for name in ("self_attn.qkv_proj", "self_attn.o_proj", "mlp.gate_up_proj", "mlp.down_proj"):
        lin = model.get_submodule(f"model.layers.0.{name}")
        assert isinstance(lin, QuantizedLinear) and lin.adapters.a.dtype == dtype
        x = torch.randn(1, T, lin.in_features, generator=torch.Generator().manual_seed(T)).to(dtype).to(device)
        with torch.no_grad():
            y = lin(x)
            with aset.rows(index):
                got = lin(x)
            assert torch.equal(lin(x), y) and got.dtype == dtype
        bank = lin.adapters
        want, mag = exact(dict(x=x[0], y=y[0], a=bank.a, b=bank.b, index=index, scale=bank.scale, parts=bank.parts, dy=y[0]))
        check(got[0], want, mag, lin.in_features, name)
        assert torch.equal(got[0][index < 0], y[0][index < 0])


@pytest.mark.parametrize("fmt", ["int8", "nf4"])
@pytest.mark.parametrize("dtype,param_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_projections(fmt, dtype, param_dtype):
    model = quantized(fmt, dtype, param_dtype=param_dtype)      # rows are of the first type, whatever the parameters that are left are of
    aset = loaded(model)
    run_projections(model, aset, 7, dtype)
    with torch.no_grad(), aset.rows(torch.zeros(8, dtype=torch.int32)):
        assert torch.isfinite(model(input_ids=torch.arange(8)[None], apply_lm_head=False).last_hidden_state).all()


def test_a_row_parallel_projection_of_one_rank_has_its_adapter(monkeypatch):
    from easydel_b200.parallel import tp

    monkeypatch.setattr(tp, "all_reduce", lambda y, group: y)
    model = quantized("int8", torch.float32)
    aset = loaded(model)
    for name in ("self_attn.o_proj", "mlp.down_proj"):
        lin = model.get_submodule(f"model.layers.0.{name}")
        lin.tp_group, lin.parallel_style = object(), "row"
    run_projections(model, aset, 5, torch.float32)
