"""Loading adapters: factors of their own per projection, and what a load that fails leaves."""

import json

import pytest
import torch
from safetensors.torch import save_file

from easydel_b200.layers.adapters import AdapterBank, AdapterSet
from easydel_b200.modules.llama import LlamaConfig, LlamaForCausalLM


def _set(count=1, rank=8):
    cfg = LlamaConfig(vocab_size=64, hidden_size=32, intermediate_size=48, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2,
                      max_position_embeddings=64)
    return AdapterSet(LlamaForCausalLM(cfg, dtype=torch.float32, param_dtype=torch.float32).eval(), count, rank)


def _pair(path, k, n, r, seed=0):
    g = torch.Generator().manual_seed(seed)
    return {f"model.layers.0.{path}.lora_A.weight": torch.randn(r, k, generator=g), f"model.layers.0.{path}.lora_B.weight": torch.randn(n, r, generator=g)}


def _product(bank, slot, part, rank):
    lo = sum(bank.parts[:part])
    a, b = bank.a[slot, part * rank:(part + 1) * rank].double(), bank.b[slot, lo:lo + bank.parts[part]].double()
    return float(bank.scale[slot]) * (b @ a)


@pytest.mark.parametrize("alphas", [(0, 8, 2), (8, 0, 2), (8, 3, 0), (0, 0, 0), (3, 8, 2), (0.1, 100, 7)])
def test_factors_of_parts(tmp_path, alphas):
    tensors = {**_pair("self_attn.q_proj", 32, 32, 4), **_pair("self_attn.v_proj", 32, 16, 2, 1), **_pair("mlp.down_proj", 48, 32, 4, 2)}
    save_file(tensors, str(tmp_path / "adapter_model.safetensors"))
    (tmp_path / "adapter_config.json").write_text(json.dumps({"lora_alpha": 2, "alpha_pattern": {"q_proj": alphas[0], "v_proj": alphas[1], "down_proj": alphas[2]}}))
    aset = _set()
    slot = aset.load("x", tmp_path)
    for path, leaf, part, r, alpha in (("self_attn.qkv_proj", "self_attn.q_proj", 0, 4, alphas[0]), ("self_attn.qkv_proj", "self_attn.v_proj", 2, 2, alphas[1]),
                                       ("mlp.down_proj", "mlp.down_proj", 0, 4, alphas[2])):
        bank = aset.banks[f"model.layers.0.{path}"]
        want = alpha / r * tensors[f"model.layers.0.{leaf}.lora_B.weight"].double() @ tensors[f"model.layers.0.{leaf}.lora_A.weight"].double()
        # b, its factor and their product are each rounded to 32 bits
        assert torch.allclose(_product(bank, slot, part, aset.rank), want, rtol=0, atol=3 * 2.0 ** -24 * float(want.abs().max() + 1e-30) * 4)


def test_a_load_that_fails_gives_its_slot_back(monkeypatch):
    aset = _set()
    put = AdapterBank.put

    def fails(self, *a):
        put(self, *a)
        raise torch.OutOfMemoryError("no room")

    for _ in range(3):
        monkeypatch.setattr(AdapterBank, "put", fails)
        with pytest.raises(torch.OutOfMemoryError):
            aset.load("x", _pair("self_attn.q_proj", 32, 32, 4))
        assert aset._free == [0] and not aset.slots
    monkeypatch.setattr(AdapterBank, "put", put)
    aset.load("x", _pair("mlp.down_proj", 48, 32, 4))
    assert not aset.banks["model.layers.0.self_attn.qkv_proj"].b.any()      # nothing of the loads before


@pytest.mark.parametrize("scale", [float("nan"), float("inf")])
def test_factors_that_are_no_numbers_are_refused(scale):
    aset = _set()
    with pytest.raises(ValueError, match="factor"):
        aset.load("x", _pair("mlp.down_proj", 48, 32, 4), scale)
    assert aset._free == [0]


def test_a_projection_that_is_named_twice_is_refused():
    q, qkv = _pair("self_attn.q_proj", 32, 32, 4), _pair("self_attn.qkv_proj", 32, 64, 4)
    aset = _set()
    for both in ({**q, **qkv}, {**qkv, **q}, {**q, **{f"base_model.model.{k}": v for k, v in q.items()}},
                 {**q, **{k.replace("lora_A.weight", "lora_A.default.weight"): v for k, v in q.items()}}):
        with pytest.raises(ValueError, match="twice"):
            aset.load("x", both)
        assert aset._free == [0]
    aset.load("x", qkv)
