"""Adapters beside quantised projections on the GPU kernels: single tokens (the fused product) and prompts, alone and through the engine."""

import pytest
import torch
from test_adapter_quantized_cpu import loaded, quantized, run_projections

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["int8", "nf4"])
@pytest.mark.parametrize("T", [1, 7, 300, 700])
def test_projections(fmt, T):
    model = quantized(fmt, torch.bfloat16, "cuda")
    run_projections(model, loaded(model, device="cuda"), T, torch.bfloat16, "cuda")


def test_engine(monkeypatch):
    from easydel_b200.inference import SamplingParams
    from easydel_b200.inference.esurge import eSurge
    from easydel_b200.modules.llama import LlamaConfig, LlamaForCausalLM

    outs = []
    for graphs in ("1", "0"):
        monkeypatch.setenv("EDL_ESURGE_CUDA_GRAPHS", graphs)
        cfg = LlamaConfig(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                          head_dim=128, max_position_embeddings=1024, eos_token_id=511, initializer_range=0.1)
        model = LlamaForCausalLM.sequential_init(cfg, dtype=torch.bfloat16, param_dtype=torch.bfloat16, device="cuda", seed=3).eval().quantize("int8")
        eng = eSurge(model, max_model_len=512, max_num_seqs=4, max_num_batched_tokens=256, num_pages=32, max_adapters=2)
        g = torch.Generator().manual_seed(1)
        for i in range(2):
            eng.load_adapter(f"a{i}", {f"{n}.lora_{k}": torch.randn(*s, generator=g) * s[1] ** -0.5 for n, b in eng.adapters.banks.items()
                                       for k, s in (("a", (8, b.a.shape[2])), ("b", (sum(b.parts), 8)))})
        sp = SamplingParams(max_tokens=8, temperature=0.0, ignore_eos=True)
        prompts = [[3, 4, 5], list(range(10, 150)), [3, 4, 5]]
        outs.append([o.outputs[0].token_ids for o in eng.generate(prompts, sp, adapter=["a0", "a1", None])])
        eng.close()
    assert outs[0] == outs[1] and outs[0][0] != outs[0][2]
