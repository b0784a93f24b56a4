"""Adapters of a model whose other weights, embeddings included, are frozen get gradients when layers are recomputed."""

import pytest
import torch

from easydel_b200.modules.llama import LlamaConfig, LlamaForCausalLM


@pytest.mark.parametrize("policy", ["nothing_saveable", "dots_saveable"])
def test_gradients_with_frozen_embeddings(policy):
    ids = torch.randint(0, 90, (2, 12), generator=torch.Generator().manual_seed(0))
    grads = []
    for p in ("", policy):
        cfg = LlamaConfig(vocab_size=90, hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                          max_position_embeddings=64, gradient_checkpointing=p)
        torch.manual_seed(0)
        model = LlamaForCausalLM(cfg, dtype=torch.float32, param_dtype=torch.float32).apply_lora_to_layers(4)
        torch.manual_seed(1)
        with torch.no_grad():
            for w in model.split_lora_params().values():
                w.copy_(torch.randn(w.shape) * 0.1)
        model.train()
        _, metrics = model.compute_loss(input_ids=ids, labels=ids)
        metrics.loss.backward()
        grads.append({n: w.grad for n, w in model.split_lora_params().items()})
    assert all(g is not None and g.any() for g in grads[0].values())
    for n, g in grads[0].items():
        assert torch.allclose(grads[1][n], g, rtol=1e-5, atol=1e-7), n
