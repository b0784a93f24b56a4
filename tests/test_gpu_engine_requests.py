"""Adapters and token rules through layers, training and the engine, on the GPU kernels."""

import pytest
import torch
from adapter_cases import check, exact

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _model(layers=2, **kw):
    from easydel_b200.modules.llama import LlamaConfig, LlamaForCausalLM

    cfg = LlamaConfig(vocab_size=4096, hidden_size=512, intermediate_size=1408, num_hidden_layers=layers, num_attention_heads=8,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=4096, eos_token_id=4095, initializer_range=0.08, **kw)
    return LlamaForCausalLM.sequential_init(cfg, dtype=BF, param_dtype=BF, device="cuda", seed=3)


def _adapter(model, seed, rank):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = {}
    for i in range(len(model.model.layers)):
        layer = model.model.layers[i]
        for n, lin in (("self_attn.qkv_proj", layer.self_attn.qkv_proj), ("self_attn.o_proj", layer.self_attn.o_proj),
                       ("mlp.gate_up_proj", layer.mlp.gate_up_proj), ("mlp.down_proj", layer.mlp.down_proj)):
            out[f"model.layers.{i}.{n}.lora_a"] = torch.randn(rank, lin.in_features, generator=g, device="cuda") * lin.in_features ** -0.5
            out[f"model.layers.{i}.{n}.lora_b"] = torch.randn(lin.out_features, rank, generator=g, device="cuda") * 0.3
    return out


@pytest.mark.parametrize("rank", [8, 5])
@pytest.mark.parametrize("T", [6, 300])
def test_training_layer(rank, T):
    from easydel_b200.layers.linears import ColumnParallelLinear, eLoRA

    torch.manual_seed(0)
    base = ColumnParallelLinear(256, (128, 64), dtype=BF).cuda()
    layer = eLoRA(base, rank, alpha=2 * rank)
    with torch.no_grad():
        layer.lora_b.normal_(std=0.3)
    x = torch.randn(2, T // 2, 256, device="cuda").to(BF).requires_grad_()
    dy = torch.randn(2, T // 2, 192, device="cuda").to(BF)
    out = layer(x)
    out.backward(dy)
    c = dict(x=x.detach().view(T, 256), y=base(x.detach()).view(T, 192), a=layer.lora_a.detach()[None], b=layer.lora_b.detach()[None], index=None, scale=2.0,
             parts=(192,), dy=dy.view(T, 192))
    val, mag = exact(c, grads=True)
    check(out.detach().view(T, 192), val["out"], mag["out"], 256, "out")
    check(layer.lora_a.grad[None], val["da"], mag["da"], T + 192, "da")
    check(layer.lora_b.grad[None], val["db"], mag["db"], T + 256, "db")
    assert base.weight.grad is None
    # dx is the sum of the base's and the adapter's part, each rounded, and their sum rounded
    want = val["dx"] + dy.view(T, 192).double().cpu() @ base.weight.detach().double().cpu()
    size = mag["dx"] + dy.view(T, 192).double().cpu().abs() @ base.weight.detach().double().cpu().abs()
    assert ((x.grad.view(T, 256).double().cpu() - want).abs() <= 3 * 2.0 ** -8 * (want.abs() + val["dx"].abs()) + 2.0 ** -14 * size).all()


def test_training_step_with_recomputed_layers_gives_the_same_gradients():
    ids = torch.randint(0, 4000, (2, 300), generator=torch.Generator().manual_seed(1)).cuda()
    grads = []
    for policy in ("nothing_saveable", "everything_saveable"):
        model = _model(gradient_checkpointing=policy).apply_lora_to_layers(8, lora_alpha=16)
        g = torch.Generator(device="cuda").manual_seed(2)
        with torch.no_grad():
            for p in model.split_lora_params().values():
                p.copy_(torch.randn(p.shape, generator=g, device="cuda") * 0.05)
        _, metrics = model.compute_loss(input_ids=ids, labels=ids)
        metrics.loss.backward()
        grads.append({n: p.grad for n, p in model.split_lora_params().items()})
    assert all(v is not None and torch.isfinite(v).all() and v.any() for v in grads[0].values())
    # the recomputed forward is the same kernels on the same inputs
    for n in grads[0]:
        a, b = grads[0][n].double(), grads[1][n].double()
        assert (a - b).norm() <= 2.0 ** -7 * b.norm(), n


def test_projection_of_a_step_adds_each_row_its_adapter():
    from easydel_b200.layers.adapters import AdapterSet

    model = _model().eval()
    aset = AdapterSet(model, 3, 16)
    for i, rank in enumerate((16, 5)):
        aset.load(f"a{i}", _adapter(model, i, rank), scale=0.5 + i)
    for T in (7, 300):
        idx = (torch.arange(T, device="cuda") % 4 - 1).clamp(max=1).to(torch.int32)
        for lin in (model.model.layers[1].self_attn.qkv_proj, model.model.layers[0].mlp.down_proj):
            x = torch.randn(1, T, lin.in_features, device="cuda").to(BF)
            with torch.no_grad():
                y = lin(x)
                with aset.rows(idx):
                    got = lin(x)
                assert torch.equal(lin(x), y)
            bank = lin.adapters
            c = dict(x=x[0], y=y[0], a=bank.a, b=bank.b, index=idx, scale=bank.scale, parts=bank.parts, dy=y[0])
            want, mag = exact(c)
            check(got[0], want, mag, lin.in_features)
            assert torch.equal(got[0][idx < 0], y[0][idx < 0])
    aset.detach()


def _run(graphs, monkeypatch, asynchronous=True):
    from easydel_b200.inference import SamplingParams
    from easydel_b200.inference.esurge import eSurge

    monkeypatch.setenv("EDL_ESURGE_CUDA_GRAPHS", "1" if graphs else "0")
    eng = eSurge(_model().eval(), max_model_len=1024, max_num_seqs=8, max_num_batched_tokens=512, num_pages=64, max_adapters=3, max_adapter_rank=16,
                 async_scheduling=asynchronous)
    for i, rank in enumerate((16, 4, 8)):
        eng.load_adapter(f"a{i}", _adapter(eng.model, i, rank), scale=1.0)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 4000, (n,), generator=g).tolist() for n in (3, 50, 400, 17)]
    greedy = SamplingParams(max_tokens=12, temperature=0.0, ignore_eos=True)
    outs = []
    for names in (["a0", "a1", None, "a2"], ["a2", None, "a0", "a0"], None):
        outs.append([o.outputs[0].token_ids for o in eng.generate(prompts, greedy, adapter=names)])
    assert bool(eng.runner._graphs) == bool(eng.runner._adapter_graphs) == graphs
    ruled = [SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True, logit_bias={77: 1000.0}),
             SamplingParams(max_tokens=6, temperature=1.0, seed=5, ignore_eos=True, allowed_token_ids=[10, 20, 4000]),
             SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True, repetition_penalty=1.5, guided_decoding=lambda p, o: [len(o), 100 + len(o)]), greedy]
    outs.append([o.outputs[0].token_ids for o in eng.generate(prompts, ruled, adapter=["a0", None, "a1", "a2"])])
    eng.close()
    return outs


def test_engine_runs_adapters_and_rules_in_replayed_and_eager_steps(monkeypatch):
    a, b = _run(True, monkeypatch), _run(False, monkeypatch)
    assert a == b
    assert a[0][0] != a[2][0] and a[0][0] != a[1][0]          # adapters change what comes out
    assert a[3][0] == [77] * 6 and set(a[3][1]) <= {10, 20, 4000} and all(t in (i, 100 + i) for i, t in enumerate(a[3][2]))


def test_requests_without_an_adapter_are_served_as_by_an_engine_without_room_for_any(monkeypatch):
    from easydel_b200.inference import SamplingParams
    from easydel_b200.inference.esurge import eSurge

    outs = []
    for room in (0, 2):
        eng = eSurge(_model().eval(), max_model_len=1024, max_num_seqs=8, max_num_batched_tokens=512, num_pages=64, max_adapters=room)
        outs.append([o.outputs[0].token_ids for o in eng.generate([[5, 6, 7], list(range(200))], SamplingParams(max_tokens=10, temperature=0.0, ignore_eos=True))])
        eng.close()
    assert outs[0] == outs[1]


@pytest.mark.parametrize("vocab", [100, 50257])
def test_rows_that_rules_leave_nothing_still_give_a_token(vocab):
    from easydel_b200.ops import serving as S

    z = torch.randn(5, vocab, device="cuda")
    bits = torch.zeros(1, (vocab + 31) // 32, dtype=torch.int32, device="cuda")
    rows = torch.tensor([-1, 0, -1, 0, -1], dtype=torch.int32, device="cuda")
    z = S.adjust_logits(z, mask=(bits, rows))
    assert (z[1] == -float("inf")).all() and torch.isfinite(z[0]).all()
    for t in (0.0, 0.8):
        kw = {} if not t else dict(temperature=torch.full((5,), t, device="cuda"), top_p=torch.full((5,), 0.9, device="cuda"),
                                   min_p=torch.zeros(5, device="cuda"), top_k=torch.zeros(5, dtype=torch.int32, device="cuda"),
                                   seeds=torch.arange(5, device="cuda"), steps=torch.zeros(5, dtype=torch.int32, device="cuda"))
        tokens, _ = S.sample(z, **kw)
        assert ((tokens >= 0) & (tokens < vocab)).all()
