"""Requests that bring adapters and token rules through the engine, on CPU: each gets what it would get alone."""

import copy
import json

import numpy as np
import pytest
import torch

from easydel_b200.inference import SamplingParams
from easydel_b200.inference.esurge import eSurge
from easydel_b200.inference.token_rules import TokenRules, collect, pack_tokens
from easydel_b200.layers.adapters import AdapterSet
from easydel_b200.modules.llama import LlamaConfig, LlamaForCausalLM

PROMPTS = [list(range(3, 40)), list(range(60, 64)), list(range(3, 40)), [5, 9]]


def _model():
    cfg = LlamaConfig(vocab_size=200, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, max_position_embeddings=2048, eos_token_id=199, initializer_range=0.2)
    torch.manual_seed(0)
    return LlamaForCausalLM(cfg, dtype=torch.float32, param_dtype=torch.float32).eval()


def _engine(model, asynchronous=False, **kw):
    return eSurge(model, max_model_len=512, max_num_seqs=4, max_num_batched_tokens=64, num_pages=32, async_scheduling=asynchronous, **kw)


def _peft(seed, rank=3, layers=2):
    """Single projections under the names that checkpoints of adapters use."""
    g = torch.Generator().manual_seed(seed)
    sizes = {"self_attn.q_proj": (64, 64), "self_attn.k_proj": (64, 32), "self_attn.v_proj": (64, 32), "self_attn.o_proj": (64, 64),
             "mlp.gate_proj": (64, 128), "mlp.up_proj": (64, 128), "mlp.down_proj": (128, 64)}
    out = {}
    for i in range(layers):
        for n, (k, m) in sizes.items():
            out[f"base_model.model.model.layers.{i}.{n}.lora_A.weight"] = torch.randn(rank, k, generator=g) * 0.3
            out[f"base_model.model.model.layers.{i}.{n}.lora_B.weight"] = torch.randn(m, rank, generator=g) * 0.3
    return out


def _merged(model, tensors, scale):
    model = copy.deepcopy(model)
    at = {"q_proj": ("qkv_proj", 0, 64), "k_proj": ("qkv_proj", 64, 96), "v_proj": ("qkv_proj", 96, 128), "o_proj": ("o_proj", 0, 64),
          "gate_proj": ("gate_up_proj", 0, 128), "up_proj": ("gate_up_proj", 128, 256), "down_proj": ("down_proj", 0, 64)}
    with torch.no_grad():
        for key in [k for k in tensors if "lora_A" in k]:
            path = key[len("base_model.model."):-len(".lora_A.weight")]
            owner, _, leaf = path.rpartition(".")
            name, lo, hi = at[leaf]
            delta = tensors[key.replace("lora_A", "lora_B")].double() @ tensors[key].double() * scale
            w = model.get_submodule(f"{owner}.{name}").weight
            w[lo:hi] = (w[lo:hi].double() + delta).float()
    return model


@pytest.mark.parametrize("asynchronous", [False, True])
def test_requests_of_a_batch_run_with_their_own_adapters(asynchronous):
    model = _model()
    one, two = _peft(1), _peft(2, rank=5)
    sp = SamplingParams(max_tokens=8, temperature=0.0, ignore_eos=True)
    want = [_engine(_merged(model, t, s) if t else model).generate(p, sp)[0].outputs[0].token_ids
            for p, (t, s) in zip(PROMPTS, [(one, 0.5), (two, 0.25), (None, 0), (two, 0.25)])]
    eng = _engine(model, asynchronous, max_adapters=2, max_adapter_rank=8)
    eng.load_adapter("one", one, scale=0.5)
    eng.load_adapter("two", two, scale=0.25)
    for _ in range(2):      # the second time the prompts are in the prefix cache
        got = [o.outputs[0].token_ids for o in eng.generate(PROMPTS, sp, adapter=["one", "two", None, "two"])]
        assert got == want
    assert want[0] != want[2]
    eng.close()
    assert _engine(model).generate(PROMPTS[2], sp)[0].outputs[0].token_ids == want[2]


def test_pages_of_one_adapter_serve_no_other_and_a_reloaded_name_starts_anew():
    model, one, two = _model(), _peft(1), _peft(2)
    prompt = list(range(1, 150)) + list(range(1, 150))      # more than two pages
    sp = SamplingParams(max_tokens=4, temperature=0.0, ignore_eos=True)
    want = [_engine(_merged(model, t, 0.5)).generate(prompt, sp)[0].outputs[0].token_ids for t in (one, two)]
    eng = _engine(model, max_adapters=2, max_adapter_rank=4)
    eng.generate(prompt, sp)
    eng.load_adapter("x", one, scale=0.5)
    out = eng.generate(prompt, sp, adapter="x")[0]
    assert out.num_cached_tokens == 0 and out.outputs[0].token_ids == want[0]
    assert eng.generate(prompt, sp, adapter="x")[0].num_cached_tokens > 0
    eng.unload_adapter("x")
    eng.load_adapter("x", two, scale=0.5)
    out = eng.generate(prompt, sp, adapter="x")[0]
    assert out.num_cached_tokens == 0 and out.outputs[0].token_ids == want[1]


def test_adapters_of_training_and_of_directories(tmp_path):
    from safetensors.torch import save_file

    model = _model()
    trained = copy.deepcopy(model).apply_lora_to_layers(4, lora_alpha=8)
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        for n, p in trained.split_lora_params().items():
            p.copy_(torch.randn(p.shape, generator=g) * 0.2)
    sp = SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True)
    tensors = {k: v.detach().clone() for k, v in trained.split_lora_params().items()}
    want = _engine(trained.merge_lora_params()).generate(PROMPTS[0], sp)[0].outputs[0].token_ids
    eng = _engine(model, max_adapters=2, max_adapter_rank=4)
    eng.load_adapter("trained", tensors, scale=2.0)
    assert eng.generate(PROMPTS[0], sp, adapter="trained")[0].outputs[0].token_ids == want

    one = _peft(1, rank=4)
    save_file(one, str(tmp_path / "adapter_model.safetensors"))
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 6, "use_rslora": True}))
    eng.load_adapter("dir", tmp_path)
    want = _engine(_merged(model, one, 3.0)).generate(PROMPTS[0], sp)[0].outputs[0].token_ids
    assert eng.generate(PROMPTS[0], sp, adapter="dir")[0].outputs[0].token_ids == want
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 6, "use_dora": True}))
    with pytest.raises(NotImplementedError, match="use_dora"):
        AdapterSet(copy.deepcopy(_model()), 1, 4).load("dir", tmp_path)


def test_refusals_of_adapters():
    model, one = _model(), _peft(1)
    with pytest.raises(RuntimeError, match="max_adapters"):
        _engine(model).load_adapter("one", one)
    eng = _engine(model, max_adapters=1, max_adapter_rank=4)
    with pytest.raises(RuntimeError, match="another engine"):
        _engine(model, max_adapters=1)
    with pytest.raises(ValueError, match="not loaded"):
        eng.generate(PROMPTS[0], adapter="one")
    for bad, words in (({}, "no adapter weights"), ({"x": torch.zeros(1)}, "is no adapter weight"),
                       ({k.replace("q_proj", "r_proj"): v for k, v in one.items()}, "no projection"),
                       ({k: v for k, v in one.items() if "lora_A" in k}, "one of its two"), (_peft(1, rank=9), "room for 8"),
                       ({k: v[:, :-1] for k, v in one.items()}, "do not fit")):
        with pytest.raises(ValueError, match=words):
            eng.load_adapter("bad", bad)
    assert eng.adapter_names == [] and eng.adapters._free == [0]
    eng.load_adapter("one", one)
    with pytest.raises(ValueError, match="loaded already"):
        eng.load_adapter("one", one)
    with pytest.raises(RuntimeError, match="slots are taken"):
        eng.load_adapter("two", one)
    eng.add_request(PROMPTS[0], SamplingParams(max_tokens=2), adapter="one")
    with pytest.raises(RuntimeError, match="in use"):
        eng.unload_adapter("one")
    while eng.scheduler.has_unfinished() or eng._inflight is not None:
        eng.step()
    eng.unload_adapter("one")
    with pytest.raises(KeyError):
        eng.unload_adapter("one")
    with pytest.raises(ValueError, match="merge or unwrap"):
        AdapterSet(copy.deepcopy(_model()).apply_lora_to_layers(2), 1, 4)


# ------------------------------------------------------------------------------------------------------------ rules
@pytest.mark.parametrize("asynchronous", [False, True])
def test_rules_of_requests(asynchronous):
    model = _model()
    eng = _engine(model, asynchronous)
    sps = [SamplingParams(max_tokens=5, temperature=0.0, ignore_eos=True, logit_bias={7: 1000.0}),
           SamplingParams(max_tokens=5, temperature=0.0, ignore_eos=True, allowed_token_ids=[11, 12]),
           SamplingParams(max_tokens=9, temperature=0.0, min_tokens=4, logit_bias={199: 1000.0}),
           SamplingParams(max_tokens=5, temperature=0.0, ignore_eos=True)]
    outs = [o.outputs[0] for o in eng.generate(PROMPTS, sps)]
    plain = _engine(model).generate(PROMPTS[3], sps[3])[0].outputs[0].token_ids
    assert outs[0].token_ids == [7] * 5 and set(outs[1].token_ids) <= {11, 12}
    assert len(outs[2].token_ids) == 5 and outs[2].token_ids[-1] == 199 and 199 not in outs[2].token_ids[:4] and outs[2].finish_reason == "stop"
    assert outs[3].token_ids == plain


@pytest.mark.parametrize("asynchronous", [False, True])
def test_a_grammar_sees_every_token(asynchronous):
    eng = _engine(_model(), asynchronous)
    seen = []

    def count_up(prompt, output):
        seen.append(list(output))
        assert prompt == PROMPTS[0] and -1 not in output
        nxt = (output[-1] if output else 20) + 1
        return [nxt] if len(output) % 2 else pack_tokens([nxt, 150], 200)

    sp = SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True, guided_decoding=count_up, logit_bias={150: -1000.0})
    other = SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True)
    a, b = eng.generate(PROMPTS[:2], [sp, other])
    assert a.outputs[0].token_ids == [21, 22, 23, 24, 25, 26]
    assert b.outputs[0].token_ids == _engine(_model()).generate(PROMPTS[1], other)[0].outputs[0].token_ids
    assert seen[-1] == [21, 22, 23, 24, 25]


def test_rules_with_penalties_and_sampling():
    model = _model()
    sp = dict(max_tokens=12, temperature=0.0, ignore_eos=True, repetition_penalty=1.7, presence_penalty=0.5, frequency_penalty=0.3)
    free = _engine(model).generate(PROMPTS[0], SamplingParams(**sp))[0].outputs[0].token_ids
    ruled = _engine(model).generate(PROMPTS[0], SamplingParams(**sp, logit_bias={free[3]: 0.0}))[0].outputs[0].token_ids
    assert ruled == free            # a bias of zero only takes the other road
    banned = _engine(model).generate(PROMPTS[0], SamplingParams(**sp, logit_bias={free[3]: -float("inf")}))[0].outputs[0].token_ids
    assert banned[:3] == free[:3] and free[3] not in banned
    drawn = _engine(model).generate(PROMPTS[0], SamplingParams(max_tokens=12, temperature=1.5, ignore_eos=True, seed=3, allowed_token_ids=[4, 5, 6]))
    assert set(drawn[0].outputs[0].token_ids) <= {4, 5, 6}


def test_layout_of_rules():
    class Req:
        def __init__(self, out):
            self.prompt_token_ids, self.output_token_ids = [1], out

    sps = [SamplingParams(logit_bias={9: 1.0, 2: -float("inf")}, min_tokens=2, max_tokens=5), SamplingParams(), SamplingParams(allowed_token_ids=[0, 33])]
    rules = [TokenRules.of(sp, 40, [5]) for sp in sps]
    assert rules[1] is None
    got = collect(rules, [Req([7]), Req([]), Req([])], "cpu")
    assert got["bias"][0].tolist() == [0, 3, 3, 3] and got["bias"][1].tolist() == [2, 5, 9]
    assert got["bias"][2].tolist() == [-float("inf"), -float("inf"), 1.0]
    assert got["mask"][1].tolist() == [-1, -1, 0] and got["mask"][0].tolist() == [[1, 2]]
    assert collect(rules[:1], [Req([7, 8])], "cpu")["bias"][1].tolist() == [2, 9]
    assert collect([None], [Req([])], "cpu") == {}
    assert pack_tokens([31], 40).tolist() == [-(1 << 31), 0] and np.int32 == pack_tokens([], 40).dtype


@pytest.mark.parametrize("kw", [dict(logit_bias={200: 1.0}), dict(logit_bias={-1: 1.0}), dict(logit_bias={3: float("nan")}),
                                dict(allowed_token_ids=[]), dict(allowed_token_ids=[200])])
def test_refusals_of_rules(kw):
    with pytest.raises(ValueError):
        _engine(_model()).add_request(PROMPTS[0], SamplingParams(**kw))


@pytest.mark.parametrize("asynchronous", [False, True])
@pytest.mark.parametrize("last", [2, 5])
def test_a_grammar_that_fails_ends_its_own_request(asynchronous, last):
    def raises(prompt, output):
        if len(output) == last:
            raise KeyError("state")
        return [30]

    def dead_end(prompt, output):
        return [31] if len(output) < last else []

    def outside(prompt, output):
        return [32] if len(output) < last else [200]

    mk = lambda g: SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True, guided_decoding=g)  # noqa: E731
    eng = _engine(_model(), asynchronous)
    outs = [o.outputs[0] for o in eng.generate(PROMPTS[:4], [mk(raises), mk(dead_end), mk(outside), mk(None)])]
    for o, t, what in zip(outs, (30, 31, 32), ("KeyError", "no token", "vocabulary")):
        assert o.token_ids == [t] * last and o.finish_reason.startswith("error") and what in o.finish_reason
    assert outs[3].token_ids == _engine(_model()).generate(PROMPTS[3], mk(None))[0].outputs[0].token_ids
    assert not eng.scheduler.has_unfinished() and len(eng._free_slots) == eng.runner.max_num_seqs


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_rules_that_leave_nothing_still_give_a_token(temperature):
    sp = SamplingParams(max_tokens=3, temperature=temperature, allowed_token_ids=[7], logit_bias={7: -float("inf")}, ignore_eos=True)
    o = _engine(_model()).generate(PROMPTS[0], sp)[0].outputs[0]
    assert len(o.token_ids) == 3 and all(0 <= t < 200 for t in o.token_ids)
