"""A grammar and the other rules of its request: what is left together, not what the mask names, has to hold a token."""

import numpy as np
import pytest
import torch

from easydel_b200.inference import SamplingParams
from easydel_b200.inference.esurge import eSurge
from easydel_b200.inference.token_rules import TokenRules, pack_tokens
from easydel_b200.modules.llama import LlamaConfig, LlamaForCausalLM


def _rules(grammar, vocab=90, ends=(2,), **kw):
    return TokenRules.of(SamplingParams(max_tokens=8, guided_decoding=grammar, **kw), vocab, list(ends))


@pytest.mark.parametrize("kw,short", [(dict(min_tokens=4), True), (dict(logit_bias={2: -float("inf")}), True), (dict(logit_bias={2: -1e30}), False),
                                      (dict(min_tokens=4, logit_bias={5: -float("inf")}), True), (dict(allowed_token_ids=[3, 5]), True), (dict(), False)])
def test_a_token_that_other_rules_forbid_is_none(kw, short):
    r = _rules(lambda p, o: [2], **kw)
    r.mask([1], [])
    assert (r.error is not None) is short
    if short:
        assert "allows no token" in str(r.error)


def test_min_tokens_lets_the_end_pass_later():
    r = _rules(lambda p, o: [2, 5] if len(o) < 4 else [2], min_tokens=4)
    for n in range(6):
        assert r.mask([1], [5] * n) is not None and r.error is None
    r = _rules(lambda p, o: [2, 5] if len(o) < 3 else [2], min_tokens=4)
    for n in range(4):
        r.mask([1], [5] * n)
        assert (r.error is not None) == (n == 3)


@pytest.mark.parametrize("vocab", [64, 90, 95])
def test_bits_behind_the_vocabulary_are_no_tokens(vocab):
    words = np.zeros((vocab + 31) // 32, np.int32)
    words[-1] = -(1 << 31)                                  # bit 31 of the last word: token 95 of 96
    r = _rules(lambda p, o: words, vocab=vocab)
    m = r.mask([1], [])
    if vocab == 64:
        assert r.error is None and np.array_equal(m, pack_tokens([63], 64))
    else:
        assert r.error is not None
    assert words[-1] == -(1 << 31)
    full = np.full((vocab + 31) // 32, -1, np.int32)
    r = _rules(lambda p, o: torch.from_numpy(full), vocab=vocab)
    assert np.array_equal(r.mask([1], []), pack_tokens(range(vocab), vocab)) and r.error is None


@pytest.mark.parametrize("asynchronous", [False, True])
def test_a_request_whose_rules_leave_its_grammar_nothing_ends_with_the_error(asynchronous):
    cfg = LlamaConfig(vocab_size=200, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, max_position_embeddings=2048, eos_token_id=199, initializer_range=0.2)
    torch.manual_seed(0)
    eng = eSurge(LlamaForCausalLM(cfg, dtype=torch.float32, param_dtype=torch.float32).eval(), max_model_len=512, max_num_seqs=4,
                 max_num_batched_tokens=64, num_pages=32, async_scheduling=asynchronous)
    seen = []

    def ends(prompt, output):
        seen.append(list(output))
        return [7] if len(output) < 2 else [199]

    mk = lambda n: SamplingParams(max_tokens=6, temperature=0.0, min_tokens=n, guided_decoding=ends)  # noqa: E731
    a, b = (o.outputs[0] for o in eng.generate([[5, 6], [7, 8]], [mk(4), mk(2)]))
    assert a.token_ids == [7, 7] and a.finish_reason.startswith("error") and "allows no token" in a.finish_reason
    assert b.token_ids == [7, 7, 199] and b.finish_reason == "stop"
    assert all(set(o) <= {7, 199} for o in seen)
    assert not eng.scheduler.has_unfinished() and len(eng._free_slots) == eng.runner.max_num_seqs
