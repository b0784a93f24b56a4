"""What a request says about its next token beyond penalties: biases, an allowed set, forbidden end tokens, a grammar.

:class:`TokenRules` holds a request's rules as arrays, made once; :func:`collect` lays the rules of a step's rows out for
``ops.serving.adjust_logits``: sorted entries per row for single tokens, one bit per token for sets.

A grammar is a callable in ``SamplingParams.guided_decoding``: ``f(prompt_token_ids, output_token_ids)`` returns the tokens allowed next (ids,
or packed int32 words with bit ``t % 32`` of word ``t // 32`` for token t), or None where everything is. Requests with one are read back after
every step, since the next mask needs the token. One that raises, or allows nothing that ``allowed_token_ids``, ``min_tokens`` and biases of minus
infinity leave, ends its own request with that error. (Where those alone leave nothing, every token is forbidden and the sampler gives token 0.)
"""

from __future__ import annotations

import typing as tp

import numpy as np
import torch

from .sampling_params import InvalidRequest

_NONE = np.zeros(0, np.int32), np.zeros(0, np.float32)


def pack_tokens(ids: tp.Iterable[int], vocab: int) -> np.ndarray:
    """Packed words that allow exactly ``ids``."""
    bits = np.zeros((vocab + 31) // 32 * 32, np.uint8)
    at = np.fromiter(ids, np.int64)
    if at.size and not (0 <= at.min() and at.max() < vocab):
        raise InvalidRequest(f"token ids from {at.min()} to {at.max()} for a vocabulary of {vocab}")
    bits[at] = 1
    return np.packbits(bits, bitorder="little").view(np.int32)


def _entries(bias: tp.Mapping[int, float]) -> tuple[np.ndarray, np.ndarray]:
    ids = np.fromiter(bias.keys(), np.int32, len(bias))
    order = np.argsort(ids, kind="stable")
    return ids[order], np.fromiter(bias.values(), np.float32, len(bias))[order]


class TokenRules:
    """Rules of one request; None from :meth:`of` if it has none."""

    def __init__(self, sp, vocab: int, end_tokens: tp.Sequence[int]):
        self.vocab, self.grammar, self.min_tokens = vocab, sp.guided_decoding if callable(sp.guided_decoding) else None, sp.min_tokens
        bias = {int(t): float(v) for t, v in (sp.logit_bias or {}).items()}
        if any(not 0 <= t < vocab or v != v for t, v in bias.items()):
            raise InvalidRequest(f"logit_bias names a token outside the vocabulary of {vocab}, or is not a number")
        self.bias = _entries(bias) if bias else _NONE
        ends = {int(t): -np.inf for t in end_tokens if 0 <= t < vocab} if sp.min_tokens else {}
        self.bias_short = _entries({**bias, **ends}) if ends else self.bias      # while there are fewer than min_tokens
        self.allowed = None if sp.allowed_token_ids is None else pack_tokens(sp.allowed_token_ids, vocab)
        if self.allowed is not None and not self.allowed.any():
            raise InvalidRequest("allowed_token_ids is empty")
        self._tokens = pack_tokens(range(vocab), vocab) if self.grammar is not None else None      # the last word's other bits name none
        self.error: Exception | None = None      # of the grammar

    @classmethod
    def of(cls, sp, vocab: int, end_tokens: tp.Sequence[int]) -> "TokenRules | None":
        if not (sp.logit_bias or sp.allowed_token_ids is not None or sp.min_tokens or callable(sp.guided_decoding)):
            return None
        return cls(sp, vocab, end_tokens)

    def entries(self, n_out: int) -> tuple[np.ndarray, np.ndarray]:
        return self.bias_short if n_out < self.min_tokens else self.bias

    def active(self, n_out: int) -> bool:
        return bool(self.entries(n_out)[0].size) or self.allowed is not None or self.grammar is not None

    def mask(self, prompt: list[int], output: list[int]) -> np.ndarray | None:
        m = self.allowed
        if self.grammar is None or self.error is not None:
            return m
        try:
            return self._grammar_mask(m, prompt, output)
        except Exception as e:  # the user's code: other requests of the step go on
            self.error = e
            return m

    def _grammar_mask(self, m: np.ndarray | None, prompt: list[int], output: list[int]) -> np.ndarray | None:
        g = self.grammar(prompt, output)
        if g is None:
            return m
        if isinstance(g, torch.Tensor):
            g = g.cpu().numpy()
        if isinstance(g, np.ndarray) and g.dtype == np.int32 and g.ndim == 1 and g.size == (self.vocab + 31) // 32:
            g = g & self._tokens
        else:
            g = pack_tokens((int(t) for t in g), self.vocab)
        g = g if m is None else m & g
        ids, values = self.entries(len(output))
        left, gone = g.view(np.uint32).copy(), ids[values == -np.inf].astype(np.int64)
        np.bitwise_and.at(left, gone // 32, ~(np.uint32(1) << (gone % 32).astype(np.uint32)))
        if not left.any():
            raise ValueError("the grammar allows no token" + (" that the request's other rules leave" if g.any() else ""))
        return g


def collect(rules: tp.Sequence["TokenRules | None"], requests: tp.Sequence, device) -> dict[str, tuple]:
    """Arguments ``bias`` and ``mask`` of ``adjust_logits`` for a step's rows; empty if no row has a rule now."""
    entries = [r.entries(len(q.output_token_ids)) if r is not None else _NONE for r, q in zip(rules, requests)]
    masks = [r.mask(q.prompt_token_ids, q.output_token_ids) if r is not None else None for r, q in zip(rules, requests)]
    out: dict[str, tuple] = {}
    up = lambda a: torch.from_numpy(a).to(device)  # noqa: E731
    if any(e[0].size for e in entries):
        ptr = np.zeros(len(entries) + 1, np.int32)
        np.cumsum([e[0].size for e in entries], out=ptr[1:])
        out["bias"] = up(ptr), up(np.concatenate([e[0] for e in entries])), up(np.concatenate([e[1] for e in entries]))
    if any(m is not None for m in masks):
        at, kept = np.full(len(masks), -1, np.int32), []
        for i, m in enumerate(masks):
            if m is not None:
                at[i] = len(kept)
                kept.append(m)
        out["mask"] = up(np.stack(kept)), up(at)
    return out
