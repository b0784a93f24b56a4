"""Serving low-rank adapters of many requests beside one model.

An :class:`AdapterSet` gives every attention and feed-forward projection of a model room for ``count`` adapters of rank up to ``rank``. While a
step runs with :meth:`AdapterSet.rows` set, each projection adds, row by row, the product of that row's adapter (``ops.adapters.lora_add``:
one launch for all adapters of the step); otherwise the model is what it was. The model's own weights and state dict are not touched.
"""

from __future__ import annotations

import contextlib
import json
import math
import os
import re
import threading
import typing as tp

import torch
from torch import nn

from ..ops.adapters import MAX_RANK, lora_add
from ..utils.parameters_transformation import FUSED_SPLITS
from .attention import Attention
from .linears import ParallelLinear, eLoRA
from .mlp import GatedMLP, PlainMLP
from .quantization import QuantizedLinear

#: names of the projections that a merged one holds, in the order of its parts
MERGED = {k: FUSED_SPLITS[k] for k in ("qkv_proj", "gate_up_proj")}
_LAYER = re.compile(r"(^|.*\.)layers\.\d+\.")


def _none():
    return None


class AdapterBank:
    """Weights of a projection's adapters: ``a [count, parts * rank, in]``, ``b [count, out, rank]``, unused ranks zero."""

    def __init__(self, owner: "AdapterSet", linear: nn.Module, count: int, rank: int, dtype: torch.dtype, device):
        self.owner = owner
        self.parts = tuple(linear.local_out_splits() or (linear.out_features,))
        self.a = torch.zeros(count, len(self.parts) * rank, linear.in_features, dtype=dtype, device=device)
        self.b = torch.zeros(count, linear.out_features, rank, dtype=dtype, device=device)
        self.scale = torch.zeros(count, dtype=torch.float32, device=device)

    def __reduce__(self):      # a copied or pickled model comes without the engine's adapters
        return _none, ()

    def add(self, y: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        """``y`` (the projection of ``x``, which nobody else holds) plus the products of the step's adapters."""
        rows = self.owner.index
        if rows is None:
            return y
        return lora_add(y, x, self.a, self.b, rows, self.scale, parts=self.parts, out=None if torch.is_grad_enabled() else y)

    def clear(self, slot: int) -> None:
        for t in (self.a, self.b, self.scale):
            t[slot].zero_()

    def put(self, slot: int, part: int | None, a: torch.Tensor, b: torch.Tensor, scale: float) -> None:
        """``part`` None: one adapter for the whole packed output, its ``a`` shared by all parts."""
        rank = self.b.shape[2]
        r, at = a.shape[0], 0
        for p, width in enumerate(self.parts):
            if part is None or part == p:
                self.a[slot, p * rank:p * rank + r].copy_(a)
                self.b[slot, at:at + width, :r].copy_(b[at:at + width] if part is None else b)
            at += width
        self.scale[slot] = scale


class AdapterSet:
    """``count`` adapters of rank up to ``rank`` for the projections of ``model``."""

    def __init__(self, model: nn.Module, count: int, rank: int):
        spec = getattr(model, "spec", None)
        if count < 1 or not 1 <= rank <= MAX_RANK:
            raise ValueError(f"{count} adapters of rank {rank}: at least one, of a rank from 1 to {MAX_RANK}")
        if getattr(spec, "residual_f32", False):
            raise NotImplementedError("models with a 32-bit residual stream run their projections without their modules: no adapters")
        self.count, self.rank = count, -(-rank // 8) * 8
        self._step = threading.local()      # a model may run in other threads meanwhile: their steps are not this one's
        self.slots: dict[str, int] = {}
        self.banks: dict[str, AdapterBank] = {}
        for name, m in model.named_modules():
            if not _LAYER.match(name) or type(m) not in (Attention, GatedMLP, PlainMLP):
                continue
            for leaf, lin in m.named_children():
                if isinstance(lin, eLoRA):
                    raise ValueError(f"{name}.{leaf} carries an adapter in training: merge or unwrap it first")
                if not isinstance(lin, (ParallelLinear, QuantizedLinear)):
                    continue
                if getattr(lin, "tp_size", 1) > 1:
                    raise NotImplementedError("adapters of requests: tensor parallelism 1")
                if len(lin.local_out_splits() or ()) * self.rank > MAX_RANK:
                    raise ValueError(f"{name}.{leaf}: rank {self.rank} in {len(lin.local_out_splits())} parts; at most {MAX_RANK} together")
                if lin.adapters is not None:
                    raise RuntimeError(f"{name}.{leaf} has adapters of another engine: close that one first")
                w = getattr(lin, "weight", None)
                dtype, device = (w.dtype, w.device) if w is not None else (model.dtype, lin.codes.device)      # that of the rows
                self.banks[f"{name}.{leaf}"] = AdapterBank(self, lin, count, self.rank, dtype, device)
        if not self.banks:
            raise NotImplementedError(f"{type(model).__name__} has no attention or feed-forward projections that take adapters")
        self._free = list(range(count - 1, -1, -1))
        self._model = model
        for name, bank in self.banks.items():
            model.get_submodule(name).adapters = bank

    def detach(self) -> None:
        """Takes the adapters off the model again."""
        for name, bank in self.banks.items():
            lin = self._model.get_submodule(name)
            if lin.adapters is bank:
                lin.adapters = None

    @contextlib.contextmanager
    def rows(self, index: torch.Tensor | None):
        """Runs what is inside with ``index[t]`` (int32; negative: none) naming the slot of the adapter of row t."""
        before, self._step.index = self.index, index
        try:
            yield self
        finally:
            self._step.index = before

    @property
    def index(self) -> torch.Tensor | None:
        return getattr(self._step, "index", None)

    # ------------------------------------------------------------------ loading
    def load(self, name: str, source: str | os.PathLike | tp.Mapping[str, torch.Tensor], scale: float | None = None) -> int:
        """Puts an adapter into a free slot and returns the slot. ``source``: a directory with ``adapter_config.json`` and
        ``adapter_model.safetensors`` (``.bin``), or tensors by name: ``<module>.lora_A.weight`` / ``lora_B.weight`` of single or merged projections,
        or what ``split_lora_params`` gives (``<module>.lora_a`` / ``lora_b``). ``scale``: factor of the product (None: ``lora_alpha`` over the
        rank, over its root for rank-stabilised ones, or 1 for tensors without a configuration)."""
        if name in self.slots:
            raise ValueError(f"adapter {name!r} is loaded already")
        if not self._free:
            raise RuntimeError(f"all {self.count} adapter slots are taken: unload one, or make more")
        tensors, config = (source, {}) if isinstance(source, tp.Mapping) else _read(source)
        # everything is checked before anything is written. A bank has one factor per adapter: parts with factors of their own have them in b
        todo: dict[int, list] = {}
        for path, bank, part, a, b in self._match(tensors):
            s = float(_scale(config, path, a.shape[0]) if scale is None else scale)
            if not math.isfinite(s):
                raise ValueError(f"{path!r}: its factor is {s}")
            todo.setdefault(id(bank), []).append((bank, part, a, b, s))
        slot = self._free.pop()
        try:
            for bank in self.banks.values():
                bank.clear(slot)
            for puts in todo.values():
                same = all(s == puts[0][4] for *_, s in puts)
                for bank, part, a, b, s in puts:
                    bank.put(slot, part, a, b if same else b.float() * s, s if same else 1.0)
        except BaseException:
            self._free.append(slot)
            raise
        self.slots[name] = slot
        return slot

    def unload(self, name: str) -> None:
        if name not in self.slots:
            raise KeyError(f"no adapter {name!r}")
        self._free.append(self.slots.pop(name))

    def _match(self, tensors: tp.Mapping[str, torch.Tensor]):
        pairs: dict[str, dict[str, torch.Tensor]] = {}
        for key, t in tensors.items():
            m = re.fullmatch(r"(?:base_model\.model\.)?(.+?)\.(?:lora_(A|B)(?:\.[^.]+)?\.weight|lora_(a|b))", key)
            if m is None:
                raise ValueError(f"{key!r} is no adapter weight")
            pair, letter = pairs.setdefault(m[1], {}), (m[2] or m[3]).lower()
            if letter in pair:
                raise ValueError(f"{m[1]!r} has its weight {letter} twice")
            pair[letter] = t
        if not pairs:
            raise ValueError("no adapter weights")
        taken: dict[int, list[int | None]] = {}      # parts of a bank (None: all)
        for path, w in pairs.items():
            owner, _, leaf = path.rpartition(".")
            merged = next((k for k, parts in MERGED.items() if leaf in parts), None)
            bank = self.banks.get(path) or (self.banks.get(f"{owner}.{merged}") if merged else None)
            if bank is None:
                raise ValueError(f"the model has no projection {path!r} that takes adapters")
            part = MERGED[merged].index(leaf) if path not in self.banks else (0 if len(bank.parts) == 1 else None)
            if len(w) != 2:
                raise ValueError(f"{path!r} has one of its two adapter weights")
            a, b = w["a"], w["b"]
            out = sum(bank.parts) if part is None else bank.parts[part]
            if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or a.shape[1] != bank.a.shape[2] or b.shape[0] != out:
                raise ValueError(f"{path!r}: adapter weights {tuple(a.shape)} and {tuple(b.shape)} do not fit a projection of {bank.a.shape[2]} to {out}")
            if a.shape[0] > self.rank:
                raise ValueError(f"{path!r}: rank {a.shape[0]}; there is room for {self.rank}")
            others = taken.setdefault(id(bank), [])
            if others and (part is None or None in others or part in others):
                raise ValueError(f"{path!r} is adapted twice, by itself and as a part of a merged projection")
            others.append(part)
            yield path, bank, part, a, b


def _scale(config: dict, path: str, rank: int) -> float:
    if not config:
        return 1.0
    alpha = config.get("lora_alpha", rank)
    for pattern, value in (config.get("alpha_pattern") or {}).items():
        if re.search(rf"(^|\.){pattern}$", path):
            alpha = value
    return alpha / (rank ** 0.5 if config.get("use_rslora") else rank)


def _read(path: str | os.PathLike) -> tuple[dict[str, torch.Tensor], dict]:
    with open(os.path.join(path, "adapter_config.json")) as f:
        config = json.load(f)
    for key in ("use_dora", "modules_to_save", "layer_replication"):
        if config.get(key):
            raise NotImplementedError(f"adapters with {key} cannot be served")
    if config.get("bias", "none") != "none":
        raise NotImplementedError("adapters with biases cannot be served")
    weights = os.path.join(path, "adapter_model.safetensors")
    if os.path.exists(weights):
        from safetensors.torch import load_file

        return load_file(weights), config
    return torch.load(os.path.join(path, "adapter_model.bin"), map_location="cpu", weights_only=True), config
