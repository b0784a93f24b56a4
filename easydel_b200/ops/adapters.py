"""Low-rank adapters of many requests beside a shared projection (``csrc/lora.cu``).

Every row of a batch may bring an adapter of its own. The shared projection runs for all rows at once; :func:`lora_add` adds

    ``out[t, c] = y[t, c] + scale[i] * (x[t] @ a[i, p].T) @ b[i, c]``,  ``i = index[t]``, ``p`` the part of the output that ``c`` is in

in one launch, whatever the rows' order: which rows go together is found on the device, so a captured graph follows the indexes of
each replay. Packed projections (queries / keys / values, gate / up) have one adapter per part, stored together. Differentiable in
``y``, ``x``, ``a`` and ``b``. CPU tensors run the plain form.
"""

from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib

vp, i32, i64, f32 = _lib.vp, _lib.i32, _lib.i64, _lib.f32
_lib.register("edl_lora_apply", i32, [vp, i64, vp, i64, vp, i64, vp, i64, i64, vp, i64, i64, vp, vp, f32, vp, i64, vp, i32, i32,
                                      i32, i32, i32, i32, vp, i32, i32, i32, vp, vp])
_lib.register("edl_lora_grads", i32, [vp, i64, vp, i64, vp, vp, vp, vp, i64, i64, vp, i64, i64, i32, i32, i32, i32, i32, i32, vp, i32,
                                      i32, i32, vp, vp])

MAX_RANK = 512       # ranks of all parts together
MAX_PARTS = 8
FEW_ROWS = 256       # up to here the inner value stays in shared memory


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows ``[T, width]`` with neighbouring elements side by side: a view where it has such a layout."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _weights(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _check(y, x, a, b, index, scale, parts, out):
    sx, sy, sa, sb, dev, dt = x.shape, y.shape, a.shape, b.shape, x.device, x.dtype
    if len(sa) != 3 or len(sb) != 3 or sa[0] != sb[0]:
        raise ValueError(f"adapters are [n, parts * r, in] and [n, out, r], got {tuple(sa)} and {tuple(sb)}")
    n, N, r = sb
    if n < 1 or N < 1 or r < 1 or sa[2] < 1:
        raise ValueError("adapters without elements")
    if parts is None:
        parts = (N,)
    elif sum(parts) != N or min(parts) < 1 or len(parts) > MAX_PARTS:
        raise ValueError(f"parts {parts} (at most {MAX_PARTS}, none empty) do not add up to the {N} output columns")
    if sa[1] != len(parts) * r:
        raise ValueError(f"{sa[1]} ranks contract x, {len(parts)} part(s) of rank {r} need {len(parts) * r}")
    if sa[1] > MAX_RANK:
        raise ValueError(f"{sa[1]} ranks over all parts; at most {MAX_RANK}")
    if not sx or sx[-1] != sa[2]:
        raise ValueError(f"rows of x have {sx[-1] if sx else 0} elements, the adapters take {sa[2]}")
    if sy[:-1] != sx[:-1] or len(sy) != len(sx) or sy[-1] != N:
        raise ValueError(f"y is {tuple(sy)}, x and the adapters ask for {(*sx[:-1], N)}")
    if dt not in (torch.bfloat16, torch.float32) or a.dtype != dt or b.dtype != dt:
        raise TypeError(f"x and its adapters are all bfloat16 or all float32, got {dt}, {a.dtype}, {b.dtype}")
    if y.dtype != dt and y.dtype != torch.float32:
        raise TypeError(f"y is of x's type or float32, got {y.dtype} beside {dt}")
    if index is None:
        if n != 1:
            raise ValueError(f"{n} adapters need an index per row")
    elif index.dtype != torch.int32 or index.numel() * sx[-1] != x.numel() or not index.is_contiguous() or index.device != dev:
        raise ValueError(f"index is a contiguous int32 tensor on {dev} with an entry for each of the {x.numel() // sx[-1]} rows")
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.shape != (n,) or not scale.is_contiguous() or scale.device != dev:
            raise ValueError(f"scale is a number or a contiguous float32 tensor [{n}] on {dev}")
        if scale.requires_grad:
            raise NotImplementedError("there is no gradient for the scales of adapters")
    if y.device != dev or a.device != dev or b.device != dev:
        raise ValueError(f"x is on {dev}, y on {y.device}, its adapters on {a.device} and {b.device}")
    if out is not None and (out.shape != sy or out.dtype != y.dtype or out.device != dev):
        raise ValueError(f"out is {tuple(out.shape)} of {out.dtype} on {out.device}, y {tuple(sy)} of {y.dtype} on {dev}")
    return parts


@functools.lru_cache(maxsize=256)
def _widths(parts: tuple[int, ...]):
    return (C.c_int * len(parts))(*parts)


def _inner(x: torch.Tensor, r: int, parts: int, result: torch.dtype, backward: bool = False) -> torch.Tensor:
    """Memory for the scaled inner value ``s x a^T`` (``s dy b`` of the backward pass) of rows ``x`` as bf16 parts ``[parts of a value, T, ranks]``."""
    cols = -(-parts * r // 16) * 16 if backward else parts * (-(-r // 16) * 16)
    return x.new_empty((3 if result == torch.float32 else 2, x.shape[0], cols), dtype=torch.bfloat16)


def _apply(x, y, out, a, b, index, scale, u, parts, backward=False):
    n, N, r = b.shape
    T, dev = x.shape[0], x.device
    if u is None and T > FEW_ROWS:
        u = _inner(x, r, len(parts), x.dtype if out is None else out.dtype, backward)
    mixed = None if index is None or T <= FEW_ROWS else index.new_empty(-(-T // FEW_ROWS))      # which blocks of rows have many adapters
    st = scale if isinstance(scale, torch.Tensor) else None
    _lib.call_on(dev, "edl_lora_apply", x.data_ptr(), x.stride(0), None if y is None else y.data_ptr(), 0 if y is None else y.stride(0),
                 None if out is None else out.data_ptr(), 0 if out is None else out.stride(0), a.data_ptr(), a.stride(0), a.stride(1),
                 b.data_ptr(), b.stride(0), b.stride(1), None if index is None else index.data_ptr(), None if st is None else st.data_ptr(),
                 0.0 if st is not None else scale, None if u is None else u.data_ptr(), 0 if u is None else u.numel(),
                 None if mixed is None else mixed.data_ptr(), T, a.shape[2], N, n, r, len(parts), _widths(parts), x.dtype == torch.float32, (x if out is None else out).dtype == torch.float32, backward,
                 _lib.status_word(dev).data_ptr())


def _grad_target(w: torch.Tensor) -> tuple[torch.Tensor, bool]:
    """The tensor that takes the gradient of adapter weights ``w``, and whether it is added to (a slice of the flat gradient buffer)."""
    mg = getattr(w, "main_grad", None)
    if mg is None:
        return torch.empty_like(w, memory_format=torch.contiguous_format), False
    return mg.view(w.shape), True


class _LoraAddFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, index, scale, parts):
        x2 = _rows(x)
        out = torch.empty_like(y, memory_format=torch.contiguous_format)
        u = _inner(x2, b.shape[2], len(parts), x.dtype) if ctx.needs_input_grad[3] else None
        _apply(x2, _rows(y), _rows(out), _weights(a), _weights(b), index, scale, u, parts)
        ctx.save_for_backward(x, a, b, u, index, scale if isinstance(scale, torch.Tensor) else None)
        ctx.scale, ctx.parts = scale, parts
        return out

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise NotImplementedError("adapters have no second derivatives")
        x, a, b, u, index, st = ctx.saved_tensors
        scale, parts = st if st is not None else ctx.scale, ctx.parts
        need_y, need_x, need_a, need_b = ctx.needs_input_grad[:4]
        dy2, x2 = _rows(dy), _rows(x)
        n, N, r = b.shape
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
        g = _inner(x2, r, len(parts), x.dtype, True) if need_a else None
        if need_x or need_a:
            _apply(dy2, None, _rows(dx) if need_x else None, _weights(a), _weights(b), index, scale, g, parts, True)
        da, a_added = _grad_target(a) if need_a else (None, False)
        db, b_added = _grad_target(b) if need_b else (None, False)
        # one launch for both, unless only one of them is added to a flat buffer
        for ta, tb, added in ((da, db, a_added or b_added),) if da is None or db is None or a_added == b_added else \
                ((da, None, a_added), (None, db, b_added)):
            if ta is None and tb is None:
                continue
            _lib.call_on(x.device, "edl_lora_grads", x2.data_ptr(), x2.stride(0), dy2.data_ptr(), dy2.stride(0), _lib.ptr(g), _lib.ptr(u),
                         _lib.ptr(index), _lib.ptr(ta), 0 if ta is None else ta.stride(0), 0 if ta is None else ta.stride(1), _lib.ptr(tb),
                         0 if tb is None else tb.stride(0), 0 if tb is None else tb.stride(1), x2.shape[0], a.shape[2], N, n, r, len(parts),
                         _widths(parts), x.dtype == torch.float32, (ta if tb is None else tb).dtype == torch.float32, added,
                         _lib.status_word(x.device).data_ptr())
        if a_added:
            a.grad_added_to_main_grad = True
        if b_added:
            b.grad_added_to_main_grad = True
        return dy if need_y else None, dx, None if a_added else da, None if b_added else db, None, None, None


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor | None = None,
             scale: float | torch.Tensor = 1.0, *, parts: tuple[int, ...] | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """``y`` plus each row's adapter product.

    ``y [..., N]``: output of the shared projection of ``x [..., K]`` (bfloat16 or float32; ``y`` may be float32 beside bfloat16
    rows); ``a [n, P * r, K]``, ``b [n, N, r]``: the adapters' weights, of x's type; ``index``: int32, an adapter per row, negative
    for none (None: one adapter for all rows); ``scale``: a number, or float32 ``[n]``; ``parts``: widths of the P parts of a
    packed output, whose ranks follow one another in ``a``. Adapters of a smaller rank are padded with zeros. ``out``: where to write
    (``y`` itself for in place; inference only). An index of ``n`` or more counts as none and sets the status word that
    ``_lib.check_status`` reads.
    """
    parts = _check(y, x, a, b, index, scale, None if parts is None else tuple(parts), out)
    grad = torch.is_grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad or y.requires_grad)
    if grad and out is not None:
        raise ValueError("out= is for inference: a gradient needs y as it was")
    if not _lib.use_kernels(x):
        o = lora_add_reference(y, x, a, b, index, scale, parts=parts)
        return o if out is None else out.copy_(o)
    if not isinstance(scale, torch.Tensor):
        scale = float(scale)
    if grad:
        if y.dtype != x.dtype:
            raise NotImplementedError("float32 outputs beside bfloat16 rows have no backward pass")
        return _LoraAddFn.apply(y, x, a, b, index, scale, parts)
    res = torch.empty_like(y, memory_format=torch.contiguous_format) if out is None else out
    if res.dim() == 2 and (res.stride(1) == 1 or res.shape[1] == 1):
        o2 = res
    elif res.is_contiguous():
        o2 = res.view(-1, res.shape[-1])
    else:      # no rows with neighbouring elements to write to
        return res.copy_(lora_add(y, x, a, b, index, scale, parts=parts))
    _apply(_rows(x), o2 if res is y else _rows(y), o2, _weights(a), _weights(b), index, scale, None, parts)
    return res


def lora_add_reference(y, x, a, b, index=None, scale=1.0, *, parts=None) -> torch.Tensor:
    """Plain form (differentiable): products in 32 bits or more, rounded once."""
    wide = torch.promote_types(torch.promote_types(x.dtype, y.dtype), torch.float32)
    n, N, r = b.shape
    parts = (N,) if parts is None else parts
    x2, flat = x.reshape(-1, x.shape[-1]).to(wide), y.reshape(-1, N).to(wide)
    idx = torch.zeros(x2.shape[0], dtype=torch.int64, device=x.device) if index is None else index.reshape(-1).long()
    st = scale.to(wide) if isinstance(scale, torch.Tensor) else torch.full((n,), float(scale), dtype=wide, device=x.device)
    out = flat
    for i in range(n):
        at = (idx == i).nonzero()[:, 0]
        u = (x2[at] @ a[i].to(wide).t()).view(-1, len(parts), r) * st[i]
        z = torch.cat([u[:, p] @ w.t() for p, w in enumerate(b[i].to(wide).split(parts))], -1)
        out = out.index_add(0, at, z)
    return out.reshape(y.shape).to(y.dtype)
