"""Low-rank adapters of many requests beside a shared projection (``csrc/lora.cu``).

Every row of a batch may bring an adapter of its own. The shared projection runs for all rows at once; :func:`lora_add` adds

    ``out[t, c] = y[t, c] + scale[i] * (x[t] @ a[i, p].T) @ b[i, c]``,  ``i = index[t]``, ``p`` the part of the output that ``c`` is in

in one launch, whatever the rows' order: which rows go together is found on the device, so a captured graph follows the indexes of
each replay. Packed projections (queries / keys / values, gate / up) have one adapter per part, stored together. Differentiable in
``y``, ``x``, ``a`` and ``b``. CPU tensors run the plain form.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib

vp, i32, i64, f32 = _lib.vp, _lib.i32, _lib.i64, _lib.f32
_lib.register("edl_lora_apply", i32, [vp, i64, vp, i64, vp, i64, vp, i64, i64, vp, i64, i64, vp, vp, f32, vp, i64, i32, i32, i32,
                                      i32, i32, i32, vp, i32, i32, i32, vp, vp])
_lib.register("edl_lora_grads", i32, [vp, i64, vp, i64, vp, vp, vp, vp, i64, i64, vp, i64, i64, i32, i32, i32, i32, i32, i32, vp, i32,
                                      i32, i32, vp])

MAX_RANK = 512       # ranks of all parts together
MAX_PARTS = 8
FEW_ROWS = 256       # up to here the inner value stays in shared memory


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows ``[T, width]`` with neighbouring elements side by side: a view where it has such a layout."""
    t2 = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    return t2 if t2.stride(1) == 1 or t2.shape[1] == 1 else t2.contiguous()


def _weights(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _check(y, x, a, b, index, scale, parts, out):
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0]:
        raise ValueError(f"adapters are [n, parts * r, in] and [n, out, r], got {tuple(a.shape)} and {tuple(b.shape)}")
    n, N, r = b.shape
    parts = (N,) if parts is None else tuple(int(p) for p in parts)
    if min(n, N, r, a.shape[2]) < 1:
        raise ValueError("adapters without elements")
    if sum(parts) != N or min(parts) < 1 or len(parts) > MAX_PARTS:
        raise ValueError(f"parts {parts} (at most {MAX_PARTS}, none empty) do not add up to the {N} output columns")
    if a.shape[1] != len(parts) * r:
        raise ValueError(f"{a.shape[1]} ranks contract x, {len(parts)} part(s) of rank {r} need {len(parts) * r}")
    if a.shape[1] > MAX_RANK:
        raise ValueError(f"{a.shape[1]} ranks over all parts; at most {MAX_RANK}")
    if x.dim() < 1 or x.shape[-1] != a.shape[2]:
        raise ValueError(f"rows of x have {x.shape[-1] if x.dim() else 0} elements, the adapters take {a.shape[2]}")
    if tuple(y.shape) != (*x.shape[:-1], N):
        raise ValueError(f"y is {tuple(y.shape)}, x and the adapters ask for {(*x.shape[:-1], N)}")
    if x.dtype not in (torch.bfloat16, torch.float32) or a.dtype != x.dtype or b.dtype != x.dtype:
        raise TypeError(f"x and its adapters are all bfloat16 or all float32, got {x.dtype}, {a.dtype}, {b.dtype}")
    if y.dtype != x.dtype and y.dtype != torch.float32:
        raise TypeError(f"y is of x's type or float32, got {y.dtype} beside {x.dtype}")
    T = x.numel() // x.shape[-1]
    if index is None:
        if n != 1:
            raise ValueError(f"{n} adapters need an index per row")
    elif index.dtype != torch.int32 or index.numel() != T or not index.is_contiguous():
        raise ValueError(f"index is a contiguous int32 tensor with an entry for each of the {T} rows")
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.shape != (n,) or not scale.is_contiguous():
            raise ValueError(f"scale is a number or a contiguous float32 tensor [{n}]")
        if scale.requires_grad:
            raise NotImplementedError("there is no gradient for the scales of adapters")
    if out is not None and (out.shape != y.shape or out.dtype != y.dtype):
        raise ValueError(f"out is {tuple(out.shape)} of {out.dtype}, y {tuple(y.shape)} of {y.dtype}")
    for t in (x, a, b, index, scale, out):
        if isinstance(t, torch.Tensor) and t.device != y.device:
            raise ValueError(f"tensors on {y.device} and {t.device}")
    return parts


def _inner(T: int, r: int, parts: int, result: torch.dtype, device, backward: bool = False) -> torch.Tensor:
    """Memory for the scaled inner value ``s x a^T`` (``s dy b`` of the backward pass) as bf16 parts ``[parts of a value, T, ranks]``."""
    cols = (parts * r + 15) // 16 * 16 if backward else parts * ((r + 15) // 16 * 16)
    return torch.empty((3 if result == torch.float32 else 2, T, cols), dtype=torch.bfloat16, device=device)


def _apply(x, y, out, a, b, index, scale, u, parts, backward=False):
    n, N, r = b.shape
    if u is None and x.shape[0] > FEW_ROWS:
        u = _inner(x.shape[0], r, len(parts), out.dtype, x.device, backward)
    st = scale if isinstance(scale, torch.Tensor) else None
    ld = [0 if t is None else t.stride(0) if t.shape[0] > 1 else t.shape[1] for t in (x, y, out)]
    with _lib.on_device(x.device):
        _lib.call("edl_lora_apply", x.data_ptr(), ld[0], _lib.ptr(y), ld[1], _lib.ptr(out), ld[2], a.data_ptr(), a.stride(0), a.stride(1),
                  b.data_ptr(), b.stride(0), b.stride(1), _lib.ptr(index), _lib.ptr(st), 0.0 if st is not None else float(scale),
                  _lib.ptr(u), 0 if u is None else u.numel(), x.shape[0], a.shape[2], N, n, r, len(parts), (C.c_int * len(parts))(*parts),
                  int(x.dtype == torch.float32), int((out if out is not None else x).dtype == torch.float32), int(backward),
                  _lib.status_word(x.device).data_ptr(), _lib.stream_ptr())


def _grad_target(w: torch.Tensor):
    """(tensor that takes the gradient of adapter weights ``w``, whether it is added to, whether autograd gets it)."""
    mg = getattr(w, "main_grad", None)
    if mg is not None and mg.dtype == torch.float32 and mg.stride(-1) == 1:
        return mg.view(w.shape) if mg.shape != w.shape else mg, True
    return torch.empty(w.shape, dtype=w.dtype, device=w.device), False


class _LoraAddFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, index, scale, parts):
        y2, x2, a2, b2 = _rows(y), _rows(x), _weights(a), _weights(b)
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
        u = _inner(x2.shape[0], b.shape[2], len(parts), x.dtype, x.device) if ctx.needs_input_grad[3] else None
        _apply(x2, y2, out.view(-1, out.shape[-1]), a2, b2, index, scale, u, parts)
        ctx.save_for_backward(x, a, b, u, index, scale if isinstance(scale, torch.Tensor) else None)
        ctx.scale, ctx.parts = scale, parts
        ctx.targets = [getattr(w, "main_grad", None) is not None for w in (a, b)]
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, a, b, u, index, st = ctx.saved_tensors
        scale, parts = st if st is not None else ctx.scale, ctx.parts
        need_y, need_x, need_a, need_b = ctx.needs_input_grad[:4]
        dy2, x2 = _rows(dy), _rows(x)
        T, (n, N, r) = x2.shape[0], b.shape
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        g = _inner(T, r, len(parts), x.dtype, x.device, True) if need_a else None
        if need_x or need_a:
            _apply(dy2, None, None if dx is None else dx.view(-1, dx.shape[-1]), _weights(a), _weights(b), index, scale, g, parts, True)
        grads = []
        jobs: dict[tuple[bool, bool], list] = {}
        for need, w, slot in ((need_a, a, 0), (need_b, b, 1)):
            if not need:
                grads.append(None)
                continue
            t, added = _grad_target(w)
            jobs.setdefault((t.dtype == torch.float32, added), [None, None])[slot] = t
            grads.append(None if added else t)
            if added:
                w.grad_added_to_main_grad = True
        with _lib.on_device(x.device):
            for (wide, added), (da, db) in jobs.items():
                _lib.call("edl_lora_grads", x2.data_ptr(), x2.stride(0) if T > 1 else x2.shape[1], dy2.data_ptr(),
                          dy2.stride(0) if T > 1 else N, _lib.ptr(g), _lib.ptr(u), _lib.ptr(index), _lib.ptr(da),
                          0 if da is None else da.stride(0), 0 if da is None else da.stride(1), _lib.ptr(db),
                          0 if db is None else db.stride(0), 0 if db is None else db.stride(1), T, a.shape[2], N, n, r, len(parts),
                          (C.c_int * len(parts))(*parts), int(x.dtype == torch.float32), int(wide), int(added), _lib.stream_ptr())
        return dy if need_y else None, dx, *grads, None, None, None


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
    parts = _check(y, x, a, b, index, scale, parts, out)
    grad = torch.is_grad_enabled() and any(t.requires_grad for t in (y, x, a, b))
    if grad and out is not None:
        raise ValueError("out= is for inference: a gradient needs y as it was")
    if not _lib.use_kernels(x):
        o = lora_add_reference(y, x, a, b, index, scale, parts=parts)
        return o if out is None else out.copy_(o)
    if grad:
        if y.dtype != x.dtype:
            raise NotImplementedError("float32 outputs beside bfloat16 rows have no backward pass")
        return _LoraAddFn.apply(y, x, a, b, index, scale, parts)
    res = torch.empty(y.shape, dtype=y.dtype, device=y.device) if out is None else out
    o2 = res if res.dim() == 2 and (res.stride(1) == 1 or res.shape[1] == 1) else res.view(-1, res.shape[-1]) if res.is_contiguous() else None
    if o2 is None:      # no rows with neighbouring elements to write to
        return res.copy_(lora_add(y, x, a, b, index, scale, parts=parts))
    y2 = o2 if res is y else _rows(y)
    _apply(_rows(x), y2, o2, _weights(a), _weights(b), index, scale, None, parts)
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
