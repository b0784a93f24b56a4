"""Low-rank adapters of many requests beside a shared projection (``csrc/lora.cu``).

Every row of a batch may bring an adapter of its own. The shared projection runs for all rows at once; :func:`lora_add` adds

    ``out[t, c] = y[t, c] + scale[i] * (x[t] @ a[i, p].T) @ b[i, c]``,  ``i = index[t]``, ``p`` the part of the output that ``c`` is in

in one launch (two or three for more than a few hundred rows), whatever the rows' order: which rows go together is found on the device, so a captured graph follows the indexes of
each replay. Packed projections (queries / keys / values, gate / up) have one adapter per part, stored together. Differentiable in
``y``, ``x``, ``a`` and ``b``. CPU tensors run the plain form.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib

vp, i32, i64, f32 = _lib.vp, _lib.i32, _lib.i64, _lib.f32


class _Shape(C.Structure):
    """``edl_lora_shape`` of ``csrc/lora.cu``."""

    _fields_ = [(k, i64) for k in ("ldx", "ldy", "ldo", "a_adapter", "lda", "b_adapter", "ldb")] + \
               [(k, i32) for k in ("T", "K", "N", "n", "r", "parts", "x_f32", "y_f32", "backward")] + [("widths", i32 * 8)]


_lib.register("edl_lora_apply", i32, [vp, vp, vp, vp, vp, vp, vp, vp, f32, vp, i64, vp, vp, vp])
_lib.register("edl_lora_backward", i32, [vp, vp, vp, vp, vp, vp, vp, vp, f32, vp, i64, vp, vp, vp, vp, vp, i32, i32, vp, vp])

MAX_RANK = 512       # ranks of all parts together
MAX_PARTS = 8
MAX_TRAINED = 65535  # adapters of a call with gradients
MAX_ROWS = 2 ** 31 - 1
BLOCK = 256          # rows that are looked through for their adapters together


def _matrix(t: torch.Tensor) -> bool:
    """Rows of neighbouring elements at one distance, apart from each other (leading dimensions, if more than one, lie one after the other)."""
    return (t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1) if t.dim() == 2 else t.is_contiguous()


def _stack(t: torch.Tensor) -> bool:
    """Matrices ``[n, rows, width]`` of such rows, apart from each other (a stack that is one matrix repeated is none)."""
    return (t.stride(2) == 1 or t.shape[2] == 1) and (t.stride(1) >= t.shape[2] or t.shape[1] == 1) and \
        (t.stride(0) >= t.stride(1) * (t.shape[1] - 1) + t.shape[2] or t.shape[0] == 1)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows ``[T, width]`` with neighbouring elements side by side: a view where it has such a layout."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if _matrix(t) else t.contiguous()


def _weights(t: torch.Tensor) -> torch.Tensor:
    return t if _stack(t) else t.contiguous()


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
    if x.numel() // sx[-1] > MAX_ROWS:
        raise ValueError(f"{x.numel() // sx[-1]} rows; at most {MAX_ROWS}")
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


def _inner_columns(r: int, parts: int, backward: bool) -> int:
    """Ranks of a row of the inner value, each part's (the backward pass: all) rounded up to 16."""
    return -(-parts * r // 16) * 16 if backward else parts * (-(-r // 16) * 16)


def _few_rows(T: int, cols: int, index: bool) -> bool:
    """``few_rows`` of ``csrc/lora.cu``: the inner value stays in shared memory."""
    return T <= 256 or T <= 512 and (index or cols <= 8192)


def pays(x: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether one adapter ``b [out, r]`` for all rows of ``x`` is faster by these kernels than by two library products and a sum.

    They have streaming forms for bfloat16 ranks up to 64 whose sizes 16-byte loads fit (8192 rows, 14336 columns to 4096, forward and backward: rank
    64 225 us, 275 by products; rank 128 709, 287), and cut float32 operands into parts for every 16 ranks (8192 rows, 14336 columns to 1024: rank
    32 1098 us, 982; to 4096: rank 16 790, 1222). Ranks or widths that those loads do not fit pay while the rows are few (512 rows, rank 14: 140
    us, 169; 8192 rows: 444, 329), of float32 with many rows too (rank 5 514 us, 697; rank 1 500, 383; rank 30 786, 731)."""
    rank, many, f32 = b.shape[1], x.numel() // x.shape[-1] > 512, x.dtype == torch.float32
    if rank % 4 == 0 and x.shape[-1] % 8 == 0 and b.shape[0] % 8 == 0:
        return rank <= (64 if not f32 else 16 if many else 32)
    return rank <= 16 and (not many or f32 and rank >= 4)


class _Plan:
    """What a call's sizes, strides and types decide: checked once, kept for the calls that follow with the same ones."""

    __slots__ = ("parts", "plain", "shape", "ref", "u_parts", "u_cols", "blocks", "T", "back", "grads")

    def __init__(self, x, y, out, a, b, parts, index, backward=False):
        n, N, r = b.shape
        # (strides along dimensions of one element mean nothing)
        rows = lambda t: 0 if t is None else t.stride(-2) if t.dim() > 1 and t.shape[-2] > 1 else t.shape[-1]  # noqa: E731
        each = lambda t: t.stride(0) if t.shape[0] > 1 else rows(t) * t.shape[1]  # noqa: E731
        res = x if out is None else out
        self.T = T = x.numel() // x.shape[-1]
        self.parts = parts
        self.shape = _Shape(rows(x), rows(y), rows(out), each(a), rows(a), each(b), rows(b), T, a.shape[2], N, n, r, len(parts),
                            x.dtype == torch.float32, res.dtype == torch.float32, backward, (i32 * 8)(*parts))
        self.ref = C.addressof(self.shape)
        self.u_parts, self.u_cols = 3 if res.dtype == torch.float32 else 2, _inner_columns(r, len(parts), backward)
        self.blocks = 0 if _few_rows(T, a.shape[2] if backward else N, index is not None) else -(-T // BLOCK)
        self.plain = False      # all operands, as the caller has them, are rows that kernels read
        self.back = self.grads = None      # the plans of the backward pass's calls, where all operands are contiguous

    def inner(self, x: torch.Tensor) -> torch.Tensor:
        """Memory for the scaled inner value (``s x a^T``, or ``s dy b`` of the backward pass) as bf16 parts ``[parts of a value, T, ranks]``."""
        return x.new_empty((self.u_parts, self.T, self.u_cols), dtype=torch.bfloat16)


def _apply(plan: _Plan, x, y, out, a, b, index, scale, u) -> None:
    u_size, mixed = 0, None
    if plan.blocks:
        if u is None:
            u = plan.inner(x)
        if index is not None:
            mixed = index.new_empty(plan.blocks)      # which blocks of rows have many adapters
    if u is not None:
        u_size, u = u.numel(), u.data_ptr()
    tensor = type(scale) is not float
    _lib.call_on(x.device, "edl_lora_apply", plan.ref, x.data_ptr(), None if y is None else y.data_ptr(), None if out is None else out.data_ptr(),
                 a.data_ptr(), b.data_ptr(), None if index is None else index.data_ptr(), scale.data_ptr() if tensor else None,
                 0.0 if tensor else scale, u, u_size, None if mixed is None else mixed.data_ptr(), _lib.status_word(x.device).data_ptr())


def _grad_target(w: torch.Tensor) -> tuple[torch.Tensor, bool]:
    """The tensor that takes the gradient of adapter weights ``w``, and whether it is added to (a slice of the flat gradient buffer)."""
    mg = getattr(w, "main_grad", None)
    if mg is None:
        return torch.empty_like(w, memory_format=torch.contiguous_format), False
    return mg.view(w.shape), True


class _LoraAddFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, index, scale, plan):
        out = torch.empty_like(y, memory_format=torch.contiguous_format)
        ctx.x_shape, a2, b2 = x.shape, a, b
        if not plan.plain:
            y, x, a2, b2 = _rows(y), _rows(x), _weights(a), _weights(b)
            plan = _Plan(x, y, out, a2, b2, plan.parts, index)
        u = plan.inner(x) if ctx.needs_input_grad[3] else None
        _apply(plan, x, y, out, a2, b2, index, scale, u)
        ctx.scale, ctx.plan = scale if type(scale) is float else None, plan
        ctx.save_for_backward(x, a, b, u, index, None if type(scale) is float else scale)
        return out

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise NotImplementedError("adapters have no second derivatives")
        x, a, b, u, index, scale = ctx.saved_tensors
        if scale is None:
            scale = ctx.scale
        plan, (need_y, need_x, need_a, need_b) = ctx.plan, ctx.needs_input_grad[:4]
        dy2 = dy if dy.is_contiguous() or _matrix(dy) else _rows(dy)
        da, a_added = _grad_target(a) if need_a else (None, False)
        db, b_added = _grad_target(b) if need_b else (None, False)
        dx = g = back = mixed = None
        g_size = 0
        if need_x or need_a:
            a2, b2 = (a, b) if plan.plain else (_weights(a), _weights(b))
            if need_x:
                dx = torch.empty_like(x) if x.shape == ctx.x_shape and x.is_contiguous() else x.new_empty(ctx.x_shape)
            usual = need_x and dy2.is_contiguous()
            back = plan.back if usual else None
            if back is None:
                back = _Plan(dy2, None, dx, a2, b2, plan.parts, index, True)
                if usual:
                    plan.back = back
            if need_a or back.blocks:
                g = back.inner(x)
                g_size = g.numel()
            if back.blocks and index is not None:
                mixed = index.new_empty(back.blocks)
        else:
            a2 = b2 = None
        # one call for all, unless only one of the weights' gradients is added to a flat buffer
        for ta, tb, added in ((da, db, a_added or b_added),) if da is None or db is None or a_added == b_added else \
                ((da, None, a_added), (None, db, b_added)):
            out = ta if tb is None else tb
            if back is None and out is None:
                continue
            usual = dy2.is_contiguous() and (ta is None or ta.is_contiguous()) and (tb is None or tb.is_contiguous())
            grads = plan.grads if usual else None
            if grads is None and out is not None:
                grads = _Plan(x, dy2, None, torch.empty_like(a, device="meta", memory_format=torch.contiguous_format) if ta is None else ta,
                              torch.empty_like(b, device="meta", memory_format=torch.contiguous_format) if tb is None else tb, plan.parts, index)
                if usual:
                    plan.grads = grads
            tensor = type(scale) is not float
            _lib.call_on(x.device, "edl_lora_backward", None if back is None else back.ref, None if grads is None else grads.ref, x.data_ptr(),
                         dy2.data_ptr(), _lib.ptr(a2), _lib.ptr(b2), _lib.ptr(index), scale.data_ptr() if tensor else None,
                         0.0 if tensor else scale, _lib.ptr(g), g_size, _lib.ptr(mixed), _lib.ptr(dx), _lib.ptr(u), _lib.ptr(ta), _lib.ptr(tb),
                         out is not None and out.dtype == torch.float32, added, _lib.status_word(x.device).data_ptr())
            back = None
        if a_added:
            a.grad_added_to_main_grad = True
        if b_added:
            b.grad_added_to_main_grad = True
        return dy if need_y else None, dx, None if a_added else da, None if b_added else db, None, None, None


_plans: dict[tuple, _Plan | None] = {}


def _plan_of(y, x, a, b, index, scale, parts, out) -> _Plan:
    """The plan of an inference call, by its sizes, strides, types and device."""
    tensor = isinstance(scale, torch.Tensor)
    key = (x.shape, x.stride(), x.dtype, x.device, y.shape, y.stride(), y.dtype, y.device, a.shape, a.stride(), a.dtype, a.device, b.shape, b.stride(),
           b.dtype, b.device, parts, index is None or (index.shape, index.dtype, index.device, index.is_contiguous()),
           (scale.shape, scale.dtype, scale.device, scale.is_contiguous(), scale.requires_grad) if tensor else None,
           0 if out is None else 1 if out is y else (out.shape, out.stride(), out.dtype, out.device))      # new rows lie side by side, y's need not
    plan = _plans.get(key)
    if plan is None:
        parts = _check(y, x, a, b, index, scale, parts, out)
        plan = _Plan(x, y, torch.empty_like(y, device="meta", memory_format=torch.contiguous_format) if out is None else out, a, b, parts, index)
        # operands whose rows have to be copied first, and results that cannot be written as rows, take the long way
        plan.plain = x.is_cuda and all(map(_matrix, (x, y) if out is None else (x, y, out))) and _stack(a) and _stack(b)
        if len(_plans) >= 4096:
            _plans.clear()
        _plans[key] = plan
    return plan


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor | None = None,
             scale: float | torch.Tensor = 1.0, *, parts: tuple[int, ...] | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """``y`` plus each row's adapter product.

    ``y [..., N]``: output of the shared projection of ``x [..., K]`` (bfloat16 or float32; ``y`` may be float32 beside bfloat16
    rows); ``a [n, P * r, K]``, ``b [n, N, r]``: the adapters' weights, of x's type; ``index``: int32, an adapter per row, negative
    for none (None: one adapter for all rows); ``scale``: a number, or float32 ``[n]``; ``parts``: widths of the P parts of a
    packed output, whose ranks follow one another in ``a``. Adapters of a smaller rank are padded with zeros. ``out``: where to write
    (``y`` itself for in place, else apart from all inputs; inference only; its rows do not overlap). An index of ``n`` or more counts as none and sets the status word that
    ``_lib.check_status`` reads. A row with infinities gives values that are not finite in that row alone; there are no second
    derivatives.
    """
    plan = _plan_of(y, x, a, b, index, scale, None if parts is None else tuple(parts), out)
    if torch.is_grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad or y.requires_grad):
        if out is not None:
            raise ValueError("out= is for inference: a gradient needs y as it was")
        if not _lib.use_kernels(x):
            return lora_add_reference(y, x, a, b, index, scale, parts=plan.parts)
        if y.dtype != x.dtype:
            raise NotImplementedError("float32 outputs beside bfloat16 rows have no backward pass")
        if b.shape[0] > MAX_TRAINED:
            raise ValueError(f"{b.shape[0]} adapters; gradients take at most {MAX_TRAINED}")
        return _LoraAddFn.apply(y, x, a, b, index, scale if isinstance(scale, torch.Tensor) else float(scale), plan)
    if plan.plain:
        res = torch.empty_like(y, memory_format=torch.contiguous_format) if out is None else out
        _apply(plan, x, y, res, a, b, index, scale if isinstance(scale, torch.Tensor) else float(scale), None)
        return res
    if not _lib.use_kernels(x):
        o = lora_add_reference(y, x, a, b, index, scale, parts=plan.parts)
        return o if out is None else out.copy_(o)
    if not isinstance(scale, torch.Tensor):
        scale = float(scale)
    if out is not None and not _matrix(out):      # no rows with neighbouring elements to write to
        return out.copy_(lora_add(y, x, a, b, index, scale, parts=plan.parts))
    res = torch.empty_like(y, memory_format=torch.contiguous_format) if out is None else out
    x2, y2, a2, b2 = _rows(x), res if res is y else _rows(y), _weights(a), _weights(b)
    _apply(_Plan(x2, y2, res, a2, b2, plan.parts, index), x2, y2, res, a2, b2, index, scale, None)
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
