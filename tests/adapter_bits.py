"""Operands that show a lost part of a 32-bit value, and the bound of a result that has all of them.

Every value is positive and its third bf16 part is as large as it can be, so nothing cancels: a result whose operand came without that part is short of
2^-17 of itself, whatever the number of products."""

from __future__ import annotations

import torch

F32 = torch.float32


def values(*shape, seed=0, device="cpu"):
    """(1 + k 2^-16 + 63 2^-23) 2^e, 128 <= k < 255, e of -1, 0, 1: first part 2^e, second k 2^(e - 16), third 63 2^(e - 23)."""
    g = torch.Generator().manual_seed(seed)
    k, e = torch.randint(128, 255, shape, generator=g).double(), torch.randint(-1, 2, shape, generator=g).double()
    return ((1 + k * 2.0 ** -16 + 63 * 2.0 ** -23) * 2.0 ** e).to(F32).to(device)


def parts(v: torch.Tensor, n: int = 3) -> list[torch.Tensor]:
    """The first ``n`` bf16 parts of float32 values, rounded to nearest."""
    out = []
    for _ in range(n):
        p = v.to(torch.bfloat16).float()
        out.append(p)
        v = v - p
    return out


def make(T, K, widths, r, n, device="cpu", seed=0):
    N, P = sum(widths), len(widths)
    v = [values(*s, seed=10 * seed + i, device=device) for i, s in enumerate(((T, K), (T, N), (n, P * r, K), (n, N, r)))]
    index = torch.randint(0, n, (T,), generator=torch.Generator().manual_seed(seed)).to(torch.int32).to(device)
    return dict(x=v[0], y=torch.zeros(T, N, device=device), dy=v[1], a=v[2], b=v[3], index=index, scale=torch.ones(n, device=device), parts=tuple(widths))


def bound(first, second, rank):
    """Relative to results whose terms are all positive. Two products follow one another: sums of ``first`` terms, then of ``second`` ones. For each,
    in units of 2^-24: the parts that are left out, 1; a group of sixteen products cut off at 2^-23 by the tensor cores, 2; a rounded sum of
    groups: of those of a warp (a sixteenth of 16-row groups fall to one of 16 warps at least), 8 warps and 8 CTAs. The factor, y and the result round."""
    each = lambda n: 3 + n / 256 + 16  # noqa: E731
    return (each(first) + (3 + rank / 16 + 1 if second is None else each(2 * second)) + 3) * 2.0 ** -24
