"""Inputs, 64-bit results and error bounds of adapter tests."""

from __future__ import annotations

import torch


def make(T, K, parts, r, n, dtype, device, index="mixed", seed=0, scale="tensor"):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s, std=1.0: (torch.randn(s, generator=g) * std).to(dtype).to(device)  # noqa: E731
    N, P = sum(parts), len(parts)
    x, y, dy = rn(T, K), rn(T, N), rn(T, N)
    a, b = rn(n, P * r, K, std=K ** -0.5), rn(n, N, r, std=r ** -0.5)
    if index == "none":
        idx = None
    elif index == "mixed":
        idx = torch.randint(-1, n, (T,), generator=g)
    elif index == "runs":
        idx = (torch.arange(T) * n) // max(T, 1)
    elif index == "bare":
        idx = torch.full((T,), -1)
    else:
        idx = torch.full((T,), int(index))
    if idx is not None:
        idx = idx.to(torch.int32).to(device)
    s = (torch.rand(n, generator=g) + 0.5).to(device) if scale == "tensor" else scale
    return dict(x=x, y=y, a=a, b=b, index=idx, scale=s, parts=tuple(parts), dy=dy)


def exact(c, grads=False):
    """The formulas in 64 bits: values, and the sums of the magnitudes that go into them."""
    x, y, a, b = (c[k].double().cpu() for k in ("x", "y", "a", "b"))
    T, n, r = x.shape[0], a.shape[0], b.shape[2]
    idx = torch.zeros(T, dtype=torch.long) if c["index"] is None else c["index"].long().cpu()
    s = c["scale"].double().cpu() if isinstance(c["scale"], torch.Tensor) else torch.full((n,), float(c["scale"])).double()
    val = dict(out=y.clone(), dx=torch.zeros_like(x), da=torch.zeros_like(a), db=torch.zeros_like(b))
    mag = {k: v.abs() for k, v in val.items()}
    dy = c["dy"].double().cpu()
    for i in range(n):
        at = (idx == i).nonzero()[:, 0]
        c0 = 0
        for p, w in enumerate(c["parts"]):
            A, B, X, D = a[i, p * r:(p + 1) * r], b[i, c0:c0 + w], x[at], dy[at, c0:c0 + w]
            for m, f in ((val, lambda t: t), (mag, torch.abs)):
                u, g = f(s[i]) * (f(X) @ f(A).t()), f(s[i]) * (f(D) @ f(B))
                m["out"][at, c0:c0 + w] += u @ f(B).t()
                m["dx"][at] += g @ f(A)
                m["da"][i, p * r:(p + 1) * r] = g.t() @ f(X)
                m["db"][i, c0:c0 + w] = f(D).t() @ u
            c0 += w
    return (val, mag) if grads else (val["out"], mag["out"])


def bound(dtype, want, mag, length):
    """One rounding of the result (half a step of its type), and of the sums: products of the tensor cores are added sixteen at a time and cut
    off at 2^-23 (six products for each where operands are fp32), 64 warps and 8 CTAs add theirs in fp32, parts of fp32 values that are left
    out are below 2^-21; the inner value enters the second product with 16 bits where the result is bf16. ``mag``: sum of the magnitudes."""
    if dtype == torch.bfloat16:
        return 2.0 ** -8 * want.abs() + (2.0 ** -15 + (length / 16 + 80) * 2.0 ** -22) * mag
    return 2.0 ** -24 * want.abs() + (2.0 ** -20 + (6 * length / 16 + 80) * 2.0 ** -22) * mag


def check(got, want, mag, length, what=""):
    off = (got.double().cpu() - want).abs()
    top = bound(got.dtype, want, mag, length)
    bad = ~(off <= top)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, by {float((off / top.clamp(min=1e-300))[bad].max()):.3g} bounds"
