"""Inputs and 64-bit results of logit rule tests."""

from __future__ import annotations

import random

import torch


def make(R, V, dtype, device, penalties=True, biases=5, masked=True, seed=0):
    g, r = torch.Generator().manual_seed(seed), random.Random(seed)
    c = dict(logits=(torch.randn(R, V, generator=g) * 3).to(dtype).to(device), kw={})
    if penalties:
        S = R + 2
        counts = torch.zeros(S, V, dtype=torch.int32)
        counts.scatter_add_(1, torch.randint(0, V, (S, 3 * V // 4), generator=g), torch.ones(S, 3 * V // 4, dtype=torch.int32))
        c["kw"].update(counts=counts.to(device), count_rows=torch.tensor([r.choice([-1, S - 1 - i]) for i in range(R)], dtype=torch.int32).to(device),
                       presence=(torch.rand(R, generator=g) * 2 - 1).to(device), frequency=torch.rand(R, generator=g).to(device),
                       repetition=(torch.rand(R, generator=g) + 0.5).to(device))
    if biases:
        n = [r.randint(0, biases) for _ in range(R)]
        ids = torch.cat([torch.randint(0, V, (k,), generator=g).sort().values for k in n]).to(torch.int32)       # the same id twice, too
        values = torch.randn(len(ids), generator=g) * 4
        values[torch.rand(len(ids), generator=g) < 0.2] = -float("inf")
        ptr = torch.tensor([sum(n[:i]) for i in range(R + 1)], dtype=torch.int32)
        c["kw"]["bias"] = (ptr.to(device), ids.to(device), values.to(device))
    if masked:
        allow = torch.rand(4, (V + 31) // 32 * 32, generator=g) < torch.tensor([0.0, 0.02, 0.5, 1.0])[:, None]
        c["kw"]["mask"] = (pack(allow).to(device), torch.tensor([r.randint(-1, 3) for _ in range(R)], dtype=torch.int32).to(device))
    return c


def pack(allow: torch.Tensor) -> torch.Tensor:
    w = (allow.view(allow.shape[0], -1, 32).long() << torch.arange(32)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def exact(c):
    """(values in 64 bits, sums of the magnitudes that go into them)."""
    z = c["logits"].double().cpu()
    kw = {k: tuple(t.cpu() if t is not None else None for t in v) if isinstance(v, tuple) else v.cpu() for k, v in c["kw"].items()}
    mag = z.abs()
    for r in range(z.shape[0]):
        if "counts" in kw:
            s = int(kw["count_rows"][r]) if "count_rows" in kw else r
            if s >= 0:
                n = kw["counts"][s, :z.shape[1]].double()
                rep, pre, fre = (float(kw[k][r]) if k in kw else d for k, d in (("repetition", 1.0), ("presence", 0.0), ("frequency", 0.0)))
                new = torch.where(z[r] > 0, z[r] / rep, z[r] * rep)
                mag[r] = torch.where(n > 0, new.abs() + abs(pre) + abs(fre) * n, mag[r])
                z[r] = torch.where(n > 0, new - pre - fre * n, z[r])
        if "bias" in kw:
            lo, hi = int(kw["bias"][0][r]), int(kw["bias"][0][r + 1])
            add: dict[int, float] = {}
            for i, v in zip(kw["bias"][1][lo:hi].tolist(), kw["bias"][2][lo:hi].double().tolist()):
                add[i] = add.get(i, 0.0) + v
                mag[r, i] += abs(v)
            for i, v in add.items():
                z[r, i] = v if v == -float("inf") else z[r, i] + v
        if "mask" in kw:
            m = r if kw["mask"][1] is None else int(kw["mask"][1][r])
            if m >= 0:
                t = torch.arange(z.shape[1])
                z[r, ((kw["mask"][0][m].long()[t // 32] >> (t % 32)) & 1) == 0] = -float("inf")
    return z, mag


def check(got, want, mag):
    """Half a step of the result's type, and a rounding to 32 bits of each of at most twelve operations (repeated ids add up)."""
    assert got.shape == want.shape
    step = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu()
    fine = torch.isfinite(want)
    odd = ~fine & ~torch.isnan(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[odd], want[odd])
    assert ((got - want).abs()[fine] <= (step * want.abs() + 12 * 2.0 ** -24 * mag)[fine]).all()
