"""What a batch of requests brings along of its own, and what its speed is tracked on: low-rank adapters of many requests beside
a shared projection (one serving step, and a training step of the adapters), and the rules for the next token (penalties, biases,
grammar masks) on the logits.

``listed()`` names the cases, ``draw(rng)`` gives one more of the same ranges, ``prepare`` makes what a program holds before the
call, ``run`` makes one pass: in plain tensor operations, or, where ``own`` is true, through the framework's entry points.
``work`` counts the bytes and operations a pass cannot do without, ``exact`` computes the same outputs in 64 bits.

Kinds: ``serve`` (adapters added to the output of a projection, no gradients), ``train`` (the same, forward and backward),
``rules`` (logits of a step's rows -> the logits that the sampler draws from).
"""

from __future__ import annotations

import math
import random

import torch

own = False

BF = torch.bfloat16
F32 = torch.float32
#: width in, widths out of the projections that carry adapters: packed queries / keys / values, output, packed gate / up, down
SHAPES = {
    "qkv": (4096, (4096, 1024, 1024)), "o": (4096, (4096,)), "gate_up": (4096, (14336, 14336)), "down": (14336, (4096,)),
    "small qkv": (1024, (1024, 256, 256)), "small down": (2816, (1024,)), "medium gate_up": (2048, (6144, 6144)),
    "shard qkv": (8192, (1024, 128, 128)), "shard down": (3584, (8192,)),
    "odd": (1001, (1003,)), "odd parts": (333, (129, 65, 63)),
}


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one user waiting for the next token, the output projection
        dict(name="adapter 1 request", kind="serve", shape="o", rank=16, adapters=4, singles=1, seqs=0, tokens=0, bare=0.0, dtype="bf16"),
        # an ordinary decode step: most requests bring an adapter, a few run the bare model; the packed projection
        dict(name="adapters 48 requests", kind="serve", shape="qkv", rank=16, adapters=32, singles=48, seqs=0, tokens=0, bare=0.2,
             dtype="bf16"),
        # a full engine, adapters of a higher rank, the longest rows
        dict(name="adapters 256 requests", kind="serve", shape="down", rank=32, adapters=64, singles=256, seqs=0, tokens=0, bare=0.1,
             dtype="bf16"),
        # prompts of several requests and running ones in one step, the widest projection
        dict(name="adapters prompts 5+3", kind="serve", shape="gate_up", rank=16, adapters=8, singles=3, seqs=5, tokens=3900, bare=0.1,
             dtype="bf16"),
        # a float32 model with sizes that no vector load fits
        dict(name="adapters odd f32", kind="serve", shape="odd", rank=5, adapters=3, singles=5, seqs=2, tokens=72, bare=0.2, dtype="f32"),
        # fine-tuning one adapter on a packed sequence of the headline run
        dict(name="train 1x8192 o", kind="train", shape="o", rank=16, adapters=1, seqs=1, tokens=8192, dtype="bf16"),
        # the same with a high rank at the longest rows
        dict(name="train 1x8192 down r64", kind="train", shape="down", rank=64, adapters=1, seqs=1, tokens=8192, dtype="bf16"),
        # three short rows that train an adapter each, a small model
        dict(name="train 3x1021 qkv", kind="train", shape="small qkv", rank=8, adapters=3, seqs=3, tokens=3063, dtype="bf16"),
        # one request that answers in a grammar
        dict(name="rules 1x32000", kind="rules", rows=1, vocab=32000, dtype="bf16", penalties=0.0, biases=0, masked=1.0),
        # an ordinary step: some rows with penalties, some in a grammar, a few biases each
        dict(name="rules 64x128256", kind="rules", rows=64, vocab=128256, dtype="bf16", penalties=0.5, biases=40, masked=0.5),
        # a full engine, 32-bit logits, rules on most rows
        dict(name="rules 256x151936 f32", kind="rules", rows=256, vocab=151936, dtype="f32", penalties=0.8, biases=300, masked=0.8),
        # an odd vocabulary, no grammar
        dict(name="rules 7x50257", kind="rules", rows=7, vocab=50257, dtype="bf16", penalties=1.0, biases=8, masked=0.0),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["decode", "decode", "prompts", "train", "train", "rules", "rules"])
    if kind == "rules":
        return dict(kind="rules", rows=_log(rng, 1, 256), vocab=rng.choice([4096, 32000, 50257, 128256, 151936, rng.randint(100, 99999)]),
                    dtype=rng.choice(["bf16", "bf16", "f32"]), penalties=rng.choice([0.0, 1.0, rng.random()]),
                    biases=rng.choice([0, _log(rng, 1, 300)]), masked=rng.choice([0.0, 1.0, rng.random()]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    shape = rng.choice(list(SHAPES) if dtype == "bf16" else ["small qkv", "small down", "odd", "odd parts"])
    rank = rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)])
    if kind == "train":
        seqs = _log(rng, 1, 8)
        return dict(kind="train", shape=shape, rank=rank, adapters=rng.randint(1, seqs), seqs=seqs, tokens=max(seqs, _log(rng, 16, 8192)),
                    dtype=dtype)
    seqs = rng.randint(1, 8) if kind == "prompts" else 0
    singles = _log(rng, 1, 256) if kind == "decode" else rng.choice([0, rng.randint(1, 40)])
    return dict(kind="serve", shape=shape, rank=rank, adapters=_log(rng, 1, 64), singles=singles, seqs=seqs,
                tokens=max(seqs * 2, _log(rng, 20, 3800)) if seqs else 0, bare=rng.choice([0.0, 0.1, 0.5]), dtype=dtype)


# --------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _rn(g, *shape, std=1.0, dtype=BF):
    return torch.randn(shape, generator=g, device="cuda", dtype=F32).mul_(std).to(dtype)


def _split(total: int, parts: int, key: str) -> list[int]:
    """``parts`` ragged lengths that add up to ``total``: the same for every seed."""
    r = random.Random(key)
    w = [r.uniform(0.2, 1.0) for _ in range(parts)]
    out = [1 + int((total - parts) * x / sum(w)) for x in w]
    out[0] += total - sum(out)
    return out


def _requests(case) -> list[tuple[int, int]]:
    """(tokens, adapter or -1) of every request, single tokens first: the same for every seed. Some adapters are popular."""
    n, r = case["adapters"], random.Random(f"{case['shape']}/{case['tokens']}/{case['seqs']}/{case.get('singles')}")
    if case["kind"] == "train":
        return [(length, b % n) for b, length in enumerate(_split(case["tokens"], case["seqs"], f"t{case['tokens']}"))]
    lens = [1] * case["singles"] + (_split(case["tokens"], case["seqs"], f"p{case['tokens']}") if case["seqs"] else [])
    return [(length, -1 if r.random() < case["bare"] else int(n * r.random() ** 1.5)) for length in lens]


def _adapter_inputs(case, seed):
    g, dt = _gen(seed), BF if case["dtype"] == "bf16" else F32
    (K, parts), r, n = SHAPES[case["shape"]], case["rank"], case["adapters"]
    N, P, reqs = sum(parts), len(parts), _requests(case)
    T = sum(a for a, _ in reqs)
    index = torch.tensor(sum(([i] * a for a, i in reqs), []), dtype=torch.int32, device="cuda")
    s = dict(x=_rn(g, T, K, dtype=dt), y=_rn(g, T, N, dtype=dt), a=_rn(g, n, P * r, K, std=K ** -0.5, dtype=dt),
             b=_rn(g, n, N, r, std=0.5 * r ** -0.5, dtype=dt), index=index,
             scale=torch.rand(n, generator=g, device="cuda") + 0.5, parts=parts, kind=case["kind"])
    if case["kind"] == "train":
        s["dy"] = _rn(g, T, N, dtype=dt)
        if case["seqs"] == 1:
            s["index"] = None       # one adapter for every row
    return s


def _rules_inputs(case, seed):
    g, R, V = _gen(seed), case["rows"], case["vocab"]
    r = random.Random(f"{R}/{V}/{case['biases']}")
    logits = _rn(g, R, V, std=3.0, dtype=BF if case["dtype"] == "bf16" else F32)
    s = dict(kind="rules", logits=logits, counts=None, bias=None, mask=None)
    if case["penalties"]:
        # token counts of the engine's slots; a row points at its slot, or at none
        slots = R + 3
        text = torch.randint(0, V, (slots, 400), generator=g, device="cuda")
        counts = torch.zeros(slots, V, dtype=torch.int32, device="cuda")
        counts.scatter_add_(1, text, torch.ones_like(text, dtype=torch.int32))
        at = [(R - 1 - i) if r.random() < case["penalties"] else -1 for i in range(R)]
        s["counts"], s["count_rows"] = counts, torch.tensor(at, dtype=torch.int32, device="cuda")
        s["presence"] = torch.rand(R, generator=g, device="cuda") - 0.3
        s["frequency"] = torch.rand(R, generator=g, device="cuda") * 0.5
        s["repetition"] = torch.rand(R, generator=g, device="cuda") * 0.6 + 0.8
    if case["biases"]:
        n = [r.randint(0, min(case["biases"], V)) for _ in range(R)]
        ids = torch.cat([torch.randperm(V, generator=g, device="cuda")[:k].sort().values for k in n]).to(torch.int32)
        values = torch.randn(sum(n), generator=g, device="cuda") * 4
        values[torch.rand(sum(n), generator=g, device="cuda") < 0.1] = -math.inf        # a forbidden token
        ptr = torch.tensor([sum(n[:i]) for i in range(R + 1)], dtype=torch.int32, device="cuda")
        s["bias"] = (ptr, ids, values)
    if case["masked"]:
        # states of a grammar: some allow a handful of tokens, some all but a few; rows share them
        states, W = 6, (V + 31) // 32
        share = torch.tensor([0.001, 0.02, 0.3, 0.9, 0.002, 0.999], device="cuda")[:, None]
        allow = torch.rand(states, W * 32, generator=g, device="cuda") < share
        weights = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
        bits = (allow.view(states, W, 32).long() * weights).sum(-1)
        bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
        at = [r.randrange(states) if r.random() < case["masked"] else -1 for _ in range(R)]
        s["mask"] = (bits, torch.tensor(at, dtype=torch.int32, device="cuda"))
    return s


def prepare(case, seed):
    return _rules_inputs(case, seed) if case["kind"] == "rules" else _adapter_inputs(case, seed)


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_adapters(y, x, a, b, index, scale, parts):
    """Every row against every adapter, with the products of the others' set to zero."""
    (T, K), (n, N, r), P = x.shape, b.shape, len(parts)
    at = torch.zeros(T, dtype=torch.int64, device=x.device) if index is None else index.long()
    on = (at[:, None] == torch.arange(n, device=x.device)) * scale                       # [T, n]
    u = (x.float() @ a.float().view(n * P * r, K).t()).view(T, n, P, r)
    u = torch.where(on[:, :, None, None] != 0, u * on[:, :, None, None], 0.0)
    part = torch.repeat_interleave(torch.arange(P, device=x.device), torch.tensor(parts, device=x.device))
    wide = torch.where(part[None, :, None, None] == torch.arange(P, device=x.device)[None, None, :, None], b.float()[:, :, None], 0.0)
    return (y.float() + u.view(T, n * P * r) @ wide.permute(0, 2, 3, 1).reshape(n * P * r, N)).to(y.dtype)


def _plain_rules(s):
    z = s["logits"].float()
    R, V = z.shape
    if s["counts"] is not None:
        c = torch.where(s["count_rows"][:, None] >= 0, s["counts"][s["count_rows"].long().clamp(min=0)], 0)
        rep = s["repetition"][:, None]
        z = torch.where(c > 0, torch.where(z > 0, z / rep, z * rep) - (s["presence"][:, None] + s["frequency"][:, None] * c), z)
    if s["bias"] is not None:
        ptr, ids, values = s["bias"]
        rows = torch.repeat_interleave(torch.arange(R, device=z.device), ptr.diff().long(), output_size=ids.numel())
        add = torch.zeros_like(z).index_put_((rows, ids.long()), values, accumulate=True)
        z = torch.where(add == -math.inf, add, z + add)
    if s["mask"] is not None:
        bits, at = s["mask"]
        allow = (bits[at.long().clamp(min=0)][..., None] >> torch.arange(32, dtype=torch.int32, device=z.device)) & 1
        z = torch.where((allow.reshape(R, -1)[:, :V] == 1) | (at[:, None] < 0), z, -math.inf)
    return z


# ---------------------------------------------------------------------------------------------------------------- calls
def run(s):
    if s["kind"] == "rules":
        if own:
            from easydel_b200.ops import serving

            kw = {}
            if s["counts"] is not None:
                kw = dict(counts=s["counts"], count_rows=s["count_rows"], presence=s["presence"], frequency=s["frequency"],
                          repetition=s["repetition"])
            return serving.adjust_logits(s["logits"], bias=s["bias"], mask=s["mask"], **kw)
        return _plain_rules(s)
    if own:
        from easydel_b200.ops import adapters

        call = adapters.lora_add
    else:
        call = _plain_adapters
    if s["kind"] == "serve":
        with torch.no_grad():
            return call(s["y"], s["x"], s["a"], s["b"], s["index"], s["scale"], parts=s["parts"])
    x, a, b = (s[name].detach().requires_grad_() for name in ("x", "a", "b"))
    out = call(s["y"], x, a, b, s["index"], s["scale"], parts=s["parts"])
    out.backward(s["dy"])
    return dict(out=out.detach(), dx=x.grad, da=a.grad, db=b.grad)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "rules":
        n, e = case["rows"] * case["vocab"], 2 if case["dtype"] == "bf16" else 4
        pen = 4 * case["penalties"] * n
        return dict(bytes=n * (e + 4.0) + pen + 8.0 * case["rows"] * case["biases"] / 2 + 6 * case["vocab"] / 8 * (case["masked"] > 0),
                    flops=2.0 * n)
    (K, parts), r, reqs = SHAPES[case["shape"]], case["rank"], _requests(case)
    N, P, e = sum(parts), len(parts), 2 if case["dtype"] == "bf16" else 4
    T, active = sum(a for a, _ in reqs), sum(a for a, i in reqs if i >= 0)
    weights = len({i for _, i in reqs if i >= 0}) * r * (P * K + N)
    flops = 2.0 * active * r * (P * K + N)
    if case["kind"] == "serve":
        return dict(bytes=e * (1.0 * active * K + 2.0 * T * N + weights), flops=flops)
    return dict(bytes=e * (2.0 * T * K + 3.0 * T * N + 2.0 * weights), flops=3 * flops)


# ------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_adapters(case, seed):
    i = _adapter_inputs(case, seed)
    parts, r = i["parts"], case["rank"]
    x, y, a, b = (i[k].double() for k in ("x", "y", "a", "b"))
    dy = i["dy"].double() if case["kind"] == "train" else None
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for n in range(case["adapters"]):
        rows = torch.arange(len(x), device="cuda") if i["index"] is None else (i["index"] == n).nonzero()[:, 0]
        s, c0 = float(i["scale"][n].double()), 0
        for p, width in enumerate(parts):
            A, B = a[n, p * r:(p + 1) * r], b[n, c0:c0 + width]
            u = x[rows] @ A.t()
            y[rows, c0:c0 + width] += s * (u @ B.t())
            if dy is not None:
                d = dy[rows, c0:c0 + width]
                g = s * (d @ B)
                dx[rows] += g @ A
                da[n, p * r:(p + 1) * r] += g.t() @ x[rows]
                db[n, c0:c0 + width] += s * (d.t() @ u)
            c0 += width
    return y if dy is None else dict(out=y, dx=dx, da=da, db=db)


def _exact_rules(case, seed):
    i = _rules_inputs(case, seed)
    z, V = i["logits"].double(), case["vocab"]
    for r in range(case["rows"]):
        if i["counts"] is not None and int(i["count_rows"][r]) >= 0:
            c = i["counts"][int(i["count_rows"][r])].double()
            rep, pre, fre = (float(i[k][r]) for k in ("repetition", "presence", "frequency"))
            seen = z[r].clone()
            seen[z[r] > 0] /= rep
            seen[z[r] <= 0] *= rep
            z[r] = torch.where(c > 0, seen - pre - fre * c, z[r])
        if i["bias"] is not None:
            ptr, ids, values = i["bias"]
            lo, hi = int(ptr[r]), int(ptr[r + 1])
            z[r, ids[lo:hi].long()] += values[lo:hi].double()
        if i["mask"] is not None and int(i["mask"][1][r]) >= 0:
            w = i["mask"][0][int(i["mask"][1][r])].long() & 0xffffffff
            t = torch.arange(V, device="cuda")
            z[r, (w[t // 32] >> (t % 32)) % 2 == 0] = -math.inf
    return z


def exact(case, seed):
    return _exact_rules(case, seed) if case["kind"] == "rules" else _exact_adapters(case, seed)
