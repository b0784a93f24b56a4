"""Calls of the adapters one after the other, and rows of one block in every order, against the formulas in 64 bits."""

import pytest
import torch
from adapter_cases import check, exact, make

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _call(c, **kw):
    from easydel_b200.ops import adapters

    return adapters.lora_add(c["y"], c["x"], c["a"], c["b"], c["index"], c["scale"], parts=c["parts"], **kw)


@pytest.mark.parametrize("T", [6, 300, 700])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("order", [("new", "in place", "grad"), ("in place", "new", "grad"), ("in place", "grad", "new")])
def test_new_results_and_results_in_place_of_one_strided_y(order, dtype, T, monkeypatch):
    from easydel_b200.ops import adapters

    monkeypatch.setattr(adapters, "_plans", {})
    c = make(T, 64, (32,), 8, 3, dtype, "cuda")
    want, mag = exact(c)
    wide = torch.full((T, 64), 7.0, dtype=dtype, device="cuda")
    plain = c["y"]
    for how in order:
        wide[:, :32] = plain
        c["y"] = wide[:, :32]
        if how == "in place":
            assert _call(c, out=c["y"]) is c["y"]
            check(wide[:, :32], want, mag, 64, how)
        elif how == "new":
            got = _call(c)
            assert got.stride() == (32, 1)
            check(got, want, mag, 64, how)
        else:
            got = _call(dict(c, x=c["x"].detach().requires_grad_()))
            check(got.detach(), want, mag, 64, how)
        assert (wide[:, 32:] == 7.0).all(), how


# blocks of 256 rows: rows of an adapter side by side, and rows of others that lie apart between them, one after the other in every order
def _layouts(T):
    t, row = torch.arange(T), torch.arange(T) % 256
    pair = torch.where(t % 2 == 0, 1, -1)
    return {
        "line, apart, line": torch.where(row < 60, 0, torch.where(row < 160, pair, 2)),
        "apart, apart, line": torch.where(row < 100, t % 2, 2),
        "apart, line, apart, line": torch.where(row < 40, torch.where(t % 2 == 0, 0, -1), torch.where(row < 90, 1, torch.where(row < 140, 2, torch.where(row == 200, 0, -1)))),
        "line, apart, apart": torch.where(row < 70, 2, t % 2),
        "line, line, apart, line in turns of blocks": torch.where(t // 256 % 2 == 0, torch.where(row < 128, 0, torch.where(row < 250, t % 2 + 1, 0)), row // 100),
    }


def _close(got, want, mag, length, what):
    """`check` with operands that stay where they are."""
    from adapter_cases import bound

    off, top = (got.double() - want).abs(), bound(got.dtype, want, mag, length)
    bad = ~(off <= top)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, first row {int(bad.any(1).nonzero()[0])}"


def _exact(x, y, a, b, index, scale, parts, dy=None):
    """out and its magnitudes, or dx and its: 64 bits, on the device."""
    r, n = b.shape[2], b.shape[0]
    x, a, b = x.double(), a.double(), b.double()
    val = y.double().clone() if dy is None else torch.zeros_like(x)
    mag = val.abs()
    for i in range(n):
        at, c0 = (index == i).nonzero()[:, 0], 0
        for p, w in enumerate(parts):
            A, B = a[i, p * r:(p + 1) * r], b[i, c0:c0 + w]
            for m, f in ((val, lambda t: t), (mag, torch.abs)):
                s = f(scale[i].double())
                if dy is None:
                    m[at, c0:c0 + w] += s * (f(x[at]) @ f(A).t()) @ f(B).t()
                else:
                    m[at] += s * (f(dy[at, c0:c0 + w].double()) @ f(B)) @ f(A)
            c0 += w
    return val, mag


@pytest.mark.parametrize("rank", [8, 16, 64])
@pytest.mark.parametrize("T,parts", [(600, (64,)), (1500, (128,)), (1500, (1344,)), (3900, (896, 128, 128)), (2100, (14336, 14336))])
def test_rows_side_by_side_and_apart_in_one_block(T, parts, rank):
    for name, index in _layouts(T).items():
        c = make(T, 64, parts, rank, 3, BF, "cuda", "bare", seed=T + rank)
        c["index"] = index.to(torch.int32).cuda()
        want, mag = _exact(c["x"], c["y"], c["a"], c["b"], c["index"], c["scale"], parts)
        got = _call(c)
        _close(got, want, mag, 64, name)
        for _ in range(4):
            assert torch.equal(got, _call(c)), name
        y = c["y"].clone()
        assert torch.equal(_call(dict(c, y=y), out=y), got), name


@pytest.mark.parametrize("rank", [8, 16, 64])
@pytest.mark.parametrize("T,K", [(600, 64), (1500, 128), (1500, 1344), (3900, 1152), (2100, 28672)])
def test_gradients_of_rows_side_by_side_and_apart_in_one_block(T, K, rank):
    for name, index in _layouts(T).items():
        c = make(T, K, (64,), rank, 3, BF, "cuda", "bare", seed=T + rank)
        c["index"] = index.to(torch.int32).cuda()
        want, mag = _exact(c["x"], c["y"], c["a"], c["b"], c["index"], c["scale"], c["parts"], c["dy"])
        first = None
        for _ in range(4):
            x = c["x"].detach().requires_grad_()
            _call(dict(c, x=x)).backward(c["dy"])
            first = x.grad if first is None else first
            assert torch.equal(first, x.grad), name
        _close(first, want, mag, 64, name)


@pytest.mark.parametrize("T", [40, 600])
def test_threads_in_turn_with_ranks_that_take_unlike_shared_memory(T):
    import threading

    # the limit of a kernel's shared memory belongs to the process: a thread with a low rank must not lower it under one with a high rank
    cs = [make(T, 64, (64,) * 3, r, 3, BF if T > 256 else F32, "cuda", "runs", seed=r) for r in (64, 16, 64, 8)]
    turn, errors, outs = threading.Barrier(4), [], [[] for _ in cs]

    def work(i):
        for at in range(12):
            turn.wait()
            if at % 4 == i or at >= 8:
                try:
                    outs[i].append(_call(cs[i]))
                except RuntimeError as e:  # shown by the assertion below
                    errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for c, o in zip(cs, outs):
        want, mag = exact(c)
        for got in o:
            check(got, want, mag, 64)
