"""Adapter kernels against the formulas in 64 bits."""

import pytest
import torch
from adapter_cases import bound, check, exact, make

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _call(c, **kw):
    from easydel_b200.ops import adapters

    return adapters.lora_add(c["y"], c["x"], c["a"], c["b"], c["index"], c["scale"], parts=c["parts"], **kw)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [1, 7, 8, 9, 255, 256, 257, 700])
@pytest.mark.parametrize("K,parts,r,n", [
    (64, (64,), 16, 4), (1024, (256, 64, 64), 8, 5), (40, (24,), 4, 3), (33, (7,), 1, 2), (129, (65, 3, 130), 5, 300), (512, (96, 32), 64, 9),
])
def test_values(dtype, T, K, parts, r, n):
    c = make(T, K, parts, r, n, dtype, "cuda", "mixed", seed=T)
    want, mag = exact(c)
    got = _call(c)
    check(got, want, mag, K)
    assert torch.equal(got, _call(c))                 # sums in a fixed order
    y = c["y"].clone()
    c["y"] = y
    assert _call(c, out=y) is y and torch.equal(y, got)      # in place


@pytest.mark.parametrize("index", ["none", "runs", "bare", "2"])
@pytest.mark.parametrize("T", [5, 300])
def test_index_patterns(index, T):
    c = make(T, 256, (128, 64), 16, 1 if index == "none" else 3, BF, "cuda", index)
    want, mag = exact(c)
    check(_call(c), want, mag, 256)


@pytest.mark.parametrize("T", [3, 400])
@pytest.mark.parametrize("r,parts", [(128, (64,)), (256, (64, 32)), (512, (40,)), (100, (16,) * 5), (64, (8,) * 8)])
def test_high_ranks(T, r, parts):
    for dtype in (BF, F32):
        c = make(T, 96, parts, r, 2, dtype, "cuda", "mixed")
        val, mag = exact(c, grads=True)
        check(_call(c), val["out"], mag["out"], 96)
        _gradients(c, val, mag)


def test_float32_output_beside_bf16_rows():
    for T in (9, 300):
        c = make(T, 320, (64, 32), 16, 3, BF, "cuda")
        c["y"] = c["y"].float() * 1.0001
        want, mag = exact(c)
        got = _call(c)
        assert got.dtype == F32
        check(got, want, mag, 320)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [6, 290])
def test_strides_and_alignment(dtype, T):
    c = make(T, 64, (32, 16), 8, 3, dtype, "cuda")
    want, mag = exact(c)

    def pitch(t, left, right):      # the same rows inside wider ones
        wide = torch.full((*t.shape[:-1], left + t.shape[-1] + right), float("nan"), dtype=t.dtype, device="cuda")
        wide[..., left:left + t.shape[-1]] = t
        return wide[..., left:left + t.shape[-1]]

    for left, right in ((8, 8), (3, 2)):
        d = dict(c, x=pitch(c["x"], left, right), y=pitch(c["y"], left, right), a=pitch(c["a"], left, right), b=pitch(c["b"], left, right))
        check(_call(d), want, mag, 64)
        box = pitch(torch.zeros_like(c["y"]), left, right)
        whole = box._base if box._base is not None else box
        assert _call(d, out=box) is box
        check(box, want, mag, 64)
        assert torch.isnan(whole[:, :left]).all() and torch.isnan(whole[:, left + 48:]).all()
    turned = dict(c, x=c["x"].t().contiguous().t(), a=c["a"].transpose(1, 2).contiguous().transpose(1, 2))
    check(_call(turned), want, mag, 64)


def test_bad_index_sets_the_status_word_and_counts_as_none():
    from easydel_b200.ops import _lib

    c = make(20, 64, (32,), 8, 3, BF, "cuda")
    c["index"][7] = 3
    c["index"][9] = 2 ** 30
    got = _call(c)
    with pytest.raises(RuntimeError, match="index out of range"):
        _lib.check_status()
    c["index"][[7, 9]] = -1
    want, mag = exact(c)
    check(got, want, mag, 64)


@pytest.mark.parametrize("T", [30, 300])
def test_values_that_are_not_finite_stay_with_their_row_and_adapter(T):
    c = make(T, 64, (32,), 12, 4, BF, "cuda")
    c["index"][:] = torch.arange(T, dtype=torch.int32, device="cuda") % 3 - 1
    clean = _call(c)
    c["x"][4, 5], c["x"][6, 5] = float("nan"), float("inf")       # rows of adapters 0 and -1
    c["a"][3] = float("nan")                                         # an adapter that nobody uses
    got = _call(c)
    rows = torch.ones(T, dtype=torch.bool)
    rows[4] = False
    assert torch.equal(got[rows], clean[rows]) and torch.isnan(got[4]).all()
    c["x"][7, 5] = float("inf")                                     # adapter 0 again
    assert not torch.isfinite(_call(c)[7]).any()


def _gradients(c, val, mag, want_f32=False):
    from easydel_b200.ops import adapters

    leaf = {k: c[k].detach().requires_grad_() for k in ("y", "x", "a", "b")}
    out = adapters.lora_add(leaf["y"], leaf["x"], leaf["a"], leaf["b"], c["index"], c["scale"], parts=c["parts"])
    out.backward(c["dy"])
    T, N = c["x"].shape[0], sum(c["parts"])
    check(out.detach(), val["out"], mag["out"], c["x"].shape[1], "out")
    check(leaf["x"].grad, val["dx"], mag["dx"], N, "dx")
    check(leaf["a"].grad, val["da"], mag["da"], T + N, "da")
    check(leaf["b"].grad, val["db"], mag["db"], T + c["x"].shape[1], "db")
    assert torch.equal(leaf["y"].grad, c["dy"])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [1, 8, 31, 256, 1100])
@pytest.mark.parametrize("K,parts,r,n,index", [
    (64, (64,), 16, 1, "none"), (320, (256, 64, 64), 8, 3, "runs"), (40, (24,), 4, 3, "mixed"), (33, (7, 5), 3, 2, "mixed"), (264, (520,), 64, 2, "mixed"),
])
def test_gradients(dtype, T, K, parts, r, n, index):
    c = make(T, K, parts, r, n, dtype, "cuda", index, seed=T)
    _gradients(c, *exact(c, grads=True))


def test_gradients_against_differences():
    from easydel_b200.ops import adapters

    c = make(40, 48, (32, 16), 8, 2, F32, "cuda")
    leaf = {k: c[k].detach().requires_grad_() for k in ("x", "a", "b")}
    adapters.lora_add(c["y"], leaf["x"], leaf["a"], leaf["b"], c["index"], c["scale"], parts=c["parts"]).backward(c["dy"])
    g = torch.Generator(device="cuda").manual_seed(1)
    for k, t in leaf.items():
        d = torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64)

        def f(h):
            m = {**{j: c[j].double() for j in ("y", "x", "a", "b")}}
            m[k] = m[k] + h * d
            o = adapters.lora_add_reference(m["y"], m["x"], m["a"], m["b"], c["index"], c["scale"], parts=c["parts"])
            return (o * c["dy"].double()).sum()

        slope = (f(1e-3) - f(-1e-3)) / 2e-3          # the outputs are linear in each: no error but rounding
        along = (t.grad.double() * d).sum()
        # every element of the gradient is within 2^-18 of its magnitudes (see the bound): along d their errors add up to at most that
        size = (t.grad.double().abs() * d.abs()).sum()
        assert abs(slope - along) <= 2.0 ** -16 * size


def test_rows_without_an_adapter_pass_no_gradient_and_unused_adapters_get_zeros():
    from easydel_b200.ops import adapters

    c = make(50, 64, (32,), 8, 4, BF, "cuda", "1")
    c["index"][10:20] = -1
    leaf = {k: c[k].detach().requires_grad_() for k in ("x", "a", "b")}
    adapters.lora_add(c["y"], leaf["x"], leaf["a"], leaf["b"], c["index"], c["scale"]).backward(c["dy"])
    assert not leaf["x"].grad[10:20].any() and leaf["x"].grad[:10].any()
    for w in ("a", "b"):
        assert not leaf[w].grad[[0, 2, 3]].any() and leaf[w].grad[1].any()


@pytest.mark.parametrize("frozen", ["a", "b", "x"])
def test_frozen_inputs(frozen):
    from easydel_b200.ops import adapters

    c = make(40, 64, (32,), 8, 2, BF, "cuda")
    val, mag = exact(c, grads=True)
    leaf = {k: c[k].detach().requires_grad_(k != frozen) for k in ("x", "a", "b")}
    adapters.lora_add(c["y"], leaf["x"], leaf["a"], leaf["b"], c["index"], c["scale"]).backward(c["dy"])
    for k, name, length in (("x", "dx", 32), ("a", "da", 72), ("b", "db", 104)):
        if k == frozen:
            assert leaf[k].grad is None
        else:
            check(leaf[k].grad, val[name], mag[name], length, name)


@pytest.mark.parametrize("T", [40, 600])
def test_gradients_are_added_to_main_grad(T):
    from easydel_b200.ops import adapters

    c = make(T, 64, (32,), 8, 2, BF, "cuda")
    val, mag = exact(c, grads=True)
    a, b = (c[k].detach().requires_grad_() for k in ("a", "b"))
    a.main_grad, b.main_grad = torch.full(a.shape, 2.0, device="cuda"), torch.zeros(b.shape, device="cuda")
    for _ in range(2):
        adapters.lora_add(c["y"], c["x"], a, b, c["index"], c["scale"]).backward(c["dy"])
    assert a.grad is None and b.grad is None and a.grad_added_to_main_grad and b.grad_added_to_main_grad
    # two passes onto 2: each sum is rounded to 32 bits
    for got, name, base in ((a.main_grad, "da", 2.0), (b.main_grad, "db", 0.0)):
        want = base + 2 * val[name]
        off = (got.double().cpu() - want).abs()
        inner = 2.0 ** -15 * 2 * mag[name]         # the factor from the forward or backward product has fp32 sums, the second product 24 bits
        assert (off <= 2.0 ** -22 * (want.abs() + base) + inner).all()


def test_captured_and_replayed_with_other_indexes():
    from easydel_b200.ops import adapters

    c = make(48, 256, (128, 64), 16, 6, BF, "cuda")
    out = torch.empty_like(c["y"])
    call = lambda: adapters.lora_add(c["y"], c["x"], c["a"], c["b"], c["index"], c["scale"], parts=c["parts"], out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for fill in (5, -1, None):
        if fill is None:
            c["index"].copy_(torch.arange(48, device="cuda") % 6)
        else:
            c["index"].fill_(fill)
        graph.replay()
        want, mag = exact(c)
        check(out, want, mag, 256)


def test_two_streams_at_once():
    cs = [make(300, 512, (256,), 16, 3, BF, "cuda", seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for c, s, o in zip(cs, streams, outs):
            with torch.cuda.stream(s):
                o.append(_call(c))
    torch.cuda.synchronize()
    for c, o in zip(cs, outs):
        want, mag = exact(c)
        for t in o:
            check(t, want, mag, 512)


def test_no_rows():
    from easydel_b200.ops import adapters

    c = make(0, 64, (32,), 8, 2, BF, "cuda")
    leaf = {k: c[k].detach().requires_grad_() for k in ("x", "a", "b")}
    out = adapters.lora_add(c["y"], leaf["x"], leaf["a"], leaf["b"], c["index"], c["scale"])
    out.backward(c["dy"])
    assert out.shape == (0, 32) and not leaf["a"].grad.any() and not leaf["b"].grad.any()


def test_refuses_gradients_of_float32_outputs_beside_bf16_rows():
    c = make(4, 64, (32,), 8, 2, BF, "cuda")
    c["y"] = c["y"].float()
    c["x"].requires_grad_()
    with pytest.raises(NotImplementedError):
        _call(c)


@pytest.mark.parametrize("T", [40, 600])
def test_broadcast_inputs_and_gradients(T):
    from easydel_b200.ops import adapters

    # one row for all, one first matrix for all adapters, and a gradient that is one row repeated
    c = make(T, 64, (32, 16), 8, 3, BF, "cuda")
    c["x"], c["a"], c["dy"] = c["x"][:1].expand(T, 64), c["a"][:1].expand(3, -1, -1), c["dy"][:1].expand(T, -1)
    val, mag = exact(c, grads=True)
    check(_call(c), val["out"], mag["out"], 64)
    x, a, b = (c[k].detach().requires_grad_() for k in ("x", "a", "b"))
    shared = a[:1].detach().clone().requires_grad_()
    out = adapters.lora_add(c["y"], x, shared.expand(3, -1, -1), b, c["index"], c["scale"], parts=c["parts"])
    (out * c["dy"][0]).sum(0).backward(torch.ones(48, device="cuda", dtype=BF))
    check(x.grad, val["dx"], mag["dx"], 48, "dx")
    check(b.grad, val["db"], mag["db"], T + 64, "db")
    # the adapters' gradients are rounded, then their sum is
    want, size = val["da"].sum(0, keepdim=True), mag["da"].sum(0, keepdim=True)
    assert ((shared.grad.double().cpu() - want).abs() <= bound(BF, want, size, T + 48) + 2.0 ** -8 * size).all()
    out = adapters.lora_add(c["y"], x, a.detach(), b, c["index"], c["scale"], parts=c["parts"])
    x.grad = None
    out.backward(c["dy"])      # strides (0, 1)
    check(x.grad, val["dx"], mag["dx"], 48, "dx")


def test_many_blocks_of_many_adapters_repeat():
    # more blocks than a cluster takes turns for, all of them single tokens of many adapters
    c = make(256 * 90 + 17, 64, (64,), 16, 40, BF, "cuda", "mixed")
    want, mag = exact(c)
    got = _call(c)
    check(got, want, mag, 64)
    for _ in range(20):
        assert torch.equal(got, _call(c))


@pytest.mark.parametrize("n", [4, 9, 70])
def test_gradients_of_blocks_of_many_adapters(n):
    c = make(1300, 128, (64, 32), 16, n, BF, "cuda", "mixed")
    c["index"][256:700] = 1      # among them blocks of one
    _gradients(c, *exact(c, grads=True))


@pytest.mark.parametrize("r", [8, 24])
def test_training_step_captured_and_replayed(r):
    from easydel_b200.ops import adapters

    c = make(600, 128, (96, 32), r, 3, BF, "cuda", "runs")
    grad = {k: torch.zeros(c[k].shape, device="cuda", dtype=BF) for k in ("x", "a", "b")}

    def step():
        leaf = {k: c[k].detach().requires_grad_() for k in ("x", "a", "b")}
        out = adapters.lora_add(c["y"], leaf["x"], leaf["a"], leaf["b"], c["index"], c["scale"], parts=c["parts"])
        for k, g in zip(leaf, torch.autograd.grad(out, list(leaf.values()), c["dy"])):
            grad[k].copy_(g)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for fill in (None, 2, -1):
        if fill is not None:
            c["index"].fill_(fill)
        c["dy"].mul_(-1)
        graph.replay()
        val, mag = exact(c, grads=True)
        for k, length in (("x", 128), ("a", 728), ("b", 728)):
            check(grad[k], val["d" + k], mag["d" + k], length, "d" + k)


def test_refuses_gradients_of_too_many_adapters():
    c = make(4, 8, (8,), 1, 65536, BF, "cuda", "3")
    _call(c)
    c["x"].requires_grad_()
    with pytest.raises(ValueError, match="65535"):
        _call(c)


@pytest.mark.parametrize("T", [512, 513, 900])
@pytest.mark.parametrize("index", ["none", "runs", "bare", "2"])
def test_index_patterns_of_many_rows(index, T):
    test_index_patterns(index, T)


@pytest.mark.parametrize("r,parts", [(128, (64,)), (256, (64, 32)), (512, (40,)), (100, (16,) * 5), (64, (8,) * 8), (12, (24, 16))])
def test_high_and_odd_ranks_of_many_rows(r, parts):
    test_high_ranks(600, r, parts)


def test_float32_output_beside_many_bf16_rows():
    for T, r, parts in ((600, 16, (64, 32)), (900, 72, (96,)), (900, 4, (40,))):
        c = make(T, 320, parts, r, 3, BF, "cuda")
        c["y"] = c["y"].float() * 1.0001
        want, mag = exact(c)
        check(_call(c), want, mag, 320)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_and_alignment_of_many_rows(dtype):
    test_strides_and_alignment(dtype, 700)


def test_values_that_are_not_finite_stay_with_their_row_and_adapter_among_many():
    test_values_that_are_not_finite_stay_with_their_row_and_adapter(700)


@pytest.mark.parametrize("T", [256, 257, 512, 513])
@pytest.mark.parametrize("index", ["none", "runs"])
def test_wide_outputs_on_both_sides_of_the_forms(T, index):
    c = make(T, 64, (8200,), 16, 1 if index == "none" else 3, BF, "cuda", index)
    want, mag = exact(c)
    check(_call(c), want, mag, 64)
    c = make(T, 8200, (64,), 16, 1 if index == "none" else 3, BF, "cuda", index)      # the backward pass is the wide one
    _gradients(c, *exact(c, grads=True))


def test_frozen_rows_of_a_wide_input():
    from easydel_b200.ops import adapters

    for K, N in ((8200, 64), (64, 8200)):
        c = make(300, K, (N,), 16, 1, BF, "cuda", "none")
        val, mag = exact(c, grads=True)
        a, b = (c[k].detach().requires_grad_() for k in ("a", "b"))
        adapters.lora_add(c["y"], c["x"], a, b, None, c["scale"]).backward(c["dy"])
        check(a.grad, val["da"], mag["da"], 300 + N, "da")
        check(b.grad, val["db"], mag["db"], 300 + K, "db")


def test_many_rows_captured_and_replayed_with_other_indexes():
    from easydel_b200.ops import adapters

    c = make(1500, 128, (96, 32), 16, 12, BF, "cuda", "mixed")
    out = torch.empty_like(c["y"])
    call = lambda: adapters.lora_add(c["y"], c["x"], c["a"], c["b"], c["index"], c["scale"], parts=c["parts"], out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    rows = torch.arange(1500, device="cuda")
    for index in (rows * 0 + 11, rows * 12 // 1500, rows % 12 - 1, rows * 0 - 1, torch.where(rows < 256, rows % 12, 3)):
        c["index"].copy_(index)
        graph.replay()
        want, mag = exact(c)
        check(out, want, mag, 128)


def test_many_rows_on_two_streams_and_in_two_threads():
    import threading

    from easydel_b200.ops import adapters

    cs = [make(900 + 100 * i, 256, (128,), 16, 6, BF, "cuda", ("mixed", "runs")[i], seed=i) for i in range(2)]
    torch.cuda.synchronize()
    outs, grads, errors = [[], []], [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    leaf = {k: cs[i][k].detach().requires_grad_() for k in ("x", "a", "b")}
                    o = adapters.lora_add(cs[i]["y"], leaf["x"], leaf["a"], leaf["b"], cs[i]["index"], cs[i]["scale"])
                    grads[i].append(torch.autograd.grad(o, list(leaf.values()), cs[i]["dy"]))
                    outs[i].append(o.detach())
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # shown by the assertion below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for c, o, g in zip(cs, outs, grads):
        val, mag = exact(c, grads=True)
        for t, (dx, da, db) in zip(o, g):
            assert torch.equal(t, o[0]) and torch.equal(dx, g[0][0]) and torch.equal(da, g[0][1]) and torch.equal(db, g[0][2])
        check(o[0], val["out"], mag["out"], 256)
        check(g[0][0], val["dx"], mag["dx"], 128)
        check(g[0][1], val["da"], mag["da"], 1100)
        check(g[0][2], val["db"], mag["db"], 1300)


@pytest.mark.parametrize("K,N", [(14336, 64), (64, 14336)])
def test_offsets_beyond_32_bits(K, N):
    from easydel_b200.ops import adapters

    T, last = 160000, 300      # 2.3e9 elements; the last rows have an adapter of their own
    g = torch.Generator(device="cuda").manual_seed(0)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=BF)  # noqa: E731
    x, y, dy = rn(T, K), rn(T, N), rn(T, N)
    a, b = rn(2, 8, K) * K ** -0.5, rn(2, N, 8) * 8 ** -0.5
    index = torch.zeros(T, dtype=torch.int32, device="cuda")
    index[-last:] = 1
    leaf = [t.requires_grad_() for t in (x, a, b)]
    out = adapters.lora_add(y, *leaf, index, 0.5)
    dx, da, db = torch.autograd.grad(out, leaf, dy)
    c = dict(x=x.detach()[-last:], y=y[-last:], a=a.detach()[1:], b=b.detach()[1:], index=None, scale=0.5, parts=(N,), dy=dy[-last:])
    val, mag = exact(c, grads=True)
    check(out.detach()[-last:], val["out"], mag["out"], K, "out")
    check(dx[-last:], val["dx"], mag["dx"], N, "dx")
    check(da[1:], val["da"], mag["da"], last + N, "da")
    check(db[1:], val["db"], mag["db"], last + K, "db")
    c = dict(c, x=x.detach()[:last], y=y[:last], a=a.detach()[:1], b=b.detach()[:1], dy=dy[:last])
    val, mag = exact(c, grads=True)
    check(out.detach()[:last], val["out"], mag["out"], K, "out")
    check(dx[:last], val["dx"], mag["dx"], N, "dx")
