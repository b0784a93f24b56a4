"""Logit rules kernel against the formulas in 64 bits."""

import pytest
import torch
from logit_rule_cases import check, exact, make

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 31), (2, 64), (5, 4095), (4, 4096), (3, 4104), (9, 10001), (2, 50257), (130, 512)])
@pytest.mark.parametrize("what", [dict(), dict(penalties=False, biases=0), dict(biases=0, masked=False), dict(penalties=False, masked=False, biases=400)])
def test_values(dtype, R, V, what):
    from easydel_b200.ops import serving

    c = make(R, V, dtype, "cuda", seed=R + V, **what)
    want, mag = exact(c)
    for out in (None, torch.empty(R, V, device="cuda"), torch.empty(R, V, device="cuda", dtype=BF)):
        check(serving.adjust_logits(c["logits"], out=out, **c["kw"]), want, mag)
    z = c["logits"].clone()
    assert serving.adjust_logits(z, out=z, **c["kw"]) is z
    check(z, want, mag)


def test_strides_and_alignment():
    from easydel_b200.ops import serving

    for left, pitch in ((8, 600), (3, 531)):
        c = make(6, 512, BF, "cuda")
        want, mag = exact(c)
        wide = torch.full((6, pitch), float("nan"), dtype=BF, device="cuda")
        wide[:, left:left + 512] = c["logits"]
        view = wide[:, left:left + 512]
        c["kw"]["counts"] = torch.nn.functional.pad(c["kw"]["counts"], (0, 5))
        c["kw"]["mask"] = (torch.nn.functional.pad(c["kw"]["mask"][0], (0, 3)), c["kw"]["mask"][1])
        check(serving.adjust_logits(view, **c["kw"]), want, mag)
        serving.adjust_logits(view, out=view, **c["kw"])
        check(view, want, mag)
        assert torch.isnan(wide[:, :left]).all() and torch.isnan(wide[:, left + 512:]).all()
        turned = c["logits"].t().contiguous().t()
        check(serving.adjust_logits(turned, **c["kw"]), want, mag)


def test_rows_that_forbid_everything_and_odd_values():
    from easydel_b200.ops import serving

    for V in (4104, 4111):
        z = torch.full((3, V), float("nan"), device="cuda")
        z[1], z[2] = float("inf"), torch.finfo(F32).min
        bits = torch.zeros(1, (V + 31) // 32, dtype=torch.int32, device="cuda")
        got = serving.adjust_logits(z, mask=(bits, torch.zeros(3, dtype=torch.int32, device="cuda")))
        assert (got == -float("inf")).all()
        assert serving.sample(got)[0].tolist() == [0, 0, 0]
        bits[0, 3] = -(1 << 31)          # one token: 127
        z[:, 127] = 1.0
        got = serving.adjust_logits(z, mask=(bits, torch.zeros(3, dtype=torch.int32, device="cuda")))
        assert serving.sample(got)[0].tolist() == [127] * 3
        ptr = torch.tensor([0, 1, 1, 1], dtype=torch.int32, device="cuda")
        got = serving.adjust_logits(z, bias=(ptr, torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), -float("inf"), device="cuda")))
        assert got[0, 0] == -float("inf") and torch.isnan(got[0, 1]) and got[1, 0] == float("inf") and got[2, 0] == torch.finfo(F32).min


def test_entries_out_of_range_count_as_absent_and_set_the_status_word():
    from easydel_b200.ops import _lib, serving

    for V in (512, 515):
        c = make(4, V, F32, "cuda")
        kw = c["kw"]

        def told():
            got = serving.adjust_logits(c["logits"], **kw)
            with pytest.raises(RuntimeError, match="index out of range"):
                _lib.check_status()
            return got

        kw["count_rows"][1] = 99
        got = told()
        kw["count_rows"][1] = -1
        assert torch.equal(got, serving.adjust_logits(c["logits"], **kw))
        kw["mask"][1][2] = 4
        got = told()
        kw["mask"][1][2] = -1
        assert torch.equal(got, serving.adjust_logits(c["logits"], **kw))
        ptr, ids, values = kw["bias"] = (torch.tensor([0, 2, 2, 2, 3], dtype=torch.int32, device="cuda"),
                                         torch.tensor([-1, V, 7], dtype=torch.int32, device="cuda"), torch.ones(3, device="cuda"))
        got = told()
        kw["bias"] = (torch.tensor([0, 0, 0, 0, 1], dtype=torch.int32, device="cuda"), ids[2:].clone(), values[2:].clone())
        assert torch.equal(got, serving.adjust_logits(c["logits"], **kw))
        kw["bias"][0][4] = 5              # behind the entries
        got = told()
        del kw["bias"]
        assert torch.equal(got, serving.adjust_logits(c["logits"], **kw))


def test_neutral_penalties_and_rows_without_rules_are_copied():
    from easydel_b200.ops import serving

    c = make(5, 1000, BF, "cuda", biases=0, masked=False)
    kw = c["kw"]
    kw["presence"].zero_(), kw["frequency"].zero_(), kw["repetition"].fill_(1.0)
    assert torch.equal(serving.adjust_logits(c["logits"], **kw), c["logits"].float())
    assert torch.equal(serving.adjust_logits(c["logits"]), c["logits"].float())


def test_agrees_with_the_sampler_s_penalties():
    from easydel_b200.ops import serving

    c = make(8, 2048, F32, "cuda", biases=0, masked=False)
    kw = dict(c["kw"])
    rows = kw.pop("count_rows").clamp(min=0)
    counts = kw.pop("counts").index_select(0, rows.long())
    z = serving.adjust_logits(c["logits"], counts=counts, **kw)
    assert torch.equal(serving.sample(z)[0], serving.sample(c["logits"], counts=counts, **kw)[0])


def test_captured_and_replayed_with_other_masks():
    from easydel_b200.ops import serving

    c = make(6, 1000, BF, "cuda")
    out = torch.empty(6, 1000, device="cuda")
    serving.adjust_logits(c["logits"], out=out, **c["kw"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serving.adjust_logits(c["logits"], out=out, **c["kw"])
    for m in (0, 1, 2, -1):
        c["kw"]["mask"][1].fill_(m)
        graph.replay()
        check(out, *exact(c))


def test_no_rows():
    from easydel_b200.ops import serving

    assert serving.adjust_logits(torch.zeros(0, 100, device="cuda")).shape == (0, 100)
