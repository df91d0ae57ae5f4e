"""A weight that is not finite quantises to a row whose logits are not finite, and
to nothing else."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ctx():
    from tests.gpu_util import ctx
    return ctx()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
def test_one_value(value, group, mins, dtype):
    from zllm_amd.head import Q4Head, q4_quantize
    gen = torch.Generator("cuda").manual_seed(2)
    W = torch.randn((70, 256), device="cuda", generator=gen).to(dtype)
    good = q4_quantize(_ctx(), W, group, mins)
    W[3, 0], W[40, 255], W[41, 131] = float(value), float(value), float(value)
    bad = [3, 40, 41]
    rest = [v for v in range(70) if v not in bad]
    codes, scales, lows = q4_quantize(_ctx(), W, group, mins)
    for a, b in ((codes, good[0]), (scales, good[1])) + (((lows, good[2]),) if mins else ()):
        assert torch.equal(a[rest], b[rest])
    assert (~scales.isfinite()).sum().item() == 3
    assert not scales[3, 0].isfinite() and not scales[40, 255 // group].isfinite() and not scales[41, 131 // group].isfinite()
    if value == "nan":
        assert scales[3, 0].isnan() and scales[40, 255 // group].isnan() and scales[41, 131 // group].isnan()
    head, whole = Q4Head(_ctx(), codes, scales, lows), Q4Head(_ctx(), *good)
    for B in (1, 9, 20, 70):
        for t in (torch.float32, torch.bfloat16):
            h = torch.randn((B, 256), device="cuda", generator=gen).to(t)
            z = head.logits(h)
            assert not z[:, bad].isfinite().any() and torch.equal(z[:, rest], whole.logits(h)[:, rest])


def test_all_of_a_group():
    from zllm_amd.head import q4_quantize
    W = torch.full((4, 64), float("nan"), device="cuda")
    for mins in (False, True):
        assert bool(q4_quantize(_ctx(), W, 32, mins)[1].isnan().all())
