"""f32 states of a 4-bit head are multiplied as two f16, to 2^-22 of each: by w, not
by the larger number that stands for w among the operands.

One value x = X 2^e a group, and codes that stand for w = 0: the operands' product
x^ (16 + q) and the sum that the products start from, -x^ (16 + q), are of the same x^.
X = A 2^13 + r, A of 11 bits, r odd and 2^11 < r < 2^12: the first f16 has A, the second
has 11 of r's 12 bits, by a tie a multiple of 4, so x^ is not x and has 22 bits, and 24
x^ = 3 x^ 2^3 has 24. The start (-24 x^, or -16 x^) and the partial sums (less the
first part's product they are minus the second's) are f32 numbers: the result is 0."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("B", [1, 16, 17, 40, 65])
def test_weights_of_zero(B, group, mins):
    from tests.gpu_util import ctx
    from zllm_amd.head import Q4Head
    V, n = 50, 4
    gen = torch.Generator("cuda").manual_seed(B + group)
    h = torch.zeros((B, n * group), device="cuda")
    X = torch.randint(1024, 2048, (B, n), device="cuda", generator=gen) * 8192
    X += torch.randint(1024, 2048, (B, n), device="cuda", generator=gen) * 2 + 1
    x = X.float() * torch.tensor([1.0, -1.0, 0.5, 64.0], device="cuda") * 2.0 ** -24
    x[0] = 1.0 + 2.0 ** -12 + 2.0 ** -23
    h[:, torch.arange(n, device="cuda") * group + torch.tensor([0, 5, 17, 31], device="cuda")] = x
    codes = torch.full((V, n * group // 2), 0x00 if mins else 0x88, dtype=torch.uint8, device="cuda")
    scales = torch.rand((V, n), device="cuda", generator=gen).add_(0.5).half()
    lows = torch.zeros_like(scales) if mins else None
    got = Q4Head(ctx(), codes, scales, lows).logits(h)
    assert bool((got == 0.0).all()), f"{int((got != 0).sum())} of {got.numel()}, up to {float(got.abs().max()):.3g}"
