"""f32 heads some of whose ids are banned by a number in a column that all states
share (states of 1 there), down to the type's lowest, or whose rows are of very unlike
size: few rows and many give what 64 bits give.

Where the weight is multiplied as two f16, each of its rows is scaled by a power of
two of its own, so a number leaves at most 2^-22 of it or 2^-39 of its row's largest,
w_v. States likewise (t, of their row). A logit is within ez = (D + 20) 2^-24 A_v + 2^-39
sum_d (|h_d| w_v + |W_vd| t) of itself, A_v = sum_d |h_d W_vd|; the banned ids' errors
are of numbers without mass. The states' gradient takes d_v 2^-s_v, s_v the weight row's
power, as two f16 of numbers scaled by their largest or twice that, T 2^-13 at most with
T = max_v |d_v| w_v: they leave 2^-39 of that, which W_vd 2^s_v, at most 2^15 |W_vd| / w_v,
makes 2^-37 T |W_vd| / w_v; the weight's own remainders give 2^-39 |d_v| w_v. The rest as in
tests/test_gpu_head.py."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def near(got, want, tol, what):
    e = (got.double() - want).abs()
    assert bool((e <= tol).all()), f"{what}: {int((~(e <= tol)).sum())} of {e.numel()}, worst {float((e / tol).nan_to_num(1e9).max()):.3g}"


def check(h, W, labels, g, what):
    from tests.gpu_util import ctx
    from zllm_amd.head import head_loss, head_loss_grad
    (N, D), V = h.shape, W.shape[0]
    print(f"[case] {what} N={N} V={V} D={D}", flush=True)
    hd, Wd, gd = h.double(), W.double(), g.double()
    at = torch.arange(N, device="cuda")
    z = hd @ Wd.T
    w, t = Wd.abs().amax(1), hd.abs().amax(1)
    ez = (D + 20) * 2.0 ** -24 * (hd.abs() @ Wd.abs().T) + 2.0 ** -39 * (hd.abs().sum(1)[:, None] * w + t[:, None] * Wd.abs().sum(1))
    L = torch.logsumexp(z, 1)
    p = (z - L[:, None]).exp()
    # (what ids without mass are off by is nothing: e^-80 of a unit)
    ez = torch.where(z < L[:, None] - 100 - ez, 0.0, ez)
    ex = ez.amax(1)
    el = ex + 2.0 ** -17
    loss = L - z[at, labels]
    l1, lse = head_loss(ctx(), h, W, labels)
    l2, dh, dw = head_loss_grad(ctx(), h, W, labels, g)
    for x in (l1, l2):
        near(x, loss, el + ex + 2.0 ** -23 * loss, "loss")
    near(lse, L, el + 2.0 ** -23 * L.abs(), "lse")
    d = p * gd[:, None]
    e = d.abs() * (2 * el + ex + 2.0 ** -21)[:, None] + 2.0 ** -126
    d[at, labels] -= gd
    e += d.abs() * 2.0 ** -24
    W0 = torch.where(w[:, None] > 1e30, 0.0, Wd)           # (no mass, and so none of the gradient: their entries are 0 exactly)
    live = (w <= 1e30).double()
    d, e = d * live, e * live
    w0 = w * live
    T = (d.abs() * w0).amax(1, keepdim=True)
    th = e @ W0.abs() + (V + 12) * 2.0 ** -24 * (d.abs() @ W0.abs()) + 2.0 ** -24 * (d @ W0).abs() + 2.0 ** -126
    th += 2.0 ** -37 * T * (W0.abs() / w0.clamp_min(1e-300)[:, None]).sum(0) + 2.0 ** -39 * (d.abs() @ w0)[:, None]
    near(dh, d @ W0, th, "dhidden")
    tw = e.T @ hd.abs() + (N + 12) * 2.0 ** -24 * (d.abs().T @ hd.abs()) + 2.0 ** -24 * (d.T @ hd).abs() + 2.0 ** -126
    near(dw, d.T @ hd, tw, "dweight")


def inputs(N, V, D, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    W = torch.randn((V, D), device="cuda", generator=gen) * D ** -0.5
    h = torch.randn((N, D), device="cuda", generator=gen)
    h[:, 0] = 1.0
    W[:, 0] *= 0.1
    labels = torch.randint(0, V, (N,), device="cuda", generator=gen)
    return h, W, labels, torch.randn(N, device="cuda", generator=gen) / N


@pytest.mark.parametrize("low", [-1e4, -1e9, -1e30, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("N,V,D", [(1, 700, 96), (20, 700, 97), (192, 700, 96), (193, 700, 96), (300, 1500, 257), (520, 4099, 64)])
def test_banned_ids(N, V, D, low):
    h, W, labels, g = inputs(N, V, D, N + D)
    W[5::9, 0] = low
    W[V - 1, 0] = low
    labels[(labels % 9 == 5) | (labels == V - 1)] = 0
    check(h, W, labels, g, f"banned by {low}")


@pytest.mark.parametrize("N", [100, 300])
@pytest.mark.parametrize("spread", [20, 60, 120])
def test_rows_of_unlike_size(N, spread):
    """From row to row any power of two, labels among them."""
    h, W, labels, g = inputs(N, 900, 128, N + spread)
    rng = np.random.default_rng(spread)
    W *= torch.from_numpy(2.0 ** rng.integers(-spread, 1, (900, 1))).float().cuda()
    check(h, W, labels, g, f"rows over 2^{spread}")


@pytest.mark.parametrize("N", [100, 300])
def test_rows_of_zeros(N):
    """Ids that a vocabulary is filled up with: the others keep their digits."""
    h, W, labels, g = inputs(N, 1024, 96, N)
    W[1000:] = 0.0
    W[::7] = 0.0
    labels[:3] = 7
    check(h, W, labels, g, "rows of zeros")


def test_a_weight_far_apart():
    """Few rows whose weight is copied all the same: it lies further apart than the products reach."""
    h, W, labels, g = inputs(100, 6, 64, 4)
    W[3, 0] = torch.finfo(torch.float32).min
    labels[labels == 3] = 2
    buf = torch.zeros((6, 5_000_000), device="cuda")
    buf[:, 100:164] = W
    check(h, buf[:, 100:164], labels, g, "far")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N", [20, 100, 300])
def test_banned_ids_of_16_bits(N, dtype):
    """They come out as if they were not there."""
    from tests.gpu_util import ctx
    from zllm_amd.head import head_loss_grad
    h, W, labels, g = inputs(N, 700, 96, N)
    h, W = h.to(dtype), W.to(dtype)
    W[5::9, 0] = torch.finfo(dtype).min
    ids = torch.arange(700, device="cuda")
    kept = ids[ids % 9 != 5]
    labels[labels % 9 == 5] = 0
    loss, dh, dw = head_loss_grad(ctx(), h, W, labels, g)
    want = head_loss_grad(ctx(), h, W[kept].contiguous(), torch.searchsorted(kept, labels), g)
    # two calls of the same products in other tiles: f32 sums in another order, entries rounded by EPS and 2^-11
    eps = torch.finfo(dtype).eps
    assert float((loss - want[0]).abs().max()) <= 2.0 ** -16
    d = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())
    assert d(dh, want[1]) <= 2 * eps and d(dw[kept], want[2]) <= 2 * eps
    assert not dw[5::9].any()
