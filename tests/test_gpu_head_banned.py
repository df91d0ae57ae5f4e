"""f32 heads some of whose ids are banned by a number in a column that all states
share (states of 1 there), down to the type's lowest: what 64 bits give.

A logit is within ez = (D + 20) 2^-24 A_v of itself, A_v = sum_d |h_d W_vd|; the banned
ids' errors are of numbers without mass. The rest as in tests/test_gpu_head.py."""
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
    w = Wd.abs().amax(1)
    ez = (D + 20) * 2.0 ** -24 * (hd.abs() @ Wd.abs().T)
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
    d, e = d * (w <= 1e30), e * (w <= 1e30)
    th = e @ W0.abs() + (V + 12) * 2.0 ** -24 * (d.abs() @ W0.abs()) + 2.0 ** -24 * (d @ W0).abs() + 2.0 ** -126
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
@pytest.mark.parametrize("N,V,D", [(1, 700, 96), (20, 700, 97), (192, 700, 96)])
def test_banned_ids(N, V, D, low):
    h, W, labels, g = inputs(N, V, D, N + D)
    W[5::9, 0] = low
    W[V - 1, 0] = low
    labels[(labels % 9 == 5) | (labels == V - 1)] = 0
    check(h, W, labels, g, f"banned by {low}")


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
