"""f32 weights and states whose numbers span many powers of two, in rows and from row
to row, where they are multiplied as two f16 of numbers scaled by a power of two.

Scaled, the largest number lies in [2^14, 2^15): f16's smallest step, 2^-24, is at
most 2^-38 of it, so what a number leaves is at most 2^-22 of it or 2^-39 of the
largest: of its row of the weight (w_v) and of states (t). A logit is so within ez = (D +
20) 2^-24 A + 2^-39 sum_d (|h_d| w_v + |W_vd| t); the rest as tests/test_gpu_head.py has
it, with what tests/test_gpu_head_banned.py derives more for the states' gradient, T =
max_v |d_v| w_v: 2^-37 T sum_v |W_vd| / w_v + 2^-39 sum_v |d_v| w_v. (The weight's is of
three bf16, of any size.)"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def case(N, V, D, seed, spread):
    rng = np.random.default_rng(seed)
    W = rng.normal(0, 1 / np.sqrt(D), (V, D)) * 2.0 ** rng.uniform(-spread, 0, (V, D))
    h = rng.normal(0, 1, (N, D)) * 2.0 ** rng.uniform(-spread, 0, (N, D)) * 2.0 ** rng.uniform(-20, 3, (N, 1))
    # some ids far below the others, and columns whose size the states and the weight share out unlike
    W[::7] *= 2.0 ** -25
    W[:, 3] *= 2.0 ** 12
    h[:, 3] *= 2.0 ** -12
    labels = rng.integers(0, V, N)
    put = lambda x: torch.from_numpy(x.astype(np.float32)).cuda()
    return put(h), put(W), torch.from_numpy(labels).cuda(), put(rng.normal(0, 1, N))


@pytest.mark.parametrize("spread", [0, 8, 16, 30])
@pytest.mark.parametrize("N,V,D", [(200, 1500, 96), (300, 600, 515), (150, 1500, 96)])
def test_spread(N, V, D, spread):
    from tests.gpu_util import ctx
    from zllm_amd.head import head_loss, head_loss_grad
    print(f"[case] range N={N} V={V} D={D} spread={spread}", flush=True)
    h, W, labels, g = case(N, V, D, N + spread, spread)
    hd, Wd, gd = h.double(), W.double(), g.double()
    at = torch.arange(N, device="cuda")
    z = hd @ Wd.T
    A = (hd.abs() @ Wd.abs().T).amax(1)
    w, t = Wd.abs().amax(1), hd.abs().amax(1)
    ez = (D + 20) * 2.0 ** -24 * A + 2.0 ** -39 * (hd.abs().sum(1) * w.amax() + t * Wd.abs().sum(1).amax())
    el = ez + 2.0 ** -17
    L = torch.logsumexp(z, 1)
    loss = L - z[at, labels]
    l1, lse = head_loss(ctx(), h, W, labels)
    l2, dh, dw = head_loss_grad(ctx(), h, W, labels, g)
    for x in (l1, l2):
        assert bool(((x.double() - loss).abs() <= el + ez + 2.0 ** -23 * loss).all())
    assert bool(((lse.double() - L).abs() <= el + 2.0 ** -23 * L.abs()).all())
    p = (z - L[:, None]).exp() * gd[:, None]
    e = p.abs() * (2 * el + ez + 2.0 ** -21)[:, None]
    d = p.clone()
    d[at, labels] -= gd
    e += d.abs() * 2.0 ** -24
    th = e @ Wd.abs() + (V + 12) * 2.0 ** -24 * (d.abs() @ Wd.abs()) + 2.0 ** -24 * (d @ Wd).abs() + 2.0 ** -126
    T = (d.abs() * w).amax(1, keepdim=True)
    th += 2.0 ** -37 * T * (Wd.abs() / w[:, None]).sum(0) + 2.0 ** -39 * (d.abs() @ w)[:, None]
    tw = e.T @ hd.abs() + (N + 12) * 2.0 ** -24 * (d.abs().T @ hd.abs()) + 2.0 ** -24 * (d.T @ hd).abs() + 2.0 ** -126
    for got, want, tol, what in ((dh, d @ Wd, th, "dhidden"), (dw, d.T @ hd, tw, "dweight")):
        x = (got.double() - want).abs()
        assert bool((x <= tol).all()), f"{what}: {int((x > tol).sum())} of {x.numel()}, worst {float((x / tol).max()):.3g}"
