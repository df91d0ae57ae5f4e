"""Rows that are all but certain of their label: a small loss, the label's entry of
the gradient, and that the row's entries balance.

With R = sum over the other ids of exp(z_v - z_label), the loss is ln(1 + R), the
label's entry -g R / (1 + R) and the others' g exp(z_v - z_label) / (1 + R): all are
made of differences of logits of one kind, so an error of the logits is a relative
error of each. A logit is within ez = (D + 20) 2^-24 A of itself (A the row's
largest sum of |h_d W_vd|; 16-bit operands: D + 8), the exponentials and their sum
within 2^-17 more: r = exp(2 ez) (1 + 2^-17) - 1, relative, of R, of the loss (the
slope of ln(1 + R) over R is below ln(1 + R) / R) and of each entry. A 16-bit type's
exponentials are kept as f16 (2^-11, and 2^-40 of the largest other), its entries
rounded once (EPS, f16 also 2^-39 of the largest of all rows); f32 entries as two f16
(3 * 2^-22, and 2^-39 of the row's largest). Sums over ids or rows have as many f32
additions as terms, and the outputs are rounded once."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -24, "bf16": 2.0 ** -126}


def _ctx():
    from tests.gpu_util import ctx
    return ctx()


def rows(N, V, D, dtype, seed, lo=4.0, hi=60.0):
    """States along their label's row: logits of lo to hi there, of about 0 elsewhere.
    The weight's first column is 1, so that dhidden's first is the sum of the entries."""
    rng = np.random.default_rng(seed)
    W = rng.normal(0, D ** -0.5, (V, D)).astype(np.float32)
    W[:, 0] = 1.0
    labels = rng.integers(0, V, N)
    labels[0], labels[-1] = 0, V - 1
    t = np.linspace(lo, hi, N).astype(np.float32)
    rng.shuffle(t)
    h = t[:, None] * W[labels]
    h[:, 0] = 0.0
    put = lambda x: torch.from_numpy(x).to(TYPES[dtype]).cuda()
    return put(h), put(W), torch.from_numpy(labels).cuda(), torch.full((N,), 1.0, device="cuda")


def oracle(h, W, labels, g):
    hd, Wd = h.double(), W.double()
    at = torch.arange(len(h), device="cuda")
    z = hd @ Wd.T
    x = (z - z[at, labels][:, None]).exp()
    x[at, labels] = 0.0
    R = x.sum(1)
    d = g.double()[:, None] * x / (1 + R)[:, None]
    top = d.amax(1)
    d[at, labels] = -g.double() * R / (1 + R)
    ez = (h.shape[1] + (20 if h.dtype == torch.float32 else 8)) * 2.0 ** -24 * (hd.abs() @ Wd.abs().T).amax(1)
    return torch.log1p(R), d, torch.expm1(2 * ez + 2.0 ** -17), top


def near(got, want, tol, what):
    e = (got.double() - want).abs()
    assert bool((e <= tol).all()), f"{what}: {int((~(e <= tol)).sum())} of {e.numel()}, worst {float((e / tol).nan_to_num(1e9).max()):.3g}"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,V,D", [(40, 1900, 4096), (100, 1900, 2048), (300, 1900, 4096), (300, 1031, 1000)])
def test_small_losses_and_their_gradients(N, V, D, dtype):
    from zllm_amd.head import head_loss, head_loss_grad
    print(f"[case] confident N={N} V={V} D={D} {dtype}", flush=True)
    h, W, labels, g = rows(N, V, D, dtype, seed=N + D)
    loss, d, r, top = oracle(h, W, labels, g)
    l1, lse = head_loss(_ctx(), h, W, labels)
    l2, dh, dw = head_loss_grad(_ctx(), h, W, labels, g)
    tol = loss * (r + 2.0 ** -24) + 2.0 ** -126
    near(l1, loss, tol, "loss")
    near(l2, loss, tol, "loss of the step")
    assert bool((l1 >= 0).all()) and bool((l2 >= 0).all())
    e = d.abs() * (r[:, None] + (EPS[dtype] + 2.0 ** -11 if dtype != "f32" else 3 * 2.0 ** -22))
    e += 2.0 ** -39 * torch.maximum(top, d.abs().amax(1))[:, None]
    if dtype == "f16":
        e += 2.0 ** -39 * d.abs().amax()
    Wd, hd = W.double(), h.double()
    near(dh, d @ Wd, e @ Wd.abs() + (V + 12) * 2.0 ** -24 * (d.abs() @ Wd.abs()) + EPS[dtype] * (d @ Wd).abs() + TINY[dtype], "dhidden")
    near(dw, d.T @ hd, e.T @ hd.abs() + (N + 12) * 2.0 ** -24 * (d.abs().T @ hd.abs()) + EPS[dtype] * (d.T @ hd).abs() + TINY[dtype],
         "dweight")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N", [30, 300])
def test_the_entries_of_a_row_balance(N, dtype):
    """dhidden's first column is the sum of a row's entries: 0, whatever the logits'
    errors, up to the roundings of each entry (EPS and 2^-11, f32 3 * 2^-22; 2^-39 of the
    row's largest, f16 of all rows' and 2^-40 of the exponentials' besides), of the sums
    of exponentials (2^-17) and of the column's sum."""
    from zllm_amd.head import head_loss_grad
    h, W, labels, g = rows(N, 1900, 4096, dtype, seed=7, lo=8.0, hi=24.0)
    _, d, _, _ = oracle(h, W, labels, g)
    _, dh, _ = head_loss_grad(_ctx(), h, W, labels, g)
    per = EPS[dtype] + 2.0 ** -11 if dtype != "f32" else 3 * 2.0 ** -22
    tol = d.abs().sum(1) * (per + 2.0 ** -17 + (1900 + 12) * 2.0 ** -24)
    tol += 2.0 ** -38 * 1900 * (d.abs().amax() if dtype == "f16" else d.abs().amax(1)) + TINY[dtype]
    near(dh[:, 0], torch.zeros(N, device="cuda", dtype=torch.float64), tol, "sum")


def test_labels_outside_leave_the_normaliser():
    from zllm_amd.head import head_loss, head_loss_grad
    for dtype in TYPES:
        for N in (20, 300):
            h, W, labels, g = rows(N, 700, 256, dtype, seed=9, hi=20.0)
            want = torch.logsumexp(h.double() @ W.double().T, 1)
            labels[3], labels[5] = 700, -7
            loss, lse = head_loss(_ctx(), h, W, labels)
            assert loss.isnan().nonzero()[:, 0].tolist() == [3, 5]
            assert float((lse - want).abs().max()) < 2.0 ** -10     # (276 * 2^-24 of sums under 48, and 2^-17)
            loss, dh, _ = head_loss_grad(_ctx(), h, W, labels, g)
            assert loss.isnan().nonzero()[:, 0].tolist() == [3, 5] and dh.isnan().all(1).nonzero()[:, 0].tolist() == [3, 5]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_a_label_far_below_the_others(dtype):
    """An id without mass takes part in nothing; as a label its loss is its distance."""
    from zllm_amd.head import head_loss
    for N in (20, 300):
        h, W, labels, _ = rows(N, 700, 256, dtype, seed=10, hi=20.0)
        h[:, 1] = 1.0
        W[:, 1:3] = 0.0
        W[600] = 0.0
        W[600, 1] = -3.0e4
        labels[:] = 5
        labels[2] = 600
        loss, lse = head_loss(_ctx(), h, W, labels)
        z = h.double() @ W.double().T
        want = torch.logsumexp(z, 1)
        assert float((lse - want).abs().max()) < 2.0 ** -10
        # (one product, which is exact: the normaliser's error and a rounding of 2^-24)
        assert abs(float(loss[2]) - float(want[2] - z[2, 600])) <= 2.0 ** -10 + 3.0e4 * 2.0 ** -23
