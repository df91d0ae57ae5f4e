"""Students that give next to nothing to the ids outside the teacher's list: the
tail's term against the formulas in 64 bits, with the outside ids' mass as a
log-sum-exp of their own. Tolerances as in test_gpu_distill.py: the outside
sum's logarithm is one more of the three."""
import math

import numpy as np
import pytest
import torch

import tests.test_gpu_distill as near
from tests.test_gpu_distill import TINY, TYPES, _ctx, check, ltol, rows_at

pytestmark = pytest.mark.gpu


def ref_far(x, ids, logp, labels, cfg, w):
    """Loss, gradient and the parts that its rounding goes by."""
    N, V = x.shape
    loss, grad, size = np.zeros(N), np.zeros((N, V)), np.zeros((N, V))
    T = cfg.temperature
    for r in range(N):
        if labels is not None and labels[r] == cfg.ignore_index:
            continue
        m = x[r].max()
        z = (x[r] - m) / T
        S = np.exp(z).sum()
        q, lq = np.exp(z) / S, z - np.log(S)
        ok = (ids[r] >= 0) & (ids[r] < V) & ~np.isneginf(logp[r])
        k, p = ids[r][ok], np.exp(logp[r][ok].astype(np.float64))
        pt = max(0.0, 1.0 - p.sum())
        out = np.ones(V, bool)
        out[k] = False
        mo = x[r][out].max()
        e = np.exp((x[r][out] - mo) / T)
        lqt = (mo - m) / T + np.log(e.sum()) - np.log(S)
        kl = (p * (np.log(p) - lq[k])).sum() + (pt * (np.log(pt) - lqt) if pt > 0 else 0.0)
        g = np.zeros(V)
        np.add.at(g, k, -p)
        g[out] = -pt * e / e.sum()
        s = np.abs(g)
        P = p.sum() + pt
        g = cfg.kl_weight / T * (g + P * q)
        s = abs(cfg.kl_weight) / T * (s + P * q)
        loss[r] = cfg.kl_weight * kl
        if labels is not None:
            e1 = np.exp(x[r] - m)
            one = np.zeros(V)
            one[labels[r]] = 1.0
            loss[r] += cfg.ce_weight * (np.log(e1.sum()) - (x[r][labels[r]] - m))
            g = g + cfg.ce_weight * (e1 / e1.sum() - one)
            s = s + abs(cfg.ce_weight) * (e1 / e1.sum() + one)
        grad[r], size[r] = w[r] * g, abs(w[r]) * s
    return loss, grad, size


@pytest.fixture(autouse=True)
def formulas(monkeypatch):
    monkeypatch.setattr(near, "ref", ref_far)


def students(rng, N, V, K, gap, T, left=0.3):
    """Rows whose listed ids lie `gap` T above the others' range, the list
    anywhere in the row; `left` of the teacher's mass outside."""
    x = rng.normal(0, 2, (N, V))
    ids = np.stack([rng.choice(V, K, replace=False) for _ in range(N)])
    np.put_along_axis(x, ids, gap * T + rng.normal(0, 1, (N, K)), 1)
    logp = np.log(rng.dirichlet(np.ones(K) * 4, N) * (1 - left)).astype(np.float32)
    return x.astype(np.float32), ids, logp


CFGS = [dict(tail=True), dict(tail=True, temperature=0.5, kl_weight=0.25), dict(tail=True, temperature=2.0, ce_weight=0.5),
        dict(tail=True, ce_weight=0.3, kl_weight=2.0)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gap", [30, 45, 80, 100, 110, 300, 1000])
def test_gaps(gap, dtype):
    """By passes (short rows) and a workgroup a row; labels in and outside the list."""
    from zllm_amd.distill import DistillConfig
    rng = np.random.default_rng(gap)
    for i, kw in enumerate(CFGS):
        for V in (61, 3001, 5003):
            cfg = DistillConfig(**kw)
            x, ids, logp = students(rng, 6, V, (1, 8, 50, 30)[i], gap, cfg.temperature)
            labels = ids[:, 0].copy()
            labels[1], labels[2] = (ids[1, 0] + 1) % V, -100
            while labels[1] in ids[1]:
                labels[1] = (labels[1] + 1) % V
            check(rows_at(x, dtype, (0, 1, 3, 7)[i], 2), ids, logp, cfg, labels if "ce_weight" in kw else None,
                  rng.normal(0, 1, 6), f"gap {gap}")


@pytest.mark.parametrize("dtype,V", [("f32", 40000), ("bf16", 40003), ("bf16", 151936)])
@pytest.mark.parametrize("gap", [90, 110, 400])
def test_rows_come_out_alike_in_few_and_many(gap, dtype, V):
    """The passes (95 rows) and a workgroup a row (96): the same rows, by the
    same formulas, none infinite."""
    from zllm_amd.distill import DistillConfig, distill_loss_grad
    rng = np.random.default_rng(gap + V)
    cfg = DistillConfig(tail=True, ce_weight=0.2)
    x, ids, logp = students(rng, 4, V, 20, gap, 1.0)
    x[3] = rng.normal(0, 2, V)                  # (one that is not far)
    labels = ids[:, 1].copy()
    rows = np.arange(96) % 4
    X, I, P, L = x[rows], ids[rows], logp[rows], labels[rows]
    for n in (95, 96):
        check(rows_at(X[:n], dtype, 0, 0), I[:n], P[:n], cfg, L[:n], None, f"few and many, gap {gap}")
    t = [torch.from_numpy(a).cuda() for a in (I.astype(np.int32), P, L)]
    xt, w = rows_at(X, dtype, 0, 0), torch.ones(96, device="cuda")
    few = distill_loss_grad(_ctx(), xt[:95], t[0][:95], t[1][:95], cfg, w[:95], t[2][:95])
    many = distill_loss_grad(_ctx(), xt, t[0], t[1], cfg, w, t[2])
    assert torch.isfinite(few[0]).all() and torch.isfinite(many[0]).all()
    assert ((few[0] - many[0][:95]).abs() <= 6 * 1.2 * ltol(V) + 2.0 ** -22 * few[0].abs()).all()
    assert torch.isfinite(few[1]).all() and torch.isfinite(many[1]).all()


@pytest.mark.parametrize("n", [4, 100])
def test_in_place(n):
    """The rows are read again for such sums: before anything is written over them."""
    from zllm_amd.distill import DistillConfig, distill_grad, distill_loss, distill_loss_grad
    rng = np.random.default_rng(n)
    V = 40005
    cfg = DistillConfig(tail=True, ce_weight=0.5, temperature=1.5)
    x, ids, logp = students(rng, n, V, 30, 200, 1.5)
    i, p = torch.from_numpy(ids.astype(np.int32)).cuda(), torch.from_numpy(logp).cuda()
    lab, w = torch.from_numpy(ids[:, 2].copy()).cuda(), torch.rand(n, device="cuda")
    for dtype in TYPES:
        print(f"[case] distill far in place n={n} {dtype}", flush=True)
        a, b, c = (rows_at(x, dtype, 1, 2) for _ in range(3))
        _, stats = distill_loss(_ctx(), a, i, p, cfg, lab)
        want, want2 = distill_grad(_ctx(), a, i, p, cfg, stats, w, lab), distill_loss_grad(_ctx(), a, i, p, cfg, w, lab)[1]
        assert torch.equal(distill_grad(_ctx(), b, i, p, cfg, stats, w, lab, out=b), want)
        assert torch.equal(distill_loss_grad(_ctx(), c, i, p, cfg, w, lab, out=c)[1], want2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 30])
def test_huge_gaps(n, dtype):
    """Listed ids at 1e10 to 3e38 above the others, the others ordinary or huge."""
    from zllm_amd.distill import DistillConfig
    rng = np.random.default_rng(n)
    V, K = 33001, 6
    x, ids, logp = students(rng, 4, V, K, 10, 1.0)
    for r, (v, o) in enumerate(((1e10, 0.0), (1e30, 5e29), (3e38, -1e9), (-1e9, -1e30))):
        x[r] += np.float32(o)
        x[r, ids[r]] = v
    x, ids, logp = (np.concatenate([a] * n) for a in (x, ids, logp))
    for T in (1.0, 2.0):
        check(rows_at(x, dtype, 1, 2), ids, logp, DistillConfig(tail=True, temperature=T), None, None, "huge gaps")


def test_weights_of_a_loss_scale():
    """Weights that the outside factor alone would take past the floats."""
    from zllm_amd.distill import DistillConfig
    rng = np.random.default_rng(9)
    V = 900
    for gap in (25, 31, 60):
        x, ids, logp = students(rng, 3, V, 8, gap, 1.0)
        check(rows_at(x, "f32", 0, 0), ids, logp, DistillConfig(tail=True, kl_weight=2.0 ** 60),
              None, np.full(3, 2.0 ** 40), f"weights, gap {gap}")


def test_nothing_outside_is_still_infinite():
    """No mass at all outside the list: what the teacher has there cannot be given."""
    from zllm_amd.distill import DistillConfig, distill_loss, distill_loss_grad
    N, V = 100, 40000
    x = torch.full((N, V), -float("inf"), device="cuda")
    x[:, 5:9] = torch.randn((N, 4), device="cuda")
    ids = torch.arange(5, 9, device="cuda", dtype=torch.int32).expand(N, 4).contiguous()
    logp = torch.full((N, 4), math.log(0.2), device="cuda")
    w = torch.ones(N, device="cuda")
    cfg = DistillConfig(tail=True)
    print("[case] distill nothing outside", flush=True)
    for n in (3, N):
        loss = distill_loss(_ctx(), x[:n], ids[:n], logp[:n], cfg)[0]
        l2, g = distill_loss_grad(_ctx(), x[:n], ids[:n], logp[:n], cfg, w[:n])
        assert torch.isposinf(loss).all() and torch.isposinf(l2).all()
        assert torch.isfinite(g).all() and not g[:, 9:].any()


@pytest.mark.parametrize("n", [4, 100])
def test_labels_outside_the_vocabulary(n):
    """Their rows are NaN, far ones too."""
    from zllm_amd.distill import DistillConfig, distill_grad, distill_loss, distill_loss_grad
    rng = np.random.default_rng(n)
    V = 40001
    x, ids, logp = students(rng, n, V, 9, 200, 1.0)
    xt, i, p = rows_at(x, "f32", 0, 1), torch.from_numpy(ids.astype(np.int32)).cuda(), torch.from_numpy(logp).cuda()
    lab, w = torch.from_numpy(ids[:, 0].copy()).cuda(), torch.ones(n, device="cuda")
    lab[1], lab[2] = V, -1
    print(f"[case] distill far, labels outside, n={n}", flush=True)
    for cfg in (DistillConfig(tail=True, ce_weight=0.5), DistillConfig(tail=True, ce_weight=0.5, temperature=2.0)):
        loss, stats = distill_loss(_ctx(), xt, i, p, cfg, lab)
        for l, g in ((loss, distill_grad(_ctx(), xt, i, p, cfg, stats, w, lab)),
                     distill_loss_grad(_ctx(), xt, i, p, cfg, w, lab)):
            assert torch.isnan(l[1:3]).all() and torch.isfinite(l[0]) and torch.isfinite(l[3:]).all()
            assert torch.isnan(g[1:3]).all() and torch.isfinite(g[0]).all() and torch.isfinite(g[3:]).all()


def test_gradient_against_differences():
    from zllm_amd.distill import DistillConfig, distill_loss
    rng = np.random.default_rng(3)
    V, K, h = 37, 5, 2.0 ** -5
    for gap in (60, 120):
        x, ids, logp = students(rng, 1, V, K, gap, 1.0)
        cfg = DistillConfig(tail=True)
        _, _, g = check(rows_at(x, "f32", 0, 0), ids, logp, cfg, what="differences")
        # (steps of h change every value by what it holds of it)
        up, down = x + h * np.eye(V, dtype=np.float32), x - h * np.eye(V, dtype=np.float32)
        step = (np.diagonal(up) - np.diagonal(down)).astype(np.float64)
        n = 2 * V
        loss, _ = distill_loss(_ctx(), torch.from_numpy(np.concatenate([up, down])).cuda(),
                               torch.from_numpy(ids).to(torch.int32).cuda().expand(n, K).contiguous(),
                               torch.from_numpy(logp).cuda().expand(n, K).contiguous(), cfg)
        d = ((loss[:V] - loss[V:]).double().cpu().numpy()) / step
        # third derivatives of the two ln sum exp are below 0.1 each; the losses are within 3 L and 2^-23 |loss|, over h
        tol = h * h / 6 * 0.2 + (3 * ltol(V) + 2.0 ** -23 * float(loss.abs().max())) / h
        assert (np.abs(d - g[0].double().cpu().numpy()) <= tol + TINY["f32"]).all()
