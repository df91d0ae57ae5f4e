"""A teacher's lists and the distillation loss with its gradient against the
formulas in 64 bits, the gradient against differences too.

Tolerances. A sum of exponentials is of f32 terms within 2^-22 of their exact
value each, added in chains of at most V / 256 + 64: its logarithm is within
L = (V / 256 + 64) 2^-23. A loss is a few such logarithms weighted by at most
kl_weight and ce_weight, rounded once: 3 (kl + ce) L + 2^-23 |loss|. A
gradient is weight * (f q - p): q within 2 L of itself (and the factors' 2^-22),
p within 2^-22, then rounded to the logits' type."""
import math

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


def ltol(V):
    return (V / 256 + 64) * 2.0 ** -23


def rows_at(x, dtype, shift, pad):
    R, V = x.shape
    buf = torch.full((R, shift + V + pad), float("nan"), dtype=TYPES[dtype], device="cuda")
    buf[:, shift:shift + V] = torch.from_numpy(np.asarray(x, np.float32)).to(TYPES[dtype]).cuda()
    return buf[:, shift:shift + V]


# ------------------------------------------------------------------ the teacher's lists
def check_teacher(xt, K, T, what=""):
    from zllm_amd.distill import teacher_topk
    N, V = xt.shape
    print(f"[case] teacher_topk {what} N={N} V={V} K={K} T={T} {xt.dtype} ld={xt.stride(0)}", flush=True)
    ids, logp, lse = (t.cpu().numpy() for t in teacher_topk(_ctx(), xt, K, T))
    x = xt.double().cpu().numpy()
    x = np.minimum(np.where(np.isnan(x), -np.inf, x), np.finfo(np.float32).max)
    for r in range(N):
        order = np.lexsort((np.arange(V), -x[r]))[:K]
        order = order[x[r][order] > -np.inf]
        n = len(order)
        assert ids[r, :n].tolist() == order.tolist(), r
        assert (ids[r, n:] == -1).all() and np.isneginf(logp[r, n:]).all()
        if n == 0:
            assert np.isneginf(lse[r])
            continue
        z = x[r] / T
        m = z.max()
        L = m + np.log(np.exp(z - m).sum())
        tol = ltol(V) + 2.0 ** -23 * abs(L)
        assert abs(lse[r] - L) <= tol
        want = (z[order] - m) - np.log(np.exp(z - m).sum())
        assert (np.abs(logp[r, :n] - want) <= ltol(V) + 2.0 ** -23 * np.abs(want)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,V", [(1, 1), (3, 5), (2, 130), (5, 1000), (3, 4099), (2, 50257), (2, 163841)])
def test_teacher_sizes(N, V, dtype):
    rng = np.random.default_rng(N + V)
    x = rng.normal(0, 2, (N, V))
    for K, T, shift in ((1, 1.0, 0), (min(V, 50), 2.0, 1), (min(V, 128), 0.7, 6)):
        check_teacher(rows_at(x, dtype, shift, 3), K, T)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [700, 20000, 128256])
def test_teacher_rows_of_ties_and_orders(V, dtype):
    """Equal values, sorted rows, whole numbers, more equal values at the K-th
    place than a list holds, NaN, infinities, fewer values than K."""
    rng = np.random.default_rng(V)
    x = rng.normal(0, 2, (13, V)).astype(np.float32)
    x[0].sort()
    x[1] = np.sort(x[1])[::-1]
    x[2] = 1.5
    x[3] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    x[4] = np.round(x[4])
    x[5, V // 3:V // 3 + 600] = 20.0
    x[6, ::2] = np.nan
    x[7] = -np.inf
    x[7, [0, V // 2, V - 1]] = [1.0, np.nan, 2.0]
    x[8] = np.nan
    x[9, rng.choice(V, 90, replace=False)] = np.inf
    x[10, :300] = np.linspace(20, 30, 300)
    x[11, -300:] = 12.0
    x[12] = -60000.0
    x[12, V - 1] = 60000.0
    xt = rows_at(x, dtype, 1, 2)
    for K in (1, 33, 64, 65, 128):
        check_teacher(xt, K, 1.0, "orders")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_teacher_rows_of_huge_values(dtype):
    """Rows all at a mask's finite value are even ones, equal values at the top
    of huge ones share; temperatures that make ordinary rows huge."""
    rng = np.random.default_rng(1)
    V = 9001
    x = np.empty((8, V), np.float32)
    for r, v in enumerate((-1e9, -1e10, -1e30, torch.finfo(TYPES[dtype]).min, 1e10, 3.3e38)):
        x[r] = v
    x[6] = 5e29
    x[6, [3, 77, V - 1]] = 1e30
    x[7] = -1e30
    x[7, 10:15] = rng.normal(0, 1, 5)
    for T in (1.0, 3.0, 1e20):
        check_teacher(rows_at(x, dtype, 1, 2), 100, T, "huge")
    y = np.concatenate([rng.normal(0, 1000, (2, V)), np.full((1, V), -7.0), np.zeros((1, V))])
    for T in (1e-7, 1e-12, 1e-25, 1e-34):
        check_teacher(rows_at(y, dtype, 1, 2), 100, T, "cold")


def test_teacher_rows_far_apart():
    """Rows past 4 GiB."""
    buf = torch.empty((3, 1_200_000_000), dtype=torch.float16, device="cuda")
    x = buf[:, -5000:]
    x.copy_(torch.randn((3, 5000), device="cuda"))
    check_teacher(x, 20, 1.0, "far")


# ------------------------------------------------------------------ loss and gradient
def lists(rng, x, K, full=True):
    """A teacher's list per row: ids of the largest values of x and noise."""
    N, V = x.shape
    t = np.nan_to_num(x, nan=0.0, posinf=50, neginf=-50) + rng.normal(0, 0.7, x.shape)
    ids = np.argsort(-t, axis=1)[:, :K].astype(np.int64)
    lse = np.log(np.exp(t - t.max(1, keepdims=True)).sum(1, keepdims=True)) + t.max(1, keepdims=True)
    logp = (np.take_along_axis(t, ids, 1) - lse).astype(np.float32)
    if not full:
        none = np.arange(K) >= rng.integers(0, K + 1, (N, 1))
        ids[none], logp[none] = -1, -np.inf
    return ids, logp


def ref(x, ids, logp, labels, cfg, w):
    """Loss, gradient and the parts |f q| + |p| that its rounding goes by."""
    N, V = x.shape
    loss, grad, size = np.zeros(N), np.zeros((N, V)), np.zeros((N, V))
    T = cfg.temperature
    with np.errstate(all="ignore"):
        for r in range(N):
            if labels is not None and labels[r] == cfg.ignore_index:
                continue
            m = x[r].max()
            z = (x[r] - m) / T
            q = np.exp(z) / np.exp(z).sum()
            lq = z - np.log(np.exp(z).sum())
            ok = (ids[r] >= 0) & (ids[r] < V) & ~np.isneginf(logp[r])
            k, p = ids[r][ok], np.exp(logp[r][ok].astype(np.float64))
            if not cfg.tail and p.sum() > 0:
                p = p / p.sum()
            kl = sum(pi * (np.log(pi) - lq[ki]) for pi, ki in zip(p, k) if pi > 0)
            P = p.sum()
            g = np.zeros(V)
            np.add.at(g, k, -p)
            s = np.abs(g)
            if cfg.tail:
                out = np.ones(V, bool)
                out[k] = False
                pt, qt = max(0.0, 1.0 - P), q[out].sum()
                if pt > 0:
                    kl += pt * (np.log(pt) - np.log(qt))
                if qt > 0:
                    g[out] -= pt * q[out] / qt
                    s[out] += pt * q[out] / qt
                P = P + pt
            g = cfg.kl_weight / T * (g + P * q)
            s = abs(cfg.kl_weight) / T * (s + P * q)
            loss[r] = cfg.kl_weight * kl
            if labels is not None:
                q1 = np.exp(x[r] - m) / np.exp(x[r] - m).sum()
                loss[r] += cfg.ce_weight * -np.log(q1[labels[r]])
                one = np.zeros(V)
                one[labels[r]] = 1.0
                g = g + cfg.ce_weight * (q1 - one)
                s = s + abs(cfg.ce_weight) * (q1 + one)
            grad[r], size[r] = w[r] * g, abs(w[r]) * s
    return loss, grad, size


def check(xt, ids, logp, cfg, labels=None, w=None, what="", out=None):
    from zllm_amd.distill import distill_grad, distill_loss, distill_loss_grad
    N, V = xt.shape
    dt = {v: k for k, v in TYPES.items()}[xt.dtype]
    w = np.ones(N, np.float32) if w is None else w.astype(np.float32)
    print(f"[case] distill {what} N={N} V={V} K={ids.shape[1]} {cfg} {xt.dtype} ld={xt.stride(0)}", flush=True)
    x = xt.double().cpu().numpy()
    loss, grad, size = ref(x, ids, logp, labels, cfg, w)
    t = dict(ids=torch.from_numpy(ids).to(torch.int32).cuda(), logp=torch.from_numpy(logp).cuda())
    lab = None if labels is None else torch.from_numpy(labels).cuda()
    wt = torch.from_numpy(w).cuda()
    l1, stats = distill_loss(_ctx(), xt, t["ids"], t["logp"], cfg, lab)
    g1 = distill_grad(_ctx(), xt, t["ids"], t["logp"], cfg, stats, wt, lab, out=out)
    l2, g2 = distill_loss_grad(_ctx(), xt, t["ids"], t["logp"], cfg, wt, lab)
    torch.cuda.synchronize()
    weight = abs(cfg.kl_weight) + (abs(cfg.ce_weight) if labels is not None else 0.0)
    for l in (l1, l2):
        l = l.double().cpu().numpy()
        same = (l == loss) | (np.isnan(l) & np.isnan(loss))
        assert (same | (np.abs(l - loss) <= 3 * weight * ltol(V) + 2.0 ** -23 * np.abs(loss))).all(), \
            (l, loss)
    for g in (g1, g2):
        g = g.double().cpu().numpy()
        tol = size * (2 * ltol(V) + 2.0 ** -21) + EPS[dt] * np.abs(grad) + TINY[dt]
        same = np.isnan(g) & np.isnan(grad)
        assert (same | (np.abs(g - grad) <= tol)).all(), np.nanmax(np.abs(g - grad) - tol)
    return l1, stats, g1


CFGS = [dict(), dict(temperature=2.0, kl_weight=4.0), dict(tail=True), dict(temperature=1.5, tail=True, ce_weight=0.5),
        dict(temperature=3.0, ce_weight=0.3, kl_weight=6.3), dict(tail=True, ce_weight=1.0, kl_weight=0.0),
        dict(ce_weight=0.4)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 37, 1000, 4099, 20011])
def test_formulas(V, dtype):
    from zllm_amd.distill import DistillConfig
    rng = np.random.default_rng(V)
    N = 6
    x = rng.normal(0, 2, (N, V))
    x[:, rng.integers(0, V)] += 6.0
    for i, kw in enumerate(CFGS):
        K = min(V, (1, 5, 50, 128)[i % 4])
        xt = rows_at(x, dtype, (0, 1, 4, 7)[i % 4], i)
        ids, logp = lists(rng, x, K, full=i % 2 == 0)
        labels = rng.integers(0, V, N)
        labels[2] = -100
        check(xt, ids, logp, DistillConfig(**kw), labels if kw.get("ce_weight") else None, rng.normal(0, 1, N), f"cfg {i}")


@pytest.mark.parametrize("N,V,dtype", [(2, 151936, "bf16"), (3, 151937, "f32"), (300, 32000, "f16"), (1, 262147, "bf16"),
                                       (2, 400001, "f32"), (1, 1048576, "bf16")])
def test_large_rows(N, V, dtype):
    from zllm_amd.distill import DistillConfig
    rng = np.random.default_rng(V)
    n = min(N, 3)
    x = rng.normal(0, 2, (n, V)).astype(np.float32)
    x[:, :20] += 8.0
    ids, logp = lists(rng, x, 64)
    x, ids, logp = (np.concatenate([a] * (N // n)) for a in (x, ids, logp))
    labels = ids[:, 3].copy()
    check(rows_at(x, dtype, 0, 0), ids, logp, DistillConfig(tail=True, ce_weight=0.2, temperature=1.3), labels,
          np.full(N, 0.25), "large")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tail", [False, True])
def test_lists_that_go_wrong(tail, dtype):
    """Empty lists, ids outside the vocabulary, ids listed twice, probabilities
    over 1 in all, entries of no probability, neighbours in one 16-byte vector,
    the first and the last id, the label in and outside the list."""
    from zllm_amd.distill import DistillConfig
    rng = np.random.default_rng(7)
    N, V, K = 9, 501, 16
    x = rng.normal(0, 2, (N, V))
    ids, logp = lists(rng, x, K)
    ids[0], logp[0] = -1, -np.inf
    ids[1, ::2] = [V, V + 7, 2 ** 31 - 1, -1, -2, V, V, V]
    ids[2, 5] = ids[2, 4]
    ids[2, 9:12] = ids[2, 4]
    logp[3] = -0.5
    logp[4, 3:] = -np.inf
    logp[4, 1] = -200.0
    ids[5] = np.arange(K)
    ids[6] = V - 1 - np.arange(K)
    logp[7] = -300.0
    labels = ids[:, 0].copy()
    labels[0], labels[1], labels[6] = 3, 9, V - 1
    for shift in (0, 1, 5):
        for T in (1.0, 2.0):
            check(rows_at(x, dtype, shift, 1), ids, logp, DistillConfig(temperature=T, tail=tail, ce_weight=0.5), labels,
                  None, f"lists shift={shift}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 57])
def test_students_of_huge_values(n, dtype):
    """Rows all at a mask's finite value are even ones; huge values beside
    ordinary ones; by passes and (513 rows) a workgroup a row."""
    from zllm_amd.distill import DistillConfig
    rng = np.random.default_rng(n)
    V, K = 4500, 12
    x = np.empty((9, V), np.float32)
    for r, v in enumerate((-1e9, -1e10, -1e30, torch.finfo(TYPES[dtype]).min, 1e10, 3.3e38)):
        x[r] = v
    x[6] = -1e30
    x[6, 10:400] = rng.normal(0, 1, 390)
    x[7] = -2e10
    x[7, 4000] = -1e10
    x[8] = 1e12 + 1e11 * rng.normal(0, 1, V)
    ids, logp = lists(rng, rng.normal(0, 2, (9, V)), K)
    ids[6] = 10 + np.arange(K)
    labels = ids[:, 2].copy()
    x, ids, logp, labels = (np.concatenate([a] * n) for a in (x, ids, logp, labels))
    for kw in (dict(), dict(tail=True), dict(tail=True, temperature=2.0, ce_weight=0.5), dict(temperature=1e-3)):
        check(rows_at(x, dtype, 1, 2), ids, logp, DistillConfig(**kw), labels if "ce_weight" in kw else None, None, "huge")


@pytest.mark.parametrize("n", [3, 520])
def test_lists_of_all_there_is(n):
    """Lists that have every id, or every id that is allowed: what rounding
    leaves of 1 is no tail that the student would have to have."""
    from zllm_amd.distill import DistillConfig, distill_loss, distill_loss_grad
    rng = np.random.default_rng(n)
    V, K = 4200 if n > 100 else 60, 60
    t, x = rng.normal(0, 2, (n, K)), rng.normal(0, 2, (n, K))
    logp = (t - np.log(np.exp(t).sum(1, keepdims=True))).astype(np.float32)
    logp -= np.float32(2.0 ** -22)               # (what is left is positive in every row)
    ids = np.stack([rng.choice(V, K, replace=False) for _ in range(n)])
    full = np.full((n, V), -np.inf, np.float32)
    np.put_along_axis(full, ids, x.astype(np.float32), 1)
    p = np.exp(logp.astype(np.float64))
    assert (p.sum(1) < 1).all() and (1 - p.sum(1) < 2.0 ** -20).all()
    x = x.astype(np.float32).astype(np.float64)
    lq = x - np.log(np.exp(x).sum(1, keepdims=True))
    want = (p * (logp - lq)).sum(1)
    xt, it, lt = torch.from_numpy(full).cuda(), torch.from_numpy(ids).to(torch.int32).cuda(), torch.from_numpy(logp).cuda()
    cfg = DistillConfig(tail=True)
    print(f"[case] distill lists of all n={n} V={V}", flush=True)
    loss = distill_loss(_ctx(), xt, it, lt, cfg)[0]
    l2, g = distill_loss_grad(_ctx(), xt, it, lt, cfg, torch.ones(n, device="cuda"))
    for l in (loss, l2):
        assert (np.abs(l.double().cpu().numpy() - want) <= 3 * ltol(V) + 2.0 ** -23 * np.abs(want)).all()
    g = g.double().cpu().numpy()
    at = np.take_along_axis(g, ids, 1)
    assert (np.abs(at - (np.exp(lq) - p)) <= (np.exp(lq) + p) * (2 * ltol(V) + 2.0 ** -21) + TINY["f32"]).all()
    np.put_along_axis(g, ids, 0.0, 1)
    assert not g.any()


@pytest.mark.parametrize("n", [5, 515])
def test_terms_of_no_weight(n):
    """A term of weight 0 has no part in the loss, were it infinite; labels
    outside the vocabulary are still NaN."""
    from zllm_amd.distill import DistillConfig, distill_loss, distill_loss_grad
    V = 4100
    x = torch.randn((n, V), device="cuda")
    x[:, 9] = -float("inf")
    labels = torch.full((n,), 9, device="cuda")
    labels[1], labels[2] = V, -100
    ids = torch.tensor([[3, 4, 5]], dtype=torch.int32, device="cuda").expand(n, 3).contiguous()
    logp = torch.full((n, 3), -1.2, device="cuda")
    far = torch.full((n, 3), 9, dtype=torch.int32, device="cuda")
    w = torch.ones(n, device="cuda")
    print(f"[case] distill weights of 0 n={n}", flush=True)
    for cfg, i, lab in ((DistillConfig(ce_weight=0.0), ids, 9), (DistillConfig(kl_weight=0.0, ce_weight=1.0), far, 3)):
        labels[labels == 9] = lab
        loss = distill_loss(_ctx(), x, i, logp, cfg, labels)[0]
        l2, g = distill_loss_grad(_ctx(), x, i, logp, cfg, w, labels)
        for l in (loss, l2):
            assert torch.isnan(l[1]) and l[2] == 0
            assert torch.isfinite(l[0]) and torch.isfinite(l[3:]).all() and (l[3:] != 0).all()
        assert torch.isnan(g[1]).all() and torch.isfinite(g[0]).all() and torch.isfinite(g[2:]).all()


@pytest.mark.parametrize("V,dtype", [(4096, "bf16"), (4099, "f32"), (16385, "f32"), (32761, "bf16"), (50257, "f16"),
                                     (65537, "bf16"), (100003, "f32"), (151936, "bf16"), (196597, "f32")])
def test_many_rows(V, dtype):
    """As many rows as a training step has (a workgroup a row there): 10 rows
    that go wrong in their own ways, 52 times each. Copies that begin alike in
    their 16 bytes (which orders the sums) come out bit for bit alike, all of
    them by the formulas; into other places and in place alike."""
    from zllm_amd.distill import DistillConfig, distill_loss_grad
    rng = np.random.default_rng(V)
    n, times, K = 10, 52, 40
    x = rng.normal(0, 2, (n, V)).astype(np.float32)
    ids, logp = lists(rng, x, K)
    ids[0, ::4] = [V, V + 7, 2 ** 31 - 1, -1, -2, V, V, V, -1, V]
    ids[1, 5:9] = ids[1, 4]
    ids[2], logp[2] = -1, -np.inf
    ids[3, :20], ids[3, 20:] = np.arange(20), V - 1 - np.arange(20)
    x[4, ids[4]] += 30.0                        # learnt
    x[5, rng.random(V) < 0.6] = -np.inf
    ids[5] = rng.choice(np.flatnonzero(np.isfinite(x[5])), K, replace=False)
    x[6, V // 2] = np.nan
    x[7, V - 1], x[8, 0] = 25.0, 25.0           # the row's ends
    ids[7, 0], ids[8, 0] = V - 1, 0
    labels = ids[:, 1].copy()
    labels[0], labels[1], labels[2], labels[7], labels[8], labels[9] = V - 1, 77, 0, V - 1, 0, -100
    w = rng.normal(0, 1, n).astype(np.float32)
    X, I, P, L, W = (torch.from_numpy(np.concatenate([a] * times)).cuda() for a in (x, ids.astype(np.int32), logp, labels, w))
    for k, kw in enumerate((dict(tail=True, ce_weight=0.5, temperature=1.5), dict(tail=True, ce_weight=0.3), dict(),
                            dict(ce_weight=0.2, temperature=2.0))):
        cfg = DistillConfig(**kw)
        lab = L if "ce_weight" in kw else None
        base = torch.full((n * times, V + (0, 3, 8, 5)[k]), float("nan"), dtype=TYPES[dtype], device="cuda")
        xt = base[:, (0, 1, 8, 2)[k]:][:, :V]
        xt.copy_(X)
        print(f"[case] distill many rows V={V} {dtype} {cfg} ld={xt.stride(0)}", flush=True)
        loss, g = distill_loss_grad(_ctx(), xt, I, P, cfg, W, lab)
        loss64, grad, size = ref(xt[:n].double().cpu().numpy(), ids, logp, None if lab is None else labels, cfg, w)
        bits = lambda t: t.contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16)
        alike = 16 // math.gcd(16, n * xt.stride(0) * xt.element_size())      # copies from one to the next alike
        for a in (bits(loss).view(times, n), bits(g).view(times, n, V)):
            assert all(torch.equal(a[c], a[c % alike]) for c in range(times))
        weight = 1.0 + kw.get("ce_weight", 0.0)
        for c in range(alike):
            l, d = (t[c * n:(c + 1) * n].double().cpu().numpy() for t in (loss, g))
            ok = (l == loss64) | (np.isnan(l) & np.isnan(loss64))
            assert (ok | (np.abs(l - loss64) <= 3 * weight * ltol(V) + 2.0 ** -23 * np.abs(loss64))).all(), (l, loss64)
            tol = size * (2 * ltol(V) + 2.0 ** -21) + EPS[dtype] * np.abs(grad) + TINY[dtype]
            assert ((np.isnan(d) & np.isnan(grad)) | (np.abs(d - grad) <= tol)).all(), np.nanmax(np.abs(d - grad) - tol)
        out = torch.zeros((n * times, V + 9), dtype=TYPES[dtype], device="cuda")
        distill_loss_grad(_ctx(), xt, I, P, cfg, W, lab, out=out[:, 3:V + 3])
        assert torch.equal(bits(out[:, 3:V + 3]), bits(g)) and not out[:, :3].any() and not out[:, V + 3:].any()
        del out
        distill_loss_grad(_ctx(), xt, I, P, cfg, W, lab, out=xt)
        assert torch.equal(bits(xt), bits(g))
        lo = (0, 1, 8, 2)[k]
        assert torch.isnan(base[:, :lo]).all() and torch.isnan(base[:, lo + V:]).all()


def test_student_that_has_learnt_the_list():
    """Next to no mass outside the list: what is outside is summed by itself."""
    from zllm_amd.distill import DistillConfig
    rng = np.random.default_rng(5)
    N, V, K = 4, 3001, 8
    x = rng.normal(0, 1, (N, V))
    ids = np.stack([rng.choice(V, K, replace=False) for _ in range(N)])
    np.put_along_axis(x, ids, 28.0 + rng.normal(0, 1, (N, K)), 1)     # e^-28 V outside
    logp = np.log(np.full((N, K), 0.9 / K)).astype(np.float32)
    check(rows_at(x, "f32", 0, 0), ids, logp, DistillConfig(tail=True), None, None, "learnt")


def test_no_numbers_come_out():
    """NaN and infinities of the student are not hidden; labels outside the
    vocabulary are NaN; ignored rows are not read."""
    from zllm_amd.distill import DistillConfig, distill_grad, distill_loss, distill_loss_grad
    N, V = 6, 1000
    x = torch.randn((N, V), device="cuda")
    x[0, 7] = float("nan")
    x[1, 9] = float("inf")
    x[2] = float("nan")
    x[3, 11:500] = -float("inf")
    ids = torch.arange(4, device="cuda", dtype=torch.int32).expand(N, 4).contiguous()
    logp = torch.full((N, 4), -1.5, device="cuda")
    labels = torch.tensor([1, 1, -100, 1, V, 1], device="cuda")
    cfg = DistillConfig(tail=True, ce_weight=0.5)
    w = torch.ones(N, device="cuda")
    loss, stats = distill_loss(_ctx(), x, ids, logp, cfg, labels)
    for l, g in ((loss, distill_grad(_ctx(), x, ids, logp, cfg, stats, w, labels)),
                 distill_loss_grad(_ctx(), x, ids, logp, cfg, w, labels)):
        assert torch.isnan(l).tolist() == [True, True, False, False, True, False]
        assert torch.isnan(g[0]).all() and torch.isnan(g[1]).any() and torch.isnan(g[4]).all()
        assert l[2] == 0 and not g[2].any()
        assert torch.isfinite(l[3]) and torch.isfinite(g[3]).all() and not g[3, 11:500].any()
    assert not stats[2].any()


def test_gradient_against_differences():
    from zllm_amd.distill import DistillConfig, distill_loss
    rng = np.random.default_rng(2)
    V, K, h = 37, 5, 2.0 ** -5
    x = rng.normal(0, 1.5, (1, V)).astype(np.float32)
    ids, logp = lists(rng, x, K)
    for kw in (dict(tail=True, ce_weight=0.5, temperature=1.5), dict(ce_weight=0.3), dict(temperature=2.0, tail=True)):
        cfg = DistillConfig(**kw)
        labels = np.array([int(ids[0, 2])])
        _, _, g = check(rows_at(x, "f32", 0, 0), ids, logp, cfg, labels, what="differences")
        both = np.concatenate([x + h * np.eye(V, dtype=np.float32), x - h * np.eye(V, dtype=np.float32)])
        n = 2 * V
        loss, _ = distill_loss(_ctx(), torch.from_numpy(both).cuda(), torch.from_numpy(ids).to(torch.int32).cuda().expand(n, K)
                               .contiguous(), torch.from_numpy(logp).cuda().expand(n, K).contiguous(), cfg,
                               torch.from_numpy(labels).cuda().expand(n).contiguous())
        d = ((loss[:V] - loss[V:]).double() / (2 * h)).cpu().numpy()
        # third derivatives of ln sum exp are below 0.1 and there are at most three of them: h^2 / 6 * 0.3; the
        # losses are within 3 (kl + ce) L and 2^-23 |loss|, over h
        tol = h * h / 6 * 0.3 + (3 * 1.5 * ltol(V) + 2.0 ** -23 * float(loss.abs().max())) / h
        assert (np.abs(d - g[0].double().cpu().numpy()) <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gradient_in_place_and_at_other_places(dtype):
    """Into the logits themselves, and into rows that begin elsewhere in their 16 bytes."""
    from zllm_amd.distill import DistillConfig, distill_grad, distill_loss, distill_loss_grad
    rng = np.random.default_rng(6)
    N, V, K = 5, 4003, 20
    x = rng.normal(0, 2, (N, V))
    ids, logp = lists(rng, x, K)
    cfg = DistillConfig(tail=True, ce_weight=0.1, temperature=1.7)
    labels = rng.integers(0, V, N)
    i, p, l = torch.from_numpy(ids).to(torch.int32).cuda(), torch.from_numpy(logp).cuda(), torch.from_numpy(labels).cuda()
    w = torch.rand(N, device="cuda")
    for shift in (0, 3):
        xt = rows_at(x, dtype, shift, 2)
        _, stats, _ = check(xt, ids, logp, cfg, labels)
        want = distill_grad(_ctx(), xt, i, p, cfg, stats, w, l)
        _, want2 = distill_loss_grad(_ctx(), xt, i, p, cfg, w, l)
        for o_shift in (0, 1, 3):
            out = rows_at(np.zeros((N, V)), dtype, o_shift, 5)
            assert torch.equal(distill_grad(_ctx(), xt, i, p, cfg, stats, w, l, out=out), want)
            assert torch.isnan(out._base[:, V + o_shift:]).all() and torch.isnan(out._base[:, :o_shift]).all()
            assert torch.equal(distill_loss_grad(_ctx(), xt, i, p, cfg, w, l, out=out)[1], want2)
            assert torch.isnan(out._base[:, V + o_shift:]).all() and torch.isnan(out._base[:, :o_shift]).all()
        a, b = rows_at(x, dtype, shift, 2), rows_at(x, dtype, shift, 2)
        assert torch.equal(distill_grad(_ctx(), a, i, p, cfg, stats, w, l, out=a), want)
        assert torch.equal(distill_loss_grad(_ctx(), b, i, p, cfg, w, l, out=b)[1], want2)


def test_autograd():
    """DistillLoss under autograd: a mean (one value broadcast to the rows), a
    weighted sum, and frozen logits."""
    from zllm_amd.distill import DistillConfig, DistillLoss, distill_grad, distill_loss
    rng = np.random.default_rng(11)
    N, V, K = 7, 900, 12
    x = rng.normal(0, 2, (N, V))
    ids, logp = lists(rng, x, K)
    i, p = torch.from_numpy(ids).to(torch.int32).cuda(), torch.from_numpy(logp).cuda()
    labels = torch.randint(0, V, (N,), device="cuda")
    cfg = DistillConfig(tail=True, ce_weight=0.5)
    f = DistillLoss(_ctx(), cfg)
    for dtype in TYPES.values():
        xt = torch.from_numpy(x).cuda().to(dtype).requires_grad_()
        loss, stats = distill_loss(_ctx(), xt.detach(), i, p, cfg, labels)
        f(xt, i, p, labels).mean().backward()
        w = torch.full((N,), 1.0 / N, device="cuda")
        assert torch.equal(xt.grad, distill_grad(_ctx(), xt.detach(), i, p, cfg, stats, w, labels))
        assert torch.equal(xt.grad, distill_grad(_ctx(), xt.detach(), i, p, cfg, stats, w[0], labels))
        xt.grad = None
        w = torch.rand(N, device="cuda")
        (f(xt, i, p, labels) * w).sum().backward()
        assert torch.equal(xt.grad, distill_grad(_ctx(), xt.detach(), i, p, cfg, stats, w, labels))
        assert torch.equal(f(xt.detach(), i, p, labels), loss)


def test_streams_and_graph():
    """The same results from a stream of its own and from a captured graph replayed between other work."""
    from zllm_amd.distill import DistillConfig, distill_loss_grad, teacher_topk
    gen = torch.Generator(device="cuda").manual_seed(3)
    N, V, K = 12, 30011, 16
    xs = [torch.randn((N, V), device="cuda", generator=gen).to(torch.bfloat16) for _ in range(3)]
    cfg = DistillConfig(tail=True)
    w = torch.full((N,), 1.0 / N, device="cuda")

    def both(x):
        ids, logp, lse = teacher_topk(_ctx(), x, K, 2.0)
        loss, g = distill_loss_grad(_ctx(), x, ids, logp, cfg, w)
        return ids, logp, lse, loss, g

    want = [both(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(xs[0])
        x = xs[0].clone()
        both(x)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = both(x)
    for k in (1, 2, 0, 1):
        x.copy_(xs[k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want[k])), k
        torch.randn(1000, device="cuda").sum()


# ------------------------------------------------------------------ refusals
def test_refusals():
    from zllm_amd._lib import ZsError
    from zllm_amd.distill import DistillConfig, distill_grad, distill_loss, distill_loss_grad, teacher_topk
    c = _ctx()
    x = torch.zeros((4, 100), device="cuda")
    ids, logp = torch.zeros((4, 8), dtype=torch.int32, device="cuda"), torch.zeros((4, 8), device="cuda")
    w, st = torch.ones(4, device="cuda"), torch.zeros((4, 4), device="cuda")
    cfg = DistillConfig()
    bad = [
        lambda: teacher_topk(c, x, 0), lambda: teacher_topk(c, x, 101), lambda: teacher_topk(c, x.double(), 3),
        lambda: teacher_topk(c, torch.zeros((2, 500), device="cuda"), 129), lambda: teacher_topk(c, x.cpu(), 3),
        lambda: teacher_topk(c, x.t(), 3), lambda: teacher_topk(c, x[0], 3),
        lambda: distill_loss(c, x, ids.long(), logp, cfg), lambda: distill_loss(c, x, ids[:3], logp, cfg),
        lambda: distill_loss(c, x, ids, logp[:, :4], cfg), lambda: distill_loss(c, x, ids, logp, cfg, w),
        lambda: distill_loss(c, x, ids.repeat(1, 17), logp.repeat(1, 17), cfg),
        lambda: distill_loss(c, x, ids, logp, cfg, torch.zeros(3, dtype=torch.int64, device="cuda")),
        lambda: distill_grad(c, x, ids, logp, cfg, st[:, :3], w), lambda: distill_grad(c, x, ids, logp, cfg, st, w[:3]),
        lambda: distill_grad(c, x, ids, logp, cfg, st, w.double()),
        lambda: distill_grad(c, x, ids, logp, cfg, st, w, out=x.half()),
        lambda: distill_loss_grad(c, x, ids, logp, cfg, w, out=torch.zeros((100, 4), device="cuda").t()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    for kw, text in ((dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
                     (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
                     (dict(kl_weight=float("inf")), "weights"), (dict(ce_weight=float("nan")), "weights")):
        with pytest.raises(ZsError, match=text):
            distill_loss(c, x, ids, logp, DistillConfig(**kw))
    with pytest.raises(ZsError, match="temperature"):
        teacher_topk(c, x, 3, 0.0)
    # rows of none are no error
    e = torch.zeros((0, 100), device="cuda")
    assert teacher_topk(c, e, 3)[0].shape == (0, 3)
    assert distill_loss(c, e, ids[:0], logp[:0], cfg)[0].shape == (0,)


def test_entry_point_refusals():
    """The C entry points' own checks: nothing is launched."""
    import ctypes as C

    from zllm_amd._lib import Distill, Teacher, ZS_EINVAL, ZS_ELIMIT, lib
    c, L = _ctx(), lib()
    n = C.c_uint64()
    for a in ((1, 10, 0), (1, 10, 11), (1, 0, 1), (1, 1000, 129), (1, (1 << 20) + 1, 1)):
        assert L.zs_teacher_topk_work(*a, C.byref(n)) == ZS_EINVAL, a
    x = torch.zeros((4, 1000), device="cuda")
    st = torch.full((4, 4), 7.0, device="cuda")
    i32 = torch.zeros((4, 8), dtype=torch.int32, device="cuda")
    assert L.zs_teacher_topk_work(4, 1000, 8, C.byref(n)) == 0
    work = torch.empty(max(n.value, 1 << 20), dtype=torch.uint8, device="cuda")

    def teach(**kw):
        a = Teacher(N=4, V=1000, K=8, ld=1000, d_logits=x.data_ptr(), temperature=1.0, d_ids=i32.data_ptr(),
                    d_logp=i32.data_ptr(), d_lse=st.data_ptr(), d_work=work.data_ptr(), work_bytes=work.numel())
        for k, v in kw.items():
            setattr(a, k, v)
        return L.zs_teacher_topk(c.h, C.byref(a), None)

    for kw in (dict(K=0), dict(K=129), dict(K=8, V=7), dict(V=(1 << 20) + 1)):
        assert teach(**kw) == ZS_ELIMIT, kw
    for kw in (dict(dtype=3), dict(ld=999), dict(d_logits=None), dict(d_logits=x.data_ptr() + 1), dict(d_ids=None),
               dict(d_lse=None), dict(temperature=0.0), dict(temperature=float("nan"))):
        assert teach(**kw) == ZS_EINVAL, kw
    assert teach(N=0) == 0

    def dist(fn, **kw):
        a = Distill(N=4, V=1000, K=8, ld=1000, d_logits=x.data_ptr(), d_ids=i32.data_ptr(), d_logp=i32.data_ptr(),
                    temperature=1.0, kl_weight=1.0, d_loss=st.data_ptr(), d_stats=st.data_ptr(),
                    d_row_grad=st.data_ptr(), row_grad_stride=1, d_grad=x.data_ptr(), ld_grad=1000,
                    d_work=work.data_ptr(), work_bytes=work.numel())
        for k, v in kw.items():
            setattr(a, k, v)
        return getattr(L, fn)(c.h, C.byref(a), None)

    for fn in ("zs_distill_loss", "zs_distill_grad", "zs_distill_loss_grad"):
        for kw in (dict(K=0), dict(K=129), dict(V=0)):
            assert dist(fn, **kw) == ZS_ELIMIT, kw
        for kw in (dict(dtype=3), dict(ld=999), dict(d_logits=None), dict(flags=2), dict(d_ids=None), dict(d_logp=None),
                   dict(temperature=0.0), dict(kl_weight=float("inf")), dict(ce_weight=float("nan"))):
            assert dist(fn, **kw) == ZS_EINVAL, kw
        assert dist(fn, N=0) == 0
    assert dist("zs_distill_loss", d_loss=None) == ZS_EINVAL and dist("zs_distill_loss", d_stats=None) == ZS_EINVAL
    assert dist("zs_distill_loss", d_stats=st.data_ptr() + 4) == ZS_EINVAL
    for kw in (dict(d_grad=None), dict(d_row_grad=None), dict(ld_grad=999), dict(d_grad=x.data_ptr() + 2),
               dict(ld_grad=1001)):
        assert dist("zs_distill_grad", **kw) == ZS_EINVAL and dist("zs_distill_loss_grad", **kw) == ZS_EINVAL, kw
    assert dist("zs_distill_grad", d_stats=None) == ZS_EINVAL
    torch.cuda.synchronize()
    assert not x.any() and (st == 7.0).all() and not i32.any()
