"""Cross entropy of the vocabulary head and its gradients against the formulas
in 64 bits, the gradients against differences too.

Tolerances. With A the row's largest sum of |h_d W_vd| over d, a logit is a sum
of D exact products (f32 operands: of products within 3 * 2^-22, two f16 each)
added in f32: it is within ez = (D + 8) 2^-24 A of itself (f32: D + 20). The normaliser is the logarithm of a sum
of exponentials, each within 2^-21 + ez, added in chains of 64 at most:
el = ez + 2^-17. The loss is normaliser - logit of the label + z_weight * its
square, rounded once: el (1 + 2 z |L|) + ez + 2^-23 |loss|. A gradient of a
logit d = g (k p - [label]) is within |g k p| (2 el + ez + 2 z el / k + 2^-21)
of itself, 16-bit types a rounding of the exponential (2^-11) and of d (EPS)
more and, below f16's normal numbers, 2^-39 of the largest factor. (Exponentials
are kept as f16 of 2^15 e, e <= 1: under 2^-29 in steps of 2^-24 / 2^15, so
within 2^-40, and a factor of at most |g k| takes them to d.) The sums over ids
or rows are of as many f32 additions as terms (f32 states' gradient: of products
within 3 * 2^-22), then rounded to the type."""
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


def rows_at(x, dtype, shift=0, pad=0, fill=float("nan")):
    """x on the GPU, its rows behind `shift` and in front of `pad` other values."""
    R, D = x.shape
    buf = torch.full((R, shift + D + pad), fill, dtype=TYPES[dtype], device="cuda")
    buf[:, shift:shift + D] = torch.as_tensor(x).to(TYPES[dtype]).cuda()
    return buf[:, shift:shift + D]


def inputs(N, V, D, dtype, seed=0, shift=0, pad=0, ignored=0.0, up=6.0, scale=1.0):
    rng = np.random.default_rng(seed)
    W = rng.normal(0, scale / np.sqrt(D), (V, D)).astype(np.float32)
    labels = (rng.random(N) ** 3 * V).astype(np.int64)
    h = (rng.normal(0, 1, (N, D)) + rng.random((N, 1)) * up * W[labels]).astype(np.float32)
    labels[rng.random(N) < ignored] = -100
    g = torch.from_numpy((rng.normal(0, 1, N) / N).astype(np.float32)).cuda()
    return rows_at(h, dtype, shift, pad), rows_at(W, dtype, shift, pad), torch.from_numpy(labels).cuda(), g


def oracle(h, W, labels, g, z, ignore=-100):
    """(loss, lse, dh, dw, and bounds of their errors) in 64 bits on the GPU."""
    dtype = {v: k for k, v in TYPES.items()}[h.dtype]
    D, V, N = h.shape[1], W.shape[0], h.shape[0]
    keep = (labels != ignore).nonzero()[:, 0]
    hd, Wd = h[keep].double(), W.double()
    n = len(keep)
    y = hd @ Wd.T
    A = (hd.abs() @ Wd.abs().T).amax(1) if n else torch.zeros(0, device="cuda", dtype=torch.float64)
    lab = labels[keep]
    L = torch.logsumexp(y, 1) if n else A
    rows = torch.arange(n, device="cuda")
    yl = y[rows, lab] if n else A
    loss, lse = (torch.zeros(N, dtype=torch.float64, device="cuda") for _ in range(2))
    tl, te = torch.zeros_like(loss), torch.zeros_like(loss)
    loss[keep], lse[keep] = L - yl + z * L * L, L
    wide = 12 if dtype == "f32" else 0           # (3 * 2^-22, in 2^-24)
    ez = (D + 8 + wide) * 2.0 ** -24 * A
    el = ez + 2.0 ** -17
    tl[keep] = el * (1 + 2 * z * L.abs()) + ez + 2.0 ** -23 * loss[keep].abs()
    te[keep] = el + 2.0 ** -23 * L.abs()
    gg = g.double().expand(N)[keep][:, None]
    k = 1 + 2 * z * L[:, None]
    p = (y - L[:, None]).exp()
    d = gg * k * p
    rel = 2 * el + ez + 2 * z * el / k[:, 0].abs().clamp_min(1e-9) + 2.0 ** -21
    e = d.abs() * (rel[:, None] + (2.0 ** -11 if dtype != "f32" else 0.0))
    if dtype != "f32":
        e += 2.0 ** -40 * (gg * k).abs()
    d[rows, lab] -= gg[:, 0]
    e += d.abs() * EPS[dtype]
    if dtype == "f16" and n:
        e += 2.0 ** -39 * (gg.abs() * k.abs().clamp_min(1.0)).max()
    dh, th = torch.zeros((N, D), dtype=torch.float64, device="cuda"), torch.zeros((N, D), dtype=torch.float64, device="cuda")
    dh[keep] = d @ Wd
    th[keep] = e @ Wd.abs() + (V + wide) * 2.0 ** -24 * (d.abs() @ Wd.abs())
    dw = d.T @ hd
    tw = e.T @ hd.abs() + n * 2.0 ** -24 * (d.abs().T @ hd.abs())
    th += EPS[dtype] * dh.abs() + TINY[dtype]
    tw += EPS[dtype] * dw.abs() + TINY[dtype]
    return loss, lse, dh, dw, tl, te, th, tw


def near(got, want, tol, what):
    d = (got.double() - want).abs()
    assert got.shape == want.shape and bool((d <= tol).all()), \
        f"{what}: {int((~(d <= tol)).sum())} of {d.numel()}, worst {float((d / tol.clamp_min(1e-300)).nan_to_num(1e9).max()):.3g} of the bound"


def check(h, W, labels, g, z=0.0, what="", **needs):
    from zllm_amd.head import HeadLossConfig, head_loss, head_loss_grad
    print(f"[case] {what} N={h.shape[0]} V={W.shape[0]} D={h.shape[1]} {h.dtype} z={z} {h.stride()} {W.stride()}", flush=True)
    cfg = HeadLossConfig(z_weight=z)
    loss, lse, dh, dw, tl, te, th, tw = oracle(h, W, labels, g, z)
    a, b = head_loss(_ctx(), h, W, labels, cfg)
    near(a, loss, tl, "loss")
    near(b, lse, te, "lse")
    l2, gh, gw = head_loss_grad(_ctx(), h, W, labels, g, cfg, **needs)
    near(l2, loss, tl, "loss of the step")
    if gh is not None:
        assert gh.dtype == h.dtype
        near(gh, dh, th, "dhidden")
    if gw is not None:
        assert gw.dtype == h.dtype
        near(gw, dw, tw, "dweight")
    return l2, gh, gw


# ------------------------------------------------------------------ sizes
SIZES = [(1, 1, 1), (3, 5, 7), (1, 256, 32), (2, 130, 8), (5, 1000, 64), (257, 300, 136), (40, 4099, 200), (300, 515, 1001),
         (64, 20000, 96), (130, 2049, 520), (513, 8200, 256)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,V,D", SIZES)
def test_sizes(N, V, D, dtype):
    check(*inputs(N, V, D, dtype, seed=N + V + D), what="sizes")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 72, 99])
@pytest.mark.parametrize("shift,pad", [(0, 8), (1, 2), (8, 0), (3, 5), (8, 24)])
def test_views(shift, pad, D, dtype):
    """Rows of longer rows whose other values are NaN, at any element."""
    check(*inputs(77, 600, D, dtype, seed=D + shift, shift=shift, pad=pad), z=1e-3, what="views")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_large_vocabulary(dtype):
    check(*inputs(33, 151936, 128, dtype, seed=1), what="vocabulary")


def test_many_hidden():
    check(*inputs(9, 300, 9000, "bf16", seed=2), what="hidden")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_in_pieces(dtype):
    """More rows than a piece of either call holds."""
    check(*inputs(66000, 200, 24, dtype, seed=3, ignored=0.3), z=1e-3, what="pieces")


def test_rows_behind_the_last_label():
    """Pieces of which the device finds out that they are empty."""
    h, W, labels, g = inputs(66000, 200, 24, "bf16", seed=4)
    labels[100:] = -100
    check(h, W, labels, g, what="empty pieces")


# ------------------------------------------------------------------ rows that go wrong in their own ways
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("share", [0.1, 0.5, 0.99, 1.0])
def test_ignored_rows(share, dtype):
    h, W, labels, g = inputs(300, 700, 80, dtype, seed=5, ignored=share)
    h[labels == -100] = float("nan")
    h[(labels == -100).nonzero()[:1, 0]] = float("inf")
    g[labels == -100] = float("nan")
    _, gh, _ = check(h, W, labels, g, what="ignored")
    assert bool((gh[labels == -100] == 0).all())


def test_another_ignore_index():
    from zllm_amd.head import HeadLossConfig, head_loss_grad
    h, W, labels, g = inputs(50, 300, 64, "bf16", seed=6)
    labels[::3] = 7
    want = oracle(h, W, labels, g, 0.0, ignore=7)
    loss, gh, gw = head_loss_grad(_ctx(), h, W, labels, g, HeadLossConfig(ignore_index=7))
    near(loss, want[0], want[4], "loss")
    near(gh, want[2], want[6], "dhidden")
    near(gw, want[3], want[7], "dweight")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_labels_outside_give_nan(dtype):
    from zllm_amd.head import head_loss, head_loss_grad
    h, W, labels, g = inputs(40, 300, 64, dtype, seed=7)
    labels[3], labels[9] = 300, -1
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[3] = bad[9] = True
    loss, lse = head_loss(_ctx(), h, W, labels)
    assert bool((loss.isnan() == bad).all()) and bool(lse.isfinite().all())
    loss, gh, gw = head_loss_grad(_ctx(), h, W, labels, g)
    assert bool((loss.isnan() == bad).all()) and bool((gh.isnan() == bad[:, None]).all()) and bool(gw.isnan().all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_values_that_are_not_finite(dtype):
    """A row of NaN or of infinities spoils its own loss and gradient, and the weight's."""
    from zllm_amd.head import head_loss_grad
    h, W, labels, g = inputs(40, 300, 64, dtype, seed=8)
    h[3], h[9, 5] = float("nan"), float("inf")
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[3] = bad[9] = True
    loss, gh, gw = head_loss_grad(_ctx(), h, W, labels, g)
    assert bool((loss.isfinite() != bad).all())
    assert bool((gh.isfinite().all(1) != bad).all())
    want = oracle(h[~bad], W, labels[~bad], g[~bad], 0.0)
    near(loss[~bad], want[0], want[4], "loss")
    near(gh[~bad], want[2], want[6], "dhidden")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_far_logits(dtype):
    """Rows whose logits lie hundreds apart, the label first, last or between."""
    h, W, labels, g = inputs(64, 900, 64, dtype, seed=9, scale=30.0, up=0.0)
    y = h.float() @ W.float().T
    labels[:20] = y[:20].argmax(1)
    labels[20:40] = y[20:40].argmin(1)
    check(h, W, labels, g, what="far")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_equal_logits(dtype):
    h, W, labels, g = inputs(20, 1030, 64, dtype, seed=10)
    h[:10] = 0.0
    W[:] = W[:1].clone()
    check(h, W, labels, g, what="equal")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 3e4])
def test_sizes_of_the_rows_weights(size, dtype):
    """Row weights that f16 cannot hold, one far above the others, zeros."""
    h, W, labels, g = inputs(60, 700, 64, dtype, seed=11)
    g = g / g.abs().max()
    g[:30] *= 1e-3
    g[5] = 0.0
    check(h, W, labels, g * size if dtype == "bf16" or size < 1e4 else g * 100.0, z=0.01, what=f"weights {size}")


def test_one_weight_for_all_rows():
    h, W, labels, _ = inputs(60, 700, 64, "bf16", seed=12)
    check(h, W, labels, torch.tensor(1 / 60, device="cuda"), what="scalar")
    check(h, W, labels, torch.tensor([1 / 60], device="cuda").expand(60), what="expanded")
    check(h, W, labels, torch.rand(120, device="cuda")[::2], what="strided")


@pytest.mark.parametrize("z", [1e-4, 0.5, -0.1])
def test_z_weight(z):
    check(*inputs(60, 700, 64, "f32", seed=13), z=z, what="z")
    check(*inputs(60, 700, 64, "f16", seed=13), z=z, what="z")


def test_one_gradient_alone():
    args = inputs(60, 700, 64, "bf16", seed=14)
    both = check(*args)
    assert torch.equal(check(*args, need_weight=False)[1], both[1])
    assert torch.equal(check(*args, need_hidden=False)[2], both[2])


@pytest.mark.parametrize("D,shift,pad", [(96, 0, 0), (100, 4, 4), (100, 1, 3), (97, 0, 0), (1, 0, 0), (3, 2, 0), (1030, 0, 2)])
@pytest.mark.parametrize("N", [1, 64, 65, 129, 192, 193])
def test_f32_rows_where_the_way_changes(N, D, shift, pad):
    """A few rows take an f32 weight as it lies, by 16 bytes or number by number, more
    of them a copy."""
    check(*inputs(N, 1101, D, "f32", seed=N + D, shift=shift, pad=pad, ignored=0.1 if N > 1 else 0.0), what="f32 rows")


@pytest.mark.parametrize("D", [64, 70])
def test_one_gradient_of_few_f32_rows(D):
    args = inputs(70, 700, D, "f32", seed=D)
    both = check(*args)
    assert torch.equal(check(*args, need_weight=False)[1], both[1])
    assert torch.equal(check(*args, need_hidden=False)[2], both[2])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("N", [63, 65, 127, 128, 129])
def test_rows_where_the_tiles_change(N, dtype):
    check(*inputs(N, 2000, 136, dtype, seed=N), what="tiles")


@pytest.mark.parametrize("N", [5, 100, 300])
def test_f32_rows_far_apart(N):
    """Further than the products' offsets reach: copied whatever the rows' number."""
    h, W, labels, g = inputs(N, 6, 64, "f32", seed=N)
    buf = torch.full((6, 5_000_000), float("nan"), device="cuda")
    buf[:, 100:164] = W
    check(h, buf[:, 100:164], labels, g, what="far f32 weight")


def test_same_results_every_time():
    args = inputs(700, 5000, 256, "bf16", seed=15, ignored=0.2)
    from zllm_amd.head import head_loss_grad
    first = head_loss_grad(_ctx(), *args)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, head_loss_grad(_ctx(), *args)))


def test_rows_far_apart():
    """Rows past 4 GiB, of the states and of the weight."""
    h, W, labels, g = inputs(3, 5, 64, "bf16", seed=16)
    buf = torch.empty((3, 1_200_000_000), dtype=torch.bfloat16, device="cuda")
    buf[:, -64:] = h
    check(buf[:, -64:], W, labels, g, what="far states")
    del buf
    buf = torch.empty((5, 1_200_000_000), dtype=torch.bfloat16, device="cuda")
    buf[:, -64:] = W
    check(h, buf[:, -64:], labels, g, what="far weight")


def test_a_weight_past_4_gib():
    """262144 rows of 8200 columns; checked at some of them."""
    from zllm_amd.head import head_loss_grad
    V, D, N = 262144, 8200, 20
    W = torch.empty((V, D), dtype=torch.bfloat16, device="cuda").normal_(0, D ** -0.5, generator=torch.Generator("cuda").manual_seed(1))
    labels = torch.randint(0, V, (N,), device="cuda")
    labels[0] = V - 1
    h = (torch.randn((N, D), device="cuda") + 6 * W[labels].float()).bfloat16()
    g = torch.full((N,), 0.05, device="cuda")
    loss, gh, gw = head_loss_grad(_ctx(), h, W, labels, g)
    y = torch.cat([h.double() @ w.double().T for w in W.split(16384)], 1)
    L = torch.logsumexp(y, 1)
    rows = torch.arange(N, device="cuda")
    assert float((loss - (L - y[rows, labels])).abs().max()) < 1e-4
    d = 0.05 * (y - L[:, None]).exp()
    d[rows, labels] -= 0.05
    want = sum(d[:, i:i + 16384] @ W[i:i + 16384].double() for i in range(0, V, 16384))
    assert float((gh.double() - want).norm() / want.norm()) < 0.01     # (three bf16 roundings)
    some = torch.cat([labels, torch.tensor([0, 1, 255, 256, 131071, 262143], device="cuda")])
    want = d[:, some].T @ h.double()
    assert bool(((gw[some].double() - want).norm(dim=1) <= 0.01 * want.norm(dim=1)).all())


# ------------------------------------------------------------------ how it is called
def test_no_rows():
    from zllm_amd.head import head_loss, head_loss_grad
    W = torch.randn((40, 16), device="cuda", dtype=torch.bfloat16)
    h, labels = W[:0], torch.empty(0, dtype=torch.int64, device="cuda")
    assert head_loss(_ctx(), h, W, labels)[0].shape == (0,)
    loss, gh, gw = head_loss_grad(_ctx(), h, W, labels, torch.empty(0, device="cuda"))
    assert loss.shape == (0,) and gh.shape == (0, 16) and bool((gw == 0).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_autograd(dtype):
    from zllm_amd.head import HeadLoss, HeadLossConfig
    h, W, labels, _ = inputs(50, 900, 72, dtype, seed=17, ignored=0.2)
    for need in ((True, True), (True, False), (False, True)):
        a, b = h.detach().clone().requires_grad_(need[0]), W.detach().clone().requires_grad_(need[1])
        loss = HeadLoss(_ctx(), HeadLossConfig(z_weight=1e-3))(a, b, labels)
        loss.mean().backward()
        want = oracle(h, W, labels, torch.full((50,), 1 / 50, device="cuda"), 1e-3)
        near(loss.detach(), want[0], want[4], "loss")
        if need[0]:
            near(a.grad, want[2], want[6], "dhidden")
        if need[1]:
            near(b.grad, want[3], want[7], "dweight")


def test_gradients_against_differences():
    from zllm_amd.head import HeadLossConfig, head_loss, head_loss_grad
    h, W, labels, g = inputs(6, 40, 16, "f32", seed=18)
    cfg = HeadLossConfig(z_weight=0.01)
    _, gh, gw = head_loss_grad(_ctx(), h, W, labels, g, cfg)
    gen = torch.Generator("cuda").manual_seed(1)
    for x, grad in ((h, gh), (W, gw)):
        for _ in range(5):
            u = torch.randn(x.shape, device="cuda", generator=gen)
            f = []
            for step in (1e-2, -1e-2):
                args = (h + step * u, W) if x is h else (h, W + step * u)
                f.append(float((head_loss(_ctx(), *args, labels, cfg)[0].double() * g).sum()))
            # differences of a smooth function: error of the third order, and of the losses' rounding over the step
            assert abs((f[0] - f[1]) / 2e-2 - float((grad.double() * u).sum())) < 1e-3


def test_in_a_graph_beside_eager_calls():
    """A captured step replayed, inputs changed between, eager work beside it."""
    from zllm_amd.head import head_loss_grad
    args = inputs(130, 3000, 128, "bf16", seed=19, ignored=0.1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        head_loss_grad(_ctx(), *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = head_loss_grad(_ctx(), *args)
    for seed in range(4):
        for x, y in zip(args, inputs(130, 3000, 128, "bf16", seed=20 + seed, ignored=0.3 * seed)):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        want = head_loss_grad(_ctx(), *args)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_on_two_streams_at_once():
    from zllm_amd.head import head_loss_grad
    cases = [inputs(200, 4000, 128, "bf16", seed=30), inputs(333, 1500, 96, "f16", seed=31)]
    want = [head_loss_grad(_ctx(), *c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(head_loss_grad(_ctx(), *cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for g in got[i] for x, y in zip(g, want[i]))


def test_refusals():
    from zllm_amd.head import HeadLossConfig, head_loss, head_loss_grad
    c = _ctx()
    h, W, labels, g = inputs(10, 50, 16, "bf16", seed=40)
    for args in ((h.float(), W, labels), (h, W[:, :8], labels), (h[0], W, labels), (h, W, labels[:9]), (h, W, labels.int()),
                 (h.cpu(), W, labels), (h, W.cpu(), labels), (h, W, labels.cpu()), (h.T, W, labels), (h.double(), W.double(), labels),
                 (h, W[:0], labels), (h[:, :0], W[:, :0], labels), (h, W[:1].expand(50, 16), labels)):
        with pytest.raises(ValueError):
            head_loss(c, *args)
        with pytest.raises(ValueError):
            head_loss_grad(c, *args, g)
    for rg in (g[:9], g.double(), g.cpu(), g[:, None]):
        with pytest.raises(ValueError):
            head_loss_grad(c, h, W, labels, rg)
    with pytest.raises(ValueError):
        head_loss_grad(c, h, W, labels, g, need_hidden=False, need_weight=False)
    from zllm_amd._lib import ZsError
    with pytest.raises(ZsError, match="z_weight"):
        head_loss(c, h, W, labels, HeadLossConfig(z_weight=float("nan")))
