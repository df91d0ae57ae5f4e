"""Logits of a head held in 4 bits against the formula in 64 bits; quantising
against the same steps in torch, bit for bit.

Tolerance. In a group, products of x by numbers of at most 31 and 24 are exact
and summed in f32, 2 G additions under partial sums of at most 55 X_g (X_g = sum
|x|): (2 G + 8) 2^-24 55 X_g, times the scale. The groups' sums are then added,
each under the whole's 15 s_g X_g + |min_g| X_g: (groups + 8) 2^-24 of that. f32
states are multiplied as two f16: 2^-22 of 31 s_g X_g more (numbers below 2^-18 of
the row's largest: 2^-40 of that, G times a group)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ctx():
    from tests.gpu_util import ctx
    return ctx()


def parts(V, D, group, mins, seed=0):
    """Codes, scales, minima: codes of every value, scales of every size."""
    gen = torch.Generator("cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (V, D // 2), device="cuda", generator=gen, dtype=torch.int32).to(torch.uint8)
    rand = lambda: torch.randn((V, D // group), device="cuda", generator=gen)
    scales = (0.02 * rand().exp()).half()
    return codes, scales, (0.1 * rand()).half() if mins else None


def weight(codes, scales, mins):
    V, D = codes.shape[0], 2 * codes.shape[1]
    q = torch.stack([codes & 15, codes >> 4], 2).view(V, scales.shape[1], -1).double()
    w = q * scales.double()[:, :, None] + mins.double()[:, :, None] if mins is not None else (q - 8) * scales.double()[:, :, None]
    return w.view(V, D)


def bound(h, scales, mins, group):
    G, n = group, scales.shape[1]
    x = h.double().abs().view(h.shape[0], n, G).sum(2)
    s = scales.double().abs()
    whole = 15 * s + (mins.double().abs() if mins is not None else 0.0)
    wide = h.dtype == torch.float32
    tol = x @ (s * ((2 * G + 8) * 55 * 2.0 ** -24 + (31 * 2.0 ** -22 if wide else 0.0)) + (n + 8) * 2.0 ** -24 * whole).T
    if wide:
        tol += 2.0 ** -40 * h.double().abs().nan_to_num(0.0, 0.0, 0.0).amax(1, keepdim=True) * G * 31 * s.sum(1)
    return tol


def states(B, D, dtype, shift=0, pad=0, seed=1):
    gen = torch.Generator("cuda").manual_seed(seed)
    buf = torch.full((B, shift + D + pad), float("nan"), device="cuda", dtype=TYPES[dtype])
    h = buf[:, shift:shift + D]
    h.copy_(torch.randn((B, D), device="cuda", generator=gen))
    return h


def check(B, V, D, group, mins, dtype, shift=0, pad=0, out=None):
    from zllm_amd.head import Q4Head
    print(f"[case] q4 B={B} V={V} D={D} group={group} mins={mins} {dtype} shift={shift} pad={pad}", flush=True)
    p = parts(V, D, group, mins, seed=V + D)
    h = states(B, D, dtype, shift, pad)
    got = Q4Head(_ctx(), *p).logits(h, out)
    assert got.shape == (B, V) and got.dtype == torch.float32
    d = (got.double() - h.double() @ weight(*p).T).abs()
    tol = bound(h, p[1], p[2], group)
    assert bool((d <= tol).all()), f"{int((~(d <= tol)).sum())} of {d.numel()}, worst {float((d / tol).nan_to_num(1e9).max()):.3g}"
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_groups(group, mins, dtype):
    for B, V, n in ((1, 1, 1), (1, 17, 3), (5, 1000, 4), (16, 515, 9), (17, 64, 33), (33, 300, 2), (64, 130, 5), (65, 2000, 8), (130, 777, 4)):
        check(B, V, n * group, group, mins, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B", [1, 2, 3, 4, 7, 8, 15, 16, 31, 32, 47, 48, 63, 96, 128, 129, 320])
def test_rows(B, dtype):
    check(B, 4099, 256, 32, False, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift,pad", [(0, 8), (1, 2), (8, 0), (3, 5)])
@pytest.mark.parametrize("B", [1, 3, 40])
def test_views(B, shift, pad, dtype):
    check(B, 600, 192, 64, True, dtype, shift, pad)


def test_large():
    check(3, 151936, 4096, 32, False, "bf16")
    check(70, 100003, 1024, 128, True, "f16")
    check(2, 300, 65536, 128, False, "bf16")


def test_rows_past_4_gib_of_logits():
    from zllm_amd.head import Q4Head
    p = parts(1048576, 32, 32, False)
    h = states(1100, 32, "bf16")
    got = Q4Head(_ctx(), *p).logits(h)
    some = [0, 1, 500, 1023, 1024, 1025, 1099]
    d = (got[some].double() - h[some].double() @ weight(*p).T).abs()
    assert bool((d <= bound(h[some], p[1], p[2], 32)).all())


def test_a_head_past_4_gib():
    from zllm_amd.head import Q4Head
    V, D = 300000, 32768
    p = parts(V, D, 128, False)
    h = states(2, D, "bf16")
    got = Q4Head(_ctx(), *p).logits(h)
    some = torch.tensor([0, 1, 131071, 262143, 262144, 299983, 299999], device="cuda")
    q = tuple(t[some] if t is not None else None for t in p)
    d = (got[:, some].double() - h.double() @ weight(*q).T).abs()
    assert bool((d <= bound(h, q[1], None, 128)).all())


def test_out_keeps_what_lies_around_it():
    buf = torch.full((7, 1011), -3.0, device="cuda")
    got = check(5, 1000, 128, 32, False, "bf16", out=buf[1:6, 5:1005])
    assert got.data_ptr() == buf[1:6, 5:1005].data_ptr()
    buf[1:6, 5:1005] = -3.0
    assert bool((buf == -3.0).all())


def test_rows_that_are_not_finite_spoil_only_themselves():
    from zllm_amd.head import Q4Head
    p = parts(500, 128, 32, True)
    for dtype in TYPES:
        h = states(20, 128, dtype)
        head = Q4Head(_ctx(), *p)
        want = head.logits(h)
        h[3, 7], h[18] = float("inf"), float("nan")
        got = head.logits(h)
        keep = [r for r in range(20) if r not in (3, 18)]
        assert torch.equal(got[keep], want[keep]) and not got[[3, 18]].isfinite().any()


def test_no_rows():
    from zllm_amd.head import Q4Head
    assert Q4Head(_ctx(), *parts(50, 64, 32, False)).logits(torch.empty((0, 64), device="cuda")).shape == (0, 50)


# ------------------------------------------------------------------ quantising
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantise(group, mins, dtype):
    from zllm_amd.head import Q4Head, q4_quantize
    V, D = 333, 384
    w = states(V, D, dtype, shift=3, pad=6, seed=5)
    w[0] = 0.0
    w[1] = 1.5
    w[2, :group] = 3.0e-9
    w[3] = torch.arange(D, device="cuda") % 15 - 7.0
    w[4, 5] = 3.0e4
    codes, scales, lows = q4_quantize(_ctx(), w, group, mins)
    x = w.float().view(V, D // group, group)
    if mins:
        lo, hi = x.amin(2, keepdim=True), x.amax(2, keepdim=True)
        s, m = ((hi - lo) / torch.full_like(lo, 15.0)).half(), lo.half()   # (a number would be divided by as * (1 / 15))
        assert torch.equal(lows, m[:, :, 0])
        q = ((x - m.float()) / s.float()).round()
    else:
        top = x.abs().amax(2, keepdim=True)
        s = (top / torch.full_like(top, 7.0)).half()
        q = (x / s.float()).round() + 8
    q = torch.where(s == 0, 0.0 if mins else 8.0, q).clamp(0, 15).view(V, D).to(torch.uint8)
    assert torch.equal(scales, s[:, :, 0]) and torch.equal(codes, q[:, 0::2] | q[:, 1::2] << 4)
    h = states(4, D, "bf16")
    assert torch.equal(Q4Head.quantize(_ctx(), w, group, mins).logits(h), Q4Head(_ctx(), codes, scales, lows).logits(h))
    # a step of the code is as far as rounding goes: half of it, and f16's rounding of scale and minimum
    back = weight(codes, scales, lows).view(V, D // group, group)
    err = (back - x.double()).abs()
    tol = (0.5 + 16 * 2.0 ** -11) * s.double() + (m.double().abs() * 2.0 ** -11 if mins else 0.0) + 2.0 ** -24 * 16
    assert bool((err <= tol).all())


# ------------------------------------------------------------------ how it is called
@pytest.mark.parametrize("temp,top_k", [(0.0, 0), (0.8, 0), (0.7, 40)])
def test_lanes_step_from_hidden_states(temp, top_k):
    """The lanes with a head take hidden states and choose what they choose
    from the head's logits, step for step, as streams come and go."""
    from zllm_amd.engine import LaneBatcher, LaneSeq, SamplingParams
    from zllm_amd.head import Q4Head
    V, D = 5001, 256
    head = Q4Head(_ctx(), *parts(V, D, 64, True))
    runs = []
    for with_head in (True, False):
        lanes = LaneBatcher(_ctx(), head=head if with_head else None)
        for i in range(5):
            lanes.add(LaneSeq(id=i, params=SamplingParams(temp=temp, top_k=top_k, top_p=0.9 if top_k else 1.0), base_seed=7 + i,
                              max_tokens=2 + i, eos=0))
        got, t = [], 0
        while lanes.active:
            h = states(len(lanes.active), D, "bf16", seed=100 + t)
            got.append(lanes.step(h if with_head else head.logits(h)))
            t += 1
        runs.append(got)
    assert runs[0] == runs[1] and len(runs[0]) >= 2


def test_the_loss_and_the_head_in_4_bits_together():
    """A head trained by head_loss_grad, then held in 4 bits: its logits give
    the losses that head_loss gives of the weight they stand for; the sampler
    and the lanes read them."""
    from zllm_amd.engine import LaneBatcher, LaneSeq, SamplingParams
    from zllm_amd.head import Q4Head, head_loss, head_loss_grad, q4_quantize
    N, V, D = 60, 1003, 128
    gen = torch.Generator("cuda").manual_seed(3)
    W = torch.randn((V, D), device="cuda", generator=gen) * D ** -0.5
    h = torch.randn((N, D), device="cuda", generator=gen)
    labels = torch.randint(0, V, (N,), device="cuda", generator=gen)
    g = torch.tensor(1.0 / N, device="cuda")
    for _ in range(3):
        _, dh, dw = head_loss_grad(_ctx(), h, W, labels, g)
        W -= 5.0 * dw
        h -= 5.0 * dh
    p = q4_quantize(_ctx(), W, 32)
    head = Q4Head(_ctx(), *p)
    z = head.logits(h)
    stands = weight(*p).float()
    loss, lse = head_loss(_ctx(), h, stands, labels)
    z64 = h.double() @ weight(*p).T
    want = torch.logsumexp(z64, 1)
    # (logits of either kind are within some 2^-17 of themselves at these sizes: D 2^-24 of sums under 2^5)
    assert float((lse - want).abs().max()) < 2.0 ** -14
    assert float((loss - (want - z64[torch.arange(N, device="cuda"), labels])).abs().max()) < 2.0 ** -13
    lanes = LaneBatcher(_ctx(), head=head)
    for i in range(8):
        lanes.add(LaneSeq(id=i, params=SamplingParams(temp=0.0), base_seed=i, max_tokens=1, eos=-1))
    assert [t for _, t, _ in lanes.step(h[:8])] == z[:8].argmax(1).tolist()


def test_in_a_graph():
    from zllm_amd.head import Q4Head
    for dtype in ("bf16", "f32"):
        head = Q4Head(_ctx(), *parts(3000, 256, 32, False))
        h = states(9, 256, dtype)
        head.logits(h)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = head.logits(h)
        for seed in range(4):
            h.copy_(states(9, 256, dtype, seed=seed))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, head.logits(h))


def test_on_two_streams_at_once():
    from zllm_amd.head import Q4Head
    head = Q4Head(_ctx(), *parts(20000, 512, 64, False))
    hs = [states(3, 512, "f32", seed=1), states(40, 512, "bf16", seed=2)]
    want = [head.logits(h) for h in hs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(head.logits(hs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_refusals():
    from zllm_amd.head import Q4Head, q4_quantize
    c = _ctx()
    codes, scales, mins = parts(50, 128, 32, True)
    for args in ((codes.int(), scales), (codes, scales.float()), (codes, scales[:, :3]), (codes[:, :40], scales),
                 (codes, scales[:49]), (codes, scales, mins[:, :2]), (codes.cpu(), scales), (codes, scales.cpu()), (codes[0], scales),
                 (codes.T.contiguous().T, scales), (codes[:0], scales[:0]), (codes[:, :0], scales)):
        with pytest.raises(ValueError):
            Q4Head(c, *args)
    head = Q4Head(c, codes, scales, mins)
    h = states(3, 128, "bf16")
    for bad in (h[:, :64], h.double(), h.cpu(), h[0], h.T):
        with pytest.raises(ValueError):
            head.logits(bad)
    for out in (torch.empty((3, 49), device="cuda"), torch.empty((3, 50), device="cuda", dtype=torch.bfloat16),
                torch.empty((3, 50)), torch.empty((50, 3), device="cuda").T, torch.empty((1, 50), device="cuda").expand(3, 50)):
        with pytest.raises(ValueError):
            head.logits(h, out)
    w = states(10, 128, "bf16")
    for args in ((w, 16), (w[:, :96], 64), (w.double(), 32), (w.cpu(), 32), (w.T, 32), (w[:0], 32)):
        with pytest.raises(ValueError):
            q4_quantize(c, *args)


def test_writing_in_place_is_known_to_autograd():
    from zllm_amd.head import Q4Head
    head = Q4Head(_ctx(), *parts(50, 64, 32, False))
    x = torch.randn((2, 50), device="cuda", requires_grad=True)
    y = x * 2.0
    z = (y * y).sum()
    head.logits(states(2, 64, "bf16"), out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
