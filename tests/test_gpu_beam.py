"""Beam search: zs_beam_select against the definition evaluated in 64 bits
candidate by candidate, zs_beam_reorder against indexing (bit for bit).

Scores: the sum of exponentials is of f32 terms, each within 2^-22 of its
exact value for the differences that matter (the argument's rounding and the
hardware exponential's) and added in chains of at most V / 256 + 64 terms, so
ln of it is within (V / 256 + 64) 2^-23; the score is rounded to f32 once."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

NINF = -np.inf
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ctx():
    from tests.gpu_util import ctx
    return ctx()


def lse_tol(V):
    return (V / 256 + 64) * 2.0 ** -23


def rows_at(x, dtype, shift, pad):
    """x [R, V] on the GPU in `dtype`, rows beginning `shift` elements into a
    wider allocation whose other elements are NaN."""
    R, V = x.shape
    buf = torch.full((R, shift + V + pad), float("nan"), dtype=TYPES[dtype], device="cuda")
    buf[:, shift:shift + V] = torch.from_numpy(x).to(TYPES[dtype]).cuda()
    return buf[:, shift:shift + V]


def clean(x):
    """float64 values as the definition sees them."""
    x = np.where(np.isnan(x), NINF, x)
    return np.minimum(x, np.finfo(np.float32).max)


def ref_select(x, scores, pool, W, eos, alpha, early, allow=None):
    """The step in 64 bits; x [R, V] float64, pool: dict of arrays. Scores are
    rounded to f32 before they are compared, as the definition has it."""
    G = scores.shape[0]
    out = {k: v.copy() for k, v in pool.items()}
    par = np.full((G, W), -1, np.int64)
    tok = np.full((G, W), -1, np.int64)
    sco = np.full((G, W), NINF)
    V = x.shape[1]
    for g in range(G):
        if pool["done"][g]:
            continue
        cand = []
        for b in range(W):
            s = scores[g, b]
            if not np.isfinite(s):
                continue
            row = clean(x[g * W + b])
            if allow is not None:
                row = np.where(allow[g * W + b], row, NINF)
            m = row.max()
            if m == NINF:
                continue
            lns = np.log(np.exp(row - m).sum())
            order = np.lexsort((np.arange(V), -row))[:W + len(eos)]
            for v in order:
                if row[v] == NINF:
                    continue
                f = np.float32(float(s) + ((row[v] - m) - lns))
                if f > NINF:
                    cand.append((-f, b, -row[v], v))
        cand.sort()
        norm = float(pool["steps"][g] + 1) ** alpha
        fin = [(out["score"][g, i], out["length"][g, i], out["parent"][g, i], out["token"][g, i])
               for i in range(W) if out["score"][g, i] > NINF]
        n = 0
        for rank, (f, b, _, v) in enumerate(cand):
            if n == W:
                break
            if v in eos:
                if rank < W:
                    e = (np.float32(float(-f) / norm), pool["steps"][g] + 1, b, v)
                    i = sum(1 for o in fin if o[0] >= e[0])
                    fin.insert(i, e)
            else:
                par[g, n], tok[g, n], sco[g, n] = b, v, -f
                n += 1
        fin = fin[:W]
        for i in range(W):
            e = fin[i] if i < len(fin) else (NINF, 0, -1, -1)
            out["score"][g, i], out["length"][g, i], out["parent"][g, i], out["token"][g, i] = e
        out["steps"][g] += 1
        full = len(fin) == W
        out["done"][g] = int(n == 0 or (full and (early or fin[-1][0] >= np.float32(float(sco[g, 0]) / norm))))
    return par, tok, sco, out


def empty_pool(G, W):
    return dict(score=np.full((G, W), NINF), length=np.zeros((G, W), np.int64), parent=np.full((G, W), -1),
                token=np.full((G, W), -1), steps=np.zeros(G, np.int64), done=np.zeros(G, np.int64))


def to_pool(p):
    from zllm_amd.beam import BeamPool
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()
    return BeamPool(torch.from_numpy(p["score"]).float().cuda(), *(i(p[k]) for k in
                    ("length", "parent", "token", "steps", "done")))


def check(xt, scores, pool, W, eos=(), alpha=1.0, early=False, allow=None, bits=None, what=""):
    from zllm_amd.beam import beam_select
    G = scores.shape[0]
    print(f"[case] beam_select {what} G={G} W={W} V={xt.shape[1]} {xt.dtype} ld={xt.stride(0)}", flush=True)
    o = beam_select(_ctx(), xt, torch.from_numpy(scores).float().cuda(), to_pool(pool), eos, alpha, early, bits)
    torch.cuda.synchronize()
    par, tok, sco, ref = ref_select(xt.double().cpu().numpy(), scores.astype(np.float32), pool, W, set(eos), alpha,
                                    early, allow)
    assert o.parents.cpu().numpy().tolist() == par.tolist()
    assert o.tokens.cpu().numpy().tolist() == tok.tolist()
    tol = lse_tol(xt.shape[1])
    for got, want in ((o.scores, sco), (o.pool.score, ref["score"])):
        got = got.double().cpu().numpy()
        assert (np.isneginf(got) == np.isneginf(want)).all()
        f = np.isfinite(want)
        assert (np.abs(got[f] - want[f]) <= tol + np.abs(want[f]) * 2.0 ** -22).all(), np.abs(got[f] - want[f]).max()
    for k in ("length", "parent", "token", "steps", "done"):
        assert getattr(o.pool, k).cpu().numpy().tolist() == ref[k].tolist(), k
    return o


def beams(rng, G, W, live=None):
    s = -np.cumsum(rng.exponential(0.5, (G, W)), 1) - 3.0
    if live is not None:
        s[:, live:] = NINF
    return s.astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,W,V", [(1, 1, 1), (2, 1, 7), (3, 4, 50), (1, 32, 257), (5, 3, 4099), (2, 8, 50257),
                                   (2, 4, 163841)])
def test_sizes_and_types(G, W, V, dtype):
    rng = np.random.default_rng(G * 1000 + W + V)
    for shift, pad in ((0, 0), (1, 2), (5, 6)):
        x = rng.normal(0, 2, (G * W, V)).astype(np.float32)
        xt = rows_at(x, dtype, shift, pad)
        check(xt, beams(rng, G, W), empty_pool(G, W), W, eos=(0,), what=f"shift={shift}")


def test_ties_between_beams_and_ids():
    """Equal rows and scores: the lower beam first, then the lower id; -0 and
    +0 are one value; a run of equal logits longer than any list."""
    G, W, V = 2, 4, 3001
    x = np.full((G * W, V), -4.0, np.float32)
    x[:, 2000:2600] = 1.5
    x[4:, 17] = 0.0
    x[4:, 16] = -0.0
    x[4:, 2000:2600] = -3.0
    scores = np.zeros((G, W), np.float32)
    for dtype in TYPES:
        o = check(rows_at(x, dtype, 3, 0), scores, empty_pool(G, W), W, what="ties")
        assert o.parents[0].tolist() == [0] * 4 and o.tokens[0].tolist() == [2000, 2001, 2002, 2003]
        assert o.parents[1].tolist() == [0, 0, 1, 1] and o.tokens[1].tolist() == [16, 17, 16, 17]


@pytest.mark.parametrize("W,eos", [(11, ()), (13, (1,)), (32, ()), (32, tuple(range(8)))])
def test_wide_beams_of_every_shape(W, eos):
    """Many candidates at one score (more than are placed at once), a beam that
    has all of the next ones, beams of a few candidates each, whole numbers,
    EOS ids first in every beam."""
    rng = np.random.default_rng(W + len(eos))
    G, V = 7, 900
    x = rng.normal(0, 2, (G, W, V)).astype(np.float32)
    s = beams(rng, G, W)
    x[0], s[0] = -1.0, 0.0
    x[1], s[1] = np.round(rng.normal(0, 1, (1, V))), -2.0
    s[2, 1:] -= 200.0
    s[3, : W - 1] -= 200.0
    x[4] = -np.inf
    x[4, :, 5:8] = rng.normal(0, 1, (W, 3))
    x[5, :, :8] += 9.0
    x[6, ::2], s[6, 1::2] = -np.inf, -1.0
    for dtype in ("f32", "bf16"):
        check(rows_at(x.reshape(G * W, V), dtype, 1, 0), s, empty_pool(G, W), W, eos, what="wide")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_values_that_are_no_numbers(dtype):
    """NaN and -inf are no candidates and have no mass, +inf is the largest
    number; rows of nothing; one id left."""
    rng = np.random.default_rng(3)
    G, W, V = 3, 3, 1000
    x = rng.normal(0, 1, (G * W, V)).astype(np.float32)
    x[0, ::3] = np.nan
    x[1] = -np.inf
    x[2, 5] = np.inf
    x[3] = np.nan
    x[4] = -np.inf
    x[4, 999] = -700.0
    x[5, [7, 900]] = np.inf
    x[6:9] = -np.inf
    o = check(rows_at(x, dtype, 1, 1), beams(rng, G, W), empty_pool(G, W), W, eos=(4,), what="no numbers")
    assert o.parents[2].tolist() == [-1] * 3 and o.pool.done.tolist() == [0, 0, 1]
    assert torch.isneginf(o.scores[2]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [300, 9001])
def test_rows_of_huge_values(V, dtype):
    """Rows that are all at a mask's finite value (any from -1e9 to the type's
    lowest) are even ones; equal values at the top of huge ones share."""
    rng = np.random.default_rng(V)
    G, W = 3, 4
    x = np.empty((G * W, V), np.float32)
    for r, v in enumerate((-1e9, -1e10, -1e30, -3.3e38, 1e10, 1e30, 3.3e38, -5e9)):
        x[r] = v
    x[3] = torch.finfo(TYPES[dtype]).min
    x[7, 40] = 2.0
    x[8] = -1e30
    x[8, 10:15] = rng.normal(0, 1, 5)
    x[9] = 5e29
    x[9, [3, 77, V - 1]] = 1e30
    x[10] = 3e12 + 1e11 * rng.normal(0, 1, V)
    x[11] = rng.normal(0, 1, V)
    check(rows_at(x, dtype, 1, 2), beams(rng, G, W), empty_pool(G, W), W, (4,), what="huge")


def test_beams_that_do_not_live():
    """Beams of score -inf, NaN or +inf are not read (their rows here would
    win); requests that are done stay as they are."""
    rng = np.random.default_rng(4)
    G, W, V = 4, 4, 777
    x = rng.normal(0, 1, (G * W, V)).astype(np.float32)
    s = beams(rng, G, W, live=1)
    s[1, 2], s[1, 3] = np.nan, np.inf
    s[3] = -np.inf
    pool = empty_pool(G, W)
    pool["done"][2] = 1
    pool["score"][2, :2], pool["length"][2, :2], pool["parent"][2, :2], pool["token"][2, :2] = [-1, -2], 3, 1, 9
    pool["steps"][:] = [0, 4, 7, 2]
    o = check(rows_at(x, "f32", 0, 0), s, pool, W, eos=(9,), what="dead beams")
    assert o.pool.done.tolist() == [0, 0, 1, 1] and o.pool.steps.tolist() == [1, 5, 7, 3]


@pytest.mark.parametrize("early", [False, True])
@pytest.mark.parametrize("alpha", [0.0, 0.7, 2.0, -1.0])
def test_eos_and_pool(alpha, early):
    """EOS ids in front of, among and behind the first `width`, several of
    them, pools empty, part full and full, equal pool scores."""
    rng = np.random.default_rng(int(alpha * 10) + early + 50)
    G, W, V = 8, 4, 300
    eos = (5, 11, 250, 4000)
    x = rng.normal(0, 1, (G * W, V)).astype(np.float32)
    x[0:4, 5] = 9.0                        # every beam ends first
    x[4:8, [5, 11, 250]] = [8.0, 7.5, 7.0]   # several ends a beam
    x[8, 11] = 12.0
    x[12:16, 250] = 2.0                    # among the others
    x[16:20, 5] = -9.0                     # far behind
    x[20, 5] = 9.0
    pool = empty_pool(G, W)
    pool["steps"][:] = rng.integers(0, 40, G)
    for g, n in ((1, 4), (2, 2), (3, 3), (4, 4), (6, 4)):
        v = -np.sort(rng.uniform(0.1, 6.0, n))
        v[1] = v[0]
        pool["score"][g, :n] = v.astype(np.float32)
        pool["length"][g, :n] = rng.integers(1, 40, n)
        pool["parent"][g, :n] = rng.integers(0, W, n)
        pool["token"][g, :n] = 5
    pool["score"][6, :4] = -1000.0
    check(rows_at(x, "f32", 0, 0), beams(rng, G, W), pool, W, eos, alpha, early, what=f"eos alpha={alpha}")


def test_wide_beams_all_ending():
    rng = np.random.default_rng(8)
    G, W, V = 2, 32, 2000
    eos = tuple(range(100, 108))
    x = rng.normal(0, 1, (G * W, V)).astype(np.float32)
    x[:, 100:108] += 8.0
    pool = empty_pool(G, W)
    check(rows_at(x, "f32", 0, 0), beams(rng, G, W) * 3, pool, W, eos, 1.0, what="all end")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [31, 64, 1003, 40007])
def test_masks(V, dtype):
    """Masked ids may hold anything; bits past V are set; a row whose mask
    leaves nothing, one id, everything."""
    rng = np.random.default_rng(V)
    G, W = 3, 2
    R = G * W
    words = (V + 31) // 32 + 1
    allow = rng.random((R, words * 32)) < 0.3
    allow[0] = False
    allow[1] = False
    allow[1, V - 1] = True
    allow[2] = True
    allow[:, V:] = True
    x = rng.normal(0, 2, (R, V)).astype(np.float32)
    bad = ~allow[:, :V]
    x[bad] = rng.choice(np.array([np.nan, np.inf, 60.0, -np.inf], np.float32), bad.sum())
    bits = np.packbits(allow, axis=1, bitorder="little").view(np.int32)
    for shift in (0, 1, 3):
        check(rows_at(x, dtype, shift, 2), beams(rng, G, W), empty_pool(G, W), W, (1,), allow=allow[:, :V],
              bits=torch.from_numpy(bits).cuda(), what=f"mask shift={shift}")


def test_a_group_in_two_launches():
    """A launch ends inside a request's rows (2^22 workgroups, five a row): the
    requests on both sides come out as in a call of their own; the others are
    done and not read (68 GB, most of it never written)."""
    from zllm_amd.beam import BeamPool, beam_select
    W, V = 32, 32800
    G = (1 << 20) // W
    mid = (1 << 22) // 5 // W
    assert (1 << 22) // 5 % W
    x = torch.empty((G * W, V), dtype=torch.bfloat16, device="cuda")
    near = slice((mid - 1) * W, (mid + 2) * W)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x[near] = torch.randn((3 * W, V), device="cuda", generator=gen).to(torch.bfloat16)
    scores = torch.randn((G, W), device="cuda", generator=gen).sub_(5.0)
    pool = BeamPool.empty(G, W)
    pool.done.fill_(1)
    pool.done[mid - 1:mid + 2] = 0
    print("[case] beam_select a group in two launches", flush=True)
    o = beam_select(_ctx(), x, scores, pool, (3,))
    a = beam_select(_ctx(), x[near], scores[mid - 1:mid + 2].contiguous(), BeamPool.empty(3, W), (3,))
    for k in ("parents", "tokens", "scores"):
        assert torch.equal(getattr(o, k)[mid - 1:mid + 2], getattr(a, k)), k
    assert (a.parents >= 0).all() and (o.parents[:mid - 1] == -1).all() and (o.parents[mid + 2:] == -1).all()
    assert o.pool.steps.sum() == 3


def test_in_place_and_other_streams():
    """Outputs that are the inputs themselves; work queued on a stream of its own."""
    from zllm_amd.beam import BeamStep, beam_select
    rng = np.random.default_rng(9)
    G, W, V = 6, 4, 5000
    x = rows_at(rng.normal(0, 2, (G * W, V)).astype(np.float32), "bf16", 0, 0)
    s = torch.from_numpy(beams(rng, G, W)).cuda()
    a = beam_select(_ctx(), x, s, to_pool(empty_pool(G, W)), (3,))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pool = to_pool(empty_pool(G, W))
        s2 = s.clone()
        b = beam_select(_ctx(), x, s2, pool, (3,), out=BeamStep(torch.empty_like(a.parents), torch.empty_like(a.tokens),
                                                                s2, pool))
    side.synchronize()
    torch.cuda.synchronize()
    assert b.scores.data_ptr() == s2.data_ptr()
    for k in ("parents", "tokens", "scores"):
        assert torch.equal(getattr(a, k), getattr(b, k)), k
    for k in ("score", "length", "parent", "token", "steps", "done"):
        assert torch.equal(getattr(a.pool, k), getattr(b.pool, k)), k


def test_search_finds_what_enumeration_finds():
    """A first-order model over 6 ids searched with beams as wide as its
    states: the best sequence of all."""
    from zllm_amd.beam import BeamSearch, BeamStates, beam_reorder
    rng = np.random.default_rng(12)
    V, W, steps, eos = 6, 6, 5, 0
    T = rng.normal(0, 2, (V, V)).astype(np.float32)
    lp = T.astype(np.float64) - np.log(np.exp(T.astype(np.float64)).sum(1, keepdims=True))
    search = BeamSearch(_ctx(), 2, W, steps, eos=(eos,), length_penalty=1.0)
    seen = torch.zeros((2 * W, steps), dtype=torch.int32, device="cuda")     # the beams' own histories
    states = BeamStates([(seen, 0)], W)
    last = torch.tensor([1] * W + [2] * W, device="cuda")
    table = torch.from_numpy(T).cuda()
    t = 0
    while not search.finished():
        search.step(table[last])
        beam_reorder(_ctx(), states, search.parents)
        seen[:, t] = search.tokens.view(-1)
        last = search.tokens.view(-1).clamp_min(0).long()
        t += 1
    for g, start in ((0, 1), (1, 2)):
        best = (NINF, None)
        stack = [(start, 0.0, [])]
        while stack:
            cur, s, toks = stack.pop()
            for v in range(V):
                n, q = toks + [v], s + lp[cur, v]
                if v == eos or len(n) == steps:
                    best = max(best, (q / len(n), n))
                if v != eos and len(n) < steps:
                    stack.append((v, q, n))
        got = search.sequences()[g][0]
        assert got.tokens == best[1] and abs(got.score - best[0]) < 1e-5
    # histories that followed the parents are the traced ones
    live = {tuple(h.tokens) for g in range(2) for h in search.sequences()[g] if not h.finished}
    if live:
        assert live <= {tuple(r[:t].tolist()) for r in seen.cpu()}


# ------------------------------------------------------------------ reordering
def ref_reorder(t, d, parents, W):
    p = parents.cpu().numpy()
    idx = np.arange(p.size)
    for r in range(p.size):
        q = p[r // W, r % W]
        if 0 <= q < W:
            idx[r] = r // W * W + q
    return t.index_select(d, torch.from_numpy(idx).to(t.device))


@pytest.mark.parametrize("W", [1, 2, 3, 4, 7, 8, 13, 16, 31, 32])
def test_reorder_layouts(W):
    """Caches with rows outside, inside and last, live prefixes, odd bytes,
    single bytes, scalars a row; -1, own and out-of-range parents."""
    from zllm_amd.beam import BeamStates, beam_reorder
    gen = torch.Generator(device="cuda").manual_seed(W)
    G = 3
    R = G * W
    rnd = lambda *s: torch.randint(-100, 100, s, device="cuda", generator=gen)
    ts = [
        (rnd(2, 2, R, 3, 40, 8).to(torch.bfloat16)[:, :, :, :, :13], 2),
        (rnd(R, 77).to(torch.int32), 0),
        (rnd(R).to(torch.int32), 0),
        (rnd(R, 5).to(torch.int8), 0),
        (rnd(3, R, 7).to(torch.float16)[:, :, 1:6], 1),
        (rnd(11, R).to(torch.float32), 1),                       # rows last: single elements
        (rnd(2, 3, R, 4, 5, 6).to(torch.int16)[:, :2, :, :3, :4, :5], 2),   # more strides than two
        (rnd(R, 0).to(torch.int32), 0),
        (rnd(R, 300).to(torch.int64)[:, 4:], 0),
        (rnd(R + 1, 33).to(torch.uint8).view(-1)[7:7 + R * 33].view(R, 33), 0),
    ]
    keep = [(t._base if t._base is not None else t) for t, _ in ts]
    parents = torch.randint(0, W, (G, W), device="cuda", generator=gen, dtype=torch.int32)
    parents[1, ::2] = -1
    parents[2, 0] = W            # out of range: stays
    want = [ref_reorder(t, d, parents, W) for t, d in ts]
    around = [b.clone() for b in keep]
    print(f"[case] beam_reorder W={W}", flush=True)
    beam_reorder(_ctx(), BeamStates(ts, W), parents)
    torch.cuda.synchronize()
    for i, ((t, _), w) in enumerate(zip(ts, want)):
        assert torch.equal(t, w), i
    # nothing outside the views changed
    for (t, _), b, a in zip(ts, keep, around):
        t.zero_()
        if t._base is not None:
            c = a.as_strided(t.shape, t.stride(), t.storage_offset())
            c.zero_()
        else:
            a.zero_()
        assert torch.equal(b, a)


def test_reorder_many_arrays_and_far_offsets():
    """More arrays than one launch takes; an array past 4 GiB whose rows lie far apart."""
    from zllm_amd.beam import BeamStates, beam_reorder
    W, G = 4, 2
    layers = [torch.randn((G * W, 3, 5), device="cuda") for _ in range(130)]
    far = torch.zeros((G * W, 600_000_000), dtype=torch.int8, device="cuda")
    ends = far[:, -1000:]
    ends.copy_(torch.randint(-100, 100, ends.shape, device="cuda"))
    parents = torch.tensor([[1, 0, 0, 3], [3, 3, 3, 0]], dtype=torch.int32, device="cuda")
    want = [ref_reorder(t, 0, parents, W) for t in layers] + [ref_reorder(ends, 0, parents, W)]
    print("[case] beam_reorder 131 arrays", flush=True)
    beam_reorder(_ctx(), BeamStates([(t, 0) for t in layers] + [(ends, 0)], W), parents)
    torch.cuda.synchronize()
    for t, w in zip(layers + [ends], want):
        assert torch.equal(t, w)


# ------------------------------------------------------------------ refusals
def test_refusals():
    from zllm_amd._lib import ZsError
    from zllm_amd.beam import BeamPool, BeamSearch, BeamStates, beam_reorder, beam_select
    c = _ctx()
    x = torch.zeros((8, 100), device="cuda")
    s = torch.zeros((2, 4), device="cuda")
    pool = BeamPool.empty(2, 4)
    bad = [
        lambda: beam_select(c, x.double(), s, pool),
        lambda: beam_select(c, x.cpu(), s, pool),
        lambda: beam_select(c, x.t().contiguous().t(), s, pool),
        lambda: beam_select(c, x[:6], s, pool),
        lambda: beam_select(c, x, s.view(8), pool),
        lambda: beam_select(c, x, s.double(), pool),
        lambda: beam_select(c, x, s, BeamPool.empty(2, 3)),
        lambda: beam_select(c, x, s, pool, eos=range(9)),
        lambda: beam_select(c, x, s, pool, eos=(-1,)),
        lambda: beam_select(c, x, s, pool, allow_bits=torch.zeros((8, 3), dtype=torch.int32, device="cuda")),
        lambda: beam_select(c, torch.zeros((33, 9), device="cuda"), torch.zeros((1, 33), device="cuda"), pool),
        lambda: BeamStates([(x[:1].expand(8, 100), 0)], 4),
        lambda: BeamStates([(x, 0)], 3),
        lambda: BeamStates([(x, 0), (x, 1)], 4),
        lambda: BeamStates([(x, 2)], 4),
        lambda: BeamStates([(x, 0)], 33),
        lambda: beam_reorder(c, BeamStates([(x, 0)], 4), torch.zeros((2, 4), device="cuda")),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(ZsError, match="length_penalty"):
        beam_select(c, x, s, pool, length_penalty=float("nan"))
    with pytest.raises(ZsError, match="ld < V"):
        beam_select(c, torch.zeros(200, device="cuda").as_strided((8, 100), (10, 1)), s, pool)
    search = BeamSearch(c, 2, 4, 0)
    with pytest.raises(ValueError):
        search.step(x)


def test_entry_point_refusals():
    """The C entry points' own checks: nothing is launched."""
    import ctypes as C

    from zllm_amd._lib import Beam, BeamStateDesc, ZS_EINVAL, ZS_ELIMIT, lib
    from zllm_amd.beam import BeamPool
    c = _ctx()
    L = lib()
    n = C.c_uint64()
    assert L.zs_beam_select_work(1, 0, 10, 1, C.byref(n)) == ZS_EINVAL
    assert L.zs_beam_select_work(1, 33, 10, 1, C.byref(n)) == ZS_EINVAL
    assert L.zs_beam_select_work(1, 4, 0, 1, C.byref(n)) == ZS_EINVAL
    assert L.zs_beam_select_work(1, 4, 10, 9, C.byref(n)) == ZS_EINVAL
    assert L.zs_beam_select_work(1, 4, 1000, 1, C.byref(n)) == 0 and n.value > 0
    x = torch.zeros((4, 1000), device="cuda")
    s = torch.zeros((1, 4), device="cuda")
    work = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    pool = BeamPool.empty(1, 4)
    i32 = torch.zeros((2, 4), dtype=torch.int32, device="cuda")

    def args(**kw):
        a = Beam(groups=1, width=4, V=1000, ld=1000, d_logits=x.data_ptr(), n_eos=1, length_penalty=1.0,
                 d_scores=s.data_ptr(), d_parent=i32[0].data_ptr(), d_token=i32[1].data_ptr(), d_score=s.data_ptr(),
                 d_work=work.data_ptr(), work_bytes=n.value)
        for k in ("score", "length", "parent", "token"):
            setattr(a, "d_fin_" + k, getattr(pool, k).data_ptr())
            setattr(a, "d_fin_" + k + "_out", getattr(pool, k).data_ptr())
        for k in ("steps", "done"):
            setattr(a, "d_" + k, getattr(pool, k).data_ptr())
            setattr(a, "d_" + k + "_out", getattr(pool, k).data_ptr())
        for k, v in kw.items():
            setattr(a, k, v)
        return L.zs_beam_select(c.h, C.byref(a), None)

    assert args(width=0) == ZS_ELIMIT and args(width=33) == ZS_ELIMIT and args(V=0) == ZS_ELIMIT
    assert args(n_eos=9) == ZS_ELIMIT and args(V=(1 << 20) + 1, ld=1 << 21) == ZS_ELIMIT
    assert args(groups=1 << 20) == ZS_ELIMIT
    for kw in (dict(dtype=3), dict(ld=999), dict(d_logits=None), dict(d_logits=x.data_ptr() + 2), dict(flags=2),
               dict(d_scores=None), dict(d_parent=None), dict(d_fin_token_out=None), dict(d_work=None),
               dict(work_bytes=n.value - 1), dict(d_work=work.data_ptr() + 8),
               dict(d_allow_bits=x.data_ptr(), allow_words=31)):
        assert args(**kw) == ZS_EINVAL, kw
    assert args(groups=0) == 0
    assert L.zs_beam_select(c.h, None, None) == ZS_EINVAL and L.zs_beam_select(None, None, None) == ZS_EINVAL
    st = BeamStateDesc(x.data_ptr(), 0, 0, 0, 16, 1, 1)
    re = lambda *a: L.zs_beam_reorder(c.h, *a, None)
    assert re(1, 4, i32.data_ptr(), C.byref(st), 1) == ZS_EINVAL        # rows of stride 0
    assert re(1, 33, i32.data_ptr(), C.byref(st), 1) == ZS_ELIMIT
    assert re(1, 4, None, C.byref(st), 1) == ZS_EINVAL and re(1, 4, i32.data_ptr(), None, 1) == ZS_EINVAL
    assert re(1, 4, i32.data_ptr(), None, 0) == 0
    torch.cuda.synchronize()
    assert not x.any() and pool.steps.tolist() == [0]
