"""What the speed of beam search and of draft distillation is measured on: the
calls that a serving engine and a training step make of zllm_amd.beam and
zllm_amd.distill, over the sizes that they meet.

Five operators; the kinds of case by the entry point called:

  select   beam.beam_select: one step of a beam search over rows of logits
  reorder  beam.beam_reorder: the states of the beams follow their parents
  teacher  distill.teacher_topk: a teacher's top log-probabilities per row
  loss     distill.distill_loss: the student's loss against such a list
  grad     distill.distill_grad: its gradient, from what the loss kept
  step     distill.distill_loss_grad: the loss and its gradient in one call

`own` false computes them from elementary torch operations in 32 bits. Sizes
are those of the repository's configurations and tests, or generic ones
between them (V from 20,000 to 151,936; a row for each beam or position).
"""
import functools
import math

import torch

own = False

DEV = "cuda"
EOS = 2
F32MAX = torch.finfo(torch.float32).max
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one request with four beams, one step: launches and latency are all there is
        dict(name="select_one", kind="select", groups=1, width=4, live=4, done=0, vocab=32000, dtype="f32", masked=False,
             alpha=1.0),
        # a server's batch of requests in step, a few of them finished
        dict(name="select_batch", kind="select", groups=64, width=4, live=4, done=4, vocab=128256, dtype="bf16",
             masked=False, alpha=0.6),
        # beams under a grammar, an odd vocabulary, NaN in masked places, a beam whose mask leaves nothing
        dict(name="select_grammar", kind="select", groups=13, width=8, live=8, done=0, vocab=100003, dtype="f16",
             masked=True, alpha=1.0),
        # wide beams that make a student's sequences offline
        dict(name="select_wide", kind="select", groups=32, width=32, live=32, done=0, vocab=151936, dtype="f32",
             masked=False, alpha=0.8),
        # the states of a short search: histories, grammar states, a small cache
        dict(name="reorder_short", kind="reorder", groups=8, width=4, layers=4, heads=4, dim=64, cap=128, length=37),
        # a server's caches after some thousand tokens
        dict(name="reorder_caches", kind="reorder", groups=4, width=4, layers=24, heads=8, dim=128, cap=2560,
             length=2011),
        # a few positions of an odd vocabulary for a small draft
        dict(name="teacher_few", kind="teacher", rows=24, vocab=50257, dtype="f32", top=16, temperature=1.0),
        # a long sequence's positions at once
        dict(name="teacher_many", kind="teacher", rows=2048, vocab=151936, dtype="bf16", top=64, temperature=2.0),
        # evaluation: the loss alone, tail bucket, hard labels beside it
        dict(name="loss_eval", kind="loss", rows=512, vocab=128256, dtype="f32", top=50, temperature=2.0, tail=True,
             ce=0.3, ragged=False),
        # the backward pass of a model whose loss was taken before; rows start at any element
        dict(name="grad_odd", kind="grad", rows=1023, vocab=50257, dtype="bf16", top=64, temperature=1.0, tail=False,
             ce=0.0, ragged=True),
        # a short ragged micro-batch, loss and gradient in one call
        dict(name="step_short", kind="step", rows=29, vocab=32000, dtype="f16", top=8, temperature=1.5, tail=True,
             ce=0.5, ragged=True),
        # a training step's positions over the largest vocabulary
        dict(name="step_large", kind="step", rows=4096, vocab=151936, dtype="bf16", top=64, temperature=1.0, tail=True,
             ce=0.2, ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["select", "reorder", "teacher", "loss", "grad", "step"])
    if kind == "reorder":
        case = dict(kind=kind, groups=_log(rng, 1, 16), width=rng.choice([2, 3, 4, 5, 8, 16]), layers=_log(rng, 2, 32),
                    heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 80, 128]), cap=0, length=_log(rng, 1, 2000))
        case["cap"] = case["length"] + rng.randrange(0, 200)
        # no more than the listed caches
        while case["groups"] * case["width"] * case["layers"] * case["heads"] * case["dim"] * case["cap"] > 1 << 30:
            case["layers"] = max(1, case["layers"] // 2)
            case["groups"] = max(1, case["groups"] // 2)
        return case
    vocab = rng.randrange(20000, 151937)
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "select":
        width = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 32])
        groups = _log(rng, 1, max(1, 512 // width))
        return dict(kind=kind, groups=groups, width=width, live=rng.choice([1, width, width]),
                    done=rng.choice([0, 0, groups // 8]), vocab=vocab, dtype=dtype, masked=rng.random() < 0.4,
                    alpha=rng.choice([0.0, 0.6, 1.0]))
    case = dict(kind=kind, rows=_log(rng, 1, 2048), vocab=vocab, dtype=dtype, top=_log(rng, 1, 128),
                temperature=rng.choice([1.0, 1.0, 1.5, 2.0, 4.0]))
    if kind != "teacher":
        case.update(tail=rng.random() < 0.5, ce=rng.choice([0.0, 0.3, 0.5]), ragged=rng.random() < 0.5)
    return case


# ------------------------------------------------------------------ inputs
def _logits(gen, rows, vocab, dtype):
    """N(0, 2) with 16 ids of each row raised by 15 k^-1.2."""
    x = torch.randn((rows, vocab), device=DEV, generator=gen).mul_(2.0)
    rank = torch.rand((rows, 16), device=DEV, generator=gen).argsort(1)
    ids = (torch.randint(0, vocab, (rows, 1), device=DEV, generator=gen) + rank * (vocab // 17)) % vocab
    up = 15.0 * torch.arange(1, 17, device=DEV, dtype=torch.float32) ** -1.2
    x.scatter_(1, ids, x.gather(1, ids) + up)
    return x.to(DTYPES[dtype])


def _unpack(bits, vocab):
    """[rows, words] packed allow bits -> [rows, vocab] truth values."""
    sh = torch.arange(32, device=bits.device, dtype=torch.int32)
    return ((bits[:, :, None] >> sh) & 1).reshape(bits.shape[0], -1)[:, :vocab].bool()


def _prepare_select(c, gen):
    G, W, V = c["groups"], c["width"], c["vocab"]
    x = _logits(gen, G * W, V, c["dtype"])
    # some beams are about to end
    ends = torch.rand(G * W, device=DEV, generator=gen) < 0.3
    x[ends, EOS] = 9.0
    bits = None
    if c["masked"]:
        words = (V + 31) // 32
        r = [torch.randint(-2 ** 31, 2 ** 31, (G * W, words), device=DEV, generator=gen, dtype=torch.int64).to(torch.int32)
             for _ in range(2)]
        bits = r[0] & r[1]
        bits[0] = 0                                     # a beam that may go nowhere
        bad = ~_unpack(bits, V)
        bad[:, ::2] = False
        x[bad] = float("nan")                           # what is masked out may hold anything
    steps = torch.randint(1, 60, (G,), device=DEV, generator=gen, dtype=torch.int32)
    scores = _scores(gen, c)
    # Scores of two beams that differ by less than 32 bits resolve would be
    # ordered by rounding alone: such groups' scores are drawn again.
    top, _ = _top(_masked(x, bits), min(V, W + 1))
    top = top.double() - _lse64(x, bits)[:, None]
    for _ in range(16):
        s = (scores.double()[:, None] + top).reshape(G, -1)
        s = s.masked_fill(~torch.isfinite(s), -1e9)
        beam = torch.arange(W, device=DEV).repeat_interleave(top.shape[1]).expand(G, -1)
        o = s.sort(1, descending=True)
        b = beam.gather(1, o.indices)[:, : 2 * W + 2]
        v = o.values[:, : 2 * W + 2]
        near = ((v[:, :-1] - v[:, 1:] < 4e-5) & (b[:, :-1] != b[:, 1:]) & (v[:, 1:] > -1e8)).any(1)
        scores = torch.where(near.repeat_interleave(W), _scores(gen, c), scores)
    # finished hypotheses so far: at most W, best first
    fin = torch.randn((G, W), device=DEV, generator=gen).mul_(0.3).sub_(1.5).sort(1, descending=True).values
    have = torch.randint(0, W + 1, (G, 1), device=DEV, generator=gen)
    none = torch.arange(W, device=DEV) >= have
    fin = fin.masked_fill(none, -float("inf"))
    flen = torch.randint(1, 60, (G, W), device=DEV, generator=gen, dtype=torch.int32).masked_fill(none, 0)
    fpar = torch.randint(0, W, (G, W), device=DEV, generator=gen, dtype=torch.int32).masked_fill(none, -1)
    ftok = torch.full((G, W), EOS, device=DEV, dtype=torch.int32).masked_fill(none, -1)
    done = (torch.arange(G, device=DEV) >= G - c["done"]).to(torch.int32)
    return dict(logits=x, scores=scores.view(G, W), bits=bits, steps=steps, done=done, fin=fin, flen=flen, fpar=fpar,
                ftok=ftok)


def _scores(gen, c):
    """Running log-probabilities of the beams, best first; beams from `live` on do not exist yet."""
    G, W = c["groups"], c["width"]
    base = torch.rand((G, 1), device=DEV, generator=gen).mul_(-40.0)
    gaps = -torch.log(torch.rand((G, W), device=DEV, generator=gen).clamp_min_(1e-6)) * 0.5
    s = base - gaps.cumsum(1)
    s[:, c["live"]:] = -float("inf")
    return s.reshape(-1)


def _lse64(x, bits):
    y = x.double()
    y = torch.where(torch.isnan(y), -float("inf"), y)
    if bits is not None:
        y = y.masked_fill_(~_unpack(bits, x.shape[1]), -float("inf"))
    return torch.logsumexp(y, 1)


def _prepare_reorder(c, gen):
    G, W = c["groups"], c["width"]
    R = G * W
    # caches [layers, keys/values, row, head, position, dim], live up to `length`
    cache = torch.empty((c["layers"], 2, R, c["heads"], c["cap"], c["dim"]), device=DEV, dtype=torch.bfloat16)
    cache.normal_(generator=gen)
    history = torch.randint(0, 151936, (R, c["cap"]), device=DEV, generator=gen, dtype=torch.int32)
    grammar = torch.randint(0, 2048, (R,), device=DEV, generator=gen, dtype=torch.int32)
    u = torch.rand((G, W), device=DEV, generator=gen)
    parents = (u * u * W).to(torch.int32).clamp_max_(W - 1)      # better beams have more children
    return dict(states=[cache[:, :, :, :, : c["length"]], history[:, : c["length"]], grammar], dims=[2, 0, 0],
                parents=parents, buffers=[cache, history, grammar])


def _prepare_distill(c, gen):
    N, V, K, T = c["rows"], c["vocab"], c["top"], c["temperature"]
    x = _logits(gen, N, V, c["dtype"])
    s = dict(logits=x)
    if c["kind"] == "teacher":
        return s
    # the teacher's list: its logits are the student's and noise
    t = x.float() + torch.randn((N, V), device=DEV, generator=gen).mul_(0.7)
    v, ids = t.topk(K, 1)
    logp = v / T - torch.logsumexp(t.div_(T), 1, keepdim=True)
    labels = ids[:, 0].clone()
    other = torch.rand(N, device=DEV, generator=gen) < 0.2
    labels[other] = torch.randint(0, V, (N,), device=DEV, generator=gen)[other]
    if c["ragged"]:
        # lists of fewer entries than K, and padding positions
        have = torch.randint(1, K + 1, (N, 1), device=DEV, generator=gen)
        none = torch.arange(K, device=DEV) >= have
        ids, logp = ids.masked_fill(none, -1), logp.masked_fill(none, -float("inf"))
        labels[torch.rand(N, device=DEV, generator=gen) < 0.15] = -100
    s.update(ids=ids.to(torch.int32), logp=logp.float(), labels=labels,
             row_grad=torch.rand(N, device=DEV, generator=gen).add_(0.5).div_(N))
    if c["kind"] == "grad":
        # what the forward pass keeps of a row: its maximum, the sums of exp((x - max)/T) and of exp(x - max), and
        # the first of them over the ids outside the list
        f = x.float()
        m = f.amax(1, keepdim=True)
        e = ((f - m) / T).exp()
        s["stats"] = torch.stack([m[:, 0], e.sum(1), (f - m).exp().sum(1), _outside(e, s["ids"]).sum(1)], 1)
        s["stats"][labels == -100] = 0.0
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    make = {"select": _prepare_select, "reorder": _prepare_reorder}.get(case["kind"], _prepare_distill)
    return dict(case=case, **make(case, gen))


# ------------------------------------------------------------------ the framework's calls
@functools.lru_cache(maxsize=None)
def _ctx():
    from zllm_amd.engine import Context
    return Context(0, 256, 151936)


def _config(c):
    from zllm_amd.distill import DistillConfig
    T = c["temperature"]
    return DistillConfig(temperature=T, kl_weight=(1.0 - c["ce"]) * T * T, ce_weight=c["ce"], tail=c["tail"])


def _run_own(s):
    c = s["case"]
    from zllm_amd import beam, distill
    if c["kind"] == "select":
        if "pool" not in s:
            s["pool"] = beam.BeamPool(score=s["fin"], length=s["flen"], parent=s["fpar"], token=s["ftok"],
                                      steps=s["steps"], done=s["done"])
        o = beam.beam_select(_ctx(), s["logits"], s["scores"], s["pool"], eos=(EOS,), length_penalty=c["alpha"],
                             allow_bits=s["bits"])
        p = o.pool
        return dict(parents=o.parents, tokens=o.tokens, scores=o.scores, fin=p.score, flen=p.length, fpar=p.parent,
                    ftok=p.token, steps=p.steps, done=p.done)
    if c["kind"] == "reorder":
        if "plan" not in s:
            s["plan"] = beam.BeamStates([(t, d) for t, d in zip(s["states"], s["dims"])], c["width"])
        beam.beam_reorder(_ctx(), s["plan"], s["parents"])
        return s["buffers"]
    if c["kind"] == "teacher":
        ids, logp, lse = distill.teacher_topk(_ctx(), s["logits"], c["top"], c["temperature"])
        return dict(ids=ids, logp=logp, lse=lse)
    cfg = _config(c)
    if c["kind"] == "loss":
        loss, stats = distill.distill_loss(_ctx(), s["logits"], s["ids"], s["logp"], cfg, labels=s["labels"])
        return dict(loss=loss, stats=stats)
    if c["kind"] == "grad":
        return dict(grad=distill.distill_grad(_ctx(), s["logits"], s["ids"], s["logp"], cfg, s["stats"], s["row_grad"],
                                              labels=s["labels"]))
    loss, grad = distill.distill_loss_grad(_ctx(), s["logits"], s["ids"], s["logp"], cfg, s["row_grad"],
                                           labels=s["labels"])
    return dict(loss=loss, grad=grad)


# ------------------------------------------------------------------ the plain form
def _masked(x, bits):
    """Rows in 32 bits: masked ids and NaN are -inf, +inf is the largest number."""
    x = torch.nan_to_num(x.float(), nan=-float("inf"), posinf=F32MAX, neginf=-float("inf"))
    return x if bits is None else x.masked_fill(~_unpack(bits, x.shape[1]), -float("inf"))


def _top(x, k):
    """The k largest of each row, equal ones by the lower id."""
    b = (x + 0.0).view(torch.int32).to(torch.int64)
    key = torch.where(b < 0, b ^ 0x7FFFFFFF, b)
    V = x.shape[1]
    key = key * (1 << 32) + (V - 1 - torch.arange(V, device=x.device))
    ids = V - 1 - (key.topk(k, 1).values & 0xFFFFFFFF)
    return x.gather(1, ids), ids


def _lse(x):
    m = x.amax(1, keepdim=True).clamp_min(-F32MAX)
    return m[:, 0] + (x - m).exp().sum(1).log()


def _plain_select(s):
    c = s["case"]
    G, W, V = c["groups"], c["width"], c["vocab"]
    x = _masked(s["logits"], s["bits"])
    v, ids = _top(x, W + 1)
    score = s["scores"].reshape(-1, 1) + (v - _lse(x)[:, None])
    score = torch.where(torch.isnan(score) | (v == -float("inf")), -float("inf"), score)
    # one list a group, best first; the sort keeps the order of beams and within beams
    score, at = score.reshape(G, -1).sort(dim=1, descending=True, stable=True)
    ids = ids.reshape(G, -1).gather(1, at).to(torch.int32)
    parent = (at // (W + 1)).to(torch.int32)
    real = score > -float("inf")
    ends = real & (ids == EOS)
    goes = real & ~ends
    # the next beams: the first W that do not end
    place = torch.where(goes, goes.cumsum(1) - 1, W).clamp_max(W)
    put = lambda fill, val: torch.full((G, W + 1), fill, device=x.device, dtype=val.dtype).scatter(1, place, torch.where(
        place < W, val, torch.full_like(val, fill)))[:, :W]
    ninf = -float("inf")
    new = dict(parents=put(-1, parent), tokens=put(-1, ids), scores=put(ninf, score))
    # the finished ones among the first W join the pool
    length = (s["steps"] + 1).float()
    norm = (length ** c["alpha"])[:, None]
    ok = ends[:, :W]
    cand = torch.where(ok, score[:, :W] / norm, ninf)
    fin, order = torch.cat([s["fin"], cand], 1).sort(dim=1, descending=True, stable=True)
    pick = lambda a, b: torch.cat([a, torch.where(ok, b, a.new_full((), -1))], 1).gather(1, order)[:, :W]
    fin = fin[:, :W]
    empty = fin == ninf
    flen = pick(s["flen"], (s["steps"] + 1)[:, None].expand(G, W)).masked_fill(empty, 0)
    fpar = pick(s["fpar"], parent[:, :W]).masked_fill(empty, -1)
    ftok = pick(s["ftok"], ids[:, :W]).masked_fill(empty, -1)
    best = new["scores"][:, 0]
    done = ((fin[:, W - 1] > ninf) & (fin[:, W - 1] >= best / norm[:, 0])) | (best == ninf)
    # groups that were done stay as they are
    was = s["done"].bool()
    keep = lambda a, b: torch.where(was.view([-1] + [1] * (b.dim() - 1)), a, b)
    i32 = lambda n: torch.tensor(n, device=x.device, dtype=torch.int32)
    return dict(parents=keep(i32(-1), new["parents"]), tokens=keep(i32(-1), new["tokens"]),
                scores=keep(torch.tensor(ninf, device=x.device), new["scores"]), fin=keep(s["fin"], fin),
                flen=keep(s["flen"], flen), fpar=keep(s["fpar"], fpar), ftok=keep(s["ftok"], ftok),
                steps=keep(s["steps"], s["steps"] + 1), done=keep(s["done"], done.to(torch.int32)))


def _plain_reorder(s):
    W = s["case"]["width"]
    base = torch.arange(s["parents"].shape[0], device=DEV, dtype=torch.int64)[:, None] * W
    rows = (base + s["parents"]).reshape(-1)
    [t.copy_(t.index_select(d, rows)) for t, d in zip(s["states"], s["dims"])]
    return s["buffers"]


def _plain_teacher(s):
    c = s["case"]
    x = _masked(s["logits"], None)
    v, ids = _top(x, c["top"])
    lse = _lse(x / c["temperature"])
    return dict(ids=ids.to(torch.int32), logp=v / c["temperature"] - lse[:, None], lse=lse)


def _outside(e, ids):
    """e with zeros at the listed ids (an absent entry stands for the row's first)."""
    return e.scatter(1, torch.where(ids >= 0, ids, ids[:, :1]).long(), 0.0)


def _target(s):
    """The list's probabilities and the tail's."""
    p = s["logp"].exp()
    if s["case"]["tail"]:
        return p, (1.0 - p.sum(1, keepdim=True)).clamp_min(0.0)
    return p / p.sum(1, keepdim=True), None


def _plain_loss(s, stats):
    c = s["case"]
    T, b = c["temperature"], c["ce"]
    ids = s["ids"].clamp_min(0).long()
    p, tail = _target(s)
    m, sT, s1, out = stats.unbind(1)
    z = (s["logits"].gather(1, ids).float() - m[:, None]) / T - sT.log()[:, None]
    kl = torch.where(p > 0, p * (p.clamp_min(1e-38).log() - z), 0.0).sum(1)
    if tail is not None:
        t = tail[:, 0]
        kl = kl + torch.where(t > 0, t * (t.clamp_min(1e-38).log() - (out.log() - sT.log())), 0.0)
    loss = (1.0 - b) * T * T * kl
    lab = s["labels"]
    if b:
        x = s["logits"].gather(1, lab.clamp_min(0)[:, None]).float()[:, 0]
        loss = loss + b * (s1.log() - (x - m))
    return torch.where(lab == -100, 0.0, loss)


def _plain_stats(s):
    c = s["case"]
    x = s["logits"].float()
    m = x.amax(1, keepdim=True)
    e = ((x - m) / c["temperature"]).exp()
    s1 = (x - m).exp().sum(1) if c["ce"] and c["temperature"] != 1.0 else e.sum(1)
    out = _outside(e, s["ids"]).sum(1) if c["tail"] else torch.zeros_like(s1)
    # (nothing is kept of padding positions)
    return torch.where((s["labels"] == -100)[:, None], 0.0, torch.stack([m[:, 0], e.sum(1), s1, out], 1))


def _plain_grad(s, stats):
    c = s["case"]
    T, b = c["temperature"], c["ce"]
    x = s["logits"].float()
    ids = torch.where(s["ids"] >= 0, s["ids"], s["ids"][:, :1]).long()
    m, sT, s1, out = (v[:, None] for v in stats.unbind(1))
    e = ((x - m) / T).exp()
    p, tail = _target(s)
    total = p.sum(1, keepdim=True) + (0.0 if tail is None else tail)
    g = e * (total / sT)
    if tail is not None:
        g = g - _outside(e, s["ids"]) * (tail / out)
    g = g.scatter_add_(1, ids, -p).mul_((1.0 - b) * T)
    if b:
        q = (x - m).exp() * (b / s1)
        g = g.add_(q).scatter_add_(1, s["labels"].clamp_min(0)[:, None], torch.full_like(m, -b))
    g = torch.where((s["labels"] == -100)[:, None], 0.0, g.mul_(s["row_grad"][:, None]))
    return g.to(s["logits"].dtype)


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _run_own(s)
    if kind == "select":
        return _plain_select(s)
    if kind == "reorder":
        return _plain_reorder(s)
    if kind == "teacher":
        return _plain_teacher(s)
    if kind == "grad":
        return dict(grad=_plain_grad(s, s["stats"]))
    stats = _plain_stats(s)
    if kind == "loss":
        return dict(loss=_plain_loss(s, stats), stats=stats)
    return dict(loss=_plain_loss(s, stats), grad=_plain_grad(s, stats))


# ------------------------------------------------------------------ what a pass cannot do without
def work(c):
    if c["kind"] == "reorder":
        W = c["width"]
        p = [math.sqrt((i + 1) / W) - math.sqrt(i / W) for i in range(W)]     # of each parent
        moved = W - sum(p)
        read = sum(1.0 - (1.0 - q) ** (W - 1) for q in p)
        row = c["layers"] * 2 * c["heads"] * c["length"] * c["dim"] * 2 + 4 * c["length"] + 4
        return dict(bytes=c["groups"] * (moved + read) * row + 4 * c["groups"] * W, flops=0)
    if c["kind"] == "select":
        rows = (c["groups"] - c["done"]) * c["live"]
        n = rows * c["vocab"]
        return dict(bytes=n * SIZE[c["dtype"]] + (rows * ((c["vocab"] + 31) // 32) * 4 if c["masked"] else 0) +
                    c["groups"] * (c["width"] * 48 + 16), flops=6 * n)
    n, K = c["rows"] * c["vocab"], c["rows"] * c["top"]
    size = SIZE[c["dtype"]]
    if c["kind"] == "teacher":
        return dict(bytes=n * size + 8 * K + 4 * c["rows"], flops=6 * n)
    # two exponentials a logit where the labels' distribution is another
    one = 5 * (2 if c["ce"] and c["temperature"] != 1.0 else 1)
    if c["kind"] == "loss":
        return dict(bytes=n * size + 8 * K + 28 * c["rows"], flops=one * n)
    if c["kind"] == "grad":
        return dict(bytes=2 * n * size + 8 * K + 28 * c["rows"], flops=one * n)
    return dict(bytes=2 * n * size + 8 * K + 16 * c["rows"], flops=2 * one * n)


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_select(s):
    c = s["case"]
    G, W, V = c["groups"], c["width"], c["vocab"]
    ninf = -float("inf")
    lp = s["logits"].double()
    lp[torch.isnan(lp)] = ninf
    if s["bits"] is not None:
        lp[~_unpack(s["bits"], V)] = ninf
    lp = torch.log_softmax(lp, 1).nan_to_num_(nan=ninf, neginf=ninf)
    all_ = (lp + s["scores"].double().view(-1, 1)).view(G, W * V)
    is_eos = torch.zeros(V, device=DEV, dtype=torch.bool)
    is_eos[EOS] = True
    live = all_.masked_fill(is_eos.repeat(W), ninf).topk(W, 1).values
    ends = all_.view(G, W, V)[:, :, EOS]
    rank = torch.stack([(all_ > ends[:, w: w + 1]).sum(1) for w in range(W)], 1)
    length = (s["steps"] + 1).double()[:, None] ** c["alpha"]
    joins = torch.where(rank < W, ends / length, ninf)
    fin = torch.cat([s["fin"].double(), joins], 1).sort(1, descending=True).values[:, :W]
    was = s["done"].bool()[:, None]
    return dict(parents=None, tokens=None, scores=live.masked_fill(was, ninf), fin=torch.where(was, s["fin"].double(), fin),
                flen=None, fpar=None, ftok=None, steps=None, done=None)


def _exact_rows(c, x, s):
    """Loss, gradient and kept sums of some rows, in 64 bits, from probabilities."""
    T, b, V = c["temperature"], c["ce"], c["vocab"]
    x = x.double()
    lq = torch.log_softmax(x / T, 1)
    p = s["logp"].double().exp()
    if not c["tail"]:
        p = p / p.sum(1, keepdim=True)
    col = torch.where(s["ids"] < 0, V, s["ids"].long())                  # absent entries go to a column of their own
    dense = torch.zeros((x.shape[0], V + 1), device=DEV, dtype=torch.float64).scatter_add_(1, col, p)[:, :V]
    inside = torch.zeros((x.shape[0], V + 1), device=DEV, dtype=torch.bool).scatter_(1, col, True)[:, :V]
    kl = torch.where(dense > 0, dense * (dense.clamp_min(1e-300).log() - lq), 0.0).sum(1)
    q = lq.exp()
    total = dense.sum(1, keepdim=True)
    g = -dense
    m = x.amax(1)
    out = torch.where(inside, 0.0, q).sum(1)
    if c["tail"]:
        pt = (1.0 - total[:, 0]).clamp_min(0.0)
        kl = kl + torch.where(pt > 0, pt * (pt.clamp_min(1e-300).log() - out.log()), 0.0)
        g = g - torch.where(inside, 0.0, q) * (pt / out)[:, None]
        total = total + pt[:, None]
    g = (g + total * q) * ((1.0 - b) * T)
    loss = (1.0 - b) * T * T * kl
    lab = s["labels"]
    l1 = torch.log_softmax(x, 1)
    if b:
        at = lab.clamp_min(0)[:, None]
        loss = loss - b * l1.gather(1, at)[:, 0]
        g = g + b * (l1.exp() - torch.zeros_like(x).scatter_(1, at, 1.0))
    skip = lab == -100
    g = torch.where(skip[:, None], 0.0, g * s["row_grad"].double()[:, None])
    sT, s1 = (torch.logsumexp(x / T, 1) - m / T).exp(), (torch.logsumexp(x, 1) - m).exp()
    stats = torch.stack([m, sT, s1 if b and T != 1.0 else sT, out * sT if c["tail"] else torch.zeros_like(m)], 1)
    return torch.where(skip, 0.0, loss), g, torch.where(skip[:, None], 0.0, stats)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "reorder":
        return None          # bytes move: nothing is computed
    if kind == "select":
        return _exact_select(s)
    if kind == "teacher":
        y = s["logits"].double() / case["temperature"]
        lse = torch.logsumexp(y, 1)
        return dict(ids=None, logp=y.topk(case["top"], 1).values - lse[:, None], lse=lse)
    per = max(1, (1 << 26) // case["vocab"])
    parts = []
    for r in range(0, case["rows"], per):
        cut = {k: s[k][r: r + per] for k in ("ids", "logp", "labels", "row_grad")}
        loss, g, stats = _exact_rows(case, s["logits"][r: r + per], cut)
        parts.append((loss, g if kind != "loss" else None, stats))
    loss, stats = torch.cat([p[0] for p in parts]), torch.cat([p[2] for p in parts])
    if kind == "loss":
        return dict(loss=loss, stats=stats)
    grad = torch.cat([p[1] for p in parts])
    return dict(grad=grad) if kind == "grad" else dict(loss=loss, grad=grad)
