"""Beam search over libzs: the step that selects the next beams from rows of
logits, and the reordering of the states that follow them.

    search = BeamSearch(ctx, groups, width, max_steps, eos=(2,))
    states = BeamStates([(kv_cache, 2), (grammar_state, 0)], width)
    while not search.finished():
        logits = model(search.tokens, ...)          # [groups * width, V]
        search.step(logits)
        beam_reorder(ctx, states, search.parents)
    best = search.sequences()[g][0].tokens

The reference decodes one hypothesis per request; there is no counterpart.
torch holds the device memory and the stream; the computation is libzs's.
"""
import ctypes as C
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from ._lib import Beam, BeamStateDesc, lib
from .engine import Context, _check

MAX_WIDTH = 32
MAX_EOS = 8
ZS_BEAM_EARLY = 1
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _rows(logits: torch.Tensor, what: str) -> torch.Tensor:
    """Checks a [rows, V] tensor of logits: any of the three types, any row
    stride, the values of a row adjacent."""
    if logits.dim() != 2 or logits.dtype not in DTYPES:
        raise ValueError(f"{what}: logits are [rows, V] of float32, float16 or bfloat16")
    if not logits.is_cuda:
        raise ValueError(f"{what}: logits are on {logits.device}, not on a GPU")
    if logits.shape[1] > 1 and logits.stride(1) != 1:
        raise ValueError(f"{what}: the logits of a row are not adjacent")
    return logits


def _ld(t: torch.Tensor) -> int:
    """Row stride in elements (a single row's is of no meaning)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _like(t: torch.Tensor, shape, dtype, dev, what: str, name: str) -> torch.Tensor:
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {dtype} tensor {tuple(shape)} on {dev}")
    return t


def _work(nbytes: int, dev) -> Optional[torch.Tensor]:
    """Scratch of one call, from torch's allocator: it is the current
    stream's, so calls on other streams never share it."""
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


@dataclass
class BeamPool:
    """Finished hypotheses of each request, best first ([groups, width]; absent
    ones score -inf), and the requests' state ([groups]). An entry's tokens
    are its EOS id `token` behind those of beam `parent` after `length` - 1
    steps."""
    score: torch.Tensor    # float32
    length: torch.Tensor   # int32, tokens with the EOS id
    parent: torch.Tensor   # int32
    token: torch.Tensor    # int32
    steps: torch.Tensor    # int32, tokens so far
    done: torch.Tensor     # int32, 1: the request takes no more steps

    @classmethod
    def empty(cls, groups: int, width: int, device="cuda") -> "BeamPool":
        i = lambda fill, *s: torch.full(s, fill, dtype=torch.int32, device=device)
        return cls(torch.full((groups, width), -float("inf"), device=device), i(0, groups, width), i(-1, groups, width),
                   i(-1, groups, width), i(0, groups), i(0, groups))


@dataclass
class BeamStep:
    parents: torch.Tensor  # int32 [groups, width]: beam of the group, -1 for none
    tokens: torch.Tensor   # int32 [groups, width]
    scores: torch.Tensor   # float32 [groups, width], best first
    pool: BeamPool

    @classmethod
    def alloc(cls, groups: int, width: int, device) -> "BeamStep":
        f = torch.empty((2, groups, width), device=device).unbind(0)
        i = torch.empty((5, groups, width), dtype=torch.int32, device=device).unbind(0)
        g = torch.empty((2, groups), dtype=torch.int32, device=device).unbind(0)
        return cls(i[0], i[1], f[0], BeamPool(f[1], i[2], i[3], i[4], g[0], g[1]))


def beam_select(ctx: Context, logits: torch.Tensor, scores: torch.Tensor, pool: BeamPool, eos: Sequence[int] = (),
                length_penalty: float = 1.0, early_stopping: bool = False, allow_bits: Optional[torch.Tensor] = None,
                out: Optional[BeamStep] = None) -> BeamStep:
    """One step of zs_beam_select (include/zs.h has the rules) for logits
    [groups * width, V] of any of the three types and scores [groups, width]
    (float32, -inf: no such beam). allow_bits: packed masks [rows, words] as
    ByteDfa.mask writes them; the scores are of the masked distribution. `out`
    may hold `scores` and the tensors of `pool` themselves. No host sync."""
    what = "beam_select"
    _rows(logits, what)
    dev = logits.device
    if scores.dim() != 2 or not 1 <= scores.shape[1] <= MAX_WIDTH:
        raise ValueError(f"{what}: scores are [groups, width], width 1 to {MAX_WIDTH}")
    G, W = scores.shape
    R, V = logits.shape
    if R != G * W:
        raise ValueError(f"{what}: {R} rows of logits for {G} groups of {W} beams")
    eos = [int(e) for e in eos]
    if len(eos) > MAX_EOS or any(not 0 <= e < 2 ** 32 for e in eos):
        raise ValueError(f"{what}: at most {MAX_EOS} EOS ids, not negative")
    _like(scores, (G, W), torch.float32, dev, what, "scores")
    a = Beam()
    a.groups, a.width, a.V, a.dtype, a.ld = G, W, V, DTYPES[logits.dtype], _ld(logits)
    a.d_logits = logits.data_ptr()
    if allow_bits is not None:
        if allow_bits.dim() != 2 or allow_bits.shape[0] != R or allow_bits.shape[1] * 32 < V:
            raise ValueError(f"{what}: allow_bits are [rows, ceil(V / 32)]")
        _like(allow_bits, allow_bits.shape, torch.int32, dev, what, "allow_bits")
        a.d_allow_bits, a.allow_words = allow_bits.data_ptr(), allow_bits.shape[1]
    a.n_eos = len(eos)
    for i, e in enumerate(eos):
        a.eos[i] = e
    a.length_penalty, a.flags = length_penalty, ZS_BEAM_EARLY if early_stopping else 0
    if out is None:
        out = BeamStep.alloc(G, W, dev)
    a.d_scores = scores.data_ptr()
    for p, tail in ((pool, ""), (out.pool, "_out")):
        for name in ("score", "length", "parent", "token"):
            t = _like(getattr(p, name), (G, W), torch.float32 if name == "score" else torch.int32, dev, what, "pool." + name)
            setattr(a, "d_fin_" + name + tail, t.data_ptr())
        for name in ("steps", "done"):
            setattr(a, "d_" + name + tail, _like(getattr(p, name), (G,), torch.int32, dev, what, "pool." + name).data_ptr())
    a.d_parent = _like(out.parents, (G, W), torch.int32, dev, what, "out.parents").data_ptr()
    a.d_token = _like(out.tokens, (G, W), torch.int32, dev, what, "out.tokens").data_ptr()
    a.d_score = _like(out.scores, (G, W), torch.float32, dev, what, "out.scores").data_ptr()
    need = C.c_uint64()
    _check(ctx.h, lib().zs_beam_select_work(G, W, V, len(eos), C.byref(need)), "zs_beam_select_work")
    work = _work(need.value, dev)
    if work is not None:
        a.d_work, a.work_bytes = work.data_ptr(), need.value
    _check(ctx.h, lib().zs_beam_select(ctx.h, C.byref(a), torch.cuda.current_stream(dev).cuda_stream), what)
    return out


def _blocks(t: torch.Tensor, row_dim: int) -> List[BeamStateDesc]:
    """The state array of one tensor: blocks of adjacent bytes under at most
    two strides; tensors of more strides become several arrays."""
    size = t.element_size()
    dims = sorted((t.stride(d) * size, t.shape[d]) for d in range(t.dim()) if d != row_dim and t.shape[d] > 1)
    if any(s == 0 for s, _ in dims) or (t.shape[row_dim] > 1 and t.stride(row_dim) == 0):
        raise ValueError("BeamStates: an expanded tensor has no rows of its own")
    block, rest = size, []
    for stride, n in dims:
        if stride == block and not rest:
            block *= n
        elif rest and stride == rest[-1][0] * rest[-1][1]:
            rest[-1] = (rest[-1][0], rest[-1][1] * n)
        else:
            rest.append((stride, n))
    starts = [0]
    for stride, n in rest[2:]:
        starts = [s + i * stride for s in starts for i in range(n)]
    inner, outer = (rest + [(0, 1), (0, 1)])[:2]
    return [BeamStateDesc(t.data_ptr() + s, t.stride(row_dim) * size, outer[0], inner[0], block, outer[1], inner[1])
            for s in starts]


class BeamStates:
    """The state arrays that follow their beams: (tensor, row_dim) pairs, row
    group * width + beam of each along row_dim. Any tensors and views whose
    rows are memory of their own: a cache [layers, 2, rows, heads, positions,
    dim] and its view up to the live position, histories, grammar states.
    Made once while the tensors stay where they are."""

    def __init__(self, tensors: Sequence[Tuple[torch.Tensor, int]], width: int):
        if not 1 <= width <= MAX_WIDTH:
            raise ValueError(f"BeamStates: width 1 to {MAX_WIDTH}")
        self.width = width
        self.tensors = [t for t, _ in tensors]   # kept: the arrays are their memory
        self.rows = None
        descs = []
        for t, d in tensors:
            if not t.is_cuda or not -t.dim() <= d < t.dim():
                raise ValueError("BeamStates: GPU tensors with a dimension of rows")
            d %= t.dim()
            if self.rows not in (None, t.shape[d]) or t.device != self.tensors[0].device:
                raise ValueError("BeamStates: tensors of different rows or devices")
            self.rows = t.shape[d]
            if t.numel():
                descs += _blocks(t, d)
        if self.rows is not None and self.rows % width:
            raise ValueError("BeamStates: the rows are not whole groups")
        self.n = len(descs)
        self.descs = (BeamStateDesc * max(self.n, 1))(*descs)


def beam_reorder(ctx: Context, states: BeamStates, parents: torch.Tensor) -> None:
    """Every row of every state becomes what its parent's row was, in place
    (zs_beam_reorder). parents: int32 [groups, width], beams of the group;
    negative ones stay. No host sync."""
    if not states.n:
        return
    dev = states.tensors[0].device
    _like(parents, (states.rows // states.width, states.width), torch.int32, dev, "beam_reorder", "parents")
    rc = lib().zs_beam_reorder(ctx.h, parents.shape[0], states.width, parents.data_ptr(), states.descs, states.n,
                               torch.cuda.current_stream(dev).cuda_stream)
    _check(ctx.h, rc, "beam_reorder")


@dataclass
class Hypothesis:
    tokens: List[int]
    score: float      # log-probability / length^length_penalty
    finished: bool    # ended with an EOS id


class BeamSearch:
    """The beams of `groups` requests over their steps: scores, pool and the
    (parent, token) of every step, on the device. The first step takes beam 0
    of every request (the others do not exist yet)."""

    def __init__(self, ctx: Context, groups: int, width: int, max_steps: int, eos: Sequence[int] = (),
                 length_penalty: float = 1.0, early_stopping: bool = False, device="cuda"):
        self.ctx, self.groups, self.width, self.max_steps = ctx, groups, width, max_steps
        self.eos, self.length_penalty, self.early_stopping = tuple(eos), length_penalty, early_stopping
        self.scores = torch.full((groups, width), -float("inf"), device=device)
        self.scores[:, 0] = 0.0
        self.pool = BeamPool.empty(groups, width, device)
        self._trace = torch.full((max_steps, 2, groups, width), -1, dtype=torch.int32, device=device)
        self.t = 0

    @property
    def parents(self) -> torch.Tensor:
        """Parents of the last step's beams (int32 [groups, width])."""
        return self._trace[self.t - 1, 0]

    @property
    def tokens(self) -> torch.Tensor:
        """Tokens of the last step's beams (int32 [groups, width])."""
        return self._trace[self.t - 1, 1]

    def step(self, logits: torch.Tensor, allow_bits: Optional[torch.Tensor] = None) -> None:
        if self.t >= self.max_steps:
            raise ValueError(f"BeamSearch: more than max_steps={self.max_steps} steps")
        at = self._trace[self.t]
        beam_select(self.ctx, logits, self.scores, self.pool, self.eos, self.length_penalty, self.early_stopping,
                    allow_bits, out=BeamStep(at[0], at[1], self.scores, self.pool))
        self.t += 1

    def finished(self) -> bool:
        """Whether no request takes more steps (reads the device)."""
        return self.t >= self.max_steps or bool(self.pool.done.all())

    def sequences(self) -> List[List[Hypothesis]]:
        """The requests' hypotheses, best first: the finished ones and, of
        requests that are not done, the beams as they stand."""
        trace = self._trace[: self.t].cpu().numpy()
        pool = {k: getattr(self.pool, k).cpu().numpy() for k in ("score", "length", "parent", "token", "done")}
        scores = self.scores.cpu().numpy()

        def follow(g, beam, steps):
            toks = []
            for t in range(steps - 1, -1, -1):
                toks.append(int(trace[t, 1, g, beam]))
                beam = int(trace[t, 0, g, beam])
            return toks[::-1]

        out = []
        for g in range(self.groups):
            hyps = [Hypothesis(follow(g, int(pool["parent"][g, i]), int(pool["length"][g, i]) - 1) +
                               [int(pool["token"][g, i])], float(pool["score"][g, i]), True)
                    for i in range(self.width) if np.isfinite(pool["score"][g, i])]
            if not pool["done"][g] and self.t:
                hyps += [Hypothesis(follow(g, b, self.t), float(scores[g, b]) / self.t ** self.length_penalty, False)
                         for b in range(self.width) if np.isfinite(scores[g, b])]
            out.append(sorted(hyps, key=lambda h: -h.score))
        return out
