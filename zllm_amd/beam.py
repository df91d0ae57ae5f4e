"""Beam search over libzs: the step that selects the next beams from rows of
logits, and the reordering of the states that follow them.

    search = BeamSearch(ctx, groups, width, max_steps, eos=(2,))
    states = BeamStates([(kv_cache, 2), (grammar_state, 0)], width)
    tokens = first                                  # the beams' first inputs, [groups * width]
    while not search.finished():
        search.step(model(tokens))                  # logits [groups * width, V]
        beam_reorder(ctx, states, search.parents)
        tokens = search.tokens.view(-1).clamp_min(0)
    best = search.sequences()[g][0].tokens

Absent beams have the token -1, which no model takes: their rows of logits are
not read, so any id stands for it.
The reference decodes one hypothesis per request; there is no counterpart.
torch holds the device memory and the stream; the computation is libzs's.
"""
import ctypes as C
import functools
import struct
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch
from torch.autograd.graph import increment_version

from ._lib import Beam, BeamStateDesc, ZsError, lib
from .engine import Context, _check

MAX_WIDTH = 32
MAX_EOS = 8
MAX_VOCAB = 1 << 20
ZS_BEAM_EARLY = 1
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

# The arguments are packed to bytes: a step of 4 beams over 32000 ids takes
# the host half as long as with the ctypes fields set one by one.
_BEAM = struct.Struct("=4IQ2Q2I8IfI18Q")
assert _BEAM.size == C.sizeof(Beam)


def _stream(dev: torch.device) -> int:
    """The current stream's handle (torch.cuda.current_stream makes an object
    of it first, which takes as long as a launch)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _rows(ctx: Context, logits: torch.Tensor, what: str) -> None:
    """Checks a [rows, V] tensor of logits: any of the three types, any row
    stride, the values of a row adjacent, on the context's GPU (whose kernels
    are launched; the stream is the logits')."""
    if logits.dim() != 2 or logits.dtype not in DTYPES:
        raise ValueError(f"{what}: logits are [rows, V] of float32, float16 or bfloat16")
    if logits.get_device() != ctx.device:
        raise ValueError(f"{what}: logits are on {logits.device}, not on the context's GPU {ctx.device}")
    if logits.shape[1] > 1 and logits.stride(1) != 1:
        raise ValueError(f"{what}: the logits of a row are not adjacent")


def _ld(t: torch.Tensor) -> int:
    """Row stride in elements (a single row's is of no meaning)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _like(t: torch.Tensor, shape, dtype, dev, what: str, name: str) -> torch.Tensor:
    if t.shape != shape or t.dtype != dtype or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {dtype} tensor {tuple(shape)} on {dev}")
    return t


def _work(nbytes: int, dev) -> Tuple[Optional[torch.Tensor], int]:
    """Scratch of one call and its address, from torch's allocator: it is the
    current stream's, so calls on other streams never share it."""
    if not nbytes:
        return None, 0
    t = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    return t, t.data_ptr()


@functools.lru_cache(maxsize=1024)
def _work_bytes(name: str, *sizes: int) -> int:
    need = C.c_uint64()
    rc = getattr(lib(), name)(*sizes, C.byref(need))
    if rc:
        raise ZsError(f"{name}{sizes} failed ({rc})")
    return need.value


_POOL = ("score", "length", "parent", "token", "steps", "done")


@dataclass(frozen=True)
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

    def _at(self):
        return (self.score.data_ptr(), self.length.data_ptr(), self.parent.data_ptr(), self.token.data_ptr(),
                self.steps.data_ptr(), self.done.data_ptr())

    def _pointers(self, G: int, W: int, dev, what: str):
        # In every call: a tensor may have been resized or put elsewhere since
        # the last. (In one expression 1.5 us of a call's 23, with a _like each 4.)
        s, l, p, t, n, d = self.score, self.length, self.parent, self.token, self.steps, self.done
        gw, g, i32, at = (G, W), (G,), torch.int32, -1 if dev.index is None else dev.index
        if not (s.shape == gw and l.shape == gw and p.shape == gw and t.shape == gw and n.shape == g and d.shape == g and
                s.dtype is torch.float32 and l.dtype is i32 and p.dtype is i32 and t.dtype is i32 and n.dtype is i32 and
                d.dtype is i32 and s.get_device() == at and l.get_device() == at and p.get_device() == at and
                t.get_device() == at and n.get_device() == at and d.get_device() == at and s.is_contiguous() and l.is_contiguous() and p.is_contiguous() and
                t.is_contiguous() and n.is_contiguous() and d.is_contiguous()):
            for name in _POOL:
                _like(getattr(self, name), g if name in ("steps", "done") else gw,
                      torch.float32 if name == "score" else i32, dev, what, "pool." + name)
        return self._at()


@dataclass(frozen=True)
class BeamStep:
    parents: torch.Tensor  # int32 [groups, width]: beam of the group, -1 for none
    tokens: torch.Tensor   # int32 [groups, width]
    scores: torch.Tensor   # float32 [groups, width], best first
    pool: BeamPool

    @classmethod
    def alloc(cls, groups: int, width: int, device) -> "BeamStep":
        """A step's tensors, uninitialised. (An allocation takes the host 1.6 us,
        a part of one that is taken apart 0.4.)"""
        i = torch.empty((7, groups, width), dtype=torch.int32, device=device).unbind(0)
        steps, done = torch.empty((2, groups), dtype=torch.int32, device=device).unbind(0)
        return cls(i[0], i[1], i[6].view(torch.float32),
                   BeamPool(i[5].view(torch.float32), i[2], i[3], i[4], steps, done))


def beam_select(ctx: Context, logits: torch.Tensor, scores: torch.Tensor, pool: BeamPool, eos: Sequence[int] = (),
                length_penalty: float = 1.0, early_stopping: bool = False, allow_bits: Optional[torch.Tensor] = None,
                out: Optional[BeamStep] = None) -> BeamStep:
    """One step of zs_beam_select (include/zs.h has the rules) for logits
    [groups * width, V] of any of the three types and scores [groups, width]
    (float32, -inf: no such beam). allow_bits: packed masks [rows, words] as
    ByteDfa.mask writes them; the scores are of the masked distribution. `out`
    may hold `scores` and the tensors of `pool` themselves. No host sync."""
    what = "beam_select"
    _rows(ctx, logits, what)
    dev = logits.device
    if scores.dim() != 2 or not 1 <= scores.shape[1] <= MAX_WIDTH:
        raise ValueError(f"{what}: scores are [groups, width], width 1 to {MAX_WIDTH}")
    G, W = scores.shape
    R, V = logits.shape
    if R != G * W:
        raise ValueError(f"{what}: {R} rows of logits for {G} groups of {W} beams")
    n_eos = len(eos)
    ends = n_eos <= MAX_EOS
    for e in eos:
        ends = ends and 0 <= e < 2 ** 32
    if not ends:
        raise ValueError(f"{what}: at most {MAX_EOS} EOS ids, not negative")
    _like(scores, (G, W), torch.float32, dev, what, "scores")
    allow, words = 0, 0
    if allow_bits is not None:
        if allow_bits.dim() != 2 or allow_bits.shape[0] != R or allow_bits.shape[1] * 32 < V:
            raise ValueError(f"{what}: allow_bits are [rows, ceil(V / 32)]")
        allow, words = _like(allow_bits, allow_bits.shape, torch.int32, dev, what, "allow_bits").data_ptr(), \
            allow_bits.shape[1]
    before = pool._pointers(G, W, dev, what)
    given = out is not None
    if not given:
        out = BeamStep.alloc(G, W, dev)
        after = out.pool._at()
    else:
        after = before if out.pool is pool else out.pool._pointers(G, W, dev, what)
        _like(out.parents, (G, W), torch.int32, dev, what, "out.parents")
        _like(out.tokens, (G, W), torch.int32, dev, what, "out.tokens")
        _like(out.scores, (G, W), torch.float32, dev, what, "out.scores")
    nbytes = _work_bytes("zs_beam_select_work", G, W, V, n_eos) if 0 < G * W and 0 < V <= MAX_VOCAB else 0
    work, at = _work(nbytes, dev)
    raw = _BEAM.pack(G, W, V, DTYPES[logits.dtype], _ld(logits), logits.data_ptr(), allow, words, n_eos, *eos,
                     *(0,) * (MAX_EOS - n_eos), length_penalty, ZS_BEAM_EARLY if early_stopping else 0, scores.data_ptr(),
                     *before, *after, out.parents.data_ptr(),
                     out.tokens.data_ptr(), out.scores.data_ptr(), at, nbytes)
    rc = lib().zs_beam_select(ctx.h, raw, _stream(dev))
    if rc:
        _check(ctx.h, rc, what)
    if given:   # (autograd is told of writes in place)
        p = out.pool
        increment_version((out.parents, out.tokens, out.scores, p.score, p.length, p.parent, p.token, p.steps, p.done))
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
    row = t.stride(row_dim) * size if t.shape[row_dim] > 1 else block   # (a single row's is of no meaning)
    return [BeamStateDesc(t.data_ptr() + s, row, outer[0], inner[0], block, outer[1], inner[1])
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
        self.device = self.tensors[0].device if self.tensors else None
        self.parents_shape = (self.rows // width, width) if self.tensors else None
        self.descs = (BeamStateDesc * max(self.n, 1))(*descs)


def beam_reorder(ctx: Context, states: BeamStates, parents: torch.Tensor) -> None:
    """Every row of every state becomes what its parent's row was, in place
    (zs_beam_reorder). parents: int32 [groups, width], beams of the group;
    negative ones stay. No host sync."""
    if not states.n:
        return
    dev, shape = states.device, states.parents_shape
    if dev.index != ctx.device:
        raise ValueError(f"beam_reorder: states are on {dev}, not on the context's GPU {ctx.device}")
    _like(parents, shape, torch.int32, dev, "beam_reorder", "parents")
    rc = lib().zs_beam_reorder(ctx.h, shape[0], shape[1], parents.data_ptr(), states.descs, states.n,
                               _stream(dev))
    if rc:
        _check(ctx.h, rc, "beam_reorder")
    increment_version(states.tensors)   # (autograd is told of writes in place)


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
        self.eos, self.length_penalty, self.early_stopping = tuple(int(e) for e in eos), length_penalty, early_stopping
        self.scores = torch.full((groups, width), -float("inf"), device=device)
        self.scores[:, 0] = 0.0
        self.pool = BeamPool.empty(groups, width, device)
        self._trace = torch.full((max_steps or 1, 2, groups, width), -1, dtype=torch.int32, device=device)
        self.t = 0

    @property
    def parents(self) -> torch.Tensor:
        """Parents of the last step's beams (int32 [groups, width]; -1 for
        absent ones, and in front of the first step for all)."""
        return self._trace[self.t - 1, 0]

    @property
    def tokens(self) -> torch.Tensor:
        """Tokens of the last step's beams (int32 [groups, width]; -1 as for
        parents)."""
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
