"""The vocabulary head over libzs: its cross entropy from hidden states, without
logits in memory, with the gradients; and a head held in 4 bits, whose logits the
sampler, the lanes and beam search read.

    loss_of = HeadLoss(ctx)
    loss_of(hidden, head_weight, labels).mean().backward()

or, without autograd, head_loss (evaluation, the scores of given tokens: their
log-probabilities are -loss) and head_loss_grad;

    head = Q4Head.quantize(ctx, head_weight, group=64)      # once
    lanes = LaneBatcher(ctx, head=head)
    lanes.step(hidden)                                      # the active streams' next tokens

or head.logits(hidden). The formulas are in include/zs.h. The reference trains
nothing; the loss has no counterpart.
Scratch of a call, from torch's allocator: a loss keeps 8 bytes for each row and 128
ids (32, of up to 128 rows). A step keeps an exponential for each row and id besides,
2 bytes of 16-bit types (4 up to 64 rows) and 8 to 14 of float32, of at most 4 GiB of
rows at a time: 8192 rows of 151936 ids take 2.5 GB. The gradients of more rows than
that are made in pieces, the weight's summed in float32 (4 V D bytes). A float32
weight is copied as well (4 V D) for more than 192 rows, a 16-bit one (2 V D) if its
rows do not lie at 16 bytes each.
torch holds the device memory and the stream; the computation is libzs's.
"""
import ctypes as C
import struct
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from ._lib import Ce, Q4, lib
from .beam import DTYPES, MAX_VOCAB, _ld, _like, _stream, _work, _work_bytes
from .engine import Context, _check

MAX_HIDDEN = 65536
MAX_LD = 4194304
_DHIDDEN, _DWEIGHT, _COPY, _FAR = 1, 2, 4, 8
# the arguments are packed to bytes, as zllm_amd.beam's
_CE = struct.Struct("=4I2Q3QqfI10Q")
_Q4 = struct.Struct("=4IQ2I6Q")
assert _CE.size == C.sizeof(Ce) and _Q4.size == C.sizeof(Q4)
GROUPS = (32, 64, 128)
_FEW = 16   # rows up to which Q4Head.logits may need no scratch


@dataclass(frozen=True)
class HeadLossConfig:
    """loss = cross entropy + z_weight * lse^2."""
    z_weight: float = 0.0
    ignore_index: int = -100


def _matrix(ctx: Context, t: torch.Tensor, what: str, name: str) -> None:
    if t.dim() != 2 or t.dtype not in DTYPES:
        raise ValueError(f"{what}: {name} is [rows, D] of float32, float16 or bfloat16")
    if t.get_device() != ctx.device:
        raise ValueError(f"{what}: {name} is on {t.device}, not on the context's GPU {ctx.device}")
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{what}: the values of a row of {name} are not adjacent, or its rows overlap")


def _call(ctx, entry, what, hidden, weight, labels, cfg, row_grad=None, want=(False, False)):
    _matrix(ctx, hidden, what, "hidden")
    _matrix(ctx, weight, what, "weight")
    (N, D), V, dev = hidden.shape, weight.shape[0], hidden.device
    if weight.shape[1] != D or weight.dtype != hidden.dtype:
        raise ValueError(f"{what}: hidden [N, D] and weight [V, D] are of one D and one type")
    if not 1 <= V <= MAX_VOCAB or not 1 <= D <= MAX_HIDDEN:
        raise ValueError(f"{what}: V is 1 to {MAX_VOCAB}, D 1 to {MAX_HIDDEN}")
    lab = _like(labels, (N,), torch.int64, dev, what, "labels").data_ptr()
    # (each of its own: autograd lets no view of one of several be changed in place)
    loss = torch.empty(N, dtype=torch.float32, device=dev)
    lse = torch.empty(N, dtype=torch.float32, device=dev)
    dh = torch.empty((N, D), dtype=hidden.dtype, device=dev) if want[0] else None
    dw = torch.empty((V, D), dtype=hidden.dtype, device=dev) if want[1] else None
    bits = (_DHIDDEN if want[0] else 0) | (_DWEIGHT if want[1] else 0)
    at, ldw = weight.data_ptr(), _ld(weight)
    size = hidden.element_size()
    if at % 16 or D * size % 16 or (V > 1 and ldw * size % 16):
        bits |= _COPY
    if ldw > MAX_LD:
        bits |= _FAR
    nbytes = _work_bytes("zs_ce_work", N, V, D, DTYPES[hidden.dtype], bits)
    work, work_at = _work(nbytes, dev)
    rg, rg_stride = (row_grad.data_ptr(), row_grad.stride(0) if row_grad.dim() else 0) if row_grad is not None else (0, 0)
    raw = _CE.pack(N, V, D, DTYPES[hidden.dtype], _ld(hidden), ldw, hidden.data_ptr(), at, lab, cfg.ignore_index,
                   cfg.z_weight, 0, loss.data_ptr(), lse.data_ptr(), rg, rg_stride, dh.data_ptr() if want[0] else 0,
                   dw.data_ptr() if want[1] else 0, D, D, work_at, nbytes)
    rc = getattr(lib(), entry)(ctx.h, raw, _stream(dev))
    if rc:
        _check(ctx.h, rc, what)
    return loss, lse, dh, dw


def head_loss(ctx: Context, hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
              cfg: HeadLossConfig = HeadLossConfig()) -> Tuple[torch.Tensor, torch.Tensor]:
    """Loss and normaliser ln sum exp(hidden . weight_v) of each row (float32
    [N] both; 0 for ignored rows). hidden [N, D] and weight [V, D] of one of
    the three types, any row strides; labels int64 [N]. No host sync."""
    return _call(ctx, "zs_ce_loss", "head_loss", hidden, weight, labels, cfg)[:2]


def head_loss_grad(ctx: Context, hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                   row_grad: torch.Tensor, cfg: HeadLossConfig = HeadLossConfig(), need_hidden: bool = True,
                   need_weight: bool = True
                   ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """The loss per row and the gradients of sum_r row_grad[r] * loss[r] by
    the hidden states and by the weight, in their type (None where not
    needed). row_grad: float32 [N], or of no dimension for one value for all
    rows (a mean over the rows: 1 / N). No host sync."""
    what = "head_loss_grad"
    if not need_hidden and not need_weight:
        raise ValueError(f"{what}: no gradient wanted")
    N = hidden.shape[0] if hidden.dim() else 0
    if row_grad.dtype != torch.float32 or row_grad.device != hidden.device or row_grad.dim() > 1 or \
            (row_grad.dim() == 1 and row_grad.shape[0] != N):
        raise ValueError(f"{what}: row_grad is a float32 tensor [N] (or of no dimension: one value for all rows)")
    loss, _, dh, dw = _call(ctx, "zs_ce_loss_grad", what, hidden, weight, labels, cfg, row_grad, (need_hidden, need_weight))
    return loss, dh, dw


class _HeadLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(fctx, hidden, weight, labels, ctx, cfg):
        fctx.save_for_backward(hidden, weight, labels)
        fctx.zs = (ctx, cfg)
        return head_loss(ctx, hidden, weight, labels, cfg)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(fctx, row_grad):
        hidden, weight, labels = fctx.saved_tensors
        ctx, cfg = fctx.zs
        _, dh, dw = head_loss_grad(ctx, hidden, weight, labels, row_grad.float(), cfg, fctx.needs_input_grad[0],
                                   fctx.needs_input_grad[1])
        return dh, dw, None, None, None


class HeadLoss(torch.nn.Module):
    """Loss per row, differentiable by the hidden states and the weight. Keeps
    neither logits nor exponentials between the passes: the backward pass makes
    the logits again, 8 N V D operations in all for head_loss_grad's 6. (Where the rows' weights are known before the
    loss, head_loss_grad makes them once; it is also what belongs into a captured
    HIP graph: autograd's own bookkeeping of leaves that an eager graph holds too
    does not.)"""

    def __init__(self, ctx: Context, cfg: HeadLossConfig = HeadLossConfig()):
        super().__init__()
        self.ctx, self.cfg = ctx, cfg

    def forward(self, hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        return _HeadLossFunction.apply(hidden, weight, labels, self.ctx, self.cfg)


def _group_of(V: int, D: int, groups: int, what: str) -> int:
    group = D // groups if groups else 0
    if group not in GROUPS or group * groups != D or not 1 <= V <= MAX_VOCAB or not D <= MAX_HIDDEN:
        raise ValueError(f"{what}: groups are of 32, 64 or 128 columns, V 1 to {MAX_VOCAB}, D up to {MAX_HIDDEN}")
    return group


def q4_quantize(ctx: Context, weight: torch.Tensor, group: int = 32, mins: bool = False
                ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Codes (uint8 [V, D / 2]), scales and, asked for, minima (float16 [V, D /
    group]) of a weight [V, D] of any of the three types (zs_q4_quantize). What
    is not finite in a group makes its scale so, and its row's logits."""
    what = "q4_quantize"
    _matrix(ctx, weight, what, "weight")
    V, D = weight.shape
    if group not in GROUPS:
        raise ValueError(f"{what}: groups are of 32, 64 or 128 columns")
    _group_of(V, D, D // group, what)
    dev = weight.device
    codes = torch.empty((V, D // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty((V, D // group), dtype=torch.float16, device=dev)
    lows = torch.empty_like(scales) if mins else None
    rc = lib().zs_q4_quantize(ctx.h, weight.data_ptr(), _ld(weight), DTYPES[weight.dtype], V, D, group, codes.data_ptr(),
                              scales.data_ptr(), lows.data_ptr() if mins else None, _stream(dev))
    if rc:
        _check(ctx.h, rc, what)
    return codes, scales, lows


class Q4Head:
    """A head held in 4 bits: codes uint8 [V, D / 2] (0 to 15, the even
    column's in the low half of a byte), scales float16 [V, D / group] and
    perhaps minima likewise; w = scale * (code - 8), or scale * code + min. The
    codes are laid out once, when it is made; what it is made from is not kept.
    That is done when the constructor returns (a host sync, but in a captured
    graph), so logits may be asked for on any stream from then on, and a head
    that is dropped keeps its memory until the streams that it was called on are
    through. A captured graph has its address: keep the head as long as that."""

    def __init__(self, ctx: Context, codes: torch.Tensor, scales: torch.Tensor, mins: Optional[torch.Tensor] = None):
        what = "Q4Head"
        if codes.dim() != 2 or scales.dim() != 2:
            raise ValueError(f"{what}: codes are [V, D / 2], scales [V, D / group]")
        if codes.get_device() != ctx.device:
            raise ValueError(f"{what}: codes are on {codes.device}, not on the context's GPU {ctx.device}")
        dev, (V, half), groups = codes.device, codes.shape, scales.shape[1]
        self.ctx, self.V, self.D, self.group, self.mins = ctx, V, 2 * half, _group_of(V, 2 * half, groups, what), mins is not None
        _like(codes, (V, half), torch.uint8, dev, what, "codes")
        _like(scales, (V, groups), torch.float16, dev, what, "scales")
        if mins is not None:
            _like(mins, (V, groups), torch.float16, dev, what, "mins")
        self._data = torch.empty(_work_bytes("zs_q4_bytes", V, self.D, self.group, int(self.mins)), dtype=torch.uint8, device=dev)
        rc = lib().zs_q4_pack(ctx.h, codes.data_ptr(), scales.data_ptr(), mins.data_ptr() if self.mins else None, V, self.D,
                              self.group, self._data.data_ptr(), _stream(dev))
        if rc:
            _check(ctx.h, rc, what)
        self._streams = {_stream(dev)}
        with torch.cuda.device(dev):
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()

    def _called_on(self, stream: int, dev) -> None:
        """Another stream than those so far: torch's allocator is told of it, or
        it would give the memory of a dropped head to the first stream's next
        tensor while this one still reads it."""
        with torch.cuda.device(dev):
            if not torch.cuda.is_current_stream_capturing():
                self._data.record_stream(torch.cuda.current_stream())
                self._streams.add(stream)

    @classmethod
    def quantize(cls, ctx: Context, weight: torch.Tensor, group: int = 32, mins: bool = False) -> "Q4Head":
        return cls(ctx, *q4_quantize(ctx, weight, group, mins))

    def logits(self, hidden: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """float32 [B, V] for hidden [B, D] of any of the three types and any
        row stride. Without out the rows lie 4 values' multiples apart, as
        zs_sample and zs_lane_step take them. Not differentiable. No host
        sync."""
        what = "Q4Head.logits"
        _matrix(self.ctx, hidden, what, "hidden")
        B, dev = hidden.shape[0], hidden.device
        if hidden.shape[1] != self.D:
            raise ValueError(f"{what}: hidden is [B, {self.D}]")
        if dev != self._data.device:
            raise ValueError(f"{what}: hidden is on {dev}, the head on {self._data.device}")
        given = out is not None
        if not given:
            out = torch.empty((B, (self.V + 3) // 4 * 4), dtype=torch.float32, device=dev)[:, : self.V]
        elif out.shape != (B, self.V) or out.dtype != torch.float32 or out.device != dev or \
                (self.V > 1 and out.stride(1) != 1) or (B > 1 and out.stride(0) < self.V):
            raise ValueError(f"{what}: out is float32 [{B}, {self.V}], the values of a row adjacent")
        at, ld = hidden.data_ptr(), _ld(hidden)
        copy = hidden.dtype == torch.float32 or at % 16 != 0 or (B > 1 and ld % 8 != 0)
        nbytes = _work_bytes("zs_q4_logits_work", B, self.D, DTYPES[hidden.dtype], int(copy)) if copy or B > _FEW else 0
        work, work_at = _work(nbytes, dev)
        raw = _Q4.pack(self.V, self.D, self.group, int(self.mins), self._data.data_ptr(), B, DTYPES[hidden.dtype], at, ld,
                       out.data_ptr(), _ld(out), work_at, nbytes)
        stream = _stream(dev)
        if stream not in self._streams:
            self._called_on(stream, dev)
        rc = lib().zs_q4_logits(self.ctx.h, raw, stream)
        if rc:
            _check(self.ctx.h, rc, what)
        if given:
            increment_version(out)   # (autograd is told of writes in place)
        return out
