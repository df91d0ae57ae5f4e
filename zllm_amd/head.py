"""The vocabulary head over libzs: its cross entropy from hidden states, without
logits, with the gradients.

    loss_of = HeadLoss(ctx)
    loss_of(hidden, head_weight, labels).mean().backward()

or, without autograd, head_loss (evaluation, the scores of given tokens: their
log-probabilities are -loss) and head_loss_grad. The formulas are in
include/zs.h. The reference trains nothing; there is no counterpart.
torch holds the device memory and the stream; the computation is libzs's.
"""
import ctypes as C
import struct
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from ._lib import Ce, lib
from .beam import DTYPES, MAX_VOCAB, _ld, _like, _stream, _work, _work_bytes
from .engine import Context, _check

MAX_HIDDEN = 65536
MAX_LD = 4194304
_DHIDDEN, _DWEIGHT, _COPY = 1, 2, 4
# the arguments are packed to bytes, as zllm_amd.beam's
_CE = struct.Struct("=4I2Q3QqfI10Q")
assert _CE.size == C.sizeof(Ce)


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
    out = torch.empty((2, N), dtype=torch.float32, device=dev)
    loss, lse = out.unbind(0)
    dh = torch.empty((N, D), dtype=hidden.dtype, device=dev) if want[0] else None
    dw = torch.empty((V, D), dtype=hidden.dtype, device=dev) if want[1] else None
    bits = (_DHIDDEN if want[0] else 0) | (_DWEIGHT if want[1] else 0)
    at, ldw = weight.data_ptr(), _ld(weight)
    if hidden.dtype == torch.float32 or at % 16 or D % 8 or (V > 1 and ldw % 8) or ldw > MAX_LD:
        bits |= _COPY
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
    the logits again, in pieces. (Where the rows' weights are known before the
    loss, head_loss_grad makes them once.)"""

    def __init__(self, ctx: Context, cfg: HeadLossConfig = HeadLossConfig()):
        super().__init__()
        self.ctx, self.cfg = ctx, cfg

    def forward(self, hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        return _HeadLossFunction.apply(hidden, weight, labels, self.ctx, self.cfg)
