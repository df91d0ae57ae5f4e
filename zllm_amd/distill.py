"""Distillation of a draft model from a teacher's top logits over libzs.

    ids, logp, _ = teacher_topk(ctx, teacher_logits, 64, temperature)   # once, kept with the tokens
    loss = DistillLoss(ctx, DistillConfig(temperature, tail=True))
    loss(draft_logits, ids, logp, labels).mean().backward()

or, without autograd, distill_loss / distill_grad / distill_loss_grad. The
formulas are in include/zs.h. The reference trains nothing; there is no
counterpart. torch holds the device memory and the stream; the computation is
libzs's.
"""
import ctypes as C
import struct
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from ._lib import Distill, Teacher, lib
from .beam import DTYPES, MAX_VOCAB, _ld, _like, _rows, _stream, _work, _work_bytes
from .engine import Context, _check

MAX_TOP = 128
ZS_DISTILL_TAIL = 1
# the arguments are packed to bytes, as zllm_amd.beam's
_TEACHER = struct.Struct("=4I2QfI5Q")
_DISTILL = struct.Struct("=4IQ4Qq3fI8Q")
assert _TEACHER.size == C.sizeof(Teacher) and _DISTILL.size == C.sizeof(Distill)


def teacher_topk(ctx: Context, logits: torch.Tensor, K: int, temperature: float = 1.0
                 ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The K largest of each row of logits [N, V] (ties by the lower id): ids
    int32 [N, K], ln softmax(logits / temperature) there float32 [N, K], and
    ln sum exp(logits / temperature) float32 [N] (zs_teacher_topk). Rows of
    fewer than K values above -inf end with ids -1, logp -inf. No host sync."""
    what = "teacher_topk"
    _rows(ctx, logits, what)
    N, V = logits.shape
    if not 1 <= K <= min(V, MAX_TOP):
        raise ValueError(f"{what}: K is 1 to min(V, {MAX_TOP})")
    dev = logits.device
    ids = torch.empty((N, K), dtype=torch.int32, device=dev)
    logp = torch.empty((N, K), dtype=torch.float32, device=dev)
    lse = torch.empty(N, dtype=torch.float32, device=dev)
    nbytes = _work_bytes("zs_teacher_topk_work", N, V, K) if N and V <= MAX_VOCAB else 0
    work, at = _work(nbytes, dev)
    raw = _TEACHER.pack(N, V, K, DTYPES[logits.dtype], _ld(logits), logits.data_ptr(), temperature, 0, ids.data_ptr(),
                        logp.data_ptr(), lse.data_ptr(), at, nbytes)
    rc = lib().zs_teacher_topk(ctx.h, raw, _stream(dev))
    if rc:
        _check(ctx.h, rc, what)
    return ids, logp, lse


@dataclass(frozen=True)
class DistillConfig:
    """loss = kl_weight * KL + ce_weight * CE. tail: the ids outside the list
    are one more outcome with what the teacher's list leaves; else the list is
    renormalised. (kl_weight = T^2 keeps the gradients' size over T.)"""
    temperature: float = 1.0
    kl_weight: float = 1.0
    ce_weight: float = 0.0
    tail: bool = False
    ignore_index: int = -100


def _call(ctx, entry, what, logits, ids, logp, cfg, labels, loss=0, stats=0, row_grad=0, row_grad_stride=0, grad=0,
          ld_grad=0):
    _rows(ctx, logits, what)
    N, V = logits.shape
    dev = logits.device
    if ids.dim() != 2 or ids.shape[0] != N or not 1 <= ids.shape[1] <= MAX_TOP:
        raise ValueError(f"{what}: ids are [N, K], K 1 to {MAX_TOP}")
    K = ids.shape[1]
    _like(ids, (N, K), torch.int32, dev, what, "ids")
    _like(logp, (N, K), torch.float32, dev, what, "logp")
    lab = 0 if labels is None else _like(labels, (N,), torch.int64, dev, what, "labels").data_ptr()
    nbytes = _work_bytes("zs_distill_work", N, V, K) if N and 0 < V <= MAX_VOCAB else 0
    work, at = _work(nbytes, dev)
    raw = _DISTILL.pack(N, V, K, DTYPES[logits.dtype], _ld(logits), logits.data_ptr(), ids.data_ptr(), logp.data_ptr(),
                        lab, cfg.ignore_index, cfg.temperature, cfg.kl_weight, cfg.ce_weight,
                        ZS_DISTILL_TAIL if cfg.tail else 0, loss, stats, row_grad, row_grad_stride, grad, ld_grad, at,
                        nbytes)
    rc = getattr(lib(), entry)(ctx.h, raw, _stream(dev))
    if rc:
        _check(ctx.h, rc, what)


def _grad(ctx, what, logits, row_grad, out):
    """The gradient's arguments and its tensor."""
    _rows(ctx, logits, what)
    N = logits.shape[0]
    dev = logits.device
    if row_grad.dtype != torch.float32 or row_grad.device != dev or row_grad.dim() > 1 or \
            (row_grad.dim() == 1 and row_grad.shape[0] != N):
        raise ValueError(f"{what}: row_grad is a float32 tensor [N] (or of no dimension: one value for all rows)")
    if out is None:
        out = torch.empty_like(logits)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev or \
            (out.shape[1] > 1 and out.stride(1) != 1) or (N > 1 and out.stride(0) < out.shape[1]):
        raise ValueError(f"{what}: out is like logits, the values of a row adjacent")
    # (the stride is 0 too for a value expanded over the rows)
    return dict(row_grad=row_grad.data_ptr(), row_grad_stride=row_grad.stride(0) if row_grad.dim() else 0,
                grad=out.data_ptr(), ld_grad=_ld(out)), out


def distill_loss(ctx: Context, logits: torch.Tensor, ids: torch.Tensor, logp: torch.Tensor, cfg: DistillConfig,
                 labels: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Loss per row (float32 [N]) of the student's logits [N, V] against the
    teacher's list, and what the backward pass needs of the rows (float32
    [N, 4]). labels: int64 [N], cfg.ignore_index marks rows of no loss."""
    N = logits.shape[0]
    loss = torch.empty(N, dtype=torch.float32, device=logits.device)
    stats = torch.empty((N, 4), dtype=torch.float32, device=logits.device)
    _call(ctx, "zs_distill_loss", "distill_loss", logits, ids, logp, cfg, labels, loss.data_ptr(), stats.data_ptr())
    return loss, stats


def distill_grad(ctx: Context, logits: torch.Tensor, ids: torch.Tensor, logp: torch.Tensor, cfg: DistillConfig,
                 stats: torch.Tensor, row_grad: torch.Tensor, labels: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of sum_r row_grad[r] * loss[r] by the logits, in their type;
    stats from distill_loss. out may be the logits themselves."""
    what = "distill_grad"
    given = out is not None
    kw, out = _grad(ctx, what, logits, row_grad, out)
    st = _like(stats, (logits.shape[0], 4), torch.float32, logits.device, what, "stats").data_ptr()
    _call(ctx, "zs_distill_grad", what, logits, ids, logp, cfg, labels, stats=st, **kw)
    if given:
        increment_version(out)   # (autograd is told of writes in place)
    return out


def distill_loss_grad(ctx: Context, logits: torch.Tensor, ids: torch.Tensor, logp: torch.Tensor, cfg: DistillConfig,
                      row_grad: torch.Tensor, labels: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None
                      ) -> Tuple[torch.Tensor, torch.Tensor]:
    """distill_loss and distill_grad in one call, where the rows' weights are
    known before the loss (a mean over the rows: row_grad = 1 / N)."""
    what = "distill_loss_grad"
    given = out is not None
    kw, out = _grad(ctx, what, logits, row_grad, out)
    loss = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
    _call(ctx, "zs_distill_loss_grad", what, logits, ids, logp, cfg, labels, loss.data_ptr(), **kw)
    if given:
        increment_version(out)
    return loss, out


class _DistillFunction(torch.autograd.Function):
    @staticmethod
    def forward(fctx, logits, ids, logp, labels, ctx, cfg):
        loss, stats = distill_loss(ctx, logits, ids, logp, cfg, labels)
        fctx.save_for_backward(logits, ids, logp, labels, stats)
        fctx.zs = (ctx, cfg)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(fctx, row_grad):
        logits, ids, logp, labels, stats = fctx.saved_tensors
        ctx, cfg = fctx.zs
        return distill_grad(ctx, logits, ids, logp, cfg, stats, row_grad.float(), labels), None, None, None, None, None


class DistillLoss(torch.nn.Module):
    """Loss per row, differentiable by the student's logits (the teacher's
    list is a constant)."""

    def __init__(self, ctx: Context, cfg: DistillConfig = DistillConfig()):
        super().__init__()
        self.ctx, self.cfg = ctx, cfg

    def forward(self, logits: torch.Tensor, ids: torch.Tensor, logp: torch.Tensor,
                labels: Optional[torch.Tensor] = None) -> torch.Tensor:
        return _DistillFunction.apply(logits, ids, logp, labels, self.ctx, self.cfg)
