"""Distils a draft model from a teacher's beams: the teacher decodes with beam
search (its per-beam states follow the beams), its likeliest ids are taken at
every position, and the draft learns them. Both models are tables of logits by
the last token. Prints the draft's loss before and after.

    python examples/distill_draft.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from zllm_amd.beam import BeamSearch, BeamStates, beam_reorder  # noqa: E402
from zllm_amd.distill import DistillConfig, DistillLoss, teacher_topk  # noqa: E402
from zllm_amd.engine import Context  # noqa: E402


def run(ctx, vocab=1000, groups=4, width=4, steps=12, epochs=40, seed=0):
    """(first loss, last loss), means over the teacher's tokens."""
    g = torch.Generator().manual_seed(seed)
    teacher = (2.0 * torch.randn(vocab, vocab, generator=g)).cuda()
    draft = torch.zeros(vocab, vocab, device="cuda", requires_grad=True)
    search = BeamSearch(ctx, groups, width, steps, eos=(0,))
    history = torch.zeros((groups * width, steps + 1), dtype=torch.int64, device="cuda")   # a beam's own state
    history[:, 0] = torch.arange(1, groups + 1).repeat_interleave(width).cuda()
    states = BeamStates([(history, 0)], width)
    while not search.finished():
        t = search.t
        search.step(teacher[history[:, t]])
        beam_reorder(ctx, states, search.parents)
        history[:, t + 1] = search.tokens.view(-1).clamp_min(0)
    seen, labels = history[:, : search.t].reshape(-1), history[:, 1 : search.t + 1].reshape(-1)
    ids, logp = teacher_topk(ctx, teacher[seen], 32)[:2]
    loss_of = DistillLoss(ctx, DistillConfig())
    losses = []
    for _ in range(epochs):
        loss = loss_of(draft[seen], ids, logp, labels).mean()
        draft.grad = None
        loss.backward()
        losses.append(float(loss.detach()))
        with torch.no_grad():
            draft -= 20.0 * draft.grad
    return losses[0], losses[-1]


if __name__ == "__main__":
    first, last = run(Context())
    print(f"loss {first:.4f} -> {last:.4f}")
