"""What beam search and distillation owe their callers beside their numbers:
tensors of another device than the context's."""
import types

import pytest
import torch

from tests.test_gpu_beam import _ctx

pytestmark = pytest.mark.gpu


def lists(N, V, K=4):
    ids = torch.arange(K, dtype=torch.int32, device="cuda").expand(N, K).contiguous()
    return ids, torch.full((N, K), -1.6, device="cuda")


def test_tensors_of_another_device_than_the_contexts_are_refused():
    from zllm_amd.beam import BeamPool, BeamStates, beam_reorder, beam_select
    from zllm_amd.distill import DistillConfig, distill_grad, distill_loss, distill_loss_grad, teacher_topk
    other = types.SimpleNamespace(device=1, h=None)          # a context of the second GPU
    x = torch.zeros((4, 30), device="cuda")
    ids, logp = lists(4, 30)
    w, cfg = torch.ones(4, device="cuda"), DistillConfig()
    parents = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    for f in (lambda: beam_select(other, x, torch.zeros((2, 2), device="cuda"), BeamPool.empty(2, 2)),
              lambda: beam_reorder(other, BeamStates([(x, 0)], 2), parents),
              lambda: teacher_topk(other, x, 3), lambda: distill_loss(other, x, ids, logp, cfg),
              lambda: distill_grad(other, x, ids, logp, cfg, torch.zeros((4, 4), device="cuda"), w),
              lambda: distill_loss_grad(other, x, ids, logp, cfg, w)):
        with pytest.raises(ValueError, match="context"):
            f()
