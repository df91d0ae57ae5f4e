"""What beam search and distillation owe their callers beside their numbers: the
loop that the module documents, writes that autograd sees, tensors of another
device than the context's."""
import textwrap
import types

import pytest
import torch

from tests.test_gpu_beam import _ctx

pytestmark = pytest.mark.gpu


def documented_loop():
    """The indented lines of zllm_amd.beam's docstring."""
    from zllm_amd import beam
    lines = beam.__doc__.splitlines()
    return textwrap.dedent("\n".join(l for l in lines if l.startswith("    ")))


def test_the_documented_loop_runs():
    """Under a model that takes ids of its vocabulary alone, with beams that are
    absent after the first step (fewer ids allowed than beams)."""
    from zllm_amd import beam
    V, groups, width = 50, 2, 3
    table = torch.randn((V, V), generator=torch.Generator().manual_seed(1))
    table[7:9, 3:] = -float("inf")
    table[7:9, 2] = -float("inf")           # two ids at the first step: the third beam is absent

    def model(tokens, *_):
        assert tokens.shape == (groups * width,)
        return torch.nn.functional.embedding(tokens.cpu(), table).cuda()     # (an id outside raises here)
    names = dict(vars(beam), ctx=_ctx(), groups=groups, width=width, max_steps=5, g=1, model=model,
                 first=torch.tensor([7, 8], device="cuda").repeat_interleave(width),
                 kv_cache=torch.zeros((2, 2, groups * width, 2, 5, 8), device="cuda"),
                 grammar_state=torch.zeros(groups * width, dtype=torch.int32, device="cuda"))
    print("[case] the documented loop", flush=True)
    exec(documented_loop(), names)
    assert names["best"] and all(0 <= t < V for t in names["best"])


def test_before_the_first_step_every_beam_is_absent():
    from zllm_amd.beam import BeamSearch
    for steps in (0, 1, 4):
        s = BeamSearch(_ctx(), 2, 3, steps)
        assert (s.parents == -1).all() and (s.tokens == -1).all() and s.tokens.shape == (2, 3)
        assert s.sequences() == [[], []] and s.finished() == (steps == 0)


def lists(N, V, K=4):
    ids = torch.arange(K, dtype=torch.int32, device="cuda").expand(N, K).contiguous()
    return ids, torch.full((N, K), -1.6, device="cuda")


def test_gradients_written_over_saved_logits_are_seen():
    """A backward pass over logits that were overwritten since raises, as it
    does after any in-place operation."""
    from zllm_amd.distill import DistillConfig, DistillLoss, distill_grad, distill_loss, distill_loss_grad
    N, V = 3, 40
    ids, logp = lists(N, V)
    cfg, w = DistillConfig(), torch.ones(N, device="cuda")
    for write in ("grad", "both"):
        leaf = torch.randn((N, V), device="cuda", requires_grad=True)
        logits = leaf * 1.0
        loss = DistillLoss(_ctx(), cfg)(logits, ids, logp).sum()
        over = logits.detach()
        if write == "grad":
            stats = distill_loss(_ctx(), over, ids, logp, cfg)[1]
            distill_grad(_ctx(), over, ids, logp, cfg, stats, w, out=over)
        else:
            distill_loss_grad(_ctx(), over, ids, logp, cfg, w, out=over)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_states_and_steps_written_in_place_are_seen():
    from zllm_amd.beam import BeamPool, BeamStates, BeamStep, beam_reorder, beam_select
    state = torch.randn((4, 2, 5), device="cuda")
    view = state[:, :, 1:]
    parents = torch.tensor([[1, 0], [0, 0]], dtype=torch.int32, device="cuda")
    before = state._version
    beam_reorder(_ctx(), BeamStates([(view, 0)], 2), parents)
    assert state._version > before
    logits, scores, pool = torch.randn((4, 9), device="cuda"), torch.zeros((2, 2), device="cuda"), BeamPool.empty(2, 2)
    out = BeamStep(torch.empty_like(parents), torch.empty_like(parents), scores, pool)
    written = [out.parents, out.tokens, scores] + [getattr(pool, k) for k in ("score", "length", "parent", "token", "steps",
                                                                              "done")]
    before = [t._version for t in written]
    beam_select(_ctx(), logits, scores, pool, out=out)
    assert all(t._version > b for t, b in zip(written, before))


def test_inference_tensors_are_taken():
    """(they have no version)"""
    from zllm_amd.beam import BeamStates, beam_reorder
    with torch.inference_mode():
        state = torch.arange(4, dtype=torch.int32, device="cuda")
        beam_reorder(_ctx(), BeamStates([(state, 0)], 2), torch.tensor([[1, 0], [0, 0]], dtype=torch.int32, device="cuda"))
    assert state.tolist() == [1, 0, 2, 2]


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
