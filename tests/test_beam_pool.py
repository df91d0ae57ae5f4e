"""A pool's tensors are looked at in every call (no GPU): one that was resized or
put elsewhere since the last is not written past its end."""
import pytest
import torch

from zllm_amd.beam import BeamPool

DEV = torch.device("cpu")
NAMES = ("score", "length", "parent", "token", "steps", "done")


def pool(G=3, W=4):
    p = BeamPool.empty(G, W, "cpu")
    assert p._pointers(3, 4, DEV, "step") == tuple(getattr(p, n).data_ptr() for n in NAMES)
    return p


@pytest.mark.parametrize("name", NAMES)
def test_changed_tensors_are_refused(name):
    for change in (lambda t: t.resize_(1), lambda t: t.resize_(7, 9), lambda t: t.set_(torch.empty(2, dtype=t.dtype)),
                   lambda t: setattr(t, "data", torch.empty((3, 8), dtype=t.dtype)[:, ::2]),
                   lambda t: setattr(t, "data", t.to(torch.int64)), lambda t: t.unsqueeze_(0)):
        p = pool()
        change(getattr(p, name))
        with pytest.raises(ValueError, match="pool." + name):
            p._pointers(3, 4, DEV, "step")


def test_a_pool_of_other_sizes_is_refused():
    for G, W in ((3, 3), (4, 4), (4, 3), (1, 12)):
        with pytest.raises(ValueError, match="pool"):
            pool()._pointers(G, W, DEV, "step")


def test_tensors_put_elsewhere_are_taken_there():
    p = pool()
    for n in NAMES:
        t = getattr(p, n)
        t.data = t.clone()
    assert p._pointers(3, 4, DEV, "step") == tuple(getattr(p, n).data_ptr() for n in NAMES)


def test_a_steps_own_pool():
    from zllm_amd.beam import BeamStep
    p = BeamStep.alloc(3, 4, DEV).pool
    p._pointers(3, 4, DEV, "step")
    p.token.resize_(1)
    with pytest.raises(ValueError, match="pool.token"):
        p._pointers(3, 4, DEV, "step")
