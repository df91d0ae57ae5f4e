"""HeadLoss's loss is the caller's own tensor: it may be changed in place, before
and without autograd."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _case():
    from tests.gpu_util import ctx
    gen = torch.Generator("cuda").manual_seed(1)
    h = torch.randn((20, 64), device="cuda", generator=gen)
    W = torch.randn((300, 64), device="cuda", generator=gen) / 8
    labels = torch.randint(0, 300, (20,), device="cuda", generator=gen)
    return ctx(), h, W, labels


def test_a_loss_changed_in_place():
    from zllm_amd.head import HeadLoss
    ctx, h, W, labels = _case()
    grads = []
    for inplace in (False, True):
        a, b = h.clone().requires_grad_(), W.clone().requires_grad_()
        loss = HeadLoss(ctx)(a, b, labels)
        mask = torch.arange(20, device="cuda") < 5
        if inplace:
            loss[mask] = 0.0
            loss /= 20
        else:
            loss = torch.where(mask, 0.0, loss) / 20
        loss.sum().backward()
        grads.append((a.grad, b.grad))
    assert all(torch.equal(x, y) for x, y in zip(*grads)) and bool((grads[1][0][:5] == 0).all())


def test_losses_that_take_a_gradient_in():
    """What head_loss gives is no view either: a term with a gradient may be added."""
    from zllm_amd.head import head_loss, head_loss_grad
    ctx, h, W, labels = _case()
    x = torch.ones(20, device="cuda", requires_grad=True)
    for t in (*head_loss(ctx, h, W, labels), head_loss_grad(ctx, h, W, labels, torch.tensor(0.1, device="cuda"))[0]):
        assert not t._is_view()
        t += x
        t.sum().backward()
    assert bool((x.grad == 3.0).all())
