"""The autograd forms and the buffers that the optimizer reads."""
import pytest
import torch

import megatron_dion_amd as mda

pytestmark = pytest.mark.gpu


def _loss_case():
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(20, 64, generator=g).cuda(), torch.nn.Parameter(torch.randn(100, 64, generator=g).cuda())
    t = torch.randint(0, 100, (20,), generator=g).cuda()
    loss, lse = mda.linear_cross_entropy_forward(x, w.detach(), t)
    _, want = mda.linear_cross_entropy_backward(torch.ones(20, device="cuda"), x, w.detach(), t, lse)
    return x, w, t, want


def test_loss_adds_to_the_main_grad_of_the_backward_pass():
    """A buffer that is put in place between the passes takes the gradient; the one before is left alone."""
    x, w, t, want = _loss_case()
    before = w.main_grad = torch.zeros_like(w)
    loss = mda.linear_cross_entropy(x, w, t, into_main_grad=True)
    w.main_grad = torch.zeros_like(w)
    loss.sum().backward()
    assert torch.equal(w.main_grad, want) and (before == 0).all() and w.grad is None


def test_loss_without_a_main_grad_at_the_backward_pass():
    x, w, t, _ = _loss_case()
    w.main_grad = torch.zeros_like(w)
    loss = mda.linear_cross_entropy(x, w, t, into_main_grad=True)
    w.main_grad = None
    with pytest.raises(RuntimeError, match="DION_NO_MAIN_GRAD"):
        loss.sum().backward()


def test_loss_of_a_frozen_weight_leaves_its_main_grad():
    x, w, t, _ = _loss_case()
    w.main_grad = torch.zeros_like(w)
    w.requires_grad_(False)
    xg = x.clone().requires_grad_()
    mda.linear_cross_entropy(xg, w, t, into_main_grad=True).sum().backward()
    assert (w.main_grad == 0).all() and xg.grad.abs().sum() > 0


@pytest.mark.parametrize("used_before", [False, True])
def test_loss_on_another_stream_into_main_grad(used_before):
    """Forward on a side stream that is behind, backward from the default stream, which reads main_grad next."""
    x, w, t, want = _loss_case()
    w.main_grad = torch.zeros_like(w)
    other = w.sum() if used_before else 0.0  # the parameter's own node belongs to the default stream then
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = mda.linear_cross_entropy(x, w, t, into_main_grad=True)
    torch.cuda.current_stream().wait_stream(side)
    total = loss.sum() + other
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
    total.backward()
    got = w.main_grad.clone()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
