"""The autograd forms and the buffers that the optimizer reads."""
import pytest
import torch

import megatron_dion_amd as mda
from megatron_dion_amd.optimizer import attach_dp_routing

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


@pytest.mark.parametrize("dtype,main_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_norm_adds_to_main_grad(dtype, main_dtype, p):
    g = torch.Generator().manual_seed(5)
    x, r, gy = (torch.randn(33, 72, generator=g).to(dtype).cuda() for _ in range(3))
    w = torch.nn.Parameter((1 + 0.2 * torch.randn(72, generator=g)).cuda())
    rng = (3, 4) if p else None
    f = mda.rms_norm_add_forward(x, w.detach(), r, p=p, rng=rng)
    b = mda.rms_norm_add_backward(gy, f.h, w.detach(), f.rstd, None, p=p, rng=rng,
                                  grad_weight=torch.zeros(72, dtype=main_dtype, device="cuda"))
    xg, rg = x.clone().requires_grad_(), r.clone().requires_grad_()
    before = w.main_grad = torch.zeros(72, dtype=main_dtype, device="cuda")
    y, _ = mda.rms_norm_add(xg, w, rg, p=p, rng=rng, into_main_grad=True)
    w.main_grad = torch.zeros(72, dtype=main_dtype, device="cuda")
    y.backward(gy)
    assert torch.equal(w.main_grad, b.grad_weight) and (before == 0).all() and w.grad is None
    assert torch.equal(xg.grad, b.grad_x) and torch.equal(rg.grad, b.grad_residual)
    y, h = mda.rms_norm_add(xg, w, rg, p=p, rng=rng, into_main_grad=True)
    h.sum().backward()  # only the residual stream: nothing for the weight
    assert torch.equal(w.main_grad, b.grad_weight)
    opt = mda.MegatronDion([w], lr=0.01)
    attach_dp_routing(opt, [("norm.weight", w)])
    w0 = w.detach().clone()
    opt.step()
    assert torch.isfinite(w).all() and not torch.equal(w.detach(), w0)
    del w.main_grad
    with pytest.raises(RuntimeError, match="DION_NO_MAIN_GRAD"):
        mda.rms_norm_add(xg, w, rg, p=p, rng=rng, into_main_grad=True)
