"""The training operators of `lm_ops.py` for autograd.

Thin `torch.autograd.Function`s over the explicit calls.  They are for eager training steps and refuse
to run while the current stream is being captured (`[DION_AUTOGRAD_CAPTURE]`): autograd runs a leaf's
accumulation on the stream that first used it, which a capture does not survive.  A captured step makes
the explicit forward and backward calls instead.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import lm_ops

__all__ = ["linear_cross_entropy", "rms_norm_add", "dropout_add"]


def _eager(what: str) -> None:
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"[DION_AUTOGRAD_CAPTURE] {what} under graph capture: make the explicit "
                           "*_forward / *_backward calls there")


def _held(rng):
    # a generator state on the device may move on before the backward pass needs this mask again
    return rng.clone() if isinstance(rng, torch.Tensor) else rng


def _rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    # incoming gradients have any strides (an expanded scalar, a transposed view)
    return None if t is None else t.contiguous()


def _main_grad(weight: torch.Tensor) -> torch.Tensor:
    main = getattr(weight, "main_grad", None)
    if main is None:
        raise RuntimeError("[DION_NO_MAIN_GRAD] into_main_grad: weight has no main_grad")
    return main


def _backward_waits_for(device: torch.device) -> None:
    """The caller of backward() finds main_grad written: autograd joins the streams of the gradients that it
    hands on, and this one it does not know."""
    done = torch.cuda.current_stream(device).record_event()
    torch.autograd.Variable._execution_engine.queue_callback(
        lambda: torch.cuda.current_stream(device).wait_event(done))


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, kwargs, owner):
        _eager("linear_cross_entropy")
        loss, lse = lm_ops.linear_cross_entropy_forward(hidden, weight, target, **kwargs)
        ctx.save_for_backward(hidden, weight, target, lse)
        ctx.kwargs, ctx.owner = kwargs, owner
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        _eager("linear_cross_entropy")
        hidden, weight, target, lse = ctx.saved_tensors
        need_h, need_w = ctx.needs_input_grad[:2]
        # the owner's main_grad of now: the optimizer may have been given another buffer since the forward pass
        main = _main_grad(ctx.owner) if need_w and ctx.owner is not None else None
        gh, gw = lm_ops.linear_cross_entropy_backward(
            _rows(grad_loss), hidden, weight, target, lse, grad_weight=main, accumulate=main is not None,
            need_hidden=need_h, need_weight=need_w, **ctx.kwargs)
        if main is not None:
            _backward_waits_for(main.device)
        return gh, None if main is not None else gw, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, vocab_start: int = 0,
                         vocab_size: Optional[int] = None, ignore_index: int = -100, group=None,
                         into_main_grad: bool = False) -> torch.Tensor:
    """Each token's cross entropy of `hidden @ weight.T` (fp32, target's shape), differentiable in hidden
    and weight.  `into_main_grad`: the backward pass adds weight's gradient to the `weight.main_grad` it finds,
    where the optimizer reads it, on the stream of the forward pass, and leaves `weight.grad` and the
    parameter's hooks alone: what waits for such a hook (an overlapped gradient reduction) has to be told
    otherwise."""
    if into_main_grad:
        _main_grad(weight)
    kwargs = dict(vocab_start=vocab_start, vocab_size=vocab_size, ignore_index=ignore_index, group=group)
    return _LinearCrossEntropy.apply(hidden, weight, target, kwargs, weight if into_main_grad else None)


class _RmsNormAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, p, rng, owner):
        _eager("rms_norm_add")
        f = lm_ops.rms_norm_add_forward(x, weight, residual, eps=eps, p=p, rng=rng)
        ctx.save_for_backward(f.h, weight, f.rstd)
        ctx.p, ctx.rng, ctx.stored, ctx.owner = p, _held(rng), f.h is not x, owner
        ctx.set_materialize_grads(False)
        return (f.y, f.h) if ctx.stored else f.y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_h=None):
        _eager("rms_norm_add")
        h, weight, rstd = ctx.saved_tensors
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if grad_y is None and grad_h is None:
            return (None,) * 7
        if grad_y is None:  # only the residual stream was used
            g = _rows(grad_h)
            gx = lm_ops.dropout_add_backward(g, p=ctx.p, rng=ctx.rng) if need_x and ctx.p > 0.0 else g
            return gx if need_x else None, None, g if need_r else None, None, None, None, None
        main = _main_grad(ctx.owner) if need_w and ctx.owner is not None else None
        b = lm_ops.rms_norm_add_backward(_rows(grad_y), h, weight, rstd, _rows(grad_h), p=ctx.p, rng=ctx.rng,
                                         grad_weight=main, accumulate=main is not None,
                                         need_input=need_x or need_r, need_weight=need_w, need_residual=need_r)
        if main is not None:
            _backward_waits_for(main.device)
        return (b.grad_x if need_x else None, None if main is not None else b.grad_weight,
                b.grad_residual if need_r else None, None, None, None, None)


def rms_norm_add(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-5, p: float = 0.0, rng: Optional[lm_ops.Rng] = None, into_main_grad: bool = False
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h): `h = residual + dropout(x)` and its RMS norm, differentiable in x, weight and residual.
    `into_main_grad` as in `linear_cross_entropy`.  The 8-bit output has no form here: nothing
    differentiates it, and the explicit calls give it with its gradients."""
    if into_main_grad:
        _main_grad(weight)
    out = _RmsNormAdd.apply(x, weight, residual, eps, p, rng, weight if into_main_grad else None)
    return out if isinstance(out, tuple) else (out, x)


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng):
        _eager("dropout_add")
        ctx.p, ctx.rng = p, _held(rng)
        return lm_ops.dropout_add_forward(x, residual, p=p, rng=rng)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _eager("dropout_add")
        grad = _rows(grad)
        gx = lm_ops.dropout_add_backward(grad, p=ctx.p, rng=ctx.rng) if ctx.needs_input_grad[0] else None
        return gx, grad if ctx.needs_input_grad[1] else None, None, None


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor] = None, *, p: float,
                rng: Optional[lm_ops.Rng] = None) -> torch.Tensor:
    """`residual + dropout(x)`, differentiable in both."""
    return _DropoutAdd.apply(x, residual, p, rng)
