"""The operators of this package that have a backward pass, as differentiable functions on ROCm tensors: layer norm (with
the residual added ahead of it) and routing by scores.  Forward and backward are the HIP kernels behind ``ops``; what is
saved for the backward pass is the normalised tensor with its row statistics, or the logits with the chosen indices.
Where no gradient is asked for, nothing is saved.  Double backward is not supported; forward-mode derivatives are refused.

Capturing a training step into a HIP graph: PyTorch ties a parameter's gradient accumulator to the stream on which the first
graph that reaches it was built, so capture before an eager graph of the same parameters is alive (or after it has been
dropped), or call ``ops.layer_norm_backward`` / ``ops.route_topk_backward``, which take no part in autograd."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops


def _rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.reshape(-1, t.shape[-1]).contiguous()


class _LayerNorm(torch.autograd.Function):
    """Takes and returns tensors of the caller's shape: x and residual have one gradient, and autograd copies it for the second
    of two leaves only if both get the same tensor (not each a view of it, as a reshape ahead of this would make them)."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        rows = _rows(x)
        out, total, mean, rstd = ops.layer_norm(rows, weight, bias, eps, _rows(residual), want_stats=True)
        for t in (out, total):
            if t is not None:
                t.resize_(x.shape)      # (not a view: views that a Function returns refuse to be changed in place)
        ctx.save_for_backward(rows if total is None else total, weight, mean, rstd)
        ctx.bias_type = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        return out, total

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_sum):
        h, weight, mean, rstd = ctx.saved_tensors
        want_x, want_residual, want_weight, want_bias = ctx.needs_input_grad[:4]
        if grad_out is None:      # only the residual stream was used
            return (grad_sum if want_x else None, grad_sum if want_residual else None, None, None, None)
        grad, gw, gb = ops.layer_norm_backward(_rows(grad_out), _rows(h), weight, mean, rstd, _rows(grad_sum),
                                               want_grad=want_x or want_residual, want_weight=want_weight, want_bias=want_bias,
                                               param_dtype=ctx.bias_type)
        if grad is not None:
            grad = grad.view(grad_out.shape)
        return (grad if want_x else None, grad if want_residual else None, gw, gb, None)


class _RouteTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, choice_bias, k, scoring, n_groups, kept_groups, group_score, renormalise, scale, want_counts):
        routing, indices, weights, counts = ops.route_topk(logits, k, scoring, choice_bias, n_groups, kept_groups, group_score,
                                                           renormalise, scale, want_counts)
        ctx.save_for_backward(logits, indices)
        ctx.how = (scoring, renormalise, scale)
        ctx.mark_non_differentiable(*(t for t in (indices, counts) if t is not None))
        ctx.set_materialize_grads(False)
        return routing, indices, weights, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_routing, _indices, grad_weights, _counts):
        logits, indices = ctx.saved_tensors
        grad = None
        if ctx.needs_input_grad[0] and (grad_routing is not None or grad_weights is not None):
            grad = ops.route_topk_backward(logits, indices, *ctx.how,
                                           grad_routing=None if grad_routing is None else grad_routing.contiguous(),
                                           grad_weights=None if grad_weights is None else grad_weights.contiguous())
        return (grad,) + (None,) * 9


def _wanted(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a reverse-mode gradient is asked for.  Forward mode shows in no requires_grad: a tensor with a tangent would come
    out of the kernels without one, so it is refused here (looked for inside a dual level only: 0.3 us a tensor)."""
    if getattr(forward_ad, '_current_level', 0) >= 0 and \
            any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError('layer_norm and route_topk have no forward-mode derivative')
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               residual: Optional[torch.Tensor] = None):
    """Layer norm over the last dimension of x, or of h = x + residual; returns out without a residual and (out, h) with one.
    Leading dimensions are free; strided inputs are copied."""
    shape = x.shape
    if residual is not None and residual.shape != shape:
        raise ops.abi.D2DMoEError(f'layer_norm: residual has shape {tuple(residual.shape)}, x {tuple(shape)}')
    weight, bias = (None if p is None else p.contiguous() for p in (weight, bias))
    if _wanted(x, residual, weight, bias):
        out, total = _LayerNorm.apply(x, residual, weight, bias, eps)
    else:
        out, total, _, _ = ops.layer_norm(_rows(x), weight, bias, eps, _rows(residual))
        out, total = out.view(shape), None if total is None else total.view(shape)
    return out if residual is None else (out, total)


def route_topk(logits: torch.Tensor, k: int, scoring: str = 'softmax', choice_bias: Optional[torch.Tensor] = None,
               n_groups: int = 1, kept_groups: int = 1, group_score: str = 'top2', renormalise: bool = True, scale: float = 1.0,
               want_counts: bool = False):
    """Routing by scores over the last dimension of logits (see ops.route_topk); returns (routing, indices, weights, counts)
    with the leading dimensions of logits.  routing and weights are differentiable in the logits; the choice, and with it
    choice_bias, has no gradient."""
    lead = logits.shape[:-1]
    z = logits.reshape(-1, logits.size(-1)).contiguous()
    if choice_bias is not None:
        choice_bias = choice_bias.detach().contiguous()
    args = (k, scoring, n_groups, kept_groups, group_score, renormalise, scale, want_counts)
    if _wanted(logits):
        routing, indices, weights, counts = _RouteTopk.apply(z, choice_bias, *args)
    else:
        routing, indices, weights, counts = ops.route_topk(z, k, scoring, choice_bias, *args[2:])
    return routing.view(logits.shape), indices.view(*lead, k), weights.view(*lead, k), counts
