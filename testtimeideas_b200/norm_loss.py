"""The two ends of a block and of a loss next to the attention: layer norm and
the linear cross entropy, each differentiable twice on the sm_100a kernels.

The meta step (``ttt_model.meta_step``) takes the gradient of a gradient through
every op of the inner step: the norms of each block and the token loss among
them. Both operators here follow the attention's form: an autograd Function
whose backward is itself a Function with a closed-form backward; a third
derivative raises. CUDA tensors run the kernels (C ABI in include/ttt_ops.h);
CPU tensors run the PyTorch formulation of the same value.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F
from torch import nn

from . import _lib


def _kernel_path(x: torch.Tensor) -> bool:
    """True when the call runs the CUDA kernels (every CUDA tensor)."""
    return x.is_cuda


class _LastFn(torch.autograd.Function):
    """apply(count, *outputs, *inputs): the outputs, tied to the inputs they were
    computed from by a backward that raises. (torch's once_differentiable leaves
    no path to the inputs, so torch.autograd.grad would skip its error.)"""

    @staticmethod
    def forward(ctx, count, *tensors):
        outs = tuple(t.view_as(t) for t in tensors[:count])
        return outs

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the second gradient of this op is not differentiable (a third derivative was requested)")


def _last(outputs, inputs):
    """The tensors of `outputs` (None stays None), with a third derivative made to raise."""
    if not torch.is_grad_enabled():
        return outputs
    real = [o for o in outputs if o is not None]
    tied = iter(_LastFn.apply(len(real), *real, *[t for t in inputs if t is not None]))
    return tuple(None if o is None else next(tied) for o in outputs)


# ---------------------------------------------------------------- layer norm
class _LayerNormBwdFn(torch.autograd.Function):
    """The gradient as a differentiable op: (dy, x, w) -> (dx, dw, db)."""

    @staticmethod
    def forward(ctx, dy, x, w, mean, rstd, need, p_type):
        dx, dw, db = _lib.layer_norm_bwd(dy, x, w, mean, rstd, need, p_type)
        ctx.save_for_backward(dy, x, w, mean, rstd)
        ctx.set_materialize_grads(False)
        return dx, dw, db

    @staticmethod
    def backward(ctx, ux, uw, ub):
        dy, x, w, mean, rstd = ctx.saved_tensors
        if ux is None and uw is None and ub is None:
            return (None,) * 7
        with torch.no_grad():
            gdy, gx, gw = _lib.layer_norm_bwd2(dy, x, w, mean, rstd, ux, uw, ub)
            grads = gdy.to(dy.dtype), gx, None if w is None else gw
        return (*_last(grads, (dy, x, w, ux, uw, ub)), None, None, None, None)


class LayerNormFn(torch.autograd.Function):
    """apply(x, weight, bias, eps): layer norm over the last dimension."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps: float):
        y, mean, rstd = _lib.layer_norm(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.set_materialize_grads(False)
        ctx.p_type = next((p.dtype for p in (weight, bias) if p is not None), x.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None
        x, weight, mean, rstd = ctx.saved_tensors
        need = tuple(ctx.needs_input_grad[:3])
        fn = _LayerNormBwdFn.apply if torch.is_grad_enabled() else _lib.layer_norm_bwd
        dx, dw, db = fn(dy, x, weight, mean, rstd, need, ctx.p_type)
        return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x: [..., dim] in fp16, bf16 or fp32, any strides (a layout that is not rows
    of unit stride is copied); weight, bias: [dim] in x's dtype or fp32, either
    may be None. On CUDA dim is at most 16384; statistics and sums are fp32.
    Differentiable twice in x, weight and the upstream gradient."""
    if not _kernel_path(x):
        return F.layer_norm(x, x.shape[-1:], weight, bias, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return LayerNormFn.apply(x, weight, bias, float(eps))
    return _lib.layer_norm(x, weight, bias, float(eps), False)[0]


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension (same parameters and state dict) on the kernels."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm normalizes one dimension, got {self.normalized_shape}")
        return layer_norm(x, self.weight, self.bias, self.eps)


# ---------------------------------------------------------------- linear cross entropy
class _LinearCEBwdFn(torch.autograd.Function):
    """The gradient as a differentiable op: (dloss, h, w) -> (dh, dw)."""

    @staticmethod
    def forward(ctx, dloss, h, w, state, reduction, need):
        dh, dw = _lib.linear_ce_bwd(dloss, h, w, state, reduction, need)
        ctx.save_for_backward(dloss, h, w, state)
        ctx.reduction = reduction
        ctx.set_materialize_grads(False)
        return dh, dw

    @staticmethod
    def backward(ctx, uh, uw):
        dloss, h, w, state = ctx.saved_tensors
        if uh is None and uw is None:
            return (None,) * 6
        need = tuple(ctx.needs_input_grad[:3])
        with torch.no_grad():
            grads = _lib.linear_ce_bwd2(dloss, h, w, state, ctx.reduction, uh, uw, need)
            grads = tuple(g if n else None for g, n in zip(grads, need))
        return (*_last(grads, (dloss, h, w, uh, uw)), None, None, None)


class LinearCrossEntropyFn(torch.autograd.Function):
    """apply(h, w, targets, mask, reduction, ignore_index): see linear_cross_entropy."""

    @staticmethod
    def forward(ctx, h, w, targets, mask, reduction: str, ignore_index: int):
        loss, state = _lib.linear_ce(h, w, targets, mask, reduction, ignore_index)
        ctx.save_for_backward(h, w, state)
        ctx.reduction = reduction
        ctx.set_materialize_grads(False)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        if dloss is None:
            return (None,) * 6
        h, w, state = ctx.saved_tensors
        need = tuple(ctx.needs_input_grad[:2])
        fn = _LinearCEBwdFn.apply if torch.is_grad_enabled() else _lib.linear_ce_bwd
        dh, dw = fn(dloss, h, w, state, ctx.reduction, need)
        return (dh if need[0] else None, dw if need[1] else None, None, None, None, None)


def _linear_ce_math(h, w, targets, mask, reduction, ignore_index):
    """The same value in PyTorch (CPU tensors)."""
    weight = torch.ones_like(targets, dtype=h.dtype) if mask is None else mask.to(h.dtype)
    keep = (weight != 0) & (targets != ignore_index)
    if bool(((targets < 0) | (targets >= w.shape[0]))[keep].any()):
        raise ValueError(f"linear cross entropy: a target is outside the vocabulary of {w.shape[0]}")
    h = torch.where(keep[..., None], h, torch.zeros((), dtype=h.dtype, device=h.device))
    t = torch.where(keep, targets, torch.zeros_like(targets))
    z = torch.matmul(h, w.transpose(0, 1))
    ce = torch.logsumexp(z, -1) - z.gather(-1, t[..., None])[..., 0]
    ce = torch.where(keep, ce * weight, torch.zeros_like(ce))
    if reduction == "none":
        return ce
    if reduction == "sum":
        return ce.sum()
    return ce.sum() / (max(targets.numel(), 1) if mask is None else weight.sum().clamp_min(1.0))


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                         mask: Optional[torch.Tensor] = None, *, reduction: str = "mean",
                         ignore_index: int = -100) -> torch.Tensor:
    """Token cross entropy of the logits ``hidden @ weight.T``, which are never stored.

    hidden: [..., dim]; weight: [vocab, dim] (both fp16 or both bf16 on CUDA);
    targets: integers, hidden's leading shape; mask: the targets' shape, bool or
    weights m (a position with m = 0 is left out). The position's loss is m times
    its cross entropy, 0 where the target is ``ignore_index``; the result is fp32
    (on CPU hidden's dtype):

    * "none": the positions' losses;  * "sum": their sum;
    * "mean": their sum over max(1, sum of the mask), or over the number of
      positions without a mask, as ``ttt_model.compute_loss`` divides (ignored
      targets count). A loss over no position at all is 0.

    Positions left out are not read: what ``hidden`` holds there changes nothing,
    and their gradient is exactly 0. A target outside the vocabulary raises: at
    once on CPU, at the next call of this library (or check_device_errors) on
    CUDA. Differentiable twice in hidden, weight and the upstream gradient."""
    if reduction not in _lib.LCE_REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_lib.LCE_REDUCTIONS)}, got {reduction!r}")
    if not _kernel_path(hidden):
        return _linear_ce_math(hidden, weight, targets, mask, reduction, ignore_index)
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return LinearCrossEntropyFn.apply(hidden, weight, targets, mask, reduction, int(ignore_index))
    return _lib.linear_ce(hidden, weight, targets, mask, reduction, int(ignore_index))[0]
