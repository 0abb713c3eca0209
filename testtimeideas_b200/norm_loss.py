"""The two ends of a block and of a loss next to the attention: layer norm and
the linear cross entropy, each differentiable twice on the sm_100a kernels.

The meta step (``ttt_model.meta_step``) takes the gradient of a gradient through
every op of the inner step: the norms of each block and the token loss among
them. Both operators here follow the attention's form: an autograd Function
whose backward is itself a Function with a closed-form backward (in C++,
csrc/torch_model_ops.cpp); a third derivative and, on CUDA, a forward-mode one
raise. CUDA tensors run the kernels (C ABI in include/ttt_ops.h); CPU tensors run
the PyTorch formulation of the same value.
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


def _autocast_to(dtype: Optional[torch.dtype], *tensors):
    """The tensors as autocast hands them to an op it runs in `dtype` (None: its own 16-bit type);
    unchanged outside autocast, and where they are not fp16, bf16 or fp32."""
    if not torch.is_autocast_enabled("cuda"):
        return tensors
    to = dtype or torch.get_autocast_dtype("cuda")
    low = (torch.float16, torch.bfloat16, torch.float32)
    return tuple(t.to(to) if t is not None and t.dtype in low else t for t in tensors)


# ---------------------------------------------------------------- layer norm
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x: [..., dim] in fp16, bf16 or fp32, any strides (a layout that is not rows
    of unit stride is copied); weight, bias: [dim] in x's dtype or fp32, either
    may be None. On CUDA dim is at most 16384; statistics and sums are fp32.
    Under autocast it runs in fp32, as F.layer_norm does.
    Differentiable twice in x, weight and the upstream gradient."""
    if not _kernel_path(x):
        return F.layer_norm(x, x.shape[-1:], weight, bias, eps)
    return _lib.layer_norm_ad(*_autocast_to(torch.float32, x, weight, bias), eps)


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension (same parameters and state dict) on the kernels."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm normalizes one dimension, got {self.normalized_shape}")
        return layer_norm(x, self.weight, self.bias, self.eps)


# ---------------------------------------------------------------- linear cross entropy
def _linear_ce_math(h, w, targets, mask, reduction, ignore_index):
    """The same value in PyTorch (CPU tensors); weights and sums in 32 bits or more."""
    dtype = h.dtype
    acc = torch.promote_types(dtype, torch.float32)
    weight = torch.ones_like(targets, dtype=acc) if mask is None else mask.to(acc)
    keep = (weight != 0) & (targets != ignore_index)
    if bool(((targets < 0) | (targets >= w.shape[0]))[keep].any()):
        raise ValueError(f"linear cross entropy: a target is outside the vocabulary of {w.shape[0]}")
    h = torch.where(keep[..., None], h, torch.zeros((), dtype=h.dtype, device=h.device))
    t = torch.where(keep, targets, torch.zeros_like(targets))
    z = torch.matmul(h, w.transpose(0, 1))
    ce = torch.logsumexp(z, -1) - z.gather(-1, t[..., None])[..., 0]
    ce = torch.where(keep, ce.to(acc) * weight, torch.zeros_like(weight))
    if reduction == "mean":
        ce = ce.sum() / (max(targets.numel(), 1) if mask is None else weight.sum().clamp_min(1.0))
    elif reduction == "sum":
        ce = ce.sum()
    return ce.to(dtype)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                         mask: Optional[torch.Tensor] = None, *, reduction: str = "mean",
                         ignore_index: int = -100) -> torch.Tensor:
    """Token cross entropy of the logits ``hidden @ weight.T``, which are never stored.

    hidden: [..., dim]; weight: [vocab, dim] (both fp16 or both bf16 on CUDA; autocast
    casts both to its type, as F.linear's operands);
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
    CUDA. Differentiable twice in hidden, weight and the upstream gradient; a mask that
    requires a gradient gets one on CPU and is refused on CUDA."""
    if reduction not in _lib.LCE_REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_lib.LCE_REDUCTIONS)}, got {reduction!r}")
    if not _kernel_path(hidden):
        return _linear_ce_math(hidden, weight, targets, mask, reduction, ignore_index)
    hidden, weight = _autocast_to(None, hidden, weight)
    return _lib.linear_ce_ad(hidden, weight, targets, mask, reduction, ignore_index)
