"""Layer norm over the last dimension, forward and backward.

`layer_norm` is the differentiable call; `layer_norm_fwd` and
`layer_norm_bwd` are the explicit pair for learners that capture their
update. On CPU tensors `layer_norm` runs the torch reference (ops/seq_ref.py)
after the same checks. Launches go to the current stream of x's device and are
hipGraph-capturable."""
from __future__ import annotations

import torch

from ._seq import ext
from ._seq_checks import check_norm
from .seq_ref import layer_norm_reference


def layer_norm_fwd(x: torch.Tensor, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, eps: float = 1e-5):
    """x [..., D] on a GPU (float32, bfloat16 or float16, any row stride),
    weight and bias [D] of x's type or float32, or None. Returns (y [..., D]
    of x's type, mean [rows] f32, rstd [rows] f32), rows = x.numel() / D."""
    return ext().layer_norm_fwd(x, weight, bias, eps)


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor,
                   weight: torch.Tensor | None, mean: torch.Tensor,
                   rstd: torch.Tensor, wdtype: torch.dtype | None = None,
                   needs=(True, True, True)):
    """Gradients (dx, dweight, dbias) of layer_norm_fwd for dy [..., D].
    mean and rstd as the forward call returned them. wdtype: the type of
    dweight and dbias where there is no weight (default: x's). needs: which
    of the three are computed; the others are None. The sums over rows run
    in a fixed order, so equal inputs give equal bits."""
    return ext().layer_norm_bwd(dy, x, weight, mean, rstd, wdtype, *needs)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last
    dimension, differentiable (once) in x, weight and bias. Statistics are
    held in 32 bits; y has x's type."""
    if x.is_cuda:
        return ext().layer_norm(x, weight, bias, eps)
    check_norm(x, weight, bias)
    return layer_norm_reference(x, weight, bias, eps)
