"""Layer norm (librlsched_norm.so), forward and backward.

`layer_norm` is the differentiable call; `layer_norm_fwd` and
`layer_norm_bwd` are the explicit pair that captured learners use. On CPU
tensors the torch reference (ops/seq_ref.py) runs. Launches go to the
current stream of x's device and are hipGraph-capturable."""
from __future__ import annotations

import torch

from ._seq import (F64, I32, I64, P, check, load_lib, note_leaves, ptr,
                   rows_of, same_device, type_code, where)
from .seq_ref import layer_norm_reference

_lib = None


def load():
    global _lib
    if _lib is None:
        _lib = load_lib("librlsched_norm.so", {
            "rlsched_norm_fwd": [I32] + [P] * 7 + [I64] * 3 + [F64, I32, I32],
            "rlsched_norm_parts": [I64, I64],
            "rlsched_norm_bwd": [I32] + [P] * 10 + [I64] * 4 + [I32, I32],
        })
    return _lib


def _check(x, weight, bias):
    if x.dim() < 1 or not 0 < x.shape[-1] < 1 << 31:
        raise ValueError("x must have a last dimension of 1 to 2**31 - 1, "
                         f"got shape {tuple(x.shape)}")
    code = wcode = type_code(x, "x")
    wdtype = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != x.shape[-1:]:
            raise ValueError(f"{name} must have shape {tuple(x.shape[-1:])}, "
                             f"got {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must be {x.dtype} or float32, "
                            f"got {t.dtype}")
        if wdtype is not None and t.dtype != wdtype:
            raise TypeError("weight and bias must have one type, got "
                            f"{wdtype} and {t.dtype}")
        wdtype = t.dtype
        wcode = type_code(t, name)
    same_device(x.device, weight=weight, bias=bias)
    return code, wcode


def layer_norm_fwd(x: torch.Tensor, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, eps: float = 1e-5):
    """x [..., D] (float32, bfloat16 or float16, any row stride), weight and
    bias [D] of x's type or float32, or None. Returns (y [..., D] of x's
    type, mean [rows] f32, rstd [rows] f32), rows = x.numel() / D."""
    code, wcode = _check(x, weight, bias)
    d = x.shape[-1]
    rows = x.numel() // d
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty(2, rows, dtype=torch.float32, device=x.device)
    mean, rstd = stats[0], stats[1]
    xr, stride = rows_of(x)
    if weight is not None:
        weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    dev, stream = where(x)
    check(load().rlsched_norm_fwd(
        dev, stream, xr.data_ptr(), ptr(weight), ptr(bias), y.data_ptr(),
        mean.data_ptr(), rstd.data_ptr(), rows, d, stride, eps, code, wcode),
        "rlsched_norm_fwd")
    return y, mean, rstd


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor,
                   weight: torch.Tensor | None, mean: torch.Tensor,
                   rstd: torch.Tensor, wdtype: torch.dtype | None = None,
                   needs=(True, True, True)):
    """Gradients (dx, dweight, dbias) of layer_norm_fwd for dy [..., D].
    mean and rstd as the forward call returned them. wdtype: the type of
    dweight and dbias (default: the weight's, or x's without one). needs:
    which of the three are computed; the others are None. The sums over rows
    run in a fixed order, so equal inputs give equal bits."""
    code, wcode = _check(x, weight, None)
    if weight is None and wdtype is not None:
        if wdtype not in (x.dtype, torch.float32):
            raise TypeError(f"wdtype must be {x.dtype} or float32")
        wcode = code if wdtype == x.dtype else 0
    elif weight is None:
        wdtype = x.dtype
    else:
        wdtype = weight.dtype
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("dy must have x's shape and type, got "
                         f"{tuple(dy.shape)} {dy.dtype}")
    d = x.shape[-1]
    rows = x.numel() // d
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.shape != (rows,) or t.dtype != torch.float32 \
                or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 [{rows}]")
    same_device(x.device, dy=dy, mean=mean, rstd=rstd)
    lib = load()
    dx = dw = db = partial = None
    if needs[0]:
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if needs[1]:
        dw = torch.empty(d, dtype=wdtype, device=x.device)
    if needs[2]:
        db = torch.empty(d, dtype=wdtype, device=x.device)
    if needs[1] or needs[2]:
        partial = torch.empty(2 * lib.rlsched_norm_parts(rows, d) * d,
                              dtype=torch.float32, device=x.device)
    xr, xs = rows_of(x)
    dyr, dys = rows_of(dy)
    if weight is not None:
        weight = weight.contiguous()
    dev, stream = where(x)
    check(lib.rlsched_norm_bwd(
        dev, stream, dyr.data_ptr(), xr.data_ptr(), ptr(weight),
        mean.data_ptr(), rstd.data_ptr(), ptr(dx), ptr(dw), ptr(db),
        ptr(partial), rows, d, xs, dys, code, wcode), "rlsched_norm_bwd")
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ctx.note = note_leaves(x, weight, bias)
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.wdtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_bwd(dy, x, weight, mean, rstd, ctx.wdtype,
                                    ctx.needs_input_grad[:3])
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last
    dimension, differentiable in x, weight and bias. Statistics are held in
    32 bits; y has x's type."""
    if not x.is_cuda:
        return layer_norm_reference(x, weight, bias, eps)
    if torch.is_grad_enabled() and (
            x.requires_grad
            or (weight is not None and weight.requires_grad)
            or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_fwd(x, weight, bias, eps)[0]
