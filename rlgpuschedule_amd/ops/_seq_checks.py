"""Checks of the sequence operators' arguments for CPU tensors: those of the
GPU's bindings (csrc/seq_bind.cpp), so that a call is accepted or refused alike
on both. float64, which the kernels do not know, is allowed here beside them."""
from __future__ import annotations

import torch

_FLOATS = (torch.float32, torch.bfloat16, torch.float16, torch.float64)
_FLAGS = (torch.uint8, torch.bool)
MAX_TOP_K = 64


def _require(ok, text, error=ValueError):
    if not ok:
        raise error(text)


def _float(t, name):
    _require(t.dtype in _FLOATS, f"{name} must be float32, bfloat16 or float16 "
             f"(float64 on the CPU), got {t.dtype}", TypeError)


def _state_type(t, x):
    return t.dtype == torch.float32 or t.dtype == x.dtype == torch.float64


def _same_device(x, t, name):
    _require(t.device == x.device,
             f"{name} is on {t.device}, expected {x.device}")


def check_norm(x, weight, bias):
    _require(x.dim() >= 1 and 0 < x.shape[-1] < 1 << 31, "x must have a last "
             f"dimension of 1 to 2**31 - 1, got shape {tuple(x.shape)}")
    _float(x, "x")
    first = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _require(t.dim() == 1 and t.shape[0] == x.shape[-1], f"{name} must "
                 f"have shape [{x.shape[-1]}], got {tuple(t.shape)}")
        _require(t.dtype in (x.dtype, torch.float32),
                 f"{name} must be {x.dtype} or float32, got {t.dtype}",
                 TypeError)
        _require(first is None or first == t.dtype, "weight and bias must "
                 f"have one type, got {first} and {t.dtype}", TypeError)
        _same_device(x, t, name)
        first = t.dtype


def check_scan(gate, x, h, done, dims, hname):
    """gate, x of `dims` dimensions; h of the last two; done of all but the
    last."""
    _require(x.dim() == dims and gate.shape == x.shape
             and gate.dtype == x.dtype,
             f"gate and x must have one type and one {dims}-dim shape, got "
             f"{tuple(gate.shape)} {gate.dtype} and {tuple(x.shape)} "
             f"{x.dtype}")
    _float(x, "x")
    E, H = x.shape[-2:]
    _require(E == 0 or H < (1 << 28) // E,
             f"{E} x {H} columns: fewer than 2**28 are supported")
    if h is not None:
        _require(h.shape == x.shape[-2:] and _state_type(h, x),
                 f"{hname} must be float32 [{E}, {H}], got {tuple(h.shape)} "
                 f"{h.dtype}")
        _same_device(x, h, hname)
    if done is not None:
        _require(done.shape == x.shape[:-1] and done.dtype in _FLAGS,
                 f"done must be uint8 or bool {list(x.shape[:-1])}, got "
                 f"{tuple(done.shape)} {done.dtype}")
        _same_device(x, done, "done")
    _same_device(x, gate, "gate")


def _packed(t):
    """Whether no two elements of t share memory and nothing lies between."""
    size = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape)
                            if n != 1):
        if stride != size:
            return False
        size *= n
    return True


def _may_share(a, b):
    """Whether b may share memory with a, which is contiguous: of views of
    one storage only packed ones apart from it are known not to."""
    if not (a.numel() and b.numel() and torch._C._is_alias_of(a, b)):
        return False
    if not _packed(b):
        return True
    a0, b0 = (t.storage_offset() * t.element_size() for t in (a, b))
    return (a0 < b0 + b.numel() * b.element_size()
            and b0 < a0 + a.numel() * a.element_size())


def check_step(gate, x, h, done):
    check_scan(gate, x, h, done, 2, "h")
    _require(h.is_contiguous(),
             "h is updated in place: it must be contiguous")
    for t in (gate, x, h):
        _require(torch.autograd.forward_ad.unpack_dual(t).tangent is None,
                 "gated_scan_step has no forward-mode derivative",
                 RuntimeError)
    _require(not torch.is_grad_enabled()
             or not any(t.requires_grad for t in (gate, x, h)),
             "gated_scan_step has no derivative: gate, x and h must not "
             "require a gradient (call it under torch.no_grad())")
    for t in (gate, x, done):
        _require(t is None or not _may_share(h, t), "h is updated in place: "
                 "it must not share memory with gate, x or done")


def check_logp(logits, actions, mask, top_k):
    _require(logits.dim() >= 1 and 0 < logits.shape[-1] <= 1 << 30,
             "logits must have 1 to 2**30 actions, got shape "
             f"{tuple(logits.shape)}")
    _float(logits, "logits")
    lead = logits.shape[:-1]
    _require(actions.shape == lead and actions.dtype == torch.int64,
             f"actions must be int64 {list(lead)}, got "
             f"{tuple(actions.shape)} {actions.dtype}")
    if mask is not None:
        _require(mask.shape == logits.shape and mask.dtype in _FLAGS,
                 f"mask must be uint8 or bool {list(logits.shape)}, got "
                 f"{tuple(mask.shape)} {mask.dtype}")
        _same_device(logits, mask, "mask")
    _require(0 <= top_k <= min(MAX_TOP_K, logits.shape[-1]),
             f"top_k must be 0 to {MAX_TOP_K} and at most the number of "
             f"actions, got {top_k}")
    _same_device(logits, actions, "actions")
