"""Log probabilities of actions (librlsched_logp.so): log softmax at the
taken actions over the allowed ones, the distribution's entropy, and its top
alternatives, forward and backward, for any number of actions.

An action that the mask leaves out is the same as one of logit -inf:
probability 0, no gradient, never an alternative, whatever its logit holds.
On CPU tensors the torch reference (ops/seq_ref.py) runs. Launches go to the
current stream of the logits' device and are hipGraph-capturable."""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._seq import (I32, I64, P, check, load_lib, note_leaves, ptr, rows_of,
                   same_device, type_code, where)
from .seq_ref import action_logprobs_reference

MAX_TOP_K = 64

_lib = None


class LogProbs(NamedTuple):
    """logp, entropy [...] f32; top_logp [..., k] f32 and top_index [..., k]
    i64, from the most probable down (None without top_k)."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: torch.Tensor | None
    top_index: torch.Tensor | None


def load():
    global _lib
    if _lib is None:
        _lib = load_lib("librlsched_logp.so", {
            "rlsched_logp_fwd": [I32] + [P] * 9 + [I64] * 4 + [I32, I32],
            "rlsched_logp_bwd": [I32] + [P] * 9 + [I64] * 4 + [I32],
        })
    return _lib


def _check(logits, actions, mask, top_k=0):
    if logits.dim() < 1 or not 0 < logits.shape[-1] < 1 << 31:
        raise ValueError("logits must have 1 to 2**31 - 1 actions, got shape "
                         f"{tuple(logits.shape)}")
    code = type_code(logits, "logits")
    if actions.shape != logits.shape[:-1] or actions.dtype != torch.int64:
        raise ValueError(f"actions must be int64 {list(logits.shape[:-1])}, "
                         f"got {tuple(actions.shape)} {actions.dtype}")
    if mask is not None and (mask.shape != logits.shape or mask.dtype
                             not in (torch.uint8, torch.bool)):
        raise ValueError(f"mask must be uint8 or bool {list(logits.shape)}, "
                         f"got {tuple(mask.shape)} {mask.dtype}")
    if not 0 <= top_k <= min(MAX_TOP_K, logits.shape[-1]):
        raise ValueError(f"top_k must be 0 to {MAX_TOP_K} and at most the "
                         f"number of actions, got {top_k}")
    same_device(logits.device, actions=actions, mask=mask)
    return code


def action_logprobs_fwd(logits: torch.Tensor, actions: torch.Tensor,
                        mask: torch.Tensor | None = None, top_k: int = 0):
    """logits [..., A] (float32, bfloat16 or float16, any row stride),
    actions [...] i64, mask [..., A] u8/bool (nonzero: allowed) or None.
    Returns (logp, entropy [...] f32, stats [rows, 2] f32, top_logp,
    top_index): see action_logprobs; stats is what action_logprobs_bwd needs,
    each row's maximum and the logarithm of its sum."""
    code = _check(logits, actions, mask, top_k)
    A = logits.shape[-1]
    lead = logits.shape[:-1]
    rows = logits.numel() // A
    logp, entropy = (torch.empty(lead, dtype=torch.float32,
                                 device=logits.device) for _ in range(2))
    stats = torch.empty(rows, 2, dtype=torch.float32, device=logits.device)
    top_logp = top_index = None
    if top_k:
        top_logp = torch.empty(lead + (top_k,), dtype=torch.float32,
                               device=logits.device)
        top_index = torch.empty(lead + (top_k,), dtype=torch.int64,
                                device=logits.device)
    xr, xs = rows_of(logits)
    mr, ms = (None, 0) if mask is None else rows_of(mask)
    actions = actions.contiguous()
    dev, stream = where(logits)
    check(load().rlsched_logp_fwd(
        dev, stream, xr.data_ptr(), actions.data_ptr(), ptr(mr),
        logp.data_ptr(), entropy.data_ptr(), stats.data_ptr(), ptr(top_logp),
        ptr(top_index), rows, A, xs, ms, top_k, code), "rlsched_logp_fwd")
    return logp, entropy, stats, top_logp, top_index


def action_logprobs_bwd(dlogp: torch.Tensor | None,
                        dentropy: torch.Tensor | None, logits: torch.Tensor,
                        actions: torch.Tensor, mask: torch.Tensor | None,
                        stats: torch.Tensor,
                        entropy: torch.Tensor) -> torch.Tensor:
    """dlogits [..., A] of the logits' type for dlogp and dentropy [...] f32;
    None for either stands for zeros. stats and entropy as the forward call
    returned them."""
    code = _check(logits, actions, mask)
    A = logits.shape[-1]
    rows = logits.numel() // A
    given = {"dlogp": dlogp, "dentropy": dentropy, "entropy": entropy}
    for name, t in given.items():
        if t is None and name.startswith("d"):
            continue
        if t.shape != actions.shape or t.dtype != torch.float32:
            raise ValueError(f"{name} must be float32 {list(actions.shape)}, "
                             f"got {tuple(t.shape)} {t.dtype}")
    if stats.shape != (rows, 2) or stats.dtype != torch.float32 \
            or not stats.is_contiguous():
        raise ValueError("stats must be action_logprobs_fwd's, of these "
                         "inputs")
    same_device(logits.device, stats=stats, **given)
    dlogits = torch.empty(logits.shape, dtype=logits.dtype,
                          device=logits.device)
    xr, xs = rows_of(logits)
    mr, ms = (None, 0) if mask is None else rows_of(mask)
    dlogp, dentropy, entropy, actions = (
        None if t is None else t.contiguous()
        for t in (dlogp, dentropy, entropy, actions))
    dev, stream = where(logits)
    check(load().rlsched_logp_bwd(
        dev, stream, ptr(dlogp), ptr(dentropy), xr.data_ptr(),
        actions.data_ptr(), ptr(mr), stats.data_ptr(), entropy.data_ptr(),
        dlogits.data_ptr(), rows, A, xs, ms, code), "rlsched_logp_bwd")
    return dlogits


class _ActionLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, mask, top_k):
        ctx.set_materialize_grads(False)
        ctx.note = note_leaves(logits)
        logp, entropy, stats, top_logp, top_index = action_logprobs_fwd(
            logits, actions, mask, top_k)
        ctx.save_for_backward(logits, actions, mask, stats, entropy)
        if top_k:
            ctx.mark_non_differentiable(top_logp, top_index)
        return logp, entropy, top_logp, top_index

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogp, dentropy, _dtop, _dindex):
        if dlogp is None and dentropy is None:
            return None, None, None, None
        logits, actions, mask, stats, entropy = ctx.saved_tensors
        return action_logprobs_bwd(dlogp, dentropy, logits, actions, mask,
                                   stats, entropy), None, None, None


def action_logprobs(logits: torch.Tensor, actions: torch.Tensor,
                    mask: torch.Tensor | None = None,
                    top_k: int = 0) -> LogProbs:
    """LogProbs of logits [..., A] at actions [...], over the actions that
    mask [..., A] allows; logp and entropy are differentiable in the logits.

    * A negative action is a row without one (padding): logp 0, no gradient
      through logp.
    * An action that is not allowed, of logit -inf, or >= A has logp -inf and
      no gradient through logp.
    * A row that allows nothing has entropy 0 and no gradient.
    * A row whose allowed logits hold NaN or +inf has no distribution: logp
      (of a row with an action), entropy, alternatives and its gradient are
      NaN, indices -1.
    * Alternatives of equal logit come lowest index first; where fewer than
      top_k (at most 64) have a logit above -inf, the rest are (-inf, -1)."""
    if not logits.is_cuda:
        _check(logits, actions, mask, top_k)
        return LogProbs(*action_logprobs_reference(logits, actions, mask,
                                                   top_k))
    if torch.is_grad_enabled() and logits.requires_grad:
        return LogProbs(*_ActionLogProbs.apply(logits, actions, mask, top_k))
    logp, entropy, _, top_logp, top_index = action_logprobs_fwd(
        logits, actions, mask, top_k)
    return LogProbs(logp, entropy, top_logp, top_index)
