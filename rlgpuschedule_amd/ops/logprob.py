"""Log probabilities of actions: log softmax at the taken actions over the
allowed ones, the distribution's entropy, and its top alternatives, forward
and backward, for any number of actions.

An action that the mask leaves out is the same as one of logit -inf:
probability 0, no gradient, never an alternative, whatever its logit holds.
On CPU tensors `action_logprobs` runs the torch reference (ops/seq_ref.py)
after the same checks. Launches go to the current stream of the logits' device
and are hipGraph-capturable."""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._seq import ext
from ._seq_checks import MAX_TOP_K, check_logp  # noqa: F401
from .seq_ref import action_logprobs_reference


class LogProbs(NamedTuple):
    """logp, entropy [...] f32; top_logp [..., k] f32 and top_index [..., k]
    i64, from the most probable down (None without top_k)."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: torch.Tensor | None
    top_index: torch.Tensor | None


def action_logprobs_fwd(logits: torch.Tensor, actions: torch.Tensor,
                        mask: torch.Tensor | None = None, top_k: int = 0):
    """logits [..., A] on a GPU (float32, bfloat16 or float16, any row
    stride, at most 2**30 actions), actions [...] i64, mask [..., A] u8/bool
    (nonzero: allowed) or None. Returns (logp, entropy [...] f32, stats [rows, 3] f32, top_logp,
    top_index): see action_logprobs; stats is what action_logprobs_bwd needs."""
    return ext().action_logprobs_fwd(logits, actions, mask, top_k)


def action_logprobs_bwd(dlogp: torch.Tensor | None,
                        dentropy: torch.Tensor | None, logits: torch.Tensor,
                        actions: torch.Tensor, mask: torch.Tensor | None,
                        stats: torch.Tensor) -> torch.Tensor:
    """dlogits [..., A] of the logits' type for dlogp and dentropy [...] f32;
    None for either stands for zeros. stats as the forward call returned
    them."""
    return ext().action_logprobs_bwd(dlogp, dentropy, logits, actions, mask,
                                     stats)


def action_logprobs(logits: torch.Tensor, actions: torch.Tensor,
                    mask: torch.Tensor | None = None,
                    top_k: int = 0) -> LogProbs:
    """LogProbs of logits [..., A] at actions [...], over the actions that
    mask [..., A] allows; logp and entropy are differentiable (once) in the
    logits.

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
    if logits.is_cuda:
        return LogProbs(*ext().action_logprobs(logits, actions, mask, top_k))
    check_logp(logits, actions, mask, top_k)
    return LogProbs(*action_logprobs_reference(logits, actions, mask, top_k))
