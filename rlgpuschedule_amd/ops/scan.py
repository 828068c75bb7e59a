"""Gated linear recurrence: whole sequences forward and backward, and single
steps.

    z = sigmoid(gate);  c_t = done_{t-1} ? 0 : h_{t-1}  (c_0 = h0)
    h_t = (1 - z_t) c_t + z_t x_t;  h_last = done_{T-1} ? 0 : h_{T-1}

Time-major [T, E, H] with done [T, E] u8 marking the steps that ended an
episode, as the rollout buffers have them: h_last is the carry of the next
rollout, and sequences of different lengths can lie one behind the other.
The state is float32 throughout. On CPU tensors gated_scan and
gated_scan_step run the torch reference (ops/seq_ref.py) after the same checks.
Launches go to the current stream of x's device and are hipGraph-capturable."""
from __future__ import annotations

import torch

from ._seq import ext
from ._seq_checks import check_scan, check_step
from .seq_ref import gated_scan_reference


def gated_scan_fwd(gate: torch.Tensor, x: torch.Tensor,
                   h0: torch.Tensor | None = None,
                   done: torch.Tensor | None = None,
                   keep_states: bool = True):
    """gate, x [T, E, H] on a GPU (float32, bfloat16 or float16; any strides
    of time and environment, such as the halves of one projection; fewer than
    2**28 columns E H), h0 [E, H] f32 or None (zeros), done [T, E] u8/bool or
    None. Returns (hs [T, E, H] of x's type, h_last [E, H] f32, states):
    states is what gated_scan_bwd needs (None without keep_states)."""
    return ext().gated_scan_fwd(gate, x, h0, done, keep_states)


def gated_scan_bwd(dhs: torch.Tensor | None, dh_last: torch.Tensor | None,
                   gate: torch.Tensor, x: torch.Tensor, states: torch.Tensor,
                   done: torch.Tensor | None = None, need_dh0: bool = True):
    """Gradients (dgate, dx [T, E, H] of x's type, dh0 [E, H] f32 or None)
    for dhs [T, E, H] of x's type and dh_last [E, H] f32; None for either
    stands for zeros. states as gated_scan_fwd returned them."""
    return ext().gated_scan_bwd(dhs, dh_last, gate, x, states, done, need_dh0)


def gated_scan(gate: torch.Tensor, x: torch.Tensor,
               h0: torch.Tensor | None = None,
               done: torch.Tensor | None = None):
    """(hs, h_last) of the recurrence above, differentiable (once) in gate, x
    and h0; arguments as gated_scan_fwd's."""
    if x.is_cuda:
        return ext().gated_scan(gate, x, h0, done)
    check_scan(gate, x, h0, done, 3, "h0")
    return gated_scan_reference(gate, x, h0, done)


def gated_scan_step(gate: torch.Tensor, x: torch.Tensor, h: torch.Tensor,
                    done_prev: torch.Tensor | None = None) -> torch.Tensor:
    """One acting step: gate, x [E, H]; h [E, H] f32 contiguous, UPDATED IN
    PLACE and sharing no memory with the others; done_prev [E] u8/bool marks
    environments whose state restarts from zero before this step. Returns the
    output [E, H] in x's type. Not differentiable: under grad mode gate, x and
    h that require a gradient are refused, and tangents always."""
    if x.is_cuda:
        return ext().gated_scan_step(gate, x, h, done_prev)
    check_step(gate, x, h, done_prev)
    with torch.no_grad():
        c = h if done_prev is None else h.masked_fill(
            done_prev.unsqueeze(-1) != 0, 0.0)
        hs, last = gated_scan_reference(gate[None], x[None], c)
        h.copy_(last)
    return hs[0]
