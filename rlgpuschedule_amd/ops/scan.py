"""Gated linear recurrence (librlsched_scan.so): whole sequences forward and
backward, and single steps.

    z = sigmoid(gate);  c_t = done_{t-1} ? 0 : h_{t-1}  (c_0 = h0)
    h_t = (1 - z_t) c_t + z_t x_t;  h_last = done_{T-1} ? 0 : h_{T-1}

Time-major [T, E, H] with done [T, E] u8 marking the steps that ended an
episode, as the rollout buffers have them: h_last is the carry of the next
rollout, and sequences of different lengths can lie one behind the other.
The state is float32 throughout. On CPU tensors the torch reference
(ops/seq_ref.py) runs. Launches go to the current stream of x's device and
are hipGraph-capturable."""
from __future__ import annotations

import torch

from ._seq import (I32, I64, P, check, load_lib, note_leaves, ptr,
                   same_device, type_code, where)
from .seq_ref import gated_scan_reference

KEEP = 64  # steps from one kept state to the next (csrc/gated_scan.hip)

_lib = None


def load():
    global _lib
    if _lib is None:
        _lib = load_lib("librlsched_scan.so", {
            "rlsched_scan_fwd": [I32] + [P] * 8 + [I64] * 7 + [I32],
            "rlsched_scan_bwd": [I32] + [P] * 10 + [I64] * 9 + [I32],
            "rlsched_scan_step": [I32] + [P] * 6 + [I64] * 4 + [I32],
        })
    return _lib


def _check(gate, x, h, done, dims, hname):
    """gate, x of `dims`; h of all but time; done of all but the width."""
    if x.dim() != dims or gate.shape != x.shape or gate.dtype != x.dtype:
        raise ValueError(
            f"gate and x must have one type and one {dims}-dim shape, got "
            f"{tuple(gate.shape)} {gate.dtype} and {tuple(x.shape)} {x.dtype}")
    code = type_code(x, "x")
    E, H = x.shape[-2:]
    if E * H >= 1 << 31:
        raise ValueError(f"{E} x {H} columns: fewer than 2**31 are supported")
    if h is not None and (h.shape != (E, H) or h.dtype != torch.float32):
        raise ValueError(f"{hname} must be float32 [{E}, {H}], got "
                         f"{tuple(h.shape)} {h.dtype}")
    if done is not None and (done.shape != x.shape[:-1] or done.dtype
                             not in (torch.uint8, torch.bool)):
        raise ValueError(f"done must be uint8 or bool {list(x.shape[:-1])}, "
                         f"got {tuple(done.shape)} {done.dtype}")
    same_device(x.device, gate=gate, done=done, **{hname: h})
    return code


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def gated_scan_fwd(gate: torch.Tensor, x: torch.Tensor,
                   h0: torch.Tensor | None = None,
                   done: torch.Tensor | None = None,
                   keep_states: bool = True):
    """gate, x [T, E, H] (float32, bfloat16 or float16; any strides of time
    and environment, such as the halves of one projection), h0 [E, H] f32 or
    None (zeros), done [T, E] u8/bool or None. Returns (hs [T, E, H] of x's
    type, h_last [E, H] f32, states): states is what gated_scan_bwd needs
    (None without keep_states)."""
    code = _check(gate, x, h0, done, 3, "h0")
    T, E, H = x.shape
    hs = torch.empty(T, E, H, dtype=x.dtype, device=x.device)
    h_last = torch.empty(E, H, dtype=torch.float32, device=x.device)
    states = None
    if keep_states:
        states = torch.empty(-(-T // KEEP), E, H, dtype=torch.float32,
                             device=x.device)
    gate, x = _unit(gate), _unit(x)
    if h0 is not None:
        h0 = h0.contiguous()
    if done is not None:
        done = done.contiguous()
    dev, stream = where(x)
    check(load().rlsched_scan_fwd(
        dev, stream, gate.data_ptr(), x.data_ptr(), ptr(h0), ptr(done),
        hs.data_ptr(), h_last.data_ptr(), ptr(states), T, E, H,
        gate.stride(0), gate.stride(1), x.stride(0), x.stride(1), code),
        "rlsched_scan_fwd")
    return hs, h_last, states


def gated_scan_bwd(dhs: torch.Tensor | None, dh_last: torch.Tensor | None,
                   gate: torch.Tensor, x: torch.Tensor, states: torch.Tensor,
                   done: torch.Tensor | None = None, need_dh0: bool = True):
    """Gradients (dgate, dx [T, E, H] of x's type, dh0 [E, H] f32 or None)
    for dhs [T, E, H] of x's type and dh_last [E, H] f32; None for either
    stands for zeros. states as gated_scan_fwd returned them."""
    code = _check(gate, x, dh_last, done, 3, "dh_last")
    T, E, H = x.shape
    if dhs is not None and (dhs.shape != x.shape or dhs.dtype != x.dtype):
        raise ValueError("dhs must have x's shape and type, got "
                         f"{tuple(dhs.shape)} {dhs.dtype}")
    if states.shape != (-(-T // KEEP), E, H) or not states.is_contiguous() \
            or states.dtype != torch.float32:
        raise ValueError("states must be gated_scan_fwd's, of these inputs")
    same_device(x.device, dhs=dhs, states=states)
    dgate = torch.empty(T, E, H, dtype=x.dtype, device=x.device)
    dx = torch.empty(T, E, H, dtype=x.dtype, device=x.device)
    dh0 = None
    if need_dh0:
        dh0 = torch.empty(E, H, dtype=torch.float32, device=x.device)
    gate, x = _unit(gate), _unit(x)
    st = sd = 0
    if dhs is not None:
        dhs = _unit(dhs)
        st, sd = dhs.stride(0), dhs.stride(1)
    if dh_last is not None:
        dh_last = dh_last.contiguous()
    if done is not None:
        done = done.contiguous()
    dev, stream = where(x)
    check(load().rlsched_scan_bwd(
        dev, stream, ptr(dhs), ptr(dh_last), gate.data_ptr(), x.data_ptr(),
        states.data_ptr(), ptr(done), dgate.data_ptr(), dx.data_ptr(),
        ptr(dh0), T, E, H, gate.stride(0), gate.stride(1), x.stride(0),
        x.stride(1), st, sd, code), "rlsched_scan_bwd")
    return dgate, dx, dh0


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, h0, done):
        ctx.set_materialize_grads(False)
        ctx.note = note_leaves(gate, x, h0)
        hs, h_last, states = gated_scan_fwd(gate, x, h0, done)
        ctx.save_for_backward(gate, x, states, done)
        return hs, h_last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dhs, dh_last):
        if dhs is None and dh_last is None:
            return None, None, None, None
        gate, x, states, done = ctx.saved_tensors
        dgate, dx, dh0 = gated_scan_bwd(dhs, dh_last, gate, x, states, done,
                                        ctx.needs_input_grad[2])
        return dgate, dx, dh0, None


def gated_scan(gate: torch.Tensor, x: torch.Tensor,
               h0: torch.Tensor | None = None,
               done: torch.Tensor | None = None):
    """(hs, h_last) of the recurrence above, differentiable in gate, x and
    h0; arguments as gated_scan_fwd's."""
    if not x.is_cuda:
        return gated_scan_reference(gate, x, h0, done)
    if torch.is_grad_enabled() and (
            gate.requires_grad or x.requires_grad
            or (h0 is not None and h0.requires_grad)):
        return _GatedScan.apply(gate, x, h0, done)
    return gated_scan_fwd(gate, x, h0, done, keep_states=False)[:2]


@torch.no_grad()
def gated_scan_step(gate: torch.Tensor, x: torch.Tensor, h: torch.Tensor,
                    done_prev: torch.Tensor | None = None) -> torch.Tensor:
    """One acting step: gate, x [E, H]; h [E, H] f32 contiguous, UPDATED IN
    PLACE; done_prev [E] u8/bool marks environments whose state restarts from
    zero before this step. Returns the output [E, H] in x's type. Not
    differentiable."""
    code = _check(gate, x, h, done_prev, 2, "h")
    if not h.is_contiguous():
        raise ValueError("h is updated in place: it must be contiguous")
    if not x.is_cuda:
        c = h if done_prev is None else h.masked_fill(
            done_prev.unsqueeze(-1) != 0, 0.0)
        hs, last = gated_scan_reference(gate[None], x[None], c)
        h.copy_(last)
        return hs[0]
    E, H = x.shape
    hs = torch.empty(E, H, dtype=x.dtype, device=x.device)
    gate, x = _unit(gate), _unit(x)
    if done_prev is not None:
        done_prev = done_prev.contiguous()
    dev, stream = where(x)
    check(load().rlsched_scan_step(
        dev, stream, gate.data_ptr(), x.data_ptr(), ptr(done_prev),
        h.data_ptr(), hs.data_ptr(), E, H, gate.stride(0), x.stride(0), code),
        "rlsched_scan_step")
    return hs
