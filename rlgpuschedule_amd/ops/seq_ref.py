"""Torch references of the sequence operators (any device, differentiable).

The definitions that norm.py, scan.py and logprob.py compute with HIP
kernels on the GPU; these run for CPU tensors and are what the numerics
tests hold the kernels to. They work in the inputs' type, but at least in
32 bits, and round to the output's type once."""
from __future__ import annotations

import math

import torch


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


def layer_norm_reference(x, weight=None, bias=None, eps: float = 1e-5):
    v = _wide(x)
    c = v - v.mean(-1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * _wide(weight)
    if bias is not None:
        y = y + _wide(bias)
    return y.to(x.dtype)


class _Gates(torch.autograd.Function):
    """(sigmoid(g), 1 - sigmoid(g)) and their derivatives z a and -z a, none
    of them taken as a difference from 1."""

    @staticmethod
    def forward(ctx, g):
        z, a = torch.sigmoid(g), torch.sigmoid(-g)
        ctx.save_for_backward(z, a)
        return z, a

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dz, da):
        z, a = ctx.saved_tensors
        return (dz - da) * z * a


def gated_scan_reference(gate, x, h0=None, done=None):
    T, E, H = x.shape
    g, v = _wide(gate), _wide(x)  # one cast, so one rounding of a gradient
    z, a = _Gates.apply(g)
    c = v.new_zeros(E, H) if h0 is None else h0
    hs = []
    for t in range(T):
        h = a[t] * c + z[t] * v[t]
        hs.append(h)
        # a selection: what an ended episode held is not seen again
        c = h if done is None else torch.where(
            done[t].unsqueeze(-1) != 0, torch.zeros_like(h), h)
    out = torch.stack(hs) if hs else v
    return out.to(x.dtype), c if T else c.clone()


def action_logprobs_reference(logits, actions, mask=None, top_k: int = 0):
    x = _wide(logits)
    A = x.shape[-1]
    allowed = x != -math.inf
    if mask is not None:
        allowed = allowed & (mask != 0)
    some = allowed.any(-1)
    v = torch.where(allowed, x, torch.zeros_like(x))
    m = torch.where(allowed, x, torch.full_like(x, -math.inf)).amax(-1)
    m = torch.where(some, m, torch.zeros_like(m)).detach()
    # below -1e4 a term's e^d is 0 and so is e^d d
    d = v - m.unsqueeze(-1)
    broken = (v.isnan() | (v == math.inf)).any(-1, keepdim=True)
    d = torch.where((d < -1e4) & ~broken, torch.full_like(d, -1e4), d)
    d = d + torch.zeros_like(m).unsqueeze(-1).masked_fill(broken, math.nan)
    d = torch.where(allowed, d, torch.zeros_like(d))
    e = torch.where(allowed, d.exp(), torch.zeros_like(x))
    s = torch.where(some, e.sum(-1), torch.ones_like(m))
    log_s = s.log()
    entropy = log_s - (e * d).sum(-1) / s
    act = actions.clamp(0, A - 1).unsqueeze(-1)
    hit = (actions < A) & allowed.gather(-1, act).squeeze(-1)
    lp = v.gather(-1, act).squeeze(-1) - m - log_s
    lp = torch.where(hit, lp, torch.full_like(lp, -math.inf))
    lp = torch.where(log_s.isnan(), log_s, lp)
    logp = torch.where(actions < 0, torch.zeros_like(lp), lp)
    top_logp = top_index = None
    if top_k:
        with torch.no_grad():
            w = torch.where(allowed, x, torch.full_like(x, -math.inf))
            w, ix = w.sort(dim=-1, descending=True, stable=True)
            w, ix = w[..., :top_k], ix[..., :top_k]
            lse = torch.where(some, log_s, torch.zeros_like(log_s))
            top_logp = w - m.unsqueeze(-1) - lse.unsqueeze(-1)
            gone = (w == -math.inf) | top_logp.isnan()
            top_index = ix.masked_fill(gone, -1)
            top_logp = torch.where(log_s.isnan().unsqueeze(-1),
                                   log_s.unsqueeze(-1).expand_as(top_logp),
                                   top_logp)
            top_index = top_index.masked_fill(top_logp.isnan(), -1)
    return logp, entropy, top_logp, top_index
