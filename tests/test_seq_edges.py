"""Sequence operators at the ends of their ranges, held to the same 64-bit
definitions and counted roundings as in test_seq_ops.py."""
import math

import pytest
import torch

from rlgpuschedule_amd import layer_norm
from rlgpuschedule_amd.ops.norm import layer_norm_bwd, layer_norm_fwd

from test_seq_ops import U, gen, randn


# ------------------------------------------------------ launches of 2^32 lanes
@pytest.mark.gpu
def test_norm_of_rows_past_2_26():
    """Rows so long that a lane for every element of dw's last sum would be
    more than a launch can have. Values of +-1 whose sums, by lane and over
    all, are exact in 32 bits: mean 0, variance 1, both row sums of the
    backward pass 0."""
    d = (1 << 26) + 40
    sign = torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda")
    x = sign.repeat(d // 4).view(1, d)
    w = torch.tensor([1.0, 2.0], device="cuda").repeat(d // 2)
    b = torch.zeros(d, device="cuda")
    dy = torch.tensor([1.0, 1.0, -1.0, -1.0], device="cuda").repeat(
        d // 4).view(1, d)
    r = 1 / math.sqrt(1 + 1e-5)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    # r from an exact sum by four operations, and three behind it
    for got, want in ((y, x * w), (dx, dy * w), (dw, (dy * x)[0])):
        off = (got.detach() - want.detach() * r).abs().max()
        assert float(off) <= 8 * U * 2, float(off)
    assert torch.equal(db, dy[0])
    del y, dx, dw, db
    # each share alone
    dw, = torch.autograd.grad(layer_norm(x.detach(), w, b), w, dy)
    assert float((dw - (dy * x.detach())[0] * r).abs().max()) <= 8 * U


@pytest.mark.gpu
def test_norm_of_2_22_long_rows():
    """As many rows as a launch could not have blocks for, each too long for a
    block's registers; one row of data seen again and again."""
    rows, d = (1 << 22) + 3, 16392
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("its outputs take 138 GB")
    g = gen(5)
    x, dy = (randn(g, 1, d, dtype=torch.bfloat16, device="cuda")
             for _ in range(2))
    w = randn(g, d, device="cuda")
    y1, mean1, rstd1 = layer_norm_fwd(x, w)
    dx1, _, _ = layer_norm_bwd(dy, x, w, mean1, rstd1,
                               needs=(True, False, False))
    some = torch.tensor([0, 1, 65535, 65536, 1 << 21, (1 << 22) - 1, 1 << 22,
                         rows - 1], device="cuda")
    y, mean, rstd = layer_norm_fwd(x.expand(rows, d), w)
    assert torch.equal(y[some], y1.expand(len(some), d))
    assert bool((mean == mean1).all()) and bool((rstd == rstd1).all())
    del y
    torch.cuda.empty_cache()
    dx, _, _ = layer_norm_bwd(dy.expand(rows, d), x.expand(rows, d), w, mean,
                              rstd, needs=(True, False, False))
    assert torch.equal(dx[some], dx1.expand(len(some), d))
    del dx
    torch.cuda.empty_cache()
