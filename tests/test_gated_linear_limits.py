"""What the gated projection refuses, it refuses before the forward pass: a training forward whose backward pass could not run is refused itself; and a backward
pass at the limit.  The refusals go by the sizes alone: no operand is there (the pointers are never read)."""
import math

import pytest
import torch

from cagc import _lib
from cagc.op import gated_linear

NOWHERE = 4096


def forward(n, dtype, saved):
    lib = _lib.load()
    rc = lib.cagc_gated_linear_fwd(None, NOWHERE if saved else None, None, None, None, None, None, None, 1, n, 8, 8, 8, dtype, dtype, 0, 1.0, None)
    return rc, lib.cagc_last_error().decode()


def backward(n, dtype):
    lib = _lib.load()
    rc = lib.cagc_gated_linear_bwd(NOWHERE, None, None, None, None, None, None, None, 1, n, 8, 8, 8, n, dtype, 0, 1.0, None)
    return rc, lib.cagc_last_error().decode()


@pytest.mark.parametrize("dtype, size", [(0, 4), (1, 2), (3, 2)])
def test_columns(dtype, size):
    most = ((7 << 20) // size - 16) // 2      # 2n values of dz, and a chunk, within 7 MiB
    for n in (most + 1, 1 << 24, 1 << 26):
        rc, why = forward(n, dtype, saved=True)
        assert rc != 0 and "n too large" in why
        assert "n too large" in backward(n, dtype)[1]
        assert "null pointer" in forward(n, dtype, saved=False)[1]      # without the backward pass there is no such limit
    assert "null pointer" in forward(most, dtype, saved=True)[1] and "null pointer" in backward(most, dtype)[1]


@pytest.mark.gpu
@pytest.mark.parametrize("dt, rows", [(torch.float32, 40), (torch.bfloat16, 130)], ids=str)
def test_training_with_the_most_columns(dt, rows):
    """rows of dz that are as long as the tiles' offsets reach.  Bounds: a sum of 2n terms in fp32 in any order to 2n 2^-24 of the sum of magnitudes would pass anything here; the kernel adds in
    pieces, and rounding errors are independent, so 64 sqrt(2n) 2^-24 of the root of the sum of squares is asked for, and dz's and the result's own rounding"""
    size = torch.finfo(dt).bits // 8
    n, k, g = ((7 << 20) // size - 16) // 2, 3, torch.Generator(device="cuda").manual_seed(1)
    x, w, dy = (torch.randn(*s, device="cuda", generator=g).to(dt) for s in ((rows, k), (2 * n, k), (rows, n)))
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    y = gated_linear(*leaves, scale=0.5)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    xd, wd, dyd = x.detach().double(), w.detach().double(), dy.double()
    z = torch.mm(xd, wd.t().contiguous()) * 0.5
    s = torch.sigmoid(z[:, :n])
    a, da = z[:, :n] * s, s * (1 + z[:, :n] * (1 - s))
    u, eps = z[:, n:], torch.finfo(dt).eps
    dz = torch.cat([dyd * u * da, dyd * a], 1)
    assert bool(((y.double() - a * u).abs() <= (a * u).abs() * eps + 1e-5 * (1 + u.abs())).all())
    want = torch.mm(dz, wd) * 0.5
    root = torch.mm(dz.square(), wd.square()).sqrt() * 0.5
    assert bool(((dx.double() - want).abs() <= root * (8 * eps + 64 * math.sqrt(2 * n) * 2.0 ** -24) + want.abs() * eps).all())
    want, root = torch.mm(dz.t().contiguous(), xd) * 0.5, torch.mm(dz.abs().t().contiguous(), xd.abs()) * 0.5
    assert bool(((dw.double() - want).abs() <= root * (2 * eps + (rows + 64) * 2.0 ** -24) + 1e-6).all())
