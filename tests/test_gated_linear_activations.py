"""The activation by itself: K = 2 with rows (g, 1) and the unit matrix as weight makes the pre-activations exactly g and 1, so the output is act(g) and the gradient act'(g).

Bounds in e = 2^-24.  Phi: fp32 arithmetic around 1/2 to 2.5 e, and below g = -1.25, where Phi is exp(-g^2/2) times a factor, (12 + 1.2 g^2) e of itself: the exponent g^2/2
is rounded twice, to g^2 e together (what rounding g to fp32 changes, too), the rest are a dozen roundings.  SiLU: s = 1 / (1 + e^-g) to (5 + 1.5 |g| (1 - s)) e.  Values below
2^-126 may be flushed.  The 16-bit types: half a step of the type on top, and for the gradient the 24 bits (2^-15) that are kept of g and of 1, and dz's rounding."""
import math

import pytest
import torch

from cagc.op import gated_linear

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E = 2.0 ** -24


def exact(act, g):
    """act, act', and the bounds of fp32 arithmetic on them"""
    if act == "silu":
        s, q = torch.sigmoid(g), torch.sigmoid(-g)
        a, da = g * s, s * (1 + g * q)
        es = s * (5 + 1.5 * g.abs() * q) * E
        return a, da, g.abs() * es + a.abs() * 2 * E, es * (1 + 2 * g.abs()) + (s * (1 + g.abs())) * 4 * E
    p, d = torch.special.erfc(-g / math.sqrt(2)) / 2, torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    ep = torch.where(g <= -1.25, p * (12 + 1.2 * g * g) * E, 2.5 * E * torch.ones_like(g))
    return g * p, p + g * d, g.abs() * ep + (g * p).abs() * 2 * E, ep + g.abs() * d * (8 + 1.2 * g * g) * E + (p + g.abs() * d) * 2 * E


def values(dt):
    g = torch.linspace(-14, 14, 40001).to(dt)
    return torch.cat([g, torch.randn(2000, generator=torch.Generator().manual_seed(1)).mul(1e-2).to(dt), torch.tensor([-1.25, 1.25, 0.0, -90.0, 90.0], dtype=dt)])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [24, 40007])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=str)
def test_to_the_last_bits(dt, act, rows):
    g = values(dt).cuda()
    unit, tiny = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    w = torch.eye(2, device="cuda", dtype=dt)
    for part in g.split(rows):
        x = torch.stack([part, torch.ones_like(part)], 1).requires_grad_(True)
        y = gated_linear(x, w, activation=act)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        gd, y, dx = part.double().cpu(), y.detach().cpu(), dx.cpu()
        a, da, ea, eda = exact(act, gd)
        kept = 0.0 if dt == F32 else 2.0 ** -15 * (1.2 * gd.abs() + 1 + da.abs())      # |act''| <= 1.13, and the other factor's 1
        flush = 2.0 ** -126 * (1 + gd.abs())
        worst = ((y[:, 0].double() - a).abs() / (ea + a.abs() * (0 if dt == F32 else unit) + tiny + flush)).max()
        assert float(worst) <= 1, f"{act}: {float(worst)} of the bound"
        worst = ((dx[:, 0].double() - da).abs() / (eda + kept + da.abs() * (0 if dt == F32 else 2.01 * unit) + 2 * tiny + flush)).max()
        assert float(worst) <= 1, f"{act}': {float(worst)} of the bound"
