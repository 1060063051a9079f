"""The 8-bit forms divide: scale = largest magnitude / 448 and q = value / scale, each rounded once in fp32, then q to e4m3.  A quotient in fp32 is exact to half
a step by IEEE arithmetic on either device, so every bit can be asked for, ties included."""
import pytest
import torch

from cagc.op import quantize_rows_e4m3, rms_norm, rms_norm_e4m3

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def by_definition(y):
    y = y.detach().cpu().float()
    scale = (y.abs().amax(-1) / 448).clamp_min(2.0 ** -126)
    return (y / scale[..., None]).to(torch.float8_e4m3fn).float(), scale


def same(q, scale, y):
    want, s = by_definition(y)
    assert torch.equal(scale.cpu(), s)
    assert torch.equal(q.cpu().float(), want)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=str)
def test_rows_as_they_are(dt, dev):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(700, 601, generator=g) * 3).to(dt).to(dev)
    same(*quantize_rows_e4m3(x), x)


@pytest.mark.parametrize("dev", DEVICES)
def test_ties(dev):
    """rows of t / 2^6 with every top from 1 to 448: q is the middle between two e4m3 values wherever t * 448 / top is"""
    tops = torch.arange(1, 449)
    x = (torch.arange(449)[None, :].minimum(tops[:, None]).float() / 64).to(dev)
    same(*quantize_rows_e4m3(x), x)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dim", [64, 1001, 5120])
def test_behind_the_norm(dim, dev):
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(129, dim, generator=g).to(dev), (1 + 0.2 * torch.randn(dim, generator=g)).to(dev)
    same(*rms_norm_e4m3(x, w), rms_norm(x, w))      # (fp32: the norm's output is what is quantised)


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_of_zeros_infinities_and_the_smallest_values(dev):
    x = torch.randn(5, 40, generator=torch.Generator().manual_seed(3))
    x[1], x[2, 7], x[3], x[4, 9] = 0.0, float("inf"), x[3] * 2.0 ** -130, float("nan")
    q, scale = quantize_rows_e4m3(x.to(dev))
    want, s = by_definition(x)
    assert torch.equal(scale.cpu().nan_to_num(1, 2), s.nan_to_num(1, 2)) and torch.equal(q.cpu().float().isnan(), want.isnan())
    assert torch.equal(q.cpu().float().nan_to_num(), want.nan_to_num()) and bool(want[2, 7].isnan()) and float(want[2, :7].abs().max()) == 0.0


@pytest.mark.parametrize("dev", DEVICES)
def test_every_size_of_scale(dev):
    """rows of every magnitude that fp32 holds: the quotient is the divided one where its residuals underflow too"""
    x = torch.randn(240, 333, generator=torch.Generator().manual_seed(4)) * 2.0 ** torch.linspace(-140, 122, 240).round()[:, None]
    same(*quantize_rows_e4m3(x.to(dev)), x)
