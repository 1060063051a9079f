"""The gated projection on 8-bit operands: scales of any size, both activations, every output type."""
import pytest
import torch

from cagc.op import gated_linear_e4m3

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E4M3 = torch.float8_e4m3fn
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("rows, k", [(5, 64), (100, 64), (100, 4160)])
def test_scales_whose_product_leaves_fp32(rows, k, dev):
    """the sum times one scale times the other stays in range where the scales' product does not.  x and w are small multiples of 128, so the sums are exact: what is left are the two products of
    either half, SiLU (1/2 of g here, to 6 roundings) and the product: below 24 2^-24"""
    g = torch.Generator().manual_seed(1)
    x, w = 128 * torch.randint(-3, 4, (rows, k), generator=g).float(), 128 * torch.randint(-3, 4, (64, k), generator=g).float()
    w[16:32] = 0
    xs, ws = torch.full((rows,), 1.37 * 2.0 ** -70), torch.full((64,), 1.21 * 2.0 ** -65)
    xs[1::2] = 1.37 * 2.0 ** 70
    ws[16:32] = 1.21 * 2.0 ** 65      # zero rows of a large scale: zero, not zero times infinity
    ws[32:48], ws[48:] = 1.3 * 2.0 ** 60, 1.3 * 2.0 ** -40
    y = gated_linear_e4m3(x.to(E4M3).to(dev), xs.to(dev), w.to(E4M3).to(dev), ws.to(dev), out_dtype=F32).cpu().double()
    z = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    want = (torch.nn.functional.silu(z[:, :32]) * z[:, 32:])[::2, :16]
    assert bool(((y[::2, :16] - want).abs() <= want.abs() * 24 * 2.0 ** -24).all())
    assert float(want.abs()[want != 0].min()) > 2.0 ** -126 and float(y[:, 16:].abs().nan_to_num(1).max()) == 0.0
