"""Rows any distance apart: a view of one token a sequence, or of some columns of a wide buffer, whose rows lie further apart than the tiles' 32-bit offsets reach (7 MiB), gives what its
contiguous copy gives, bit for bit (padding copies the same values, the same tiles multiply them)."""
import pytest
import torch

from cagc.op import gated_linear, gated_linear_e4m3, quantize_rows_e4m3

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def apart(t, dev, gap):
    """the rows of t, `gap` bytes and a little more apart"""
    wide = torch.empty(t.shape[0], gap // t.element_size() + 24, dtype=t.dtype, device=dev)
    view = wide[:, 16:16 + t.shape[1]]
    view.copy_(t)
    return view


def values(shape, dt, dev, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dt).to(dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dt, rows, k", [(BF16, 3, 96), (BF16, 70, 96), (F16, 70, 33), (F32, 40, 50)], ids=str)
def test_wide_rows(dt, rows, k, dev):
    x, w, b = values((rows, k), dt, dev, 1), values((24, k), dt, dev, 2), values((24,), dt, dev, 3)
    dy = values((rows, 12), dt, dev, 4)
    plain = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = gated_linear(*plain, scale=0.2)
    grads = torch.autograd.grad(want, plain, dy)
    for far_x, far_w in ((True, False), (False, True), (True, True)):
        leaves = [apart(x, dev, 8 << 20) if far_x else x.clone(), apart(w, dev, 8 << 20) if far_w else w.clone(), b.clone()]
        assert not far_x or leaves[0].stride(0) * leaves[0].element_size() > 7 << 20
        assert torch.equal(gated_linear(*leaves, scale=0.2), want)
        y = gated_linear(*[t.requires_grad_(True) for t in leaves], scale=0.2)
        assert torch.equal(y, want)
        for g, v in zip(torch.autograd.grad(y, leaves, apart(dy, dev, 8 << 20)), grads):
            assert torch.equal(g, v)


@pytest.mark.parametrize("dev", DEVICES)
def test_the_last_token_of_each_sequence(dev):
    hidden = torch.zeros(5, 2048, 2048, dtype=BF16, device=dev)      # 8 MiB a sequence
    hidden[:, -1] = values((5, 2048), BF16, dev, 1)
    w = values((32, 2048), BF16, dev, 2)
    assert torch.equal(gated_linear(hidden[:, -1], w, scale=0.02), gated_linear(hidden[:, -1].contiguous(), w, scale=0.02))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("rows", [5, 70])
def test_wide_rows_in_8_bits(rows, dev):
    q, s = quantize_rows_e4m3(values((rows, 80), F32, dev, 1))
    wq, ws = quantize_rows_e4m3(values((24, 80), F32, dev, 2))
    want = gated_linear_e4m3(q, s, wq, ws)
    assert torch.equal(gated_linear_e4m3(apart(q, dev, 8 << 20), s, wq, ws), want)
    assert torch.equal(gated_linear_e4m3(q, s, apart(wq, dev, 8 << 20), ws), want)
