"""Forward-mode derivatives of the row-wise, gated and gradient operators: a dual tensor's tangent either comes through (the composed paths on the CPU) or the call
raises; an output without a tangent would read as a derivative of zero."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from cagc.op import clip_grad_norm_, gated_linear, gated_linear_e4m3, get_total_norm, quantize_rows_e4m3, rms_norm, rms_norm_e4m3

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def tensors(dev):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(s, generator=g).to(dev) for s in ((5, 16), (5, 16), (16,), (12, 16), (12,))]


def clip(g):
    p = torch.nn.Parameter(torch.empty(g.shape, device=g.device))
    p.grad = g
    return clip_grad_norm_(p, 1.0)


def calls(x, r, w, wg, b):
    """(call, its differentiable inputs)"""
    return [(lambda x, w, r: rms_norm(x, w, residual=r), (x, w, r)), (lambda x: rms_norm(x), (x,)), (gated_linear, (x, wg, b)), (lambda x, wg: gated_linear(x, wg), (x, wg)),
            (lambda x: get_total_norm([x, w]), (x,)), (clip, (x,))]


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_on_the_gpu_raises(grad):
    n = 0
    for f, args in calls(*tensors("cuda")):
        for i in range(len(args)):
            with fwd.dual_level(), torch.set_grad_enabled(grad):
                dual = [fwd.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]
                with pytest.raises(NotImplementedError):
                    f(*dual)
            n += 1
    assert n == 11
    x, r, w, wg, b = tensors("cuda")
    with fwd.dual_level():      # without a tangent the level alone changes nothing
        inside = gated_linear(rms_norm(x, w), wg, b)
    assert torch.equal(inside, gated_linear(rms_norm(x, w), wg, b))


@pytest.mark.parametrize("dev", DEVICES)
def test_a_tangent_on_the_8_bit_forms_raises(dev):
    x, r, w, wg, b = tensors(dev)
    (q, s), (wq, ws) = quantize_rows_e4m3(x), quantize_rows_e4m3(wg)
    b16 = b.bfloat16()
    for f, args in ((lambda x, w, r: rms_norm_e4m3(x, w, residual=r), (x, w, r)), (lambda s, ws, b: gated_linear_e4m3(q, s, wq, ws, b), (s, ws, b16))):
        for i in range(len(args)):
            with fwd.dual_level():
                dual = [fwd.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]
                with pytest.raises(NotImplementedError):
                    f(*dual)


def test_tangents_of_the_composed_paths():
    """fp32 on the CPU against the difference quotient of the same path in 64 bits: ~100 terms of order 1, each 2^-24, far below 1e-4"""
    x, r, w, wg, b = tensors("cpu")
    for f, args in ((lambda x, w, r: rms_norm(x, w, residual=r)[0], (x, w, r)), (lambda x, wg, b: gated_linear(x, wg, b, scale=0.25), (x, wg, b))):
        for i in range(len(args)):
            d = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(9))
            with fwd.dual_level():
                tangent = fwd.unpack_dual(f(*[fwd.make_dual(a, d) if j == i else a for j, a in enumerate(args)])).tangent
            at = [[a.double() + (k * 1e-6 * d.double() if j == i else 0) for j, a in enumerate(args)] for k in (1, -1)]
            assert float((tangent.double() - (f(*at[0]) - f(*at[1])) / 2e-6).abs().max()) < 1e-4
