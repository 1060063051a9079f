"""cagc.op.clip_grad_norm_ / get_total_norm against the formula in 64 bits, and the training steps' max_grad_norm.

Tolerances: the norm's sums run in 64 bits, so what is left is its rounding to fp32 (2^-24); a clipped value is the value times a coefficient rounded to fp32,
rounded in fp32 and to the type: u_T + 3 2^-24."""
import math

import pytest
import torch

import cagc.model as M
from cagc import kd
from cagc.op import clip_grad_norm_, get_total_norm

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def unit(t):
    return torch.finfo(t).eps / 2


def params_with(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        out.append(p)
    return out


def gradients(sizes, types, dev, seed, scale=0.1):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(t).to(dev) for n, t in zip(sizes, types)]


def norm64(grads, kind):
    v = torch.cat([g.detach().cpu().double().reshape(-1) for g in grads])
    return float(v.abs().max()) if kind == math.inf else float(v.abs().pow(kind).sum() ** (1 / kind))


SIZES = {"one": [1], "odd": [1, 3, 7, 4095, 4097, 16385], "many": [5, 1000, 33] * 100, "empty_among": [0, 10, 0], "wide": [3_000_001, 2]}


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("types", [(F32,), (BF16,), (F16,), (F32, BF16, F16)], ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_norm_and_clip(sizes, types, kind, dev):
    sizes = SIZES[sizes]
    grads = gradients(sizes, [types[i % len(types)] for i in range(len(sizes))], dev, 1)
    before = [g.detach().cpu().double() for g in grads]
    want = norm64(grads, kind)
    norm = get_total_norm(grads, kind)
    assert norm.dtype == F32 and norm.device == grads[0].device and abs(float(norm) - want) <= 2 * E * want
    params = params_with(grads)
    assert torch.equal(clip_grad_norm_(params, 2 * want + 1, kind), norm)      # below the threshold: untouched
    assert all(torch.equal(g.cpu().double(), b) for g, b in zip(grads, before))
    got = clip_grad_norm_(params, 0.3 * want, kind)
    assert torch.equal(got, norm)
    coef = 0.3 * want / (want + 1e-6)
    for g, b in zip(grads, before):
        tol = (b * coef).abs() * (unit(g.dtype) + 3 * E) + torch.finfo(g.dtype).smallest_normal * unit(g.dtype) * 2
        assert bool(((g.cpu().double() - b * coef).abs() <= tol).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_values_whose_squares_leave_fp32(dev):
    grads = [torch.full((1000,), 1e25, device=dev), torch.full((500,), 1e-30, device=dev)]
    assert abs(float(get_total_norm(grads)) / (1e25 * math.sqrt(1000)) - 1) < 1e-6
    assert abs(float(get_total_norm(grads[1:])) / (1e-30 * math.sqrt(500)) - 1) < 1e-6
    clip_grad_norm_(params_with(grads), 1.0)
    assert abs(float(grads[0][0]) * math.sqrt(1000) - 1) < 1e-6


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", [1.0, 2.0, math.inf])
def test_nan_and_infinity(kind, dev):
    for bad in (float("nan"), float("inf"), -float("inf")):
        grads = gradients([100, 5000], [F32, BF16], dev, 1)
        grads[1][77] = bad
        ours, torchs = [g.clone() for g in grads], [g.float() for g in grads]
        norm = get_total_norm(grads, kind)
        assert bool(norm.isnan()) if bad != bad else float(norm) == math.inf
        with pytest.raises(RuntimeError):
            clip_grad_norm_(params_with(ours), 1.0, kind, error_if_nonfinite=True)
        assert all(torch.equal(a, b) or bad != bad for a, b in zip(ours, grads))      # raised before anything was scaled
        with pytest.raises(RuntimeError):
            get_total_norm(grads, kind, error_if_nonfinite=True)
        clip_grad_norm_(params_with(ours), 1.0, kind)
        torch.nn.utils.clip_grad_norm_(params_with(torchs), 1.0, kind)
        for a, b in zip(ours, torchs):
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.float().nan_to_num(), b.to(a.dtype).float().nan_to_num())


@pytest.mark.parametrize("dev", DEVICES)
def test_layouts_and_lists(dev):
    conv = torch.randn(6, 5, 3, 3, device=dev).to(memory_format=torch.channels_last)
    part = torch.randn(40, 30, device=dev)[:, 3:20]
    odd = torch.randn(101, device=dev)[1:]      # 4-byte alignment only
    half = torch.randn(101, device=dev).bfloat16()[1:]
    grads = [conv, part, odd, half]
    before, want = [g.clone() for g in grads], norm64(grads, 2)
    version = conv._version
    params = params_with(grads) + [torch.nn.Parameter(torch.zeros(3, device=dev))]      # one without a gradient
    norm = clip_grad_norm_(iter(params), 0.5 * want)
    assert abs(float(norm) - want) <= 2 * E * want and conv._version > version
    for g, b in zip(grads, before):
        assert torch.allclose(g.float(), b.float() * 0.5, rtol=unit(g.dtype) * 2 + 1e-6, atol=1e-7)
    assert float(clip_grad_norm_([], 1.0)) == 0.0 and float(clip_grad_norm_(params[-1], 1.0)) == 0.0 and float(get_total_norm([])) == 0.0
    assert abs(float(get_total_norm(odd)) - norm64([odd], 2)) < 1e-5


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    g = torch.randn(8, device=dev)
    sparse = torch.eye(3, device=dev).to_sparse()
    for bad in (lambda: get_total_norm([g], 3.0), lambda: get_total_norm([g], 0.5), lambda: get_total_norm([sparse]), lambda: clip_grad_norm_(params_with([g]), 1.0, 4)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.gpu
def test_refusals_of_the_kernels():
    g = torch.randn(64, device="cuda")
    part = torch.randn(8, 8, device="cuda")[:, 2:5]
    for bad in ([part, part], [g, g], [g[:40], g[30:]], [g, torch.randn(3)], [g.double()], [g.to(torch.float8_e4m3fn)], [g, g[5:6]]):
        with pytest.raises(RuntimeError):
            get_total_norm(bad)
        with pytest.raises(RuntimeError):
            clip_grad_norm_(params_with([t.detach() for t in bad]), 1.0)


@pytest.mark.gpu
def test_replayed_graph_and_another_stream():
    sizes, types = [70_001, 3, 4096] * 60, [F32, BF16, F16] * 60      # more than one launch holds
    grads = gradients(sizes, types, "cuda", 1)
    params = params_with(grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(params, 1.0)
    for k in range(3):
        fresh = gradients(sizes, types, "cuda", 30 + k, 0.1 if k != 1 else 1e-5)
        for g, f in zip(grads, fresh):
            g.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            want = clip_grad_norm_(params_with(fresh), 1.0)
        side.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(grads, fresh))


def _nets():
    torch.manual_seed(0)
    student = M.Generator(32, 64, 2, generator_net_shape=[12, 12, 10, 10, 7, 7, 5, 5])
    teacher = M.Generator(32, 64, 2, generator_net_shape=[24, 24, 20, 20, 16, 16, 8, 8])
    return student, teacher, M.Discriminator(32)


@pytest.mark.parametrize("dev", DEVICES)
def test_training_steps_clip(dev):
    """KDStep / TrainIteration with max_grad_norm: the gradients that Adam sees have that norm; without it, what they were"""
    B = 4
    z, mask, real = torch.randn(B, 64, generator=torch.Generator().manual_seed(1)).to(dev), kd.ellipse_mask(B, 32, dev), torch.rand(B, 3, 32, 32).to(dev)
    norms = {}
    for limit in (None, 1e9, 0.01):
        student, teacher, disc = (m.to(dev) for m in _nets())
        step = kd.TrainIteration(student, teacher, disc, latent=64, max_grad_norm=limit)
        noise = [torch.zeros(B, 1, 2 ** ((i + 5) // 2), 2 ** ((i + 5) // 2), device=dev) for i in range(student.num_layers)]
        step.g_step([z], None, mask, noise, noise)
        norms[limit] = float(get_total_norm([p.grad for p in student.parameters() if p.grad is not None]))
        assert (step.last_grad_norm is None) == (limit is None)
        step.d_step(real, [z], noise=noise)
        d = float(get_total_norm([p.grad for p in disc.parameters() if p.grad is not None]))
        assert limit != 0.01 or d <= 0.01 * (1 + 1e-5)
        step.d_reg(real)
        step.g_reg([z[:2]], noise=[n[:2] for n in noise])
        assert limit != 0.01 or float(get_total_norm([p.grad for p in student.parameters() if p.grad is not None])) <= 0.01 * (1 + 1e-5)
    # two runs of one step repeat to fp32 summation order (the convolutions' backward adds with atomics)
    assert abs(norms[None] - norms[1e9]) < 1e-4 * norms[None] and abs(norms[0.01] - 0.01) < 1e-6 and norms[None] > 0.02


@pytest.mark.gpu
def test_graphed_step_clips():
    student, teacher, disc = (m.cuda() for m in _nets())
    step = kd.GraphedKDStep(student, teacher, disc, 4, kd.ellipse_mask(4, 32, "cuda"), latent=64, random_noise=True, max_grad_norm=0.01)
    for _ in range(3):
        step.replay()
        torch.cuda.synchronize()
        assert float(step.last_grad_norm) > 0.02 and abs(float(step.flat_grad.double().norm()) - 0.01) < 1e-6
    step.close()
