"""cagc.op.gated_linear / gated_linear_e4m3 against the formula in 64 bits.

Tolerances, from the rounding of each step (u_T = finfo(T).eps / 2): a product over K terms in fp32, whatever the order, is off by at most (K + 8) 2^-24 of the
sum of magnitudes; the activation by (16 + 4 |g|) 2^-24 of |g|; the pre-activations are kept for the backward pass by cutting 8 of fp32's 24 significant bits in the
16-bit types: what is cut off is below one unit of the 16th bit, 2^-15 of the value; dz is rounded to the type; every result is rounded to the type.  |act'| <= 1.13, |act''| <= 1.13 (GELU: 2 phi(0) = 0.80; SiLU: 0.5)."""
import math

import pytest
import torch

import cagc.model as M
from cagc import _lib
from cagc.op import clip_grad_norm_, gated_linear, gated_linear_e4m3, quantize_rows_e4m3, rms_norm, rms_norm_e4m3

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def unit(t):
    return torch.finfo(t).eps / 2


def make(shape, dtype, dev, seed, scale=1.0, extra=0):
    g = torch.Generator().manual_seed(seed)
    t = (torch.randn(*shape[:-1], shape[-1] + extra, generator=g) * scale).to(dtype).to(dev)
    return t[..., :shape[-1]]


def within(got, want, tol, what):
    got, want, tol = got.detach().double().cpu(), want.cpu(), tol.cpu()
    bad = (got - want).abs() > tol
    assert got.shape == want.shape and not bool(bad.any()) and bool(torch.isfinite(got).all()), \
        f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol.clamp_min(1e-300)).max()):.3g} of the tolerance"


def act64(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    p = torch.special.ndtr(g)
    return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def reference(x, w, b, act, scale, dt, dy=None):
    """64 bits on the CPU: values and their tolerances"""
    x, w = x.detach().cpu().double(), w.detach().cpu().double()
    x = x.reshape(-1, x.shape[-1])
    k, n = x.shape[1], w.shape[0] // 2
    z, mag = x @ w.t() * scale, x.abs() @ w.abs().t() * abs(scale)
    if b is not None:
        z, mag = z + b.detach().cpu().double(), mag + b.detach().cpu().double().abs()
    dz_ = mag * (k + 8) * E
    g, u, eg, eu = z[:, :n], z[:, n:], dz_[:, :n], dz_[:, n:]
    a, da = act64(act, g)
    ea = 1.13 * eg + (16 + 4 * g.abs()) * E * g.abs()
    ut, tiny = unit(dt), torch.finfo(dt).smallest_normal * unit(dt) * 2
    out = {"y": a * u, "y_tol": (ea * u.abs() + a.abs() * eu + ea * eu) * 1.01 + (a * u).abs() * (ut + 4 * E) + tiny}
    if dy is None:
        return out
    dy = dy.detach().cpu().double().reshape(-1, n)
    keep = 0.0 if dt == F32 else 2.0 ** -15
    eg, eu = eg + keep * g.abs(), eu + keep * u.abs()
    ea = 1.13 * eg + (16 + 4 * g.abs()) * E * g.abs()
    eda = 1.13 * eg + (32 + 8 * g.abs()) * E * (1 + g.abs())
    dz = torch.cat([dy * u * da, dy * a], 1)
    edz = torch.cat([dy.abs() * (eu * da.abs() + u.abs() * eda + eu * eda), dy.abs() * ea], 1) * 1.01
    if b is not None:
        out["db"] = dz.sum(0)
        out["db_tol"] = edz.sum(0) + dz.abs().sum(0) * (len(dz) + 8) * E + out["db"].abs() * ut + tiny
    edz = edz + dz.abs() * (0.0 if dt == F32 else ut) + tiny
    top = dz.abs() + edz
    out["dx"] = dz @ w * scale
    out["dx_tol"] = (edz @ w.abs() + top @ w.abs() * (2 * n + 8) * E) * abs(scale) + out["dx"].abs() * ut + tiny
    out["dw"] = dz.t() @ x * scale
    out["dw_tol"] = (edz.t() @ x.abs() + top.t() @ x.abs() * (len(x) + 8) * E) * abs(scale) + out["dw"].abs() * ut + tiny
    return out


# rows, k, n, dtype, activation, bias, extra elements between rows of x
CASES = [
    (1, 64, 64, BF16, "silu", False, 0), (1, 1, 1, F32, "gelu", True, 0), (3, 7, 5, F16, "silu", True, 2), (16, 512, 512, F32, "silu", True, 0),
    (17, 130, 33, BF16, "gelu", True, 0), (32, 1000, 100, F16, "silu", False, 8), (33, 64, 64, F32, "gelu", False, 0), (40, 257, 130, BF16, "silu", True, 1),
    (64, 129, 257, F32, "silu", True, 3), (65, 512, 200, F16, "gelu", True, 0), (77, 1001, 273, F16, "gelu", True, 0), (128, 2048, 64, BF16, "silu", False, 0),
    (130, 96, 1030, BF16, "gelu", False, 64), (300, 640, 129, F32, "gelu", True, 0), (1000, 65, 70, BF16, "silu", True, 0), (513, 320, 640, BF16, "silu", False, 0),
]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_gradients(case, dev):
    rows, k, n, dt, act, bias, extra = case
    scale = 1 / math.sqrt(k)
    x = make((rows, k), dt, dev, 1, 1.0, extra).requires_grad_(True)
    w = make((2 * n, k), dt, dev, 2).requires_grad_(True)
    b = make((2 * n,), dt, dev, 3, 0.3).requires_grad_(True) if bias else None
    dy = make((rows, n), dt, dev, 4, 1.0, extra)
    with torch.no_grad():
        y0 = gated_linear(x, w, b, activation=act, scale=scale)
    y = gated_linear(x, w, b, activation=act, scale=scale)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    ref = reference(x, w, b, act, scale, dt, dy)
    assert torch.equal(y, y0) and y.dtype == dt
    within(y, ref["y"], ref["y_tol"], "y")
    if dev == "cpu":      # (torch's autograd of the composed path is not this package's)
        return
    within(grads[0], ref["dx"], ref["dx_tol"], "dx")
    within(grads[1], ref["dw"], ref["dw_tol"], "dw")
    if bias:
        within(grads[2], ref["db"], ref["db_tol"], "db")
    again = torch.autograd.grad(gated_linear(x, w, b, activation=act, scale=scale), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))      # fixed order of summation


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("rows, k, n, act", [(2040, 2048, 4090, "gelu"), (4100, 4090, 1030, "silu"), (1250, 700, 4400, "gelu"), (3000, 256, 900, "silu")])
def test_large_tiles(rows, k, n, act, dt):
    """sizes that the larger tiles take, with and without a split of K, in every product"""
    scale = 1 / math.sqrt(k)
    x, w, b = make((rows, k), dt, "cuda", 1).requires_grad_(True), make((2 * n, k), dt, "cuda", 2).requires_grad_(True), make((2 * n,), dt, "cuda", 4, 0.3).requires_grad_(True)
    dy = make((rows, n), dt, "cuda", 3)
    y = gated_linear(x, w, b, activation=act, scale=scale)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    xd, wd = x.detach().double(), w.detach().double()
    z = xd @ wd.t().contiguous() * scale + b.detach().double()
    a, da = act64(act, z[:, :n])
    u = z[:, n:]
    dz = torch.cat([dy.double() * u * da, dy.double() * a], 1)
    # two roundings to the type (dz, the result), each below u_T in the mean, and the fp32 sums: 2^-24 sqrt(terms) in the mean, 2^-24 * 64 at these sizes
    ut = unit(dt) + 64 * E
    for what, got, want in (("y", y, a * u), ("dx", dx, dz @ wd * scale), ("dw", dw, dz.t().contiguous() @ xd * scale), ("db", db, dz.sum(0))):
        err = (got.detach().double() - want)
        assert float(err.norm() / want.norm()) < 2 * ut, what
        assert float(err.abs().max()) < 16 * ut * float(want.abs().max()), what


@pytest.mark.gpu
def test_gradient_against_differences():
    x, w, b, dy = make((6, 40), F32, "cuda", 1), make((36, 40), F32, "cuda", 2), make((36,), F32, "cuda", 3), make((6, 18), F32, "cuda", 4)
    for act in ("silu", "gelu"):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        grads = torch.autograd.grad(gated_linear(*leaves, activation=act, scale=0.2), leaves, dy)

        def value(x, w, b):
            z = x @ w.t().contiguous() * 0.2 + b
            return (act64(act, z[:, :18])[0] * z[:, 18:] * dy.double()).sum()
        for i, g in enumerate(grads):
            d = make(g.shape, F32, "cuda", 10 + i).double()
            at = [t.double() for t in (x, w, b)]
            lo, hi = list(at), list(at)
            lo[i], hi[i] = at[i] - 1e-5 * d, at[i] + 1e-5 * d
            slope = float((value(*hi) - value(*lo)) / 2e-5)
            assert abs(float((g.double() * d).sum()) - slope) < 1e-3      # 64-bit quotient; fp32 gradients: ~1500 terms of order 1, 2^-22 each


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("case", [(1, 64, 64, BF16, False), (16, 1024, 100, BF16, True), (5, 33, 7, F16, True), (31, 200, 48, F32, False), (50, 129, 65, BF16, True),
                                  (200, 512, 300, BF16, False), (1000, 640, 1030, F32, True), (1500, 2100, 1100, BF16, True)], ids=str)
def test_e4m3(case, dev):
    rows, k, n, dt, bias = case
    xq, xs = quantize_rows_e4m3(make((rows, k), F32, dev, 1))
    wq, ws = quantize_rows_e4m3(make((2 * n, k), F32, dev, 2, 1 / math.sqrt(k)))
    b = make((2 * n,), dt, dev, 3, 0.3) if bias else None
    y = gated_linear_e4m3(xq, xs, wq, ws, b, out_dtype=dt)
    x, w = xq.double() * xs.double()[:, None], wq.double() * ws.double()[:, None]
    ref = reference(x, w, b, "silu", 1.0, dt)
    assert y.dtype == dt
    # the matrix instruction adds 128 products at a time; what it drops of the smaller ones is bounded with 2^-20 of the sum of magnitudes
    mag = (x.cpu().abs() @ w.cpu().abs().t())
    z = x.cpu() @ w.cpu().t() + (0 if b is None else b.cpu().double())
    more = (mag[:, :n] * (z[:, n:].abs() + 1) + mag[:, n:] * (z[:, :n].abs() + 1)) * 1.13 * 2.0 ** -20
    within(y, ref["y"], ref["y_tol"] + more, "y")


@pytest.mark.parametrize("dev", DEVICES)
def test_leading_dimensions_expanded_rows_and_no_rows(dev):
    w = make((24, 10), F32, dev, 2)
    x = make((2, 3, 10), F32, dev, 1)
    y = gated_linear(x, w)
    assert y.shape == (2, 3, 12) and torch.equal(y.reshape(6, 12), gated_linear(x.reshape(6, 10), w))
    assert torch.allclose(gated_linear(x.transpose(0, 1), w), y.transpose(0, 1), atol=0, rtol=1e-6)
    row = make((1, 10), F32, dev, 3)
    assert torch.equal(gated_linear(row.expand(5, 10), w), gated_linear(row.repeat(5, 1), w))
    assert gated_linear(x[0, 0], w).shape == (12,)
    e = torch.empty(0, 10, device=dev, requires_grad=True)
    wg = w.clone().requires_grad_(True)
    out = gated_linear(e, wg)
    ge, gw = torch.autograd.grad(out.sum(), (e, wg))
    assert out.shape == (0, 12) and ge.shape == (0, 10) and float(gw.abs().max()) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 40, 200])
def test_nothing_beyond_the_rows_is_read_into_them_or_written(rows):
    """NaN around the operands' rows and columns, and guards around the output"""
    k, n = 72, 50
    wide = torch.full((rows + 300, k + 24), float("nan"), device="cuda", dtype=BF16)
    wide[:rows, :k] = make((rows, k), BF16, "cuda", 1)
    wbuf = torch.full((2 * n + 300, k + 24), float("nan"), device="cuda", dtype=BF16)
    wbuf[:2 * n, :k] = make((2 * n, k), BF16, "cuda", 2)
    y = gated_linear(wide[:rows, :k], wbuf[:2 * n, :k], scale=0.1)
    assert torch.equal(y, gated_linear(wide[:rows, :k].contiguous(), wbuf[:2 * n, :k].contiguous(), scale=0.1)) and bool(torch.isfinite(y).all())
    bad = wide[:rows, :k].clone()
    bad[1, 3] = float("inf")      # one row's infinity stays in that row
    z = gated_linear(bad, wbuf[:2 * n, :k], scale=0.1)
    keep = [i for i in range(rows) if i != 1]
    assert torch.equal(z[keep], y[keep]) and not bool(torch.isfinite(z[1]).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    x, w, b = torch.randn(3, 8, device=dev), torch.randn(10, 8, device=dev), torch.randn(10, device=dev)
    q, s = quantize_rows_e4m3(x)
    wq, ws = quantize_rows_e4m3(w)
    for bad in (lambda: gated_linear(x, w[:9]), lambda: gated_linear(x, w[:, :7]), lambda: gated_linear(x, w.half()), lambda: gated_linear(x, w, b[:9]),
                lambda: gated_linear(x, w, b.half()), lambda: gated_linear(x, w, activation="relu"), lambda: gated_linear(x[:, :0], w[:, :0]),
                lambda: gated_linear(x, w[:0]), lambda: gated_linear(torch.zeros((), device=dev), w),
                lambda: gated_linear_e4m3(x, s, wq, ws), lambda: gated_linear_e4m3(q, s[:2], wq, ws), lambda: gated_linear_e4m3(q, s, wq, ws.half()),
                lambda: gated_linear_e4m3(q, s, wq, ws, b, out_dtype=BF16), lambda: gated_linear_e4m3(q, s, wq, ws, out_dtype=torch.float64)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", (F32, BF16), ids=str)
def test_gradients_of_more_rows_than_bands_of_sixteen(dt):
    """a grid holds 65535 bands of rows: 1 048 560 rows of bands of 16"""
    rows, k, n = 1100003, 5, 3
    x, w, b = (make(s, dt, "cuda", i).requires_grad_(True) for i, s in enumerate(((rows, k), (2 * n, k), (2 * n,)), 1))
    dy = make((rows, n), dt, "cuda", 4)
    grads = torch.autograd.grad(gated_linear(x, w, b, scale=0.4), (x, w, b), dy)
    ref = reference(x, w, b, "silu", 0.4, dt, dy)
    for g, name in zip(grads, ("dx", "dw", "db")):
        within(g, ref[name], ref[name + "_tol"], name)


def test_columns_beyond_a_launch_are_refused():
    """by the sizes alone: no operands are there"""
    lib = _lib.load()
    assert lib.cagc_gated_linear_fwd(None, None, None, None, None, None, None, None, 1, (1 << 26) + 1, 8, 8, 8, 3, 3, 0, 1.0, None) != 0
    assert b"bad sizes" in lib.cagc_last_error()


@pytest.mark.gpu
def test_refusals_of_the_kernels():
    with pytest.raises(RuntimeError):
        gated_linear(torch.randn(2, 8, device="cuda", dtype=torch.float64), torch.randn(4, 8, device="cuda", dtype=torch.float64))
    with pytest.raises(RuntimeError):
        gated_linear(torch.randn(2, 8, device="cuda"), torch.randn(4, 8))
    with pytest.raises(RuntimeError):      # rows beyond 7 MiB
        gated_linear(torch.zeros(1, 1 << 21, device="cuda"), torch.zeros(2, 1 << 21, device="cuda"))
    x, w = torch.randn(4, 8, device="cuda", requires_grad=True), torch.randn(4, 8, device="cuda")
    (g,) = torch.autograd.grad(gated_linear(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def _block(x, r, norm, gate, down):
    """a pre-norm gated block: the sum goes on as the next residual"""
    y, h = norm(x, residual=r)
    return torch.nn.functional.linear(gate(y), down), h


@pytest.mark.gpu
def test_together_as_a_block_trains():
    """norm -> gated projection -> down projection, twice, a loss, the backward pass and the clipped gradients, eagerly and replayed from a graph"""
    torch.manual_seed(0)
    d, f, rows = 96, 160, 70
    norms = [M.RMSNorm(d).cuda() for _ in range(2)]
    gates = [M.GatedLinear(d, f).cuda() for _ in range(2)]
    downs = [torch.nn.Parameter(torch.randn(d, f, device="cuda") / 20) for _ in range(2)]
    params = [p for m in norms + gates for p in m.parameters()] + downs
    x0 = make((rows, d), F32, "cuda", 1)
    target = make((rows, d), F32, "cuda", 2)

    def loss(wide):
        x, r = x0, torch.zeros_like(x0)
        if wide:
            x, r = x.double(), r.double()
        for m, g, p in zip(norms, gates, downs):
            if not wide:
                x, r = _block(x, r, m, g, p)
            else:
                r = x + r
                y = r * (r.square().mean(-1, keepdim=True) + m.eps) ** -0.5 * m.weight.double()
                z = y @ g.weight.double().t() * g.scale + g.bias.double()
                x = (torch.nn.functional.silu(z[:, :f]) * z[:, f:]) @ p.double().t()
        return (x + r - target).square().mean()
    want = torch.autograd.grad(loss(True), params)
    got = torch.autograd.grad(loss(False), params)
    total = math.sqrt(sum(float(g.square().sum()) for g in want))
    for a, b in zip(got, want):      # fp32 through two blocks of ~100-term sums: 2^-24 sqrt(terms) of the values, far below 1e-4 of the gradient
        assert float((a.double() - b.double()).norm()) < 1e-4 * total
    for p in params:
        p.grad = None
    loss(False).backward()
    norm = clip_grad_norm_(params, 0.5 * total)
    assert abs(float(norm) - total) < 1e-4 * total
    for p, b in zip(params, want):
        assert float((p.grad.double() - 0.5 * b.double()).norm()) < 1e-4 * total
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        static = torch.autograd.grad(loss(False), params)
    for k in range(3):
        with torch.no_grad():
            for p in params:
                p.mul_(0.97)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.autograd.grad(loss(False), params)
        assert all(torch.allclose(a, b, rtol=1e-4, atol=1e-6) for a, b in zip(static, eager))


@pytest.mark.parametrize("dev", DEVICES)
def test_together_in_8_bits(dev):
    """norm in 8 bits -> gated projection on it: the serving form of the block, against the same block in 64 bits"""
    with torch.no_grad():
        d, f, rows = 128, 96, 5
        x, r, w = make((rows, d), BF16, dev, 1), make((rows, d), BF16, dev, 2), make((2 * f, d), F32, dev, 3, 1 / math.sqrt(d))
        q, s, h = rms_norm_e4m3(x, residual=r)
        wq, ws = quantize_rows_e4m3(w)
        y = gated_linear_e4m3(q, s, wq, ws)
        hd = h.double()
        n = hd * (hd.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
        # either operand's values are off by 2^-4 of themselves at most (uniform in the mean: 2^-4 / sqrt 3 each): z by about 2^-4 sqrt(2/3) of its size 1
        z = n @ w.double().t().contiguous()
        want = torch.nn.functional.silu(z[:, :f]) * z[:, f:]
        assert float((y.double() - want).norm() / want.norm()) < 0.12


@pytest.mark.gpu
def test_another_stream_and_two_graphs_of_one_shape():
    x, w = make((200, 72), BF16, "cuda", 1), make((130, 72), BF16, "cuda", 2)
    want = gated_linear(x, w, scale=0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = gated_linear(x, w, scale=0.1)
    side.synchronize()
    assert torch.equal(got, want)
    inputs, outs, graphs = [x.clone(), x.clone()], [], []
    for t in inputs:      # K is cut (a workspace) and the rows of w are padded (another): each graph has its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(gated_linear(t[:, :71], w[:, :71], scale=0.1))
        graphs.append(g)
    for k in range(3):
        for i, t in enumerate(inputs):
            t.copy_(make((200, 72), BF16, "cuda", 10 * k + i))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for t, o in zip(inputs, outs):
            assert torch.equal(o, gated_linear(t[:, :71], w[:, :71], scale=0.1))


@pytest.mark.parametrize("dev", DEVICES)
def test_module(dev):
    torch.manual_seed(0)
    m = M.GatedLinear(40, 24, lr_mul=0.5, activation="gelu").to(dev)
    assert [(k, tuple(p.shape)) for k, p in m.named_parameters()] == [("weight", (48, 40)), ("bias", (48,))]
    with torch.no_grad():
        m.bias.copy_(make((48,), F32, dev, 3))
    x = make((7, 40), F32, dev, 1)
    ref = reference(x, m.weight, m.bias * 0.5, "gelu", m.scale, F32)
    within(m(x), ref["y"], ref["y_tol"], "module")
    assert M.GatedLinear(4, 3, bias=False).bias is None
