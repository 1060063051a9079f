"""cagc.op.rms_norm / rms_norm_e4m3 / quantize_rows_e4m3 against the formula in 64 bits.

Tolerances: a value rounded to type T is off by at most u_T = finfo(T).eps / 2 relative (half its smallest subnormal absolute).  Sums run in fp32 over
chains of at most 4 x 8 products a lane, 6 + 4 additions across lanes: below 64 roundings of 2^-24 of the sum of magnitudes.  The weight's gradient
adds `rows` terms in some order: (rows + 64) 2^-24 of the sum of magnitudes."""
import pytest
import torch

import cagc.model as M
from cagc.op import quantize_rows_e4m3, rms_norm, rms_norm_e4m3

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
EPS = 1e-6


def unit(t):
    return torch.finfo(t).eps / 2


def make(shape, dtype, dev, seed, scale=1.0, extra=0):
    g = torch.Generator().manual_seed(seed)
    t = (torch.randn(*shape[:-1], shape[-1] + extra, generator=g) * scale).to(dtype).to(dev)
    return t[..., :shape[-1]]


def within(got, want, tol, what):
    got, want, tol = got.double().cpu(), want.cpu(), tol.cpu()
    bad = (got - want).abs() > tol
    assert got.shape == want.shape and not bool(bad.any()) and bool(torch.isfinite(got).all()), \
        f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol.clamp_min(1e-300)).max()):.3g} of the tolerance"


def reference(x, w, r, dy=None, dh=None):
    """64 bits, on the sum as it is returned: dict of (value, sum of magnitudes behind it)"""
    h = (x.double() if r is None else (x.double() + r.double())).to(x.dtype).double()
    d = h.shape[-1]
    inv = (h.square().mean(-1, keepdim=True) + EPS) ** -0.5
    n = h * inv
    wd = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    out = {"h": h, "y": n * wd}
    if dy is not None:
        t = dy.double() * wd
        c = (t * n).mean(-1, keepdim=True)
        out["dx"] = inv * (t - n * c)
        out["dx_mag"] = inv * (t.abs() + n.abs() * (t * n).abs().mean(-1, keepdim=True))
        if dh is not None:
            out["dx"] = out["dx"] + dh.double()
            out["dx_mag"] = out["dx_mag"] + dh.double().abs()
        p = (dy.double() * n).reshape(-1, d)
        out["dw"], out["dw_mag"] = p.sum(0), p.abs().sum(0)
    return out


CASES = [   # shape, dtype, weight dtype (None: no weight), residual, extra elements between rows
    ((16, 512), F32, F32, False, 0), ((1, 1), F32, F32, True, 0), ((3, 7), F32, None, False, 0), ((5, 4, 33), F32, F32, True, 5),
    ((1, 2048), BF16, BF16, True, 0), ((7, 1001), BF16, F32, True, 3), ((65, 64), F16, F16, False, 0), ((9, 4095), F16, F32, True, 1),
    ((33, 5120), BF16, BF16, True, 64), ((2, 8192), F32, F32, True, 0), ((3, 16384), F32, F32, True, 0), ((3, 20001), BF16, BF16, True, 0),
    ((2, 32768), F16, F16, False, 0), ((1030, 1536), BF16, F32, True, 0), ((4099, 40), BF16, BF16, False, 0), ((2500, 2), F32, F32, True, 0),
    ((300, 6000), BF16, F32, False, 0), ((70, 513), F16, None, True, 7),
]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_gradients(case, dev):
    shape, dt, wdt, residual, extra = case
    x = make(shape, dt, dev, 1, 2.0, extra).requires_grad_(True)
    r = make(shape, dt, dev, 2, 3.0).requires_grad_(True) if residual else None
    w = (1 + 0.2 * make(shape[-1:], F32, dev, 3)).to(wdt).requires_grad_(True) if wdt else None
    dy, dh = make(shape, dt, dev, 4, 1.0, extra), (make(shape, dt, dev, 5) if residual else None)
    out = rms_norm(x, w, residual=r, eps=EPS)
    y, h = out if residual else (out, None)
    leaves = [t for t in (x, r, w) if t is not None]
    grads = torch.autograd.grad((y, h) if residual else y, leaves, (dy, dh) if residual else dy)
    ref = reference(x.detach(), None if w is None else w.detach(), None if r is None else r.detach(), dy, dh)
    u, tiny = unit(dt), torch.finfo(dt).smallest_normal * unit(dt) * 2
    if residual:
        assert torch.equal(h.detach().double(), ref["h"])
        assert torch.equal(grads[0], grads[1])
    assert y.dtype == dt and y.shape == x.shape
    # (mean of squares: 64 roundings, halved by the root; the division, the root and two products; the final rounding)
    within(y.detach(), ref["y"], ref["y"].abs() * (u + 40 * E) + tiny, "y")
    if dev == "cpu":      # torch's own autograd rounds the intermediate gradients to the type and sums in the weight's: its order is not ours to bound
        return
    within(grads[0], ref["dx"], ref["dx"].abs() * u + ref["dx_mag"] * 160 * E + tiny, "dx")
    if w is not None:
        rows = x.numel() // shape[-1]
        assert grads[-1].dtype == wdt
        within(grads[-1], ref["dw"], ref["dw"].abs() * unit(wdt) + ref["dw_mag"] * (rows + 128) * E + torch.finfo(wdt).smallest_normal * unit(wdt) * 2, "dw")


@pytest.mark.gpu
def test_gradient_against_differences():
    x, r, w = make((5, 96), F32, "cuda", 1), make((5, 96), F32, "cuda", 2), 1 + 0.2 * make((96,), F32, "cuda", 3)
    dy, dh = make((5, 96), F32, "cuda", 4), make((5, 96), F32, "cuda", 5)

    def value(x, r, w):
        h = x + r
        return (h * (h.square().mean(-1, keepdim=True) + EPS) ** -0.5 * w * dy.double() + h * dh.double()).sum()
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, h = rms_norm(leaves[0], leaves[2], residual=leaves[1], eps=EPS)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    for i, g in enumerate(grads):
        d = make(g.shape, F32, "cuda", 10 + i).double()
        at = [t.double() for t in (x, r, w)]
        lo, hi = list(at), list(at)
        lo[i], hi[i] = at[i] - 1e-5 * d, at[i] + 1e-5 * d
        slope = float((value(*hi) - value(*lo)) / 2e-5)
        # the 64-bit quotient is good to 1e-10 x the third derivative; the gradients carry fp32 rounding (x + r among it) on ~500 terms of order 1
        assert abs(float((g.double() * d).sum()) - slope) < 1e-3


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("case", [c for c in CASES if c[0][-1] > 1], ids=str)
def test_e4m3(case, dev):
    shape, dt, wdt, residual, extra = case
    x, r = make(shape, dt, dev, 1, 2.0, extra), (make(shape, dt, dev, 2, 3.0) if residual else None)
    w = (1 + 0.2 * make(shape[-1:], F32, dev, 3)).to(wdt) if wdt else None
    out = rms_norm_e4m3(x, w, residual=r, eps=EPS)
    ref = reference(x, w, r)
    q, scale = out[:2]
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == F32 and scale.shape == x.shape[:-1]
    if residual:
        assert torch.equal(out[2].double(), ref["h"])
    top = ref["y"].abs().amax(-1)
    within(scale, top / 448, top / 448 * 48 * E, "scale")
    # half a step: 2^-4 relative, or half of the smallest subnormal 2^-9; a value next to a tie may go either way, by fp32 rounding of the quotient
    s = (top / 448)[..., None]
    within(q.double() * scale.double()[..., None], ref["y"], ref["y"].abs() * (2.0 ** -4 + 128 * E) + s * 2.0 ** -10, "q")
    assert float(q.float().abs().amax()) == 448.0


@pytest.mark.parametrize("dev", DEVICES)
def test_quantize_rows(dev):
    x = make((37, 300), BF16, dev, 1, 5.0)
    x[3] = 0
    x[4] = 1e-38
    q, scale = quantize_rows_e4m3(x)
    xd = x.double()
    s = (xd.abs().amax(-1) / 448).clamp_min(2.0 ** -126)
    within(scale, s, s * 8 * E, "scale")
    within(q.double() * scale.double()[:, None], xd, xd.abs() * (2.0 ** -4 + 16 * E) + s[:, None] * 2.0 ** -10, "q")
    assert float(q[3].float().abs().max()) == 0.0


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_of_nan_inf_and_zeros_stay_their_own(dev):
    x = make((6, 200), F32, dev, 1)
    x[1, 7], x[2, 5], x[3] = float("nan"), float("inf"), 0.0
    y = rms_norm(x)
    clean = rms_norm(x[[0, 4, 5]])
    assert torch.equal(y[[0, 4, 5]], clean)
    assert bool(y[1].isnan().all()) and bool(y[2, 5].isnan()) and float(y[2, :5].abs().max()) == 0.0 and float(y[3].abs().max()) == 0.0
    q, s = rms_norm_e4m3(x)
    assert bool(s[1].isnan()) and bool(torch.isfinite(s[[0, 3, 4, 5]]).all()) and float(q[3].float().abs().max()) == 0.0


@pytest.mark.parametrize("dev", DEVICES)
def test_no_rows_and_the_sum_alone(dev):
    x = torch.empty(0, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    y = rms_norm(x, w)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == (0, 64) and gx.shape == (0, 64) and float(gw.abs().max()) == 0.0
    q, s = rms_norm_e4m3(x.detach())
    assert q.shape == (0, 64) and s.shape == (0,)
    x, r = make((4, 64), F32, dev, 1).requires_grad_(True), make((4, 64), F32, dev, 2)
    _, h = rms_norm(x, residual=r)      # only the sum is used further on
    (gx,) = torch.autograd.grad(h.sum(), x)
    assert torch.equal(gx, torch.ones_like(gx))


@pytest.mark.gpu
def test_more_rows_than_a_launch_holds():
    rows = (1 << 21) * 2 + 5
    x = torch.randn(rows, 3, device="cuda", dtype=BF16)
    r = torch.randn(rows, 3, device="cuda", dtype=BF16)
    y, h = rms_norm(x, residual=r)
    q, s, h2 = rms_norm_e4m3(x, residual=r)
    assert torch.equal(h, x + r) and torch.equal(h2, h)
    for at in (0, (1 << 21) - 2, (1 << 21) + 1, rows - 4):
        part = slice(at, at + 4)
        one, _ = rms_norm(x[part], residual=r[part])
        q1, s1, _ = rms_norm_e4m3(x[part], residual=r[part])
        assert torch.equal(y[part], one) and torch.equal(q[part].float(), q1.float()) and torch.equal(s[part], s1)


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    x, w = torch.randn(3, 8, device=dev), torch.ones(8, device=dev)
    for bad in (lambda: rms_norm(x, w[:7]), lambda: rms_norm(x, w.half()), lambda: rms_norm(x, w, residual=x[:1]), lambda: rms_norm(x, w, residual=x.half()),
                lambda: rms_norm(torch.zeros((), device=dev)), lambda: rms_norm(x[:, :0]), lambda: rms_norm_e4m3(x.clone().requires_grad_(True)),
                lambda: quantize_rows_e4m3(torch.zeros((), device=dev))):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.gpu
def test_refusals_of_the_kernels():
    for bad in (lambda: rms_norm(torch.randn(2, 8, device="cuda", dtype=torch.float64)), lambda: rms_norm(torch.randn(2, 16385, device="cuda")),
                lambda: rms_norm(torch.randn(2, 8, device="cuda"), torch.ones(8))):
        with pytest.raises(RuntimeError):
            bad()
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(rms_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


@pytest.mark.gpu
def test_another_stream_and_a_replayed_graph():
    x, r, w = make((300, 520), BF16, "cuda", 1), make((300, 520), BF16, "cuda", 2), make((520,), F32, "cuda", 3)
    want = rms_norm(x, w, residual=r)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = rms_norm(x, w, residual=r)
        rms_norm(x, w, residual=r)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    dy = make((300, 520), BF16, "cuda", 4)
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = rms_norm(xs, ws, residual=r)
        grads = torch.autograd.grad((y, h), (xs, ws), (dy, dy))
    for k in range(3):
        fresh = make((300, 520), BF16, "cuda", 20 + k)
        with torch.no_grad():
            xs.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        xe, we = fresh.clone().requires_grad_(True), w.clone().requires_grad_(True)
        ye, he = rms_norm(xe, we, residual=r)
        ge = torch.autograd.grad((ye, he), (xe, we), (dy, dy))
        assert torch.equal(y, ye) and torch.equal(h, he) and all(torch.equal(a, b) for a, b in zip(grads, ge))


@pytest.mark.parametrize("dev", DEVICES)
def test_module(dev):
    m = M.RMSNorm(48).to(dev)
    x = make((5, 48), F32, dev, 1)
    assert [k for k, _ in m.named_parameters()] == ["weight"]
    within(m(x).detach(), reference(x, None, None)["y"], reference(x, None, None)["y"].abs() * 41 * E, "module")
    y, h = m(x, residual=x)
    assert torch.equal(h, x + x) and y.shape == x.shape
    assert list(M.RMSNorm(48, weight=False).parameters()) == []
