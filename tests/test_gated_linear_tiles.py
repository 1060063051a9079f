"""Every tile and K split of the gated projection's three products, through the C entry points, with NaN around the operands, NaN in what is to be written, workspaces of exactly the size asked for
and guards around everything that is written.

Bounds as in test_gated_linear.py: a sum over K terms in fp32 to (K + 8) 2^-24 of the sum of magnitudes, the activation to (16 + 4 |g|) 2^-24 of |g|, 24 bits kept of the pre-activations
(16-bit types), dz and every result rounded to the type.  e4m3: the matrix instruction cuts each of 8 neighbouring products to a multiple of 2^-14 of the largest one's power of two, so a
group of 8 is off by less than 8 * 2^-14 of its largest product, which the largest |x| and the largest |w| of the group bound."""
import ctypes
import math

import pytest
import torch

from cagc import _lib
from cagc.op import gated_linear

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
CODE = {F32: 0, F16: 1, BF16: 3, E4M3: 4}
E = 2.0 ** -24
FORWARD, DX, DW = 0, 1, 2

# rows, n, k whose plans together are every tile, cut along K and not, in every product
CASES = {
    16: [(3, 22, 300), (20, 22, 22), (33, 22, 22), (1249, 650, 22), (65, 21, 1206), (2787, 1279, 22), (200, 7185, 136), (38, 8243, 276), (8923, 38, 276), (1041, 67, 6041), (2840, 3929, 21),
         (8329, 882, 16), (1764, 4165, 16), (2785, 202, 4470), (269, 1815, 3333), (2221, 2877, 274)],
    32: [(3, 22, 300), (20, 23, 23), (36, 23, 23), (489, 212, 20), (66, 21, 433), (619, 4270, 23), (8458, 338, 20), (40, 8467, 156), (8296, 22, 948), (34, 7248, 385), (869, 4284, 24),
         (4160, 85, 1779), (8213, 973, 23), (426, 6185, 1164), (5829, 200, 2656), (6256, 1276, 488)],
    8: [(3, 22, 300), (20, 22, 22), (33, 22, 22), (70, 22, 22), (73, 22, 2320), (5449, 321, 23), (6147, 470, 23), (1115, 130, 6852), (4139, 1522, 565), (1961, 341, 8804)],
}
TILES = {(256, 256, False), (128, 128, False), (128, 128, True), (128, 64, False), (128, 64, True), (128, 32, False), (128, 32, True)}


def bits_of(dt):
    return torch.finfo(dt).bits


def plan(product, rows, n, k, dt):
    a, b, c = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    assert _lib.load().cagc_gated_linear_plan(a, b, c, product, rows, n, k, CODE[dt]) == 0
    return a.value, b.value, c.value > 1


def aligned_k(k):
    return (k + 15) // 16 * 16


@pytest.mark.parametrize("aligned", [False, True])
@pytest.mark.parametrize("dt", [F32, BF16, F16, E4M3], ids=str)
def test_the_cases_reach_every_tile(dt, aligned):
    """(arithmetic of the host alone)"""
    for product in (FORWARD,) if dt == E4M3 else (FORWARD, DX, DW):
        seen = {plan(product, r, n, aligned_k(k) if aligned else k, dt) for r, n, k in CASES[bits_of(dt)]}
        few = {(0, 0, False)} if product == FORWARD else set()
        assert TILES | few == seen, (product, (TILES | few) ^ seen)


class Guarded:
    """tensors to be written: NaN before, 4 KB of guards on either side"""
    SIZE, MARK = 4096, 0xA5

    def __init__(self):
        self.all = []

    def __call__(self, shape, dt):
        nbytes = math.prod(shape) * torch.empty((), dtype=dt).element_size()
        buf = torch.full((nbytes + 2 * self.SIZE,), self.MARK, dtype=torch.uint8, device="cuda")
        buf[self.SIZE:self.SIZE + nbytes] = 0xFF
        self.all.append((buf, nbytes))
        return buf[self.SIZE:self.SIZE + nbytes].view(dt).view(shape)

    def check(self):
        for buf, nbytes in self.all:
            assert bool((buf[:self.SIZE] == self.MARK).all()) and bool((buf[self.SIZE + nbytes:] == self.MARK).all()), "written outside"


def framed(t, aligned):
    """t's rows in the middle of a buffer of NaN: (view, elements from row to row)"""
    side = 16 if aligned else 3
    ld = t.shape[1] + 2 * side + (0 if aligned else 1)
    buf = torch.full((t.shape[0] + 8, ld), float("nan"), device="cuda").to(t.dtype)
    view = buf[4:-4, side:side + t.shape[1]]
    view.copy_(t)
    return view, ld


def act64(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    p = torch.special.erfc(-g / math.sqrt(2)) / 2
    return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def times(a, b):
    return torch.mm(a, b.contiguous())


def forward64(x, w, b, act, scale, out, more=None):
    """z, its bound, and the output with its bound; x, w in 64 bits"""
    n = w.shape[0] // 2
    z, mag = times(x, w.t()) * scale, times(x.abs(), w.abs().t()) * scale
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    ez = mag * (x.shape[1] + 8) * E + (0 if more is None else more)
    g, u, eg, eu = z[:, :n], z[:, n:], ez[:, :n], ez[:, n:]
    a, da = act64(act, g)
    ea = 1.13 * eg + (16 + 4 * g.abs()) * E * g.abs()
    tiny = torch.finfo(out).smallest_normal * torch.finfo(out).eps
    return z, ez, a * u, (ea * u.abs() + a.abs() * eu + ea * eu) * 1.01 + (a * u).abs() * (torch.finfo(out).eps / 2 + 4 * E) + tiny


def backward64(x, w, b, act, scale, dt, z, ez, dy):
    n = w.shape[0] // 2
    ut, tiny, keep = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps, 0.0 if dt == F32 else 2.0 ** -15
    g, u, eg, eu = z[:, :n], z[:, n:], ez[:, :n] + keep * z[:, :n].abs(), ez[:, n:] + keep * z[:, n:].abs()
    a, da = act64(act, g)
    ea, eda = 1.13 * eg + (16 + 4 * g.abs()) * E * g.abs(), 1.13 * eg + (32 + 8 * g.abs()) * E * (1 + g.abs())
    dz = torch.cat([dy * u * da, dy * a], 1)
    edz = torch.cat([dy.abs() * (eu * da.abs() + u.abs() * eda + eu * eda), dy.abs() * ea], 1) * 1.01
    db = dz.sum(0)
    out = {"db": (db, edz.sum(0) + dz.abs().sum(0) * (len(dz) + 8) * E + db.abs() * ut + tiny)}
    edz = edz + dz.abs() * (0.0 if dt == F32 else ut) + tiny
    top = dz.abs() + edz
    dx, dw = times(dz, w) * scale, times(dz.t().contiguous(), x) * scale
    out["dx"] = dx, (times(edz, w.abs()) + times(top, w.abs()) * (2 * n + 8) * E) * scale + dx.abs() * ut + tiny
    out["dw"] = dw, (times(edz.t().contiguous(), x.abs()) + times(top.t().contiguous(), x.abs()) * (len(x) + 8) * E) * scale + dw.abs() * ut + tiny
    return out


def within(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)      # (a NaN is not within)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off"


def values(shape, dt, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dt)


def stream():
    return torch.cuda.current_stream().cuda_stream


def ptr(t):
    return None if t is None else t.data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("aligned", [False, True], ids=["any", "aligned"])
@pytest.mark.parametrize("dt, case", [(dt, c) for dt in (F32, F16, BF16) for c in CASES[bits_of(dt)]], ids=str)
def test_training(dt, case, aligned):
    rows, n, k = case
    k = aligned_k(k) if aligned else k
    act, code, scale = ("silu", "gelu")[rows % 2], CODE[dt], 1 / math.sqrt(k)
    x, w, b, dy = values((rows, k), dt, 1), values((2 * n, k), dt, 2), values((2 * n,), dt, 3, 0.3), values((rows, n), dt, 4)
    (xv, ldx), (wv, ldw), (dyv, lddy) = framed(x, aligned), framed(w, aligned), framed(dy, aligned)
    made, act_code = Guarded(), {"silu": 0, "gelu": 1}[act]
    out, alone = made((rows, n), dt), made((rows, n), dt)
    saved = made((2 if dt == F32 else 3, rows, n), F32 if dt == F32 else torch.int16)
    need = _lib.query("cagc_gated_linear_workspace", ptr(xv), ptr(wv), rows, n, k, ldx, ldw, code)
    for o, s in ((out, saved), (alone, None)):
        ws = made((need,), torch.uint8) if need else None
        _lib.call("cagc_gated_linear_fwd", ptr(o), ptr(s), ptr(ws), ptr(xv), ptr(wv), ptr(b), None, None, rows, n, k, ldx, ldw, code, code, act_code, scale)
    made.check()
    xd, wd = x.double(), w.double()
    z, ez, want, tol = forward64(xd, wd, b, act, scale, dt)
    within(out, want, tol, "out")
    assert torch.equal(out, alone)
    ref, full = backward64(xd, wd, b, act, scale, dt, z, ez, dy.double()), {}
    for which in (("dx", "dw", "db"), ("dx",), ("dw",), ("db",), ("dx", "db")):
        o = {m: made({"dx": (rows, k), "dw": (2 * n, k), "db": (2 * n,)}[m], dt) for m in which}
        need = _lib.query("cagc_gated_linear_bwd_workspace", ptr(xv), ptr(wv), rows, n, k, ldx, ldw, code, *(int(m in which) for m in ("dx", "dw", "db")))
        _lib.call("cagc_gated_linear_bwd", *(ptr(o.get(m)) for m in ("dx", "dw", "db")), ptr(made((need,), torch.uint8)), ptr(dyv), ptr(saved), ptr(xv), ptr(wv), rows, n, k, ldx, ldw, lddy,
                  code, act_code, scale)
        made.check()
        for m in which:
            if len(which) == 3:
                within(o[m], *ref[m], m)
                full[m] = o[m].clone()
            else:
                assert torch.equal(o[m], full[m]), (which, m)
    del made.all[:]


@pytest.mark.gpu
@pytest.mark.parametrize("aligned", [False, True], ids=["any", "aligned"])
@pytest.mark.parametrize("out_dt", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("case", CASES[8], ids=str)
def test_8_bits(case, out_dt, aligned):
    rows, n, k = case
    k = aligned_k(k) if aligned else k
    act = ("silu", "gelu")[(rows + out_dt.itemsize + aligned) % 2]
    x, w = values((rows, k), F32, 1).to(E4M3), values((2 * n, k), F32, 2).to(E4M3)
    sx, sw = values((rows,), F32, 5).abs() + 0.1, (values((2 * n,), F32, 6).abs() + 0.1) / math.sqrt(k)
    b = values((2 * n,), out_dt, 3, 0.3) if rows % 3 else None
    (xv, ldx), (wv, ldw), made = framed(x, aligned), framed(w, aligned), Guarded()
    out = made((rows, n), out_dt)
    need = _lib.query("cagc_gated_linear_workspace", ptr(xv), ptr(wv), rows, n, k, ldx, ldw, 4)
    ws = made((need,), torch.uint8) if need else None
    _lib.call("cagc_gated_linear_fwd", ptr(out), None, ptr(ws), ptr(xv), ptr(wv), ptr(b), ptr(sx), ptr(sw), rows, n, k, ldx, ldw, 4, CODE[out_dt], {"silu": 0, "gelu": 1}[act], 1.0)
    made.check()
    xd, wd = x.double() * sx.double()[:, None], w.double() * sw.double()[:, None]

    def tops(t):
        t = torch.nn.functional.pad(t.abs(), (0, -t.shape[1] % 8))
        return t.view(t.shape[0], -1, 8).amax(-1)
    more = times(tops(xd), tops(wd).t()) * 8 * 2.0 ** -14
    _, _, want, tol = forward64(xd, wd, b, act, 1.0, out_dt, more)
    within(out, want, tol, "out")


@pytest.mark.gpu
def test_two_graphs_with_k_cut():
    """the slabs of a cut K are a workspace of each call's own: two graphs of one shape, replayed in turn with eager work between, forward and backward"""
    rows, n, k = 128, 64, 2047
    assert plan(FORWARD, rows, n, k, BF16)[2]
    x, w = values((rows, k), BF16, 1), values((2 * n, k), BF16, 2)
    padded = 256 * -(-rows * (k + 1) * 2 // 256) + 256 * -(-2 * n * (k + 1) * 2 // 256)
    assert _lib.query("cagc_gated_linear_workspace", ptr(x), ptr(w), rows, n, k, k, k, 3) > padded
    inputs = [x.clone().requires_grad_(True) for _ in range(2)]
    dy, made = values((rows, n), BF16, 3), []

    def step(t):
        y = gated_linear(t, w, scale=0.02)
        return y, torch.autograd.grad(y, t, dy)[0]
    step(inputs[0])
    torch.cuda.synchronize()
    for t in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            made.append((step(t), g))
    for turn in range(4):
        with torch.no_grad():
            for i, t in enumerate(inputs):
                t.copy_(values((rows, k), BF16, 10 * turn + i))
        for _, g in made[::-1] if turn % 2 else made:
            g.replay()
        torch.cuda.synchronize()
        for t, ((y, dx), _) in zip(inputs, made):
            ey, edx = step(t)
            assert torch.equal(y, ey) and torch.equal(dx, edx)
