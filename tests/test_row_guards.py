"""The row-wise and gradient-norm entry points with NaN around what they read, exact workspaces, and guards around what they write: nothing beyond a row, a tensor or a workspace is touched."""
import ctypes
import math

import pytest
import torch

from cagc import _lib

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODE = {F32: 0, F16: 1, BF16: 3}
GUARD, MARK = 4096, 0xA5
pytestmark = pytest.mark.gpu


class Guarded:
    def __init__(self):
        self.all = []

    def __call__(self, shape, dt, shift=0):
        """a tensor to be written, all NaN before, `shift` elements off its alignment"""
        size = torch.empty((), dtype=dt).element_size()
        start, nbytes = GUARD + shift * size, math.prod(shape) * size
        buf = torch.full((nbytes + 2 * GUARD + shift * size,), MARK, dtype=torch.uint8, device="cuda")
        buf[start:start + nbytes] = 0xFF
        self.all.append((buf, start, nbytes))
        return torch.as_strided(buf.view(torch.uint8)[start:start + nbytes].view(dt), shape, [math.prod(shape[i + 1:]) for i in range(len(shape))])

    def check(self):
        for buf, start, nbytes in self.all:
            assert bool((buf[:start] == MARK).all()) and bool((buf[start + nbytes:] == MARK).all()), "written outside"


def framed(t, extra):
    buf = torch.full((t.shape[0] + 2, t.shape[1] + 8 + extra), float("nan"), device="cuda", dtype=t.dtype)
    view = buf[1:-1, 4:4 + t.shape[1]]
    view.copy_(t)
    return view, buf.stride(0)


def values(shape, dt, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dt).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


DIMS = [1, 3, 8, 63, 64, 65, 509, 520, 1023, 2049, 4099, 5125, 8191, 12301, 16384, 20003, 32767]


@pytest.mark.parametrize("rows", [1, 7, 150])
@pytest.mark.parametrize("dt, dim", [(dt, dim) for dt in (F32, F16, BF16) for dim in DIMS if dim * dt.itemsize <= 65536], ids=str)      # (a row holds 64 KiB)
def test_norm(dt, dim, rows):
    code, made = CODE[dt], Guarded()
    x, r, w, dy, dh = values((rows, dim), dt, 1), values((rows, dim), dt, 2), values((dim,), F32, 3), values((rows, dim), dt, 4), values((rows, dim), dt, 5)
    (xv, xs), (rv, rs), (wv, _), (dyv, dys), (dhv, dhs) = framed(x, 1), framed(r, 3), framed(w[None], 0), framed(dy, 2), framed(dh, 0)
    y, h, rstd = made((rows, dim), dt, 1), made((rows, dim), dt, 1), made((rows,), F32)
    _lib.call("cagc_rms_norm_fwd", ptr(y), ptr(h), ptr(rstd), ptr(xv), ptr(rv), ptr(wv), rows, dim, xs, rs, code, 0, 1e-6)
    q, scale, h2 = made((rows, dim), torch.uint8, 3), made((rows,), F32), made((rows, dim), dt, 1)
    _lib.call("cagc_rms_norm_e4m3", ptr(q), ptr(scale), ptr(h2), ptr(xv), ptr(rv), ptr(wv), rows, dim, xs, rs, code, 0, 1e-6)
    q2, scale2 = made((rows, dim), torch.uint8, 3), made((rows,), F32)
    _lib.call("cagc_quantize_rows_e4m3", ptr(q2), ptr(scale2), ptr(xv), rows, dim, xs, code)
    dx, dw = made((rows, dim), dt, 1), made((dim,), F32)
    need = _lib.query("cagc_rms_norm_bwd_workspace", rows, dim, code)
    ws = made((need,), torch.uint8) if need else None
    _lib.call("cagc_rms_norm_bwd", ptr(dx), ptr(dw), ptr(ws), ptr(dyv), ptr(dhv), ptr(h), ptr(wv), ptr(rstd), rows, dim, dys, dhs, dim, code, 0)
    made.check()
    # against 64 bits, coarsely (test_rms_norm.py holds the bounds): every element is written, and from its own row
    hd = (x.double() + r.double()).to(dt).double()
    n = hd * (hd.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
    t = dy.double() * w.double()
    want = {"h": hd, "y": n * w.double(), "dw": (dy.double() * n).sum(0),
            "dx": (t - n * (t * n).mean(-1, keepdim=True)) * (hd.square().mean(-1, keepdim=True) + 1e-6) ** -0.5 + dh.double()}
    e = torch.finfo(dt).eps
    for name, got, eps in (("h", h, 0.0), ("h", h2, 0.0), ("y", y, e), ("dx", dx, e), ("dw", dw, 1e-6)):
        mag = {"h": 0.0, "y": 1e-5, "dx": 1e-4, "dw": 1e-4 * math.sqrt(rows)}[name] * (1 + want[name].abs().max())
        assert bool(((got.double() - want[name]).abs() <= want[name].abs() * eps + mag).all()), name
    for bits, s, v in ((q, scale, want["y"]), (q2, scale2, x.double())):
        got = bits.view(torch.float8_e4m3fn).double() * s.double()[:, None]
        assert bool(((got - v).abs() <= v.abs() * (2.0 ** -4 + 1e-4) + s.double()[:, None] * 2.0 ** -9).all())


@pytest.mark.parametrize("norm_type", [0, 1, 2])
def test_gradient_norm(norm_type):
    sizes = [1, 0, 5, 4095, 4096, 4097, 70003, 3, 16384, 8] * 30      # more than one launch holds
    types = [(F32, BF16, F16)[i % 3] for i in range(len(sizes))]
    made = Guarded()
    grads = []
    for i, (n, t) in enumerate(zip(sizes, types)):
        g = made((n,), t, i % 4)
        g.copy_(values((n,), t, i))
        grads.append(g)
    before = [g.double() for g in grads]
    p = (ctypes.c_uint64 * len(grads))(*(g.data_ptr() for g in grads))
    n = (ctypes.c_int64 * len(grads))(*sizes)
    codes = (ctypes.c_int * len(grads))(*(CODE[t] for t in types))
    norm, ws = made((1,), F32), made((_lib.query("cagc_grad_norm_workspace", ctypes.addressof(n), len(grads)),), torch.uint8)
    _lib.call("cagc_clip_grad_norm", ptr(norm), ptr(ws), ctypes.addressof(p), ctypes.addressof(n), ctypes.addressof(codes), len(grads), norm_type, 2.0, 1)
    made.check()
    flat = torch.cat(before).abs()
    want = float({0: flat.max(), 1: flat.sum(), 2: flat.square().sum().sqrt()}[norm_type])
    assert abs(float(norm) - want) <= want * 2.0 ** -23
    for g, b in zip(grads, before):
        v = b * (2.0 / (want + 1e-6))
        assert bool(((g.double() - v).abs() <= v.abs() * torch.finfo(g.dtype).eps + torch.finfo(g.dtype).smallest_normal * torch.finfo(g.dtype).eps).all())
