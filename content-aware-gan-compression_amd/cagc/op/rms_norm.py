"""Root-mean-square norm of rows with the residual's addition, and its form with 8-bit output — beside the mapping network's PixelNorm
(the same norm without weight and residual).

    h = input + residual (rounded to the type: it is returned),  out = h * (mean(h^2) + eps)^-1/2 * weight

GPU tensors -> cagc_rms_norm_* (csrc/rmsnorm.hip): fp32 / fp16 / bf16, sums in fp32, weight in the input's type or fp32.  CPU tensors ->
composed PyTorch.  First-order autograd (a second derivative raises, and so does forward mode on the GPU)."""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _lib
from .._lib import ROW_DTYPE, address, launch, no_tangents, rows_of

E4M3_MAX = 448.0
_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 3}      # the types of rows, of ROW_DTYPE


def _check(name, input, weight, residual):
    shape, dtype, dev = input.shape, input.dtype, input.get_device()
    if not shape or shape[-1] < 1:
        raise RuntimeError(f"{name}: input of shape {tuple(shape)} has no rows to norm")
    if residual is not None and (residual.shape != shape or residual.dtype is not dtype or residual.get_device() != dev):
        raise RuntimeError(f"{name}: residual {tuple(residual.shape)} {residual.dtype} on {residual.device}, input {tuple(shape)} "
                           f"{dtype} on {input.device}")
    if weight is not None:
        if weight.shape != shape[-1:] or weight.get_device() != dev:
            raise RuntimeError(f"{name}: weight {tuple(weight.shape)} on {weight.device} for input {tuple(shape)} on {input.device}")
        if weight.dtype is not dtype and weight.dtype is not torch.float32:
            raise RuntimeError(f"{name}: weight {weight.dtype} for input {dtype} (the input's type or float32)")
    if dev >= 0 and dtype not in _CODES:
        raise RuntimeError(f"{name} (HIP): unsupported dtype {dtype}")
    return shape, dtype, dev


def _composed(input, weight, residual, eps):
    """(out in the wide type, h)"""
    h = input if residual is None else input + residual
    wide = h if h.dtype == torch.float64 else h.float()
    y = wide * torch.rsqrt(wide.square().mean(-1, keepdim=True) + eps)
    return (y if weight is None else y * weight.to(y.dtype)), h


def _rows(input, weight, residual, dim, code):
    """the tensors that hold the rows of input and residual, the weight, and (rows, strides, type codes) for the entry points"""
    x, n, xs = rows_of(input, dim)
    r, rs = None, 0
    if residual is not None:
        r, _, rs = rows_of(residual, dim)
    if weight is None:
        return x, r, None, n, xs, rs, code
    return x, r, weight.contiguous(), n, xs, rs, _CODES[weight.dtype]


def _forward(input, weight, residual, eps, dev, want_rstd):
    """(out, h or None, rstd or None, h as the backward pass reads it, its row stride)"""
    dim, code = input.shape[-1], _CODES[input.dtype]
    x, r, w, n, xs, rs, wcode = _rows(input, weight, residual, dim, code)
    out = torch.empty_like(input, memory_format=torch.contiguous_format)
    h = None if r is None else torch.empty_like(out)
    rstd = out.new_empty(n, dtype=torch.float32) if want_rstd else None
    launch("cagc_rms_norm_fwd", dev, out.data_ptr(), address(h), address(rstd), x.data_ptr(), address(r), address(w), n, dim, xs, rs, code, wcode, eps)
    return out, h, rstd, (x if h is None else h), (xs if h is None else dim)


class _RMSNorm(Function):
    @staticmethod
    def forward(ctx, input, weight, residual, eps, dev):
        out, h, rstd, read, stride = _forward(input, weight, residual, eps, dev, True)
        ctx.save_for_backward(read, weight, rstd)
        ctx.stride, ctx.shape, ctx.dev = stride, input.shape, dev
        ctx.set_materialize_grads(False)
        return out if h is None else (out, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        return _backward_once(ctx, dy, dh) if torch.is_grad_enabled() else _backward(ctx, dy, dh)


def _backward(ctx, dy, dh):
    h, weight, rstd = ctx.saved_tensors
    need_x, need_w, need_r, _, _ = ctx.needs_input_grad
    want_x = need_x or need_r
    dim, rows = ctx.shape[-1], rstd.shape[0]
    dx = dw = None
    if dy is None or rows == 0:      # only the sum was used, or there are no rows
        dx = dh if dy is None else torch.zeros(ctx.shape, dtype=h.dtype, device=h.device)
        dw = torch.zeros_like(weight) if need_w else None
    elif want_x or need_w:
        g, _, gs = rows_of(dy, dim)
        d, ds = None, 0
        if dh is not None:
            d, _, ds = rows_of(dh, dim)
        code = wcode = _CODES[h.dtype]
        w = ws = None
        if weight is not None:
            w, wcode = weight.contiguous(), _CODES[weight.dtype]
        if want_x:
            dx = h.new_empty(ctx.shape)
        if need_w:
            dw = torch.empty_like(w)
            need = _lib.query("cagc_rms_norm_bwd_workspace", rows, dim, code)
            ws = rstd.new_empty(need // 4) if need else None
        launch("cagc_rms_norm_bwd", ctx.dev, address(dx), address(dw), address(ws), g.data_ptr(), address(d), h.data_ptr(), address(w), rstd.data_ptr(), rows,
               dim, gs, ds, ctx.stride, code, wcode)
    return dx if need_x else None, dw, dx if need_r else None, None, None


_backward_once = once_differentiable(_backward)


def _needs_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def rms_norm(input, weight=None, residual=None, eps=1e-6):
    """Root-mean-square norm over the last dimension.  Returns out, or (out, input + residual) with a residual (of the input's shape)."""
    _, dtype, dev = _check("rms_norm", input, weight, residual)
    if dev < 0:
        y, h = _composed(input, weight, residual, eps)
        y = y.to(dtype)
        return y if residual is None else (y, h)
    no_tangents("rms_norm", (input, weight, residual))
    if _needs_grad(input, weight, residual):
        return _RMSNorm.apply(input, weight, residual, eps, dev)
    out, h, _, _, _ = _forward(input, weight, residual, eps, dev, False)
    return out if h is None else (out, h)


def _quantize(y):
    """rows of the composed path -> (e4m3, scale)"""
    y = y.float()
    scale = (y.abs().amax(-1) / E4M3_MAX).clamp_min(2.0 ** -126)
    return (y / scale[..., None]).to(torch.float8_e4m3fn), scale


def rms_norm_e4m3(input, weight=None, residual=None, eps=1e-6):
    """The same norm with its output in 8 bits: (q in float8_e4m3fn, scale [...] in fp32 with out ~ q * scale[..., None]), and input + residual
    as a third with a residual.  scale = largest magnitude of the row / 448.  For inference: inputs that require grad raise in grad mode."""
    shape, dtype, dev = _check("rms_norm_e4m3", input, weight, residual)
    if _needs_grad(input, weight, residual):
        raise RuntimeError("rms_norm_e4m3 has no backward pass: call it under torch.no_grad(), or use rms_norm")
    no_tangents("rms_norm_e4m3", (input, weight, residual))
    if dev < 0:
        y, h = _composed(input, weight, residual, eps)
        return _quantize(y) if residual is None else (*_quantize(y), h)
    dim, code = shape[-1], _CODES[dtype]
    x, r, w, n, xs, rs, wcode = _rows(input, weight, residual, dim, code)
    q = torch.empty_like(input, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    scale = q.new_empty(shape[:-1], dtype=torch.float32)
    h = None if r is None else torch.empty_like(input, memory_format=torch.contiguous_format)
    launch("cagc_rms_norm_e4m3", dev, q.data_ptr(), scale.data_ptr(), address(h), x.data_ptr(), address(r), address(w), n, dim, xs, rs, code, wcode, eps)
    return (q, scale) if h is None else (q, scale, h)


def quantize_rows_e4m3(input):
    """Rows (last dimension) in 8 bits as they are: (q, scale [...]) as in `rms_norm_e4m3` — what `gated_linear_e4m3` takes as its weight.
    Not differentiated."""
    shape, dtype, dev = _check("quantize_rows_e4m3", input, None, None)
    input = input.detach()
    if dev < 0:
        return _quantize(input)
    x, n, xs = rows_of(input, shape[-1])
    q = torch.empty_like(input, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    scale = q.new_empty(shape[:-1], dtype=torch.float32)
    launch("cagc_quantize_rows_e4m3", dev, q.data_ptr(), scale.data_ptr(), x.data_ptr(), n, shape[-1], xs, ROW_DTYPE[dtype])
    return q, scale
