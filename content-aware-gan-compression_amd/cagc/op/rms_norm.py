"""Root-mean-square norm of rows with the residual's addition, and its form with 8-bit output — beside the mapping network's PixelNorm
(the same norm without weight and residual).

    h = input + residual (rounded to the type: it is returned),  out = h * (mean(h^2) + eps)^-1/2 * weight

GPU tensors -> cagc_rms_norm_* (csrc/rmsnorm.hip): fp32 / fp16 / bf16, sums in fp32, weight in the input's type or fp32.  CPU tensors ->
composed PyTorch.  First-order autograd (a second derivative raises)."""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _lib

E4M3_MAX = 448.0
_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _check(name, input, weight, residual):
    if input.dim() < 1 or input.shape[-1] < 1:
        raise RuntimeError(f"{name}: input of shape {tuple(input.shape)} has no rows to norm")
    if residual is not None and (residual.shape != input.shape or residual.dtype != input.dtype or residual.device != input.device):
        raise RuntimeError(f"{name}: residual {tuple(residual.shape)} {residual.dtype} on {residual.device}, input {tuple(input.shape)} "
                           f"{input.dtype} on {input.device}")
    if weight is not None:
        if weight.shape != input.shape[-1:] or weight.device != input.device:
            raise RuntimeError(f"{name}: weight {tuple(weight.shape)} on {weight.device} for input {tuple(input.shape)} on {input.device}")
        if weight.dtype != input.dtype and weight.dtype != torch.float32:
            raise RuntimeError(f"{name}: weight {weight.dtype} for input {input.dtype} (the input's type or float32)")
    if input.device.type != "cpu" and input.dtype not in _TYPES:
        raise RuntimeError(f"{name} (HIP): unsupported dtype {input.dtype}")


def _composed(input, weight, residual, eps):
    """(out in the wide type, h)"""
    h = input if residual is None else input + residual
    wide = h if h.dtype == torch.float64 else h.float()
    y = wide * torch.rsqrt(wide.square().mean(-1, keepdim=True) + eps)
    return (y if weight is None else y * weight.to(y.dtype)), h


def _p(t):
    return None if t is None else t.data_ptr()


def _forward(input, weight, residual, eps, want_rstd):
    """(out, h or None, rstd or None, h as the backward pass reads it, its row stride)"""
    dim = input.shape[-1]
    x, xs = _lib.rows_of(input, dim)
    r, rs = (None, 0) if residual is None else _lib.rows_of(residual, dim)
    w = None if weight is None else weight.contiguous()
    out = torch.empty(input.shape, dtype=input.dtype, device=input.device)
    h = None if residual is None else torch.empty_like(out)
    rstd = torch.empty(x.shape[0], dtype=torch.float32, device=input.device) if want_rstd else None
    code = _lib.ROW_DTYPE[input.dtype]
    with _lib.on_device(x):
        _lib.call("cagc_rms_norm_fwd", out.data_ptr(), _p(h), _p(rstd), x.data_ptr(), _p(r), _p(w), x.shape[0], dim, xs, rs, code,
                  code if w is None else _lib.ROW_DTYPE[w.dtype], eps)
    return out, h, rstd, (x if h is None else h), (xs if h is None else dim)


class _RMSNorm(Function):
    @staticmethod
    def forward(ctx, input, weight, residual, eps):
        out, h, rstd, read, stride = _forward(input, weight, residual, eps, True)
        ctx.save_for_backward(read, weight, rstd)
        ctx.stride, ctx.shape, ctx.has_residual = stride, input.shape, residual is not None
        ctx.set_materialize_grads(False)
        return out if h is None else (out, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        want_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[2]
        want_w = weight is not None and ctx.needs_input_grad[1]
        dim = ctx.shape[-1]
        rows = rstd.shape[0]
        dx = dw = None
        if dy is None or rows == 0:      # only the sum was used, or there are no rows
            dx = dh if dy is None else torch.zeros(ctx.shape, dtype=h.dtype, device=h.device)
            dw = torch.zeros_like(weight) if want_w else None
        elif want_x or want_w:
            g, gs = _lib.rows_of(dy, dim)
            d, ds = (None, 0) if dh is None else _lib.rows_of(dh, dim)
            w = None if weight is None else weight.contiguous()
            code = _lib.ROW_DTYPE[h.dtype]
            dx = torch.empty(ctx.shape, dtype=h.dtype, device=h.device) if want_x else None
            dw = ws = None
            if want_w:
                dw = torch.empty_like(w)
                ws = torch.empty(_lib.query("cagc_rms_norm_bwd_workspace", rows, dim, code), dtype=torch.uint8, device=h.device)
            with _lib.on_device(h):
                _lib.call("cagc_rms_norm_bwd", _p(dx), _p(dw), _p(ws), g.data_ptr(), _p(d), h.data_ptr(), _p(w), rstd.data_ptr(), rows,
                          dim, gs, ds, ctx.stride, code, code if w is None else _lib.ROW_DTYPE[w.dtype])
        return (dx if ctx.needs_input_grad[0] else None, dw, dx if ctx.has_residual and ctx.needs_input_grad[2] else None, None)


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def rms_norm(input, weight=None, residual=None, eps=1e-6):
    """Root-mean-square norm over the last dimension.  Returns out, or (out, input + residual) with a residual (of the input's shape)."""
    _check("rms_norm", input, weight, residual)
    if input.device.type == "cpu":
        y, h = _composed(input, weight, residual, eps)
        y = y.to(input.dtype)
        return y if residual is None else (y, h)
    if _needs_grad(input, weight, residual):
        return _RMSNorm.apply(input, weight, residual, eps)
    out, h, _, _, _ = _forward(input, weight, residual, eps, False)
    return out if residual is None else (out, h)


def _quantize(y):
    """rows of the composed path -> (e4m3, scale)"""
    y = y.float()
    scale = (y.abs().amax(-1) * (1 / E4M3_MAX)).clamp_min(2.0 ** -126)
    return (y * (1 / scale)[..., None]).to(torch.float8_e4m3fn), scale


def rms_norm_e4m3(input, weight=None, residual=None, eps=1e-6):
    """The same norm with its output in 8 bits: (q in float8_e4m3fn, scale [...] in fp32 with out ~ q * scale[..., None]), and input + residual
    as a third with a residual.  scale = largest magnitude of the row / 448.  For inference: inputs that require grad raise in grad mode."""
    _check("rms_norm_e4m3", input, weight, residual)
    if _needs_grad(input, weight, residual):
        raise RuntimeError("rms_norm_e4m3 has no backward pass: call it under torch.no_grad(), or use rms_norm")
    if input.device.type == "cpu":
        y, h = _composed(input, weight, residual, eps)
        return _quantize(y) if residual is None else (*_quantize(y), h)
    dim = input.shape[-1]
    x, xs = _lib.rows_of(input, dim)
    r, rs = (None, 0) if residual is None else _lib.rows_of(residual, dim)
    w = None if weight is None else weight.contiguous()
    q = torch.empty(input.shape, dtype=torch.float8_e4m3fn, device=input.device)
    scale = torch.empty(input.shape[:-1], dtype=torch.float32, device=input.device)
    h = None if residual is None else torch.empty(input.shape, dtype=input.dtype, device=input.device)
    code = _lib.ROW_DTYPE[input.dtype]
    with _lib.on_device(x):
        _lib.call("cagc_rms_norm_e4m3", q.data_ptr(), scale.data_ptr(), _p(h), x.data_ptr(), _p(r), _p(w), x.shape[0], dim, xs, rs, code,
                  code if w is None else _lib.ROW_DTYPE[w.dtype], eps)
    return (q, scale) if h is None else (q, scale, h)


def quantize_rows_e4m3(input):
    """Rows (last dimension) in 8 bits as they are: (q, scale [...]) as in `rms_norm_e4m3` — what `gated_linear_e4m3` takes as its weight."""
    _check("quantize_rows_e4m3", input, None, None)
    if _needs_grad(input):
        input = input.detach()
    if input.device.type == "cpu":
        return _quantize(input)
    dim = input.shape[-1]
    x, xs = _lib.rows_of(input, dim)
    q = torch.empty(input.shape, dtype=torch.float8_e4m3fn, device=input.device)
    scale = torch.empty(input.shape[:-1], dtype=torch.float32, device=input.device)
    with _lib.on_device(x):
        _lib.call("cagc_quantize_rows_e4m3", q.data_ptr(), scale.data_ptr(), x.data_ptr(), x.shape[0], dim, xs, _lib.ROW_DTYPE[input.dtype])
    return q, scale
