"""Gated projection — beside EqualLinear, whose `scale` convention it keeps (weights of unit variance, scaled at run time):

    out = act(scale * input @ Wg.T + bg) * (scale * input @ Wu.T + bu),   weight = [Wg; Wu] of 2n rows, act = SiLU or GELU

GPU tensors -> cagc_gated_linear_* (csrc/gated.hip), one kernel for both projections, the activation and the product; fp32 / fp16 / bf16 with
fp32 sums; the backward pass rounds the pre-activations' gradients to the type (fp16: keep them below 65504).  CPU tensors -> composed PyTorch.  First-order autograd (a second derivative raises, and so does forward mode on the GPU)."""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from .. import _lib
from .._lib import ROW_DTYPE, address, launch, no_tangents, rows_of

ACTIVATIONS = {"silu": 0, "gelu": 1}      # CAGC_ACT_*
_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _check(name, input, weight, bias, activation):
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise RuntimeError(f"{name}: activation {activation!r} (one of {', '.join(ACTIVATIONS)})")
    shape, wshape, dev = input.shape, weight.shape, input.get_device()
    if not shape or len(wshape) != 2 or wshape[0] % 2 or wshape[0] == 0 or wshape[1] != shape[-1] or wshape[1] == 0:
        raise RuntimeError(f"{name}: weight {tuple(wshape)} for input {tuple(shape)} (2n rows of the input's width)")
    if weight.dtype is not input.dtype or weight.get_device() != dev:
        raise RuntimeError(f"{name}: weight {weight.dtype} on {weight.device}, input {input.dtype} on {input.device}")
    if bias is not None and (bias.shape != wshape[:1] or bias.get_device() != dev):
        raise RuntimeError(f"{name}: bias {tuple(bias.shape)} on {bias.device} for weight {tuple(wshape)} on {input.device}")
    return act, shape, wshape[0] // 2, dev


def _composed(z, activation):
    g, u = z.chunk(2, -1)
    return (F.silu(g) if activation == "silu" else F.gelu(g)) * u


def _forward(input, weight, bias, act, scale, out_dtype, shape, n, dev, save=False, x_scale=None, w_scale=None):
    """(out, pre-activations or None)"""
    k = shape[-1]
    x, rows, ldx = rows_of(input, k)
    w, _, ldw = rows_of(weight, k)
    b = None if bias is None else bias.contiguous()
    code = ROW_DTYPE[input.dtype]
    out = input.new_empty(shape[:-1] + (n,), dtype=out_dtype)
    saved = ws = None
    if save:                 # for the backward pass: fp32, or 24 bits of each in three 16-bit planes
        saved = out.new_empty((2, rows, n)) if code == 0 else out.new_empty((3, rows, n), dtype=torch.int16)
    px, pw = x.data_ptr(), w.data_ptr()
    need = _lib.query("cagc_gated_linear_workspace", px, pw, rows, n, k, ldx, ldw, code)
    if need:
        ws = out.new_empty(need, dtype=torch.uint8)
    launch("cagc_gated_linear_fwd", dev, out.data_ptr(), address(saved), address(ws), px, pw, address(b), address(x_scale), address(w_scale), rows, n, k, ldx, ldw, code,
           ROW_DTYPE[out_dtype], act, scale)
    return out, saved


class _GatedLinear(Function):
    @staticmethod
    def forward(ctx, input, weight, bias, act, scale, shape, n, dev):
        out, saved = _forward(input, weight, bias, act, scale, input.dtype, shape, n, dev, save=True)
        ctx.save_for_backward(input, weight, saved)
        ctx.how = act, scale, shape, n, dev
        return out

    @staticmethod
    def backward(ctx, dy):
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def _backward(ctx, dy):
    input, weight, saved = ctx.saved_tensors
    act, scale, shape, n, dev = ctx.how
    want_x, want_w, want_b = ctx.needs_input_grad[:3]
    k, rows = shape[-1], saved.shape[1]
    dx = dw = db = None
    if rows == 0:
        dx = torch.zeros_like(input) if want_x else None
        dw = torch.zeros_like(weight) if want_w else None
        db = weight.new_zeros(2 * n) if want_b else None
        return dx, dw, db, None, None, None, None, None
    x, _, ldx = rows_of(input, k)
    w, _, ldw = rows_of(weight, k)
    g, _, ldg = rows_of(dy, n)
    if want_x:
        dx = torch.empty_like(input, memory_format=torch.contiguous_format)
    if want_w:
        dw = torch.empty_like(weight, memory_format=torch.contiguous_format)
    if want_b:
        db = weight.new_empty(2 * n)
    code, px, pw = ROW_DTYPE[input.dtype], x.data_ptr(), w.data_ptr()
    ws = saved.new_empty(_lib.query("cagc_gated_linear_bwd_workspace", px, pw, rows, n, k, ldx, ldw, code, want_x, want_w, want_b), dtype=torch.uint8)
    launch("cagc_gated_linear_bwd", dev, address(dx), address(dw), address(db), ws.data_ptr(), g.data_ptr(), saved.data_ptr(), px, pw, rows, n, k, ldx, ldw, ldg, code, act, scale)
    return dx, dw, db, None, None, None, None, None


_backward_once = once_differentiable(_backward)


def gated_linear(input, weight, bias=None, activation="silu", scale=1.0):
    """[..., k] -> [..., n] with weight [2n, k] (n gate rows, then n up rows) and bias [2n], all of one type."""
    act, shape, n, dev = _check("gated_linear", input, weight, bias, activation)
    dtype = input.dtype
    if bias is not None and bias.dtype is not dtype:
        raise RuntimeError(f"gated_linear: bias {bias.dtype}, input {dtype}")
    if dev < 0:
        wide = dtype if dtype == torch.float64 else torch.float32
        z = F.linear(input.to(wide), weight.to(wide)) * scale
        return _composed(z if bias is None else z + bias.to(wide), activation).to(dtype)
    if dtype not in _TYPES:
        raise RuntimeError(f"gated_linear (HIP): unsupported dtype {dtype}")
    no_tangents("gated_linear", (input, weight, bias))
    if torch.is_grad_enabled() and (input.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _GatedLinear.apply(input, weight, bias, act, float(scale), shape, n, dev)
    return _forward(input, weight, bias, act, float(scale), dtype, shape, n, dev)[0]


def gated_linear_e4m3(input, input_scale, weight, weight_scale, bias=None, activation="silu", out_dtype=torch.bfloat16):
    """The gated projection on 8-bit operands: input [..., k] and weight [2n, k] in float8_e4m3fn with an fp32 scale per row (input_scale [...],
    weight_scale [2n]: `rms_norm_e4m3`, `quantize_rows_e4m3`), bias in out_dtype (fp32 / fp16 / bf16).  Sums are good to about 1.5e-5 of their
    size (the matrix cores cut 8-bit products to 14 bits below the largest of 8 neighbours).  No backward pass."""
    name = "gated_linear_e4m3"
    act, shape, n, dev = _check(name, input, weight, bias, activation)
    if input.dtype is not torch.float8_e4m3fn:
        raise RuntimeError(f"{name}: input {input.dtype} (float8_e4m3fn)")
    if out_dtype not in _TYPES or (bias is not None and bias.dtype is not out_dtype):
        raise RuntimeError(f"{name}: out_dtype {out_dtype}, bias {None if bias is None else bias.dtype}")
    for s, want, what in ((input_scale, shape[:-1], "input_scale"), (weight_scale, weight.shape[:1], "weight_scale")):
        if s.shape != want or s.dtype is not torch.float32 or s.get_device() != dev:
            raise RuntimeError(f"{name}: {what} {tuple(s.shape)} {s.dtype} on {s.device} ({tuple(want)} float32 on {input.device})")
    if torch.is_grad_enabled() and (input_scale.requires_grad or weight_scale.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad()")
    no_tangents(name, (input, input_scale, weight, weight_scale, bias))
    if dev < 0:
        z = F.linear(input.float(), weight.float()) * input_scale[..., None] * weight_scale
        return _composed(z if bias is None else z + bias.float(), activation).to(out_dtype)
    return _forward(input, weight, bias, act, 1.0, out_dtype, shape, n, dev, x_scale=input_scale.contiguous(), w_scale=weight_scale.contiguous())[0]
