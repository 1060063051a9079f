"""Gated projection — beside EqualLinear, whose `scale` convention it keeps (weights of unit variance, scaled at run time):

    out = act(scale * input @ Wg.T + bg) * (scale * input @ Wu.T + bu),   weight = [Wg; Wu] of 2n rows, act = SiLU or GELU

GPU tensors -> cagc_gated_linear_* (csrc/gated.hip), one kernel for both projections, the activation and the product; fp32 / fp16 / bf16 with
fp32 sums.  CPU tensors -> composed PyTorch.  First-order autograd (a second derivative raises)."""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from .. import _lib

ACTIVATIONS = {"silu": 0, "gelu": 1}      # CAGC_ACT_*
_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _check(name, input, weight, bias, activation):
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"{name}: activation {activation!r} (one of {', '.join(ACTIVATIONS)})")
    if input.dim() < 1 or weight.dim() != 2 or weight.shape[0] % 2 or weight.shape[0] == 0 or weight.shape[1] != input.shape[-1] or weight.shape[1] == 0:
        raise RuntimeError(f"{name}: weight {tuple(weight.shape)} for input {tuple(input.shape)} (2n rows of the input's width)")
    if weight.dtype != input.dtype or weight.device != input.device:
        raise RuntimeError(f"{name}: weight {weight.dtype} on {weight.device}, input {input.dtype} on {input.device}")
    if bias is not None and (bias.shape != weight.shape[:1] or bias.device != input.device):
        raise RuntimeError(f"{name}: bias {tuple(bias.shape)} on {bias.device} for weight {tuple(weight.shape)} on {input.device}")


def _composed(z, activation):
    g, u = z.chunk(2, -1)
    return (F.silu(g) if activation == "silu" else F.gelu(g)) * u


def _p(t):
    return None if t is None else t.data_ptr()


def _forward(name, input, weight, bias, act, scale, out_dtype, saved=None, x_scale=None, w_scale=None):
    k, n = input.shape[-1], weight.shape[0] // 2
    x, ldx = _lib.rows_of(input, k)
    w, ldw = _lib.rows_of(weight, k)
    b = None if bias is None else bias.contiguous()
    rows, code = x.shape[0], _lib.ROW_DTYPE[input.dtype]
    out = torch.empty(input.shape[:-1] + (n,), dtype=out_dtype, device=input.device)
    if saved is not None:                # pre-activations for the backward pass: fp32, or 24 bits of each in three 16-bit planes
        saved = (torch.empty(2, rows, n, dtype=torch.float32, device=input.device) if input.dtype == torch.float32 else
                 torch.empty(3, rows, n, dtype=torch.int16, device=input.device))
    with _lib.on_device(x):
        need = _lib.query("cagc_gated_linear_workspace", x.data_ptr(), w.data_ptr(), rows, n, k, ldx, ldw, code)
        ws = torch.empty(need, dtype=torch.uint8, device=input.device) if need else None
        _lib.call("cagc_gated_linear_fwd", out.data_ptr(), _p(saved), _p(ws), x.data_ptr(), w.data_ptr(), _p(b), _p(x_scale), _p(w_scale), rows, n, k,
                  ldx, ldw, code, _lib.ROW_DTYPE[out_dtype], act, scale)
    return out, saved


class _GatedLinear(Function):
    @staticmethod
    def forward(ctx, input, weight, bias, act, scale):
        out, saved = _forward("gated_linear", input, weight, bias, act, scale, input.dtype, saved=True)
        ctx.save_for_backward(input, weight, saved)
        ctx.act, ctx.scale, ctx.has_bias = act, scale, bias is not None
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        input, weight, saved = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.has_bias and ctx.needs_input_grad[2]
        k, n = input.shape[-1], weight.shape[0] // 2
        rows, dev, dt = saved.shape[1], input.device, input.dtype
        if rows == 0:
            return (torch.zeros_like(input) if want_x else None, torch.zeros_like(weight) if want_w else None,
                    torch.zeros(2 * n, dtype=dt, device=dev) if want_b else None, None, None)
        x, ldx = _lib.rows_of(input, k)
        w, ldw = _lib.rows_of(weight, k)
        g, ldg = _lib.rows_of(dy, n)
        dx = torch.empty(input.shape, dtype=dt, device=dev) if want_x else None
        dw = torch.empty(weight.shape, dtype=dt, device=dev) if want_w else None
        db = torch.empty(2 * n, dtype=dt, device=dev) if want_b else None
        code = _lib.ROW_DTYPE[dt]
        with _lib.on_device(x):
            need = _lib.query("cagc_gated_linear_bwd_workspace", x.data_ptr(), w.data_ptr(), rows, n, k, ldx, ldw, code, want_x, want_w, want_b)
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            _lib.call("cagc_gated_linear_bwd", _p(dx), _p(dw), _p(db), ws.data_ptr(), g.data_ptr(), saved.data_ptr(), x.data_ptr(), w.data_ptr(), rows, n, k,
                      ldx, ldw, ldg, code, ctx.act, ctx.scale)
        return dx, dw, db, None, None


def gated_linear(input, weight, bias=None, activation="silu", scale=1.0):
    """[..., k] -> [..., n] with weight [2n, k] (n gate rows, then n up rows) and bias [2n], all of one type."""
    _check("gated_linear", input, weight, bias, activation)
    if bias is not None and bias.dtype != input.dtype:
        raise RuntimeError(f"gated_linear: bias {bias.dtype}, input {input.dtype}")
    if input.device.type == "cpu":
        wide = input.dtype if input.dtype == torch.float64 else torch.float32
        z = F.linear(input.to(wide), weight.to(wide)) * scale
        return _composed(z if bias is None else z + bias.to(wide), activation).to(input.dtype)
    if input.dtype not in _TYPES:
        raise RuntimeError(f"gated_linear (HIP): unsupported dtype {input.dtype}")
    if torch.is_grad_enabled() and (input.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _GatedLinear.apply(input, weight, bias, ACTIVATIONS[activation], float(scale))
    return _forward("gated_linear", input, weight, bias, ACTIVATIONS[activation], float(scale), input.dtype)[0]


def gated_linear_e4m3(input, input_scale, weight, weight_scale, bias=None, activation="silu", out_dtype=torch.bfloat16):
    """The gated projection on 8-bit operands: input [..., k] and weight [2n, k] in float8_e4m3fn with an fp32 scale per row (input_scale [...],
    weight_scale [2n]: `rms_norm_e4m3`, `quantize_rows_e4m3`), bias in out_dtype (fp32 / fp16 / bf16).  No backward pass."""
    name = "gated_linear_e4m3"
    _check(name, input, weight, bias, activation)
    if input.dtype != torch.float8_e4m3fn:
        raise RuntimeError(f"{name}: input {input.dtype} (float8_e4m3fn)")
    if out_dtype not in _TYPES or (bias is not None and bias.dtype != out_dtype):
        raise RuntimeError(f"{name}: out_dtype {out_dtype}, bias {None if bias is None else bias.dtype}")
    for what, s, shape in (("input_scale", input_scale, input.shape[:-1]), ("weight_scale", weight_scale, weight.shape[:1])):
        if s.shape != shape or s.dtype != torch.float32 or s.device != input.device:
            raise RuntimeError(f"{name}: {what} {tuple(s.shape)} {s.dtype} on {s.device} ({tuple(shape)} float32 on {input.device})")
    if torch.is_grad_enabled() and (input_scale.requires_grad or weight_scale.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad()")
    if input.device.type == "cpu":
        z = F.linear(input.float(), weight.float()) * input_scale[..., None] * weight_scale
        return _composed(z if bias is None else z + bias.float(), activation).to(out_dtype)
    return _forward(name, input, weight, bias, ACTIVATIONS[activation], 1.0, out_dtype, x_scale=input_scale.contiguous(),
                    w_scale=weight_scale.contiguous())[0]
