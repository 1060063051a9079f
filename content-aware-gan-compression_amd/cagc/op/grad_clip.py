"""Norm of many gradients together and clipping by it, with the interface of torch.nn.utils.clip_grad_norm_ — what KDStep's
`max_grad_norm` calls.

GPU tensors -> cagc_clip_grad_norm (csrc/gradnorm.hip): a launch for up to 120 tensors' norm, one that joins it, one that scales (and
leaves at once where nothing is to be clipped); sums in 64 bits and in a fixed order; nothing waits for the host, so it can be captured.  CPU tensors ->
composed PyTorch."""
import ctypes

import torch

from .. import _lib

_NORMS = {1.0: 1, 2.0: 2, float("inf"): 0}


def _tensors(name, tensors):
    """the list's tensors, on one device and of types the kernels take"""
    dev = tensors[0].device
    for t in tensors:
        if t.device != dev or t.layout != torch.strided or (dev.type != "cpu" and t.dtype not in _lib.ROW_DTYPE or t.dtype == torch.float8_e4m3fn):
            raise RuntimeError(f"{name}: {t.dtype} {t.layout} tensor on {t.device} (dense fp32 / fp16 / bf16 gradients on one device)")
    return dev


def _norm_code(name, norm_type):
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise RuntimeError(f"{name}: norm_type {norm_type} (1, 2 or inf)")
    return code


def _composed_norm(tensors, code):
    if code == 0:
        return torch.stack([t.abs().amax().double() if t.numel() else t.new_zeros((), dtype=torch.float64) for t in tensors]).amax()
    s = torch.stack([t.double().abs().pow(code).sum() for t in tensors]).sum()
    return s.sqrt() if code == 2 else s


def _launch(tensors, code, max_norm, scale, dev):
    """the norm (0-dim fp32); with `scale`, the tensors are clipped in place"""
    flat = [t if t.is_contiguous() else t.contiguous() for t in tensors]
    n = len(flat)
    p = (ctypes.c_void_p * n)(*[t.data_ptr() for t in flat])
    sizes = (ctypes.c_int64 * n)(*[t.numel() for t in flat])
    types = (ctypes.c_int * n)(*[_lib.ROW_DTYPE[t.dtype] for t in flat])
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(_lib.query("cagc_grad_norm_workspace", sizes, n), dtype=torch.uint8, device=dev)
    with _lib.on_device(norm):
        _lib.call("cagc_clip_grad_norm", norm.data_ptr(), ws.data_ptr(), p, sizes, types, n, code, max_norm, scale)
    if scale:
        for t, f in zip(tensors, flat):
            if f is not t:
                t.copy_(f)
        torch.autograd.graph.increment_version(tensors)
    return norm


def _finite(name, norm, error_if_nonfinite):
    if error_if_nonfinite and not bool(torch.isfinite(norm)):
        raise RuntimeError(f"{name}: the norm of the gradients is not finite")


@torch.no_grad()
def get_total_norm(tensors, norm_type=2.0, error_if_nonfinite=False):
    """Norm of all the tensors' elements together (0-dim fp32 on their device)."""
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    code = _norm_code("get_total_norm", norm_type)
    if not tensors:
        return torch.tensor(0.0)
    dev = _tensors("get_total_norm", tensors)
    norm = _composed_norm(tensors, code).float() if dev.type == "cpu" else _launch(tensors, code, 0.0, 0, dev)
    _finite("get_total_norm", norm, error_if_nonfinite)
    return norm


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scales the parameters' gradients in place by min(1, max_norm / (norm + 1e-6)), norm taken over all of them together, and returns the
    norm before (0-dim fp32 on their device).  error_if_nonfinite waits for the norm and raises before anything is scaled."""
    name = "clip_grad_norm_"
    parameters = [parameters] if torch.is_tensor(parameters) else parameters
    grads = [p.grad for p in parameters if p.grad is not None]
    max_norm, code = float(max_norm), _norm_code(name, norm_type)
    if not grads:
        return torch.tensor(0.0)
    dev = _tensors(name, grads)
    if dev.type == "cpu":
        norm = _composed_norm(grads, code)
        _finite(name, norm, error_if_nonfinite)
        coef = (max_norm / (norm + 1e-6)).clamp(max=1.0)
        for g in grads:
            g.copy_(g * coef if g.dtype == torch.float64 else g.float() * coef.float())
        return norm.float()
    if error_if_nonfinite:
        _finite(name, _launch(grads, code, 0.0, 0, dev), True)
    return _launch(grads, code, max_norm, 1, dev)
