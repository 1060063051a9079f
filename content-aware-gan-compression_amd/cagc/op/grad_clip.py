"""Norm of many gradients together and clipping by it, with the interface of torch.nn.utils.clip_grad_norm_ — what KDStep's
`max_grad_norm` calls.

GPU tensors -> cagc_clip_grad_norm (csrc/gradnorm.hip): a launch for up to 120 tensors' norm, one that joins it, one that scales (and
leaves at once where nothing is to be clipped); sums in 64 bits and in a fixed order; nothing waits for the host, so it can be captured.  CPU tensors ->
composed PyTorch.  On the GPU two tensors of the list must not share memory (strided views of one buffer may lie between each other)."""
from array import array
from operator import attrgetter

import torch

from .. import _lib

_NORMS = {1.0: 1, 2.0: 2, float("inf"): 0}
_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 3}
_T = torch.Tensor
_dtype, _layout = attrgetter("dtype"), attrgetter("layout")


def _check(name, tensors, norm_type):
    """(number of the device that all the tensors are on, the norm's code)"""
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise RuntimeError(f"{name}: norm_type {norm_type} (1, 2 or inf)")
    devices, dtypes, layouts = set(map(_T.get_device, tensors)), set(map(_dtype, tensors)), set(map(_layout, tensors))
    dev = tensors[0].get_device()
    if len(devices) > 1 or layouts != {torch.strided} or (dev >= 0 and not dtypes <= _CODES.keys()) or not all(t.is_floating_point for t in dtypes):
        raise RuntimeError(f"{name}: tensors of {sorted(map(str, dtypes))} {sorted(map(str, layouts))} on devices {sorted(devices)} "
                           "(dense fp32 / fp16 / bf16 gradients on one device)")
    return dev, code


def _composed_norm(tensors, code):
    if code == 0:
        return torch.stack([t.abs().amax().double() if t.numel() else t.new_zeros((), dtype=torch.float64) for t in tensors]).amax()
    s = torch.stack([t.double().abs().pow(code).sum() for t in tensors]).sum()
    return s.sqrt() if code == 2 else s


def _span(t):
    """(first address, distance of the last byte, t)"""
    e = t.element_size()
    if t.is_contiguous():
        return t.data_ptr(), t.numel() * e - 1, t
    return t.data_ptr(), sum(s * (n - 1) for s, n in zip(t.stride(), t.size())) * e + e - 1, t


def _layout_of(t):
    """[(stride, count), ...] in bytes, the largest stride first: the bytes that t's elements take, from its first address on"""
    e = t.element_size()
    dims = []
    for s, n in [(1, e)] + sorted((s * e, n) for s, n in zip(t.stride(), t.size()) if n > 1 and s):
        if dims and s == dims[-1][0] * dims[-1][1]:
            dims[-1] = (dims[-1][0], dims[-1][1] * n)
        else:
            dims.append((s, n))
    return dims[::-1]


def _reach(dims):
    return sum(s * (n - 1) for s, n in dims)


def _meet(a, b, d, left):
    """whether a byte of layout `a` is one of layout `b`, which begins d behind it.  The outer dimension with the larger stride goes by; of two with the same stride only the difference of their
    indices matters, so that columns of one matrix cost the same however many rows it has.  left: steps that may be taken, then the answer is yes."""
    if d > _reach(a) or -d > _reach(b):
        return False
    if not a and not b:
        return d == 0
    left[0] -= 1
    if left[0] < 0:
        return True
    sa, sb = a[0][0] if a else 0, b[0][0] if b else 0
    s = max(sa, sb)
    a1, b1 = a[1:] if sa == s else a, b[1:] if sb == s else b
    lo = -((_reach(a1) - d) // s)                # d - m s within [-reach(b1), reach(a1)]
    hi = (d + _reach(b1)) // s
    lo, hi = max(lo, 1 - b[0][1] if sb == s else 0), min(hi, a[0][1] - 1 if sa == s else 0)
    return any(_meet(a1, b1, d - m * s, left) for m in range(lo, hi + 1))


def _share_memory(tensors):
    """whether two tensors of the list have an element's memory in common"""
    open_ = []                  # those that reach beyond where the next one begins
    for p in sorted((_span(t) for t in tensors if t.numel()), key=lambda p: p[0]):
        open_ = [q for q in open_ if q[0] + q[1] >= p[0]]
        if open_ and any(_meet(_layout_of(q[2]), _layout_of(p[2]), p[0] - q[0], [20000]) for q in open_):
            return True
        open_.append(p)
    return False


def _launch(tensors, code, max_norm, scale, dev):
    """the norm (0-dim fp32); with `scale`, the tensors are clipped in place"""
    _lib.no_tangents("clip_grad_norm_" if scale else "get_total_norm", tensors)
    flat, n = tensors, len(tensors)
    if not all(map(_T.is_contiguous, tensors)):
        if _share_memory(tensors):              # (the library sees copies)
            raise RuntimeError("cagc_clip_grad_norm: two tensors of the list share memory")
        if scale and any(s == 0 and n > 1 for t in tensors for s, n in zip(t.stride(), t.size())):
            raise RuntimeError("cagc_clip_grad_norm: elements of an expanded tensor share memory")
        flat = [t.contiguous() for t in tensors]
    p, sizes = array("Q", map(_T.data_ptr, flat)), array("q", map(_T.numel, flat))
    types = array("i", map(_CODES.__getitem__, map(_dtype, flat)))
    sizes_at = sizes.buffer_info()[0]
    norm = flat[0].new_empty((), dtype=torch.float32)
    ws = norm.new_empty(_lib.query("cagc_grad_norm_workspace", sizes_at, n) // 4)
    _lib.launch("cagc_clip_grad_norm", dev, norm.data_ptr(), ws.data_ptr(), p.buffer_info()[0], sizes_at, types.buffer_info()[0], n, code, max_norm, scale)
    if scale:
        if flat is not tensors:
            with torch.no_grad():
                for t, f in zip(tensors, flat):
                    if f is not t:
                        t.copy_(f)
        torch.autograd.graph.increment_version(tensors)
    return norm


def _finite(name, norm, error_if_nonfinite):
    if error_if_nonfinite and not bool(torch.isfinite(norm)):
        raise RuntimeError(f"{name}: the norm of the gradients is not finite")


def get_total_norm(tensors, norm_type=2.0, error_if_nonfinite=False):
    """Norm of all the tensors' elements together (0-dim fp32 on their device; not differentiated)."""
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    dev, code = _check("get_total_norm", tensors, norm_type)
    if dev < 0:
        with torch.no_grad():
            norm = _composed_norm(tensors, code).float()
    else:
        norm = _launch(tensors, code, 0.0, 0, dev)
    _finite("get_total_norm", norm, error_if_nonfinite)
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scales the parameters' gradients in place by min(1, max_norm / (norm + 1e-6)), norm taken over all of them together, and returns the
    norm before (0-dim fp32 on their device).  error_if_nonfinite waits for the norm and raises before anything is scaled."""
    name = "clip_grad_norm_"
    parameters = [parameters] if torch.is_tensor(parameters) else parameters
    grads = [g for p in parameters if (g := p.grad) is not None]
    if not grads:
        return torch.tensor(0.0)
    max_norm = float(max_norm)
    dev, code = _check(name, grads, norm_type)
    if dev < 0:
        with torch.no_grad():
            norm = _composed_norm(grads, code)
            _finite(name, norm, error_if_nonfinite)
            coef = (max_norm / (norm + 1e-6)).clamp(max=1.0)
            for g in grads:
                g.copy_(g * coef if g.dtype == torch.float64 else g.float() * coef.float())
        return norm.float()
    if error_if_nonfinite:
        _finite(name, _launch(grads, code, 0.0, 0, dev), True)
    return _launch(grads, code, max_norm, 1, dev)
