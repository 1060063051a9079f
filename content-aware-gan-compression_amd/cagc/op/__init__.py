"""Operator layer (L1) — same public names as the reference's `op` package (op/__init__.py:1-2), and the framework's own row-wise and
training operators."""
from .fused_act import FusedLeakyReLU, fused_leaky_relu
from .gated_linear import gated_linear, gated_linear_e4m3
from .grad_clip import clip_grad_norm_, get_total_norm
from .rms_norm import quantize_rows_e4m3, rms_norm, rms_norm_e4m3
from .upfirdn2d import upfirdn2d

__all__ = ["FusedLeakyReLU", "fused_leaky_relu", "upfirdn2d", "rms_norm", "rms_norm_e4m3", "quantize_rows_e4m3", "gated_linear",
           "gated_linear_e4m3", "clip_grad_norm_", "get_total_norm"]
