"""Drop-in name for the reference's `op` package (reference op/__init__.py:1-2)."""
from cagc.op import (FusedLeakyReLU, clip_grad_norm_, fused_leaky_relu, gated_linear, gated_linear_e4m3, get_total_norm,  # noqa: F401
                     quantize_rows_e4m3, rms_norm, rms_norm_e4m3, upfirdn2d)
