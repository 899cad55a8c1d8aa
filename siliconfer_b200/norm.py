"""RMS norm with the residual's addition, and e4m3 rows with one scale for every 128 columns, on the GPU.

``rms_norm`` feeds ``Q4Linear`` (its output is in the activations' type);
``rms_norm_e4m3`` and ``quantize_e4m3`` give what ``fp8_linear`` reads: e4m3
codes whose rows start at multiples of 16 bytes, and a [..., ceil(K / 128)]
fp32 scale, max|y| / 448 of each row's 128 columns.  No counterpart in
siliconfer, which norms in fp32 through MLX.  The kernels are in libsf_q4.so
(``sf_rms_norm``, ``sf_quantize_e4m3``); there is no CPU fallback, and no
gradient: outputs are detached from inputs that require one.
"""
from __future__ import annotations

from . import _lib


def rms_norm(x, weight=None, eps: float = 1e-6, residual=None, out_dtype=None):
    """x [..., K] -> y = h / sqrt(mean(h^2) + eps) * weight with h = x + residual.

    fp32 arithmetic; y has ``out_dtype`` (x's dtype by default).  With a
    ``residual`` the result is (y, h), h rounded to x's dtype: the next
    residual.  The norm itself uses h before that rounding."""
    y, _, h = _lib.ext().rms_norm(x, weight, eps, residual, out_dtype, False)
    return y if residual is None else (y, h)


def rms_norm_e4m3(x, weight=None, eps: float = 1e-6, residual=None):
    """``rms_norm`` with its output in e4m3: (codes, scales), or (codes, scales, h) with a ``residual``."""
    y, scales, h = _lib.ext().rms_norm(x, weight, eps, residual, None, True)
    return (y, scales) if residual is None else (y, scales, h)


def quantize_e4m3(x):
    """x [..., K] -> (codes float8_e4m3fn [..., K], scales fp32 [..., ceil(K / 128)])."""
    return _lib.ext().quantize_e4m3(x)


__all__ = ["rms_norm", "rms_norm_e4m3", "quantize_e4m3"]
