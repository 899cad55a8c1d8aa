"""Linear layers over e4m3 weights with one fp32 scale for every 128 x 128 block.

The 8-bit sibling of ``Q4Linear``: weights of one byte, products on the tensor
cores in e4m3, sums in fp32.  Inputs are e4m3 rows with one scale for every
128 columns, as ``rms_norm_e4m3`` and ``quantize_e4m3`` give them.  No
counterpart in siliconfer (its weights are int4 or int2).  The kernel is in
libsf_q4.so (``sf_fp8_linear``); there is no CPU fallback, and no gradient:
outputs are detached from inputs that require one.
"""
from __future__ import annotations

import torch

from . import _lib
from .norm import quantize_e4m3

BLOCK = 128
E4M3_MAX = 448.0


def quantize_weight_e4m3(w: torch.Tensor):
    """w [N, K] -> (codes float8_e4m3fn [N, K], scales fp32 [ceil(N / 128), ceil(K / 128)]), on w's device.

    scale = max|w| / 448 of the block (1 where that is 0); the codes' rows start at multiples of 16 bytes."""
    if w.dim() != 2 or not w.numel():
        raise RuntimeError("w must be a non-empty [N, K]")
    N, K = w.shape
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    blocks = torch.nn.functional.pad(w.detach().float(), (0, kb * BLOCK - K, 0, nb * BLOCK - N)).view(nb, BLOCK, kb, BLOCK)
    amax = blocks.abs().amax((1, 3))
    scales = torch.where(amax == 0, torch.ones_like(amax), (amax / E4M3_MAX).clamp_min(2.0 ** -126))
    values = (blocks / scales[:, None, :, None]).clamp_(-E4M3_MAX, E4M3_MAX).view(nb * BLOCK, kb * BLOCK)[:N, :K]
    store = torch.zeros((N, -(-K // 16) * 16), dtype=torch.uint8, device=w.device)
    store[:, :K] = values.to(torch.float8_e4m3fn).view(torch.uint8)
    return store.view(torch.float8_e4m3fn)[:, :K], scales


def fp8_linear(x, x_scales, w, w_scales, bias=None, out_dtype=torch.float32):
    """Y[..., N] = X @ W^T (+ bias) over codes and their scales, fp32 accumulation.

    x [..., K] codes with x_scales [..., ceil(K / 128)]; w [N, K] codes with
    w_scales [ceil(N / 128), ceil(K / 128)]; bias fp32 [N].  The rows of x and w
    start at multiples of 16 bytes (the quantizers' outputs do)."""
    return _lib.ext().fp8_linear(x, x_scales, w, w_scales, bias, out_dtype)


class Fp8Linear(torch.nn.Module):
    """``Fp8Linear(weight, bias)(x)``: x a float tensor (quantized here), or the (codes, scales) pair of
    ``rms_norm_e4m3``, which skips that pass."""

    def __init__(self, weight, bias=None, device=None, out_dtype=None):
        super().__init__()
        weight = torch.as_tensor(weight)
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else weight.device
        codes, scales = quantize_weight_e4m3(weight.to(device))
        self.out_features, self.in_features = codes.shape
        self.out_dtype = out_dtype
        # the whole padded rows: moving the module keeps them at multiples of 16 bytes
        self.register_buffer("codes", codes.as_strided((codes.shape[0], -(-codes.shape[1] // 16) * 16),
                                                       (-(-codes.shape[1] // 16) * 16, 1)), persistent=False)
        self.register_buffer("scales", scales, persistent=False)
        self.register_buffer("bias", None if bias is None else torch.as_tensor(bias).detach().to(
            device=device, dtype=torch.float32).contiguous(), persistent=False)

    def forward(self, x):
        dtype = self.out_dtype
        if not isinstance(x, tuple):
            dtype = dtype or x.dtype
            x = quantize_e4m3(x)
        codes, scales = x[:2]
        if codes.shape[-1] != self.in_features:
            raise RuntimeError("X/W in_features mismatch")
        return fp8_linear(codes, scales, self.codes[:, :self.in_features], self.scales, self.bias, dtype or torch.float32)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


__all__ = ["quantize_e4m3", "quantize_weight_e4m3", "fp8_linear", "Fp8Linear"]
