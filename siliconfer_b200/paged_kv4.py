"""A paged cache of keys and values in 4 bits, and attention over it.

``paged_kv``'s pages and rules with half the bytes: a head's vector is D / 2
bytes of codes and four bf16 scales, one for each quarter of the head.  Keys and
queries can be normed and turned on the way.  Element e of a vector lies in
quarter c = e // (D / 4) at place r = e % (D / 4); its code is bits 4c .. 4c + 3
of the vector's 16-bit word r (low byte first) and stands for
(code - 8) * scale[c].  No counterpart in siliconfer (its cache is int8).  The
kernels are in libsf_q4.so (``sf_paged4_append``, ``sf_paged4_attention``); there
is no CPU fallback, and no gradient: outputs are detached from inputs that
require one.

A call's new tokens are packed as in ``paged_kv``: sequence b's are rows
starts[b] .. starts[b + 1] - 1 of q, k and v (without ``starts``: the same number
for every sequence), the last of its seq_lens[b] tokens; token j of it is slot
j % page_size of page block_table[b, j // page_size].  Rows in front of a
sequence's first token, before starts[0] and from starts[batch] on are written
nowhere and see no key.
"""
from __future__ import annotations

import torch

from . import _lib


def quantize_kv4(x):
    """x [..., head_dim] -> (codes uint8 [..., head_dim / 2], scales bf16 [..., 4]), in torch operations on x's device.

    A quarter's scale is max|x| / 7.5, rounded to fp32 and then to bf16, at least
    2^-126; code - 8 is x / scale, rounded to the nearest (ties to even) and
    limited to -8 .. 7.  Four NaN scales where the vector is not finite."""
    D = x.shape[-1]
    if D % 4:
        raise RuntimeError("head_dim must be a multiple of 4")
    y = x.detach().double().unflatten(-1, (4, D // 4))
    scale = (y.abs().amax(-1) / 7.5).float().bfloat16().clamp_min(2.0 ** -126)
    finite = torch.isfinite(y).all(-1).all(-1)[..., None]
    scale = torch.where(finite, scale, float("nan"))
    n = torch.where(finite[..., None], (y / scale.double()[..., None]).round().clamp(-8, 7) + 8, 8.0).to(torch.int16)
    words = torch.stack([n[..., 0, :] | n[..., 1, :] << 4, n[..., 2, :] | n[..., 3, :] << 4], -1)
    return words.to(torch.uint8).flatten(-2), scale


def dequantize_kv4(codes, scales, dtype=torch.float32):
    """(codes [..., head_dim / 2], scales [..., 4]) -> [..., head_dim], in torch operations on their device."""
    w = codes.unflatten(-1, (-1, 2))
    n = torch.stack([w[..., 0] & 15, w[..., 0] >> 4, w[..., 1] & 15, w[..., 1] >> 4], -2)
    return ((n.float() - 8) * scales.float()[..., None]).flatten(-2).to(dtype)


def paged4_append(k, v, k_codes, k_scales, v_codes, v_scales, block_table, seq_lens, starts=None, q=None, table=None,
                  interleaved: bool = False, positions=None, axes=None, q_weight=None, k_weight=None, eps=None):
    """Writes k and v [T, n_kv_heads, head_dim] as the last tokens of their sequences.

    k, and q [T, heads, head_dim], which is returned, pass through
    ``qk_norm_rotary`` on the way: normed for each head with ``eps``, turned with
    a ``table``, by ``positions`` ([T], or [T, axes] with ``axes``) or, without
    these, by each token's place in its sequence.  Codes and scales are updated
    in place.  Two rows of one call must not be the same token."""
    return _lib.ext().paged4_append(k, v, k_codes, k_scales, v_codes, v_scales, block_table, seq_lens, starts, q, table,
                                    interleaved, positions, axes, q_weight, k_weight, eps)


def paged4_attention(q, k_codes, k_scales, v_codes, v_scales, block_table, seq_lens, starts=None, scale=None,
                     window: int = 0, out_dtype=None, return_lse: bool = False):
    """q [T, heads, head_dim] -> softmax(scale * q . k) v over each row's own and earlier tokens.

    ``scale`` defaults to head_dim^-0.5; ``window`` > 0 limits a row to its
    last ``window`` keys.  A row that sees no key gives 0.  ``return_lse`` adds
    log sum e^(scale * q . k) [T, heads] (-inf for such a row).

    Sums are in fp32.  With 16-bit queries and outputs weights are fp16 numbers,
    and long runs (head_dim 64 or 128) take keys and values rounded to 11 bits:
    a score, and the log-sum, is off by up to 2^-12 of scale * sum |q k| there.
    Scales up to 2^100, of values from 2^-60, any distance apart between tokens;
    smaller ones lose digits, and so does a quarter 2^20 and more below its
    vector's largest."""
    out, lse = _lib.ext().paged4_attention(q, k_codes, k_scales, v_codes, v_scales, block_table, seq_lens, starts, scale,
                                           window, out_dtype, return_lse)
    return (out, lse) if return_lse else out


class Paged4KVCache:
    """A pool of pages: k_codes, v_codes uint8 [num_pages, n_kv_heads, page_size, head_dim / 2] and k_scales, v_scales
    bf16 [num_pages, n_kv_heads, page_size, 4].  Which pages a sequence holds is the caller's to keep."""

    def __init__(self, num_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64, device=None):
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else "cpu"
        if head_dim % 4:
            raise RuntimeError("head_dim must be a multiple of 4")
        shape = (num_pages, n_kv_heads, page_size)
        self.page_size = page_size
        self.k_codes = torch.full((*shape, head_dim // 2), 0x88, dtype=torch.uint8, device=device)
        self.v_codes = torch.full((*shape, head_dim // 2), 0x88, dtype=torch.uint8, device=device)
        self.k_scales = torch.zeros((*shape, 4), dtype=torch.bfloat16, device=device)
        self.v_scales = torch.zeros((*shape, 4), dtype=torch.bfloat16, device=device)

    def append(self, k, v, block_table, seq_lens, starts=None, q=None, table=None, interleaved: bool = False,
               positions=None, axes=None, q_weight=None, k_weight=None, eps=None):
        return paged4_append(k, v, self.k_codes, self.k_scales, self.v_codes, self.v_scales, block_table, seq_lens,
                             starts, q, table, interleaved, positions, axes, q_weight, k_weight, eps)

    def attend(self, q, block_table, seq_lens, starts=None, scale=None, window: int = 0, out_dtype=None,
               return_lse: bool = False):
        return paged4_attention(q, self.k_codes, self.k_scales, self.v_codes, self.v_scales, block_table, seq_lens,
                                starts, scale, window, out_dtype, return_lse)


__all__ = ["quantize_kv4", "dequantize_kv4", "paged4_append", "paged4_attention", "Paged4KVCache"]
