"""A paged cache of keys and values in e4m3, and attention over it.

Beside ``kv_attention`` (one contiguous int8 cache, a scale for every vector):
here sequences share a pool of pages, and a page keeps one power-of-two scale
for each kv head, so that tokens can be added to a page, and its older codes
moved to a larger scale, without losing what they hold.  Keys and values can
be written together with the rotary positions of the step.  The kernels are in
libsf_q4.so (``sf_paged_append``, ``sf_paged_attention``); there is no CPU
fallback, and no gradient: outputs are detached from inputs that require one.

A call's new tokens are packed: sequence b's are rows starts[b] ..
starts[b + 1] - 1 of q, k and v (without ``starts``: the same number for every
sequence), and are the last of its seq_lens[b] tokens.  Token j of sequence b
is slot j % page_size of page block_table[b, j // page_size].  A sequence with
fewer tokens than rows has padding rows in front, which are not written and see
no key (a waiting slot of a decode batch: length 0 and one row).  Rows before
starts[0] and from starts[batch] on are no sequence's and are treated alike (a
captured step replayed with fewer tokens).
"""
from __future__ import annotations

import torch

from . import _lib


def paged_append(k, v, k_codes, k_scales, v_codes, v_scales, block_table, seq_lens, starts=None, q=None, table=None,
                 interleaved: bool = False):
    """Writes k and v [T, n_kv_heads, head_dim] as the last tokens of their sequences.

    With a ``table`` (``rotary_table``) k is turned by its positions first, and
    q [T, heads, head_dim], if given, is returned turned likewise.  Codes and
    scales are updated in place.  Two sequences of one call must not write to
    the same page."""
    return _lib.ext().paged_append(k, v, k_codes, k_scales, v_codes, v_scales, block_table, seq_lens, starts, q, table,
                                   interleaved)


def paged_attention(q, k_codes, k_scales, v_codes, v_scales, block_table, seq_lens, starts=None, scale=None,
                    window: int = 0, out_dtype=None, return_lse: bool = False):
    """q [T, heads, head_dim] -> softmax(scale * q . k) v over each row's own and earlier tokens.

    ``scale`` defaults to head_dim^-0.5; ``window`` > 0 limits a row to its
    last ``window`` keys.  Weights are held as fine as the finer of q's type
    and ``out_dtype`` (q's type by default).  A row that sees no key gives 0.  ``return_lse`` adds
    log sum e^(scale * q . k) [T, heads] (-inf for such a row)."""
    out, lse = _lib.ext().paged_attention(q, k_codes, k_scales, v_codes, v_scales, block_table, seq_lens, starts, scale,
                                          window, out_dtype, return_lse)
    return (out, lse) if return_lse else out


class PagedKVCache:
    """A pool of pages: k_codes, v_codes [num_pages, n_kv_heads, page_size, head_dim] float8_e4m3fn and
    k_scales, v_scales [num_pages, n_kv_heads] fp32.  Which pages a sequence holds is the caller's to keep."""

    def __init__(self, num_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64, device=None):
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else "cpu"
        shape = (num_pages, n_kv_heads, page_size, head_dim)
        self.page_size = page_size
        self.k_codes = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        self.v_codes = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        self.k_scales = torch.ones(shape[:2], dtype=torch.float32, device=device)
        self.v_scales = torch.ones(shape[:2], dtype=torch.float32, device=device)

    def append(self, k, v, block_table, seq_lens, starts=None, q=None, table=None, interleaved: bool = False):
        return paged_append(k, v, self.k_codes, self.k_scales, self.v_codes, self.v_scales, block_table, seq_lens,
                            starts, q, table, interleaved)

    def attend(self, q, block_table, seq_lens, starts=None, scale=None, window: int = 0, out_dtype=None,
               return_lse: bool = False):
        return paged_attention(q, self.k_codes, self.k_scales, self.v_codes, self.v_scales, block_table, seq_lens,
                               starts, scale, window, out_dtype, return_lse)


__all__ = ["paged_append", "paged_attention", "PagedKVCache"]
