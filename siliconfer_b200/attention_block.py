"""The attention half of a decoder layer in 8 bits: norm, projections, rotary positions, paged cache, attention.

Six kernels a call (with one more where the 8-bit cache's query and key heads
are normed or positions are given), and nothing between them: the norm's codes are the fused
projection's input, whose output's slices (queries, keys, values, not copied)
go into the cache with their positions and to the attention, and the norm after
the output projection adds the residual and hands the next layer its codes.

The cache is held in 8 bits (``PagedKVCache``) or in 4 (``Paged4KVCache``, which
norms and turns query and key heads in its append).  Keys that the 8-bit cache
gets normed, or turned by given positions, are rounded to the block's type on the
way; else, and in the 4-bit cache, they are rounded once, to their codes.

    python -m siliconfer_b200.attention_block

runs a prompt and decode steps (one CUDA graph, replayed) on random weights with
either cache and prints the time of each.
"""
from __future__ import annotations

import torch

from .fp8_linear import Fp8Linear
from .norm import quantize_e4m3, rms_norm_e4m3
from .paged_kv import PagedKVCache
from .paged_kv4 import Paged4KVCache
from .rotary import qk_norm_rotary, rotary_table


class Fp8AttentionBlock(torch.nn.Module):
    """``w_qkv`` [(heads + 2 n_kv_heads) * head_dim, hidden]: queries, keys, values; ``w_o`` [hidden, heads * head_dim];
    ``norm_in`` and ``norm_out`` [hidden] weights of the norms before the attention and after it; ``q_norm`` and ``k_norm``
    [head_dim] of norms of each query and key head (both or neither)."""

    def __init__(self, w_qkv, w_o, norm_in, norm_out, heads: int, n_kv_heads: int, eps: float = 1e-6, window: int = 0,
                 interleaved: bool = False, qkv_bias=None, dtype=torch.bfloat16, device=None, q_norm=None, k_norm=None):
        super().__init__()
        self.heads, self.n_kv_heads, self.head_dim = heads, n_kv_heads, w_qkv.shape[0] // (heads + 2 * n_kv_heads)
        if w_qkv.shape[0] != (heads + 2 * n_kv_heads) * self.head_dim or w_o.shape[1] != heads * self.head_dim:
            raise RuntimeError("w_qkv and w_o do not agree on heads and head_dim")
        self.eps, self.window, self.interleaved = eps, window, interleaved
        self.qkv = Fp8Linear(w_qkv, qkv_bias, device=device, out_dtype=dtype)
        self.o = Fp8Linear(w_o, device=device, out_dtype=dtype)
        place = dict(device=self.qkv.codes.device, dtype=torch.float32)
        self.register_buffer("norm_in", torch.as_tensor(norm_in).to(**place), persistent=False)
        self.register_buffer("norm_out", torch.as_tensor(norm_out).to(**place), persistent=False)
        if (q_norm is None) != (k_norm is None):
            raise RuntimeError("q_norm and k_norm go together")
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            self.register_buffer(name, None if w is None else torch.as_tensor(w).to(**place), persistent=False)

    def forward(self, x, cache, block_table, seq_lens, table, starts=None, positions=None, axes=None):
        """x [T, hidden], the last tokens of their sequences (``PagedKVCache`` or ``Paged4KVCache``) ->
        ((codes, scales), residual): the normed input of what follows, and x plus the attention's output.

        ``positions`` [T], or [T, axes] with ``axes`` (``rotary_axes``), in place of the tokens' places in their sequences;
        those of rows that hold no token are not looked at."""
        if axes is not None and positions is None:
            raise RuntimeError("axes need positions")
        T, H, Hkv, D = x.shape[0], self.heads, self.n_kv_heads, self.head_dim
        qkv = self.qkv(rms_norm_e4m3(x, self.norm_in, self.eps)).view(T, H + 2 * Hkv, D)
        q, k, v = qkv.split((H, Hkv, Hkv), 1)
        head_eps = None if self.q_norm is None else self.eps
        if isinstance(cache, Paged4KVCache):
            q = cache.append(k, v, block_table, seq_lens, starts, q=q, table=table, interleaved=self.interleaved,
                             positions=positions, axes=axes, q_weight=self.q_norm, k_weight=self.k_norm, eps=head_eps)
        elif positions is not None:
            q, k = qk_norm_rotary(q, k, positions, table, self.q_norm, self.k_norm, head_eps, self.interleaved, axes, seq_lens, starts)
            cache.append(k, v, block_table, seq_lens, starts)
        else:
            if head_eps is not None:
                q, k = qk_norm_rotary(q, k, q_weight=self.q_norm, k_weight=self.k_norm, eps=head_eps)
            q = cache.append(k, v, block_table, seq_lens, starts, q=q, table=table, interleaved=self.interleaved)
        y = cache.attend(q, block_table, seq_lens, starts, window=self.window)
        codes, scales, h = rms_norm_e4m3(self.o(quantize_e4m3(y.view(T, H * D))), self.norm_out, self.eps, residual=x)
        return (codes, scales), h


def main(hidden: int = 4096, heads: int = 32, n_kv_heads: int = 8, head_dim: int = 128, batch: int = 16, prompt: int = 512,
         steps: int = 64, page: int = 64):
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    weights = (rand((heads + 2 * n_kv_heads) * head_dim, hidden) * hidden ** -0.5,
               rand(hidden, heads * head_dim) * (heads * head_dim) ** -0.5, torch.ones(hidden), torch.ones(hidden))
    per = -(-(prompt + steps) // page)
    pages = torch.arange(batch * per, dtype=torch.int32, device="cuda").view(batch, per)
    table = rotary_table(per * page, head_dim)
    x, h = rand(batch * prompt, hidden).bfloat16(), rand(batch, hidden).bfloat16()
    for kind in (PagedKVCache, Paged4KVCache):
        normed = {} if kind is PagedKVCache else dict(q_norm=torch.ones(head_dim), k_norm=torch.ones(head_dim))
        block = Fp8AttentionBlock(*weights, heads, n_kv_heads, **normed)
        cache = kind(batch * per, n_kv_heads, head_dim, page)
        lens = torch.full((batch,), prompt, dtype=torch.int32, device="cuda")
        step = lambda: block(h, cache, pages, lens, table)
        block(x, cache, pages, lens, table)
        graph, events = torch.cuda.CUDAGraph(), [torch.cuda.Event(enable_timing=True) for _ in range(4)]
        step()                                   # on the last prompt token's place, which the first step takes again
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            lens.add_(1)
            step()
        for timed in (False, True):
            if timed:
                events[0].record()
            for _ in range(4):
                block(x, cache, pages, lens, table)
        events[1].record()
        events[2].record()
        for _ in range(steps):
            graph.replay()
        events[3].record()
        events[3].synchronize()
        print(f"{kind.__name__}: {batch} prompts of {prompt} tokens: {events[0].elapsed_time(events[1]) * 1e3 / 4:.1f} us; "
              f"a decode step of {batch} sequences: {events[2].elapsed_time(events[3]) * 1e3 / steps:.1f} us")


__all__ = ["Fp8AttentionBlock"]

if __name__ == "__main__":
    main()
