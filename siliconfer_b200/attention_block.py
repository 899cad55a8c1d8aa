"""The attention half of a decoder layer in 8 bits: norm, projections, rotary positions, paged cache, attention.

Six kernels a call, and nothing between them: the norm's codes are the fused
projection's input, whose output's slices (queries, keys, values, not copied)
go into the cache with their positions and to the attention, and the norm after
the output projection adds the residual and hands the next layer its codes.

    python -m siliconfer_b200.attention_block

runs a prompt and decode steps (one CUDA graph, replayed) on random weights and
prints the time of each.
"""
from __future__ import annotations

import torch

from .fp8_linear import Fp8Linear
from .norm import quantize_e4m3, rms_norm_e4m3
from .paged_kv import PagedKVCache
from .rotary import rotary_table


class Fp8AttentionBlock(torch.nn.Module):
    """``w_qkv`` [(heads + 2 n_kv_heads) * head_dim, hidden]: queries, keys, values; ``w_o`` [hidden, heads * head_dim];
    ``norm_in`` and ``norm_out`` [hidden] weights of the norms before the attention and after it."""

    def __init__(self, w_qkv, w_o, norm_in, norm_out, heads: int, n_kv_heads: int, eps: float = 1e-6, window: int = 0,
                 interleaved: bool = False, qkv_bias=None, dtype=torch.bfloat16, device=None):
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

    def forward(self, x, cache: PagedKVCache, block_table, seq_lens, table, starts=None):
        """x [T, hidden], the last tokens of their sequences (``PagedKVCache``) -> ((codes, scales), residual):
        the normed input of what follows, and x plus the attention's output."""
        T, H, Hkv, D = x.shape[0], self.heads, self.n_kv_heads, self.head_dim
        qkv = self.qkv(rms_norm_e4m3(x, self.norm_in, self.eps)).view(T, H + 2 * Hkv, D)
        q, k, v = qkv.split((H, Hkv, Hkv), 1)
        q = cache.append(k, v, block_table, seq_lens, starts, q=q, table=table, interleaved=self.interleaved)
        y = cache.attend(q, block_table, seq_lens, starts, window=self.window)
        codes, scales, h = rms_norm_e4m3(self.o(quantize_e4m3(y.view(T, H * D))), self.norm_out, self.eps, residual=x)
        return (codes, scales), h


def main(hidden: int = 4096, heads: int = 32, n_kv_heads: int = 8, head_dim: int = 128, batch: int = 16, prompt: int = 512,
         steps: int = 64, page: int = 64):
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    block = Fp8AttentionBlock(rand((heads + 2 * n_kv_heads) * head_dim, hidden) * hidden ** -0.5,
                              rand(hidden, heads * head_dim) * (heads * head_dim) ** -0.5,
                              torch.ones(hidden), torch.ones(hidden), heads, n_kv_heads)
    per = -(-(prompt + steps) // page)
    cache = PagedKVCache(batch * per, n_kv_heads, head_dim, page)
    pages = torch.arange(batch * per, dtype=torch.int32, device="cuda").view(batch, per)
    lens = torch.full((batch,), prompt, dtype=torch.int32, device="cuda")
    table = rotary_table(per * page, head_dim)
    x, h = rand(batch * prompt, hidden).bfloat16(), rand(batch, hidden).bfloat16()
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
    print(f"{batch} prompts of {prompt} tokens: {events[0].elapsed_time(events[1]) * 1e3 / 4:.1f} us; a decode step of "
          f"{batch} sequences: {events[2].elapsed_time(events[3]) * 1e3 / steps:.1f} us")


__all__ = ["Fp8AttentionBlock"]

if __name__ == "__main__":
    main()
