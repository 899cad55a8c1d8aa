"""The 8-bit attention block against its definition in 64 bits, with the same roundings to e4m3 at the same places.

Bound: with fp32 activations the two differ by fp32 roundings, until one of these puts a value on the other side of a
tie of two codes.  That moves one element of a row of at least 256 by 2^-4 of itself, at most 2^-8 of the row, and
happens for a few of a million elements; the bound is 2^-8 over the whole tensor.
"""
import types

import pytest
import torch

from test_paged_kv import append_ref, e4m3
from test_rotary import turned

BOUND = 2.0 ** -8


def quantized(y):
    T, K = y.shape
    z = torch.nn.functional.pad(y, (0, -K % 128)).view(T, -1, 128)
    s = z.abs().amax(2) / 448
    s = torch.where(s == 0, 1.0, s)
    return (e4m3(z / s[..., None]) * s[..., None]).view(T, -1)[:, :K]


def normed(h, w, eps):
    return w.double() * h / ((h * h).mean(1, keepdim=True) + eps).sqrt()


def weight(layer):
    w = layer.codes[:, :layer.in_features].double()
    full = layer.scales.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    return w * full[:w.shape[0], :w.shape[1]]


def block_ref(block, x, cache, batch, pos, table, window):
    """(normed codes' values, residual, cache of keys and values with scales) in 64 bits."""
    H, Hkv, D = block.heads, block.n_kv_heads, block.head_dim
    T = x.shape[0]
    y = quantized(normed(x.double(), block.norm_in, block.eps)) @ weight(block.qkv).T
    if block.qkv.bias is not None:
        y = y + block.qkv.bias.double()
    q, k, v = y.view(T, H + 2 * Hkv, D).split((H, Hkv, Hkv), 1)
    q, k = turned(q, pos, table, block.interleaved)[0], turned(k, pos, table, block.interleaved)[0]
    kc, ks = append_ref(cache.k_codes, cache.k_scales, batch, k)
    vc, vs = append_ref(cache.v_codes, cache.v_scales, batch, v)
    out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    for b, l, n, at in batch.rows():
        p = batch.table[b].long()
        ka, va = ((c[p] * s[p][..., None, None]).transpose(1, 2).reshape(-1, Hkv, D)[:l].repeat_interleave(H // Hkv, 1)
                  for c, s in ((kc, ks), (vc, vs)))
        for i in range(n):
            lo = max(0, l - n + i + 1 - window) if window else 0
            hi = l - n + i + 1
            w = torch.softmax(torch.einsum("hd,khd->hk", q[at + i], ka[lo:hi]) * D ** -0.5, -1)
            out[at + i] = torch.einsum("hk,khd->hd", w, va[lo:hi])
    h = x.double() + quantized(out.view(T, H * D)) @ weight(block.o).T
    return quantized(normed(h, block.norm_out, block.eps)), h


def batch_of(lens, news, table, page, Hkv):
    def rows():
        at = 0
        for b, (l, n) in enumerate(zip(lens, news)):
            yield b, l, n, at
            at += n
    return types.SimpleNamespace(rows=rows, table=table, page=page, Hkv=Hkv)


def near(a, b):
    return float((a.double() - b).norm()) <= BOUND * float(b.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,H,Hkv,D,page,window,interleaved", [(256, 4, 2, 64, 16, 0, False), (896, 14, 2, 64, 64, 0, False),
                                                                    (512, 8, 8, 128, 32, 20, True)])
def test_prompt_then_decode(cuda, hidden, H, Hkv, D, page, window, interleaved):
    from siliconfer_b200.attention_block import Fp8AttentionBlock
    from siliconfer_b200.paged_kv import PagedKVCache
    from siliconfer_b200.rotary import rotary_table
    g = torch.Generator(device="cuda").manual_seed(hidden)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    block = Fp8AttentionBlock(rand((H + 2 * Hkv) * D, hidden) * hidden ** -0.5, rand(hidden, H * D) * (H * D) ** -0.5,
                              1 + 0.1 * rand(hidden), 1 + 0.1 * rand(hidden), H, Hkv, window=window,
                              interleaved=interleaved, qkv_bias=0.1 * rand((H + 2 * Hkv) * D), dtype=torch.float32)
    lens = [37, 1, 70]
    per = -(-80 // page)
    cache = PagedKVCache(3 * per + 1, Hkv, D, page)
    pages = torch.randperm(3 * per + 1, generator=g, device="cuda")[:3 * per].view(3, per).to(torch.int32)
    table = rotary_table(80, D)
    for news in (lens, [1, 1, 1], [1, 1, 1]):
        first = news is lens
        if not first:
            lens = [l + 1 for l in lens]
        x = rand(sum(news), hidden)
        pos = torch.cat([torch.arange(l - n, l, device="cuda") for l, n in zip(lens, news)])
        ref, ref_h = block_ref(block, x, cache, batch_of(lens, news, pages, page, Hkv), pos, table, window)
        starts = torch.tensor([0, *torch.tensor(news).cumsum(0)], dtype=torch.int32, device="cuda") if first else None
        (codes, scales), h = block(x, cache, pages, torch.tensor(lens, dtype=torch.int32, device="cuda"), table, starts)
        got = codes.double() * scales.double().repeat_interleave(128, 1)[:, :hidden]
        assert near(h, ref_h) and near(got, ref)


@pytest.mark.gpu
def test_decode_step_in_a_graph(cuda):
    """A captured step reads the lengths from the device: replays extend the sequences as calls do."""
    from siliconfer_b200.attention_block import Fp8AttentionBlock
    from siliconfer_b200.paged_kv import PagedKVCache
    from siliconfer_b200.rotary import rotary_table
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    block = Fp8AttentionBlock(rand(512, 256) / 16, rand(256, 256) / 16, torch.ones(256), torch.ones(256), 4, 2)
    x, table = rand(2, 256).bfloat16(), rotary_table(64, 64)
    pages = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    results = []
    for captured in (False, True):
        cache, lens = PagedKVCache(8, 2, 64, 16), torch.tensor([0, 9], dtype=torch.int32, device="cuda")

        def step():
            lens.add_(1)
            return block(x, cache, pages, lens, table)
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            for _ in range(20):
                graph.replay()
        else:
            for _ in range(20):
                out = step()
        results.append([*out[0], out[1], cache.k_codes, cache.k_scales, cache.v_codes])
    for a, b in zip(*results):
        assert torch.equal(a.double(), b.double())


def test_refuses_weights_that_disagree():
    from siliconfer_b200.attention_block import Fp8AttentionBlock
    for w_qkv, w_o in ((torch.zeros(513, 256), torch.zeros(256, 256)), (torch.zeros(512, 256), torch.zeros(256, 192))):
        with pytest.raises(RuntimeError, match="heads"):
            Fp8AttentionBlock(w_qkv, w_o, torch.ones(256), torch.ones(256), 4, 2, device="cpu")
