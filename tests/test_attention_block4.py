"""The attention block with a 4-bit cache, with normed heads, and with positions of several axes, against its definition in 64
bits with the same roundings at the same places.

Bound: as for the 8-bit cache, 2^-8 over the whole tensor: with fp32 activations the two differ by fp32 roundings, until one
of these puts a value on the other side of a tie.  That moves an e4m3 code by 2^-4 of itself, as there, or a cached element
by a step, a seventh of its quarter's largest, of one key among many; both for a few of a million elements.
"""
import pytest
import torch

from test_attention_block import batch_of, near, normed, quantized, weight
from test_paged_kv import append_ref
from test_paged_kv4 import codes_of, value_of
from test_qk_norm_rotary import reference


def block_ref(block, x, cache, four, batch, pos, table, axes, window):
    H, Hkv, D = block.heads, block.n_kv_heads, block.head_dim
    T = x.shape[0]
    y = quantized(normed(x.double(), block.norm_in, block.eps)) @ weight(block.qkv).T
    q, k, v = y.view(T, H + 2 * Hkv, D).split((H, Hkv, Hkv), 1)
    eps = None if block.q_norm is None else block.eps
    q = reference(q, block.q_norm, eps, pos, table, block.interleaved, axes)[0]
    k = reference(k, block.k_norm, eps, pos, table, block.interleaved, axes)[0]
    if four:
        kv = []
        for codes, scales, rows in ((cache.k_codes, cache.k_scales, k), (cache.v_codes, cache.v_scales, v)):
            vals, new = value_of(codes, scales), value_of(*codes_of(rows))
            for b, l, n, at in batch.rows():
                for i in range(n):
                    p = l - n + i
                    vals[batch.table[b, p // batch.page], :, p % batch.page] = new[at + i]
            kv.append(vals)
    else:
        kv = [(c * s[..., None, None]) for c, s in (append_ref(cache.k_codes, cache.k_scales, batch, k),
                                                    append_ref(cache.v_codes, cache.v_scales, batch, v))]
    out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    for b, l, n, at in batch.rows():
        ka, va = (c[batch.table[b].long()].transpose(1, 2).reshape(-1, Hkv, D)[:l].repeat_interleave(H // Hkv, 1) for c in kv)
        for i in range(n):
            lo, hi = (max(0, l - n + i + 1 - window) if window else 0), l - n + i + 1
            w = torch.softmax(torch.einsum("hd,khd->hk", q[at + i], ka[lo:hi]) * D ** -0.5, -1)
            out[at + i] = torch.einsum("hk,khd->hd", w, va[lo:hi])
    h = x.double() + quantized(out.view(T, H * D)) @ weight(block.o).T
    return quantized(normed(h, block.norm_out, block.eps)), h


@pytest.mark.gpu
@pytest.mark.parametrize("four", [True, False])
@pytest.mark.parametrize("head_norms", [True, False])
@pytest.mark.parametrize("hidden,H,Hkv,D,page,window,interleaved,n_axes", [(256, 4, 2, 64, 16, 0, False, 0), (896, 14, 2, 64, 64, 0, True, 3),
                                                                           (512, 8, 8, 128, 32, 20, False, 2)])
def test_prompt_then_decode(cuda, hidden, H, Hkv, D, page, window, interleaved, n_axes, head_norms, four):
    from siliconfer_b200.attention_block import Fp8AttentionBlock
    from siliconfer_b200.paged_kv import PagedKVCache
    from siliconfer_b200.paged_kv4 import Paged4KVCache
    from siliconfer_b200.rotary import rotary_axes, rotary_table
    g = torch.Generator(device="cuda").manual_seed(hidden)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    norms = dict(q_norm=1 + 0.1 * rand(D), k_norm=1 + 0.1 * rand(D)) if head_norms else {}
    block = Fp8AttentionBlock(rand((H + 2 * Hkv) * D, hidden) * hidden ** -0.5, rand(hidden, H * D) * (H * D) ** -0.5,
                              1 + 0.1 * rand(hidden), 1 + 0.1 * rand(hidden), H, Hkv, window=window, interleaved=interleaved,
                              dtype=torch.float32, **norms)
    lens = [37, 1, 70]
    per = -(-80 // page)
    cache = (Paged4KVCache if four else PagedKVCache)(3 * per + 1, Hkv, D, page)
    pages = torch.randperm(3 * per + 1, generator=g, device="cuda")[:3 * per].view(3, per).to(torch.int32)
    table = rotary_table(80, D)
    axes = rotary_axes([D // 2 - n_axes + 1] + [1] * (n_axes - 1), interleaved=True) if n_axes else None
    for news in (lens, [1, 1, 1], [1, 1, 1]):
        first = news is lens
        if not first:
            lens = [l + 1 for l in lens]
        x = rand(sum(news), hidden)
        pos = torch.cat([torch.arange(l - n, l, device="cuda") for l, n in zip(lens, news)])
        given = torch.randint(0, 80, (len(pos), n_axes), generator=g, device="cuda") if n_axes else None
        ref, ref_h = block_ref(block, x, cache, four, batch_of(lens, news, pages, page, Hkv), pos if given is None else given, table,
                               axes, window)
        starts = torch.tensor([0, *torch.tensor(news).cumsum(0)], dtype=torch.int32, device="cuda") if first else None
        (codes, scales), h = block(x, cache, pages, torch.tensor(lens, dtype=torch.int32, device="cuda"), table, starts, given, axes)
        got = codes.double() * scales.double().repeat_interleave(128, 1)[:, :hidden]
        assert near(h, ref_h) and near(got, ref)


@pytest.mark.gpu
def test_decode_step_in_a_graph(cuda):
    """A captured step reads the lengths from the device: replays extend the sequences as calls do."""
    from siliconfer_b200.attention_block import Fp8AttentionBlock
    from siliconfer_b200.paged_kv4 import Paged4KVCache
    from siliconfer_b200.rotary import rotary_table
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    block = Fp8AttentionBlock(rand(512, 256) / 16, rand(256, 256) / 16, torch.ones(256), torch.ones(256), 4, 2, q_norm=rand(64),
                              k_norm=rand(64))
    x, table = rand(2, 256).bfloat16(), rotary_table(64, 64)
    pages = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    results = []
    for captured in (False, True):
        cache, lens = Paged4KVCache(8, 2, 64, 16), torch.tensor([0, 9], dtype=torch.int32, device="cuda")

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


@pytest.mark.gpu
def test_example_runs(cuda, capsys):
    from siliconfer_b200 import attention_block
    attention_block.main(hidden=256, heads=4, n_kv_heads=2, head_dim=64, batch=2, prompt=30, steps=4, page=16)
    lines = capsys.readouterr().out.splitlines()
    assert [l.split(":")[0] for l in lines] == ["PagedKVCache", "Paged4KVCache"]


def test_refuses_one_head_norm():
    from siliconfer_b200.attention_block import Fp8AttentionBlock
    with pytest.raises(RuntimeError, match="together"):
        Fp8AttentionBlock(torch.zeros(512, 256), torch.zeros(256, 256), torch.ones(256), torch.ones(256), 4, 2, device="cpu",
                          q_norm=torch.ones(64))


def test_refuses_axes_without_positions():
    from siliconfer_b200.attention_block import Fp8AttentionBlock
    block = Fp8AttentionBlock(torch.zeros(512, 256), torch.zeros(256, 256), torch.ones(256), torch.ones(256), 4, 2, device="cpu")
    with pytest.raises(RuntimeError, match="positions"):
        block(torch.zeros(1, 256), None, None, None, None, axes=torch.zeros(32, dtype=torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("four", [True, False])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("n_axes", [0, 2])
def test_positions_of_padding_rows_are_not_looked_at(cuda, n_axes, packed, four):
    """Positions outside the table in rows that hold no token: no error with either cache, and the other rows as they were."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.attention_block import Fp8AttentionBlock
    from siliconfer_b200.paged_kv import PagedKVCache
    from siliconfer_b200.paged_kv4 import Paged4KVCache
    from siliconfer_b200.rotary import rotary_axes, rotary_table
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    block = Fp8AttentionBlock(rand(512, 256) / 16, rand(256, 256) / 16, torch.ones(256), torch.ones(256), 4, 2, q_norm=rand(64),
                              k_norm=rand(64))
    table, axes = rotary_table(40, 64), rotary_axes([20, 12]) if n_axes else None
    pages = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    if packed:      # two rows before the first token, three behind the last, and two of sequence 0 before its first token
        starts, lens = torch.tensor([2, 9, 12], dtype=torch.int32, device="cuda"), torch.tensor([5, 30], dtype=torch.int32, device="cuda")
        real, T = [*range(4, 9), 9, 10, 11], 15
    else:
        starts, lens, real, T = None, torch.tensor([3, 20], dtype=torch.int32, device="cuda"), [2, 3, 4, *range(5, 10)], 10
    x = rand(T, 256).bfloat16()
    pos = torch.randint(0, 40, (T, n_axes) if n_axes else (T,), generator=g, device="cuda")
    results = []
    for fill in (None, -1, 10 ** 6):
        rest = torch.ones(T, dtype=torch.bool, device="cuda")
        rest[real] = False
        if fill is not None:
            pos[rest] = fill
        cache = (Paged4KVCache if four else PagedKVCache)(8, 2, 64, 16)
        (codes, scales), h = block(x, cache, pages, lens, table, starts, pos, axes)
        assert _lib.load().sf_q4_check_device_error() == 0
        results.append((codes[real].double(), scales[real], h[real], cache.k_codes.double(), cache.k_scales, cache.v_codes.double()))
        assert torch.isfinite(h.float()).all()
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
