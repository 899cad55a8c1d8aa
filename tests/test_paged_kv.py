"""The paged e4m3 cache and attention over it, against plain 64-bit arithmetic over the pages.

Bounds.
  * append: a page's scale is the least power of two, 2^-64 at least, that keeps its largest value within 448 (the
    rows' own and, on a page that held tokens, its former scale), so scales are compared bit for bit, and so are the
    codes of values, which divide exactly; a turned key may fall on the other side of a tie: half a code step
    (2^-4 of the value, 2^-10 of the scale when subnormal) instead of equality.
  * attention, fp32: a score of magnitude up to about 40 is off by 2^-21 of itself and the products' rounding, so a
    weight by some 2e-5 of itself, and the output by that share of max|v|: 3e-5 max|v|.  16-bit queries: weights enter
    the second product in fp16 (2^-11 each), the output is rounded to its type: 2^-10 max|v| + 2^-8 |out| (2^-11 in fp16).
    The log-sum keeps fp32: 4e-5.
"""
import math
import random

import pytest
import torch

E4M3_MAX = 448.0


class Batch:
    """Sequences of the given lengths, of which the last `news` tokens are the call's, over pages in random order."""

    def __init__(self, lens, news, H, Hkv, D, page, dtype, seed=0, ragged=True, spare=3, fill=None):
        self.lens, self.news, self.H, self.Hkv, self.D, self.page = lens, news, H, Hkv, D, page
        g = torch.Generator(device="cuda").manual_seed(seed + sum(lens) + D)
        self.g, self.dtype = g, dtype
        B, per = len(lens), max(1, max(-(-l // page) for l in lens))
        self.P = B * per + spare
        self.table = torch.randperm(self.P, generator=g, device="cuda")[:B * per].view(B, per).to(torch.int32)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.starts = torch.tensor([sum(news[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda") if ragged else None
        self.T = sum(news)
        shape = (self.P, Hkv, page, D)
        mk = lambda: (torch.randn(shape, generator=g, device="cuda") * 80).clamp(-448, 448).to(torch.float8_e4m3fn)
        sc = lambda: torch.exp2(torch.randint(-8, -4, shape[:2], generator=g, device="cuda").float())
        self.k, self.v, self.ks, self.vs = mk(), mk(), sc(), sc()
        if fill is not None:   # what lies beyond a sequence's end
            for b, l in enumerate(lens):
                for j in range(per):
                    for t in (self.k, self.v):
                        t.view(torch.uint8)[self.table[b, j], :, max(0, min(page, l - j * page)):] = fill
        self.q = (1.5 * torch.randn(self.T, H, D, generator=g, device="cuda")).to(dtype)

    def args(self):
        return self.k, self.ks, self.v, self.vs, self.table, self.seq_lens

    def rows(self):
        at = 0
        for b, (l, n) in enumerate(zip(self.lens, self.news)):
            yield b, l, n, at
            at += n

    def values(self, codes, scales, b, l):
        p = self.table[b, :-(-l // self.page)].long()
        x = codes[p].double() * scales[p].double()[:, :, None, None]
        return x.permute(1, 0, 2, 3).reshape(self.Hkv, -1, self.D)[:, :l]

    def ref(self, scale=None, window=0):
        out = torch.zeros(self.T, self.H, self.D, dtype=torch.float64, device="cuda")
        lse = torch.full((self.T, self.H), -math.inf, dtype=torch.float64, device="cuda")
        vmax = 0.0
        G = self.H // self.Hkv
        for b, l, n, at in self.rows():
            if not n or not l:
                continue
            k, v = self.values(self.k, self.ks, b, l), self.values(self.v, self.vs, b, l)
            vmax = max(vmax, float(v.abs().max()))
            q = self.q[at:at + n].double().view(n, self.Hkv, G, self.D)
            s = torch.einsum("nhgd,hjd->nhgj", q, k) * (self.D ** -0.5 if scale is None else scale)
            far = torch.arange(l - n, l, device="cuda")[:, None] - torch.arange(l, device="cuda")
            hidden = (far < 0) | ((far >= window) if window else False)
            s = s.masked_fill(hidden[:, None, None], -math.inf)
            out[at:at + n] = torch.einsum("nhgj,hjd->nhgd", s.softmax(-1), v).reshape(n, self.H, self.D)
            lse[at:at + n] = s.logsumexp(-1).reshape(n, self.H)
        return out, lse, vmax


def check_attention(batch, out_dtype=None, **kw):
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv import paged_attention
    out, lse = paged_attention(batch.q, *batch.args(), starts=batch.starts, out_dtype=out_dtype, return_lse=True, **kw)
    ref, lref, vmax = batch.ref(**kw)
    dtype = out_dtype or batch.dtype
    assert out.dtype == dtype and out.shape == ref.shape and lse.dtype == torch.float32
    bound = 3e-5 * vmax if batch.dtype == torch.float32 else 2.0 ** -10 * vmax
    bound = bound + {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype] * ref.abs()
    assert ((out.double() - ref).abs() <= bound).all()
    empty = lref == -math.inf
    assert torch.equal(empty, lse == -math.inf)
    assert ((lse.double() - lref)[~empty].abs() <= 4e-5 + 2e-6 * lref[~empty].abs()).all()
    assert _lib.load().sf_q4_check_device_error() == 0
    return out


HEADS = [(1, 1), (8, 8), (14, 2), (8, 1), (12, 4), (64, 8), (16, 1), (40, 2), (9, 3)]
LENS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 500, 1000, 2049]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("H,Hkv", HEADS)
def test_single_tokens(cuda, H, Hkv, D, dtype):
    """One new token each, a batch of every length, each page size."""
    for i, page in enumerate((16, 32, 64, 128, 256)):
        lens = LENS[i::2] if Hkv == 8 else LENS[i::3]
        check_attention(Batch(lens, [1] * len(lens), H, Hkv, D, page, dtype, seed=page, ragged=False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,D", [(14, 2, 64), (8, 8, 128), (64, 8, 128), (8, 1, 256), (20, 4, 96)])
def test_several_tokens(cuda, H, Hkv, D, dtype):
    """Ragged counts of new tokens from none to whole prompts, with empty sequences between."""
    check_attention(Batch([70, 5, 0, 300, 129, 64], [7, 5, 0, 1, 40, 64], H, Hkv, D, 32, dtype))
    check_attention(Batch([33, 257], [33, 200], H, Hkv, D, 64, dtype))
    check_attention(Batch([100, 100, 100], [4, 4, 4], H, Hkv, D, 16, dtype, ragged=False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("window", [1, 7, 16, 33, 100, 5000])
def test_window(cuda, window, dtype):
    check_attention(Batch([1, 40, 500, 130], [1, 9, 3, 130], 8, 2, 64, 32, dtype), window=window)
    check_attention(Batch([700] * 3, [1] * 3, 16, 2, 128, 64, dtype, ragged=False), window=window, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_sequences_and_uneven_batches(cuda, dtype):
    check_attention(Batch([40000], [1], 8, 1, 128, 64, dtype, ragged=False))
    check_attention(Batch([9000, 1, 0, 17, 3001], [1, 1, 0, 1, 1], 64, 8, 128, 64, dtype))
    rng = random.Random(4)
    lens = [rng.randint(1, 400) for _ in range(200)]
    check_attention(Batch(lens, [1] * 200, 4, 2, 64, 16, dtype, ragged=False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_rows_empty_and_no_rows(cuda, dtype):
    from siliconfer_b200.paged_kv import paged_attention
    b = Batch([5, 6], [1, 1], 8, 2, 64, 16, dtype, ragged=False)
    b.seq_lens.zero_()
    # a length below its number of new rows: the rows before the sequence see nothing, and nothing is out of range
    out, lse = paged_attention(b.q, *b.args(), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out = paged_attention(b.q[:0], *b.args(), starts=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 8, 64)
    b = Batch([3, 40], [5, 2], 8, 2, 64, 16, dtype)     # two of the five rows lie before their sequence
    out, lse = paged_attention(b.q, *b.args(), starts=b.starts, return_lse=True)
    assert (out[:2] == 0).all() and (lse[:2] == -math.inf).all() and torch.isfinite(lse[2:]).all()
    c = Batch([3, 40], [3, 2], 8, 2, 64, 16, dtype)
    c.q, c.k, c.v, c.ks, c.vs, c.table = b.q[2:], b.k, b.v, b.ks, b.vs, b.table
    ref, lref, vmax = c.ref()
    assert ((out[2:].double() - ref).abs() <= 2.0 ** -10 * vmax + 2.0 ** -8 * ref.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [0x7f, 0xff, 0x7e])
def test_contents_beyond_the_end_do_not_matter(cuda, fill):
    """NaN and the largest codes in every slot past a sequence's end, and in pages of no sequence."""
    for dtype in (torch.float32, torch.bfloat16):
        check_attention(Batch([1, 20, 100, 130], [1, 1, 1, 1], 14, 2, 64, 64, dtype, ragged=False, fill=fill))
        check_attention(Batch([9, 33, 65], [9, 2, 33], 8, 8, 128, 16, dtype, fill=fill))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_large_and_small_values(cuda, dtype):
    """Scores that would overflow e^s, scales far apart between pages, zero scales, queries near their type's limits."""
    b = Batch([200, 300], [1, 1], 8, 2, 64, 16, dtype, ragged=False)
    check_attention(b, scale=3.0 / 8)
    b.vs = torch.exp2(torch.randint(-40, 12, b.vs.shape, generator=b.g, device="cuda").float())
    check_attention(b)
    b.vs[::2] = 0
    check_attention(b)
    b.q = (b.q.float() * (2.0 ** -12)).to(dtype)
    check_attention(b, scale=512.0)
    if dtype != torch.float16:
        b.q = (b.q.float() * 2.0 ** 60).to(dtype)
        check_attention(b, scale=2.0 ** -54)
    b.q.zero_()
    check_attention(b)


@pytest.mark.gpu
def test_non_finite_values_stay_in_their_rows(cuda):
    from siliconfer_b200.paged_kv import paged_attention
    b = Batch([50, 60], [2, 2], 8, 2, 64, 16, torch.bfloat16, ragged=False)
    b.q[0, 3, 5] = float("nan")
    b.v.view(torch.uint8)[b.table[1, 0], 1, 3, 7] = 0x7f      # sequence 1, kv head 1, column 7
    out = paged_attention(b.q, *b.args())
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 3] = True
    bad[2:, 4:, 7] = True
    assert torch.equal(out.isnan(), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_values_that_a_row_does_not_see_cannot_reach_it(cuda, D, dtype):
    """NaN keys and values of later tokens of the same call, and of tokens before a row's window."""
    from siliconfer_b200.paged_kv import paged_attention
    b = Batch([90], [60], 8, 2, D, 16, dtype)
    ref, _, vmax = b.ref(window=10)
    k, v = b.k.view(torch.uint8), b.v.view(torch.uint8)
    for at in (40, 47, 70):
        k[b.table[0, at // 16], 1, at % 16] = 0x7f
        v[b.table[0, at // 16], 1, at % 16, 3] = 0xff
        v[b.table[0, at // 16], 0, at % 16, D - 1] = 0x7f
    out = paged_attention(b.q, *b.args(), starts=b.starts, window=10)
    pos = torch.arange(30, 90, device="cuda")
    sees = torch.zeros(60, dtype=torch.bool, device="cuda")
    for at in (40, 47, 70):
        sees |= (pos >= at) & (pos < at + 10)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[sees, 4:] = True
    bad[sees, :4, D - 1] = True
    assert torch.equal(out.isnan(), bad)
    assert (~sees).sum() > 5
    assert ((out.double() - ref).abs()[~bad] <= 2.0 ** -10 * vmax + 2.0 ** -8 * ref.abs()[~bad]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv", [(8, 2), (32, 4)])
def test_strided_queries_types_and_repeats(cuda, H, Hkv):
    b = Batch([300, 1000, 90], [1, 4, 2], H, Hkv, 128, 64, torch.bfloat16)
    first = check_attention(b, out_dtype=torch.float32)
    wide = torch.zeros(b.T, (H + 3) * 128 + 1, device="cuda", dtype=torch.bfloat16)
    q = b.q
    for off in (0, 1, 130):
        wide[:, off:off + H * 128] = q.reshape(b.T, -1)
        b.q = wide[:, off:off + H * 128].view(b.T, H, 128)
        assert torch.equal(check_attention(b, out_dtype=torch.float32), first)
    b.q = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(check_attention(b, out_dtype=torch.float32), first)
    check_attention(b, out_dtype=torch.float16)


@pytest.mark.gpu
def test_streams_and_capture(cuda):
    from siliconfer_b200.paged_kv import paged_attention
    a = Batch([3000, 10], [1, 1], 32, 4, 128, 64, torch.bfloat16, ragged=False)
    b = Batch([100, 2000, 77], [1, 1, 1], 32, 4, 128, 64, torch.bfloat16, ragged=False, seed=9)
    ra, rb = paged_attention(a.q, *a.args()), paged_attention(b.q, *b.args())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(20):
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(paged_attention(x.q, *x.args()))
    torch.cuda.synchronize()
    assert all(torch.equal(y, r) for y, r in zip(got, [ra, rb] * 20))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = paged_attention(a.q, *a.args())
    for lens in ([3000, 10], [17, 2]):       # lengths are read when the graph runs
        a.lens = lens
        a.seq_lens.copy_(torch.tensor(lens))
        graph.replay()
        torch.cuda.synchronize()
        ref, _, vmax = a.ref()
        assert ((y.double() - ref).abs() <= 2.0 ** -10 * vmax + 2.0 ** -8 * ref.abs()).all()


@pytest.mark.gpu
def test_pages_past_31_bits(cuda):
    """A pool of more than 2^31 codes: the pages at its end are read and written like the first ones."""
    from siliconfer_b200.paged_kv import paged_append
    b = Batch([40, 90], [1, 1], 8, 2, 128, 64, torch.bfloat16, ragged=False)
    P = 2 ** 31 // (2 * 64 * 128) + 40
    big = [torch.zeros(P, 2, 64, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    far = P - b.P
    for dst, src in zip(big, (b.k, b.v)):
        dst.view(torch.uint8)[far:] = src.view(torch.uint8)
    ref, _, vmax = b.ref()
    pad = lambda s: torch.cat([torch.ones(far, 2, device="cuda"), s])
    b.k, b.v, b.ks, b.vs, b.table = big[0], big[1], pad(b.ks), pad(b.vs), b.table + far
    out = check_attention(b)
    assert ((out.double() - ref).abs() <= 2.0 ** -10 * vmax + 2.0 ** -8 * ref.abs()).all()
    v = torch.full((2, 2, 128), 3.0, device="cuda", dtype=torch.bfloat16)
    paged_append(v, v, *b.args())
    p = int(b.table[1, 1])
    assert (b.v[p, :, 89 - 64].float() * b.vs[p][:, None] - 3).abs().max() <= 3 * 2.0 ** -4


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------
def e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).float().to(torch.float8_e4m3fn).double()


def append_ref(codes, scales, batch, rows):
    """rows [T, Hkv, D] in 64 bits into (codes, scales), a page at a time; returns both as 64-bit tensors."""
    c, s = codes.double(), scales.double()
    for b, l, n, at in batch.rows():
        for j in range((l - n) // batch.page, -(-l // batch.page)) if n else ():
            lo, hi = max(l - n, j * batch.page), min(l, (j + 1) * batch.page)
            p, base = int(batch.table[b, j]), j * batch.page
            new = rows[at + lo - (l - n):at + hi - (l - n)].transpose(0, 1)
            for h in range(batch.Hkv):
                fin = new[h][torch.isfinite(new[h])].abs()
                amax = float(fin.max()) if fin.numel() else 0.0
                e = -64
                if amax > 0:
                    e = math.floor(math.log2(amax)) - 9
                    while amax > E4M3_MAX * 2.0 ** e:
                        e += 1
                scale = 2.0 ** max(e, -64)
                if lo > base:
                    old = float(s[p, h])
                    scale = max(scale, old)
                    c[p, h, :lo - base] = e4m3(c[p, h, :lo - base] * (old / scale))
                c[p, h, lo - base:hi - base] = e4m3(new[h] / scale)
                s[p, h] = scale
    return c, s


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=1e9), torch.nan_to_num(b, nan=1e9))


def check_append(batch, dtype, rot=None, interleaved=False, turn=True, values=None, strided=False):
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv import paged_append
    from siliconfer_b200.rotary import rotary_table
    from test_rotary import check as check_rotary, turned
    T, Hkv, H, D = batch.T, batch.Hkv, batch.H, batch.D
    qkv = torch.randn(T, (H + 2 * Hkv) * D + 1, generator=batch.g, device="cuda").to(dtype)
    off = 1 if strided else 0
    part = lambda a, h: qkv[:, off + a * D:off + (a + h) * D].view(T, h, D)
    q, k, v = part(0, H), part(H, Hkv), part(H + Hkv, Hkv)
    if values is not None:
        values(k, v)
    pos = torch.cat([torch.arange(l - n, l, device="cuda") for _, l, n, _ in batch.rows()] or [torch.zeros(0)]).long()
    table = rotary_table(max(batch.lens) + 1, rot or D) if turn else None
    kr = (turned(k, pos, table, interleaved)[0] if turn else k.double())
    kc, kscale = append_ref(batch.k, batch.ks, batch, kr)
    vc, vscale = append_ref(batch.v, batch.vs, batch, v.double())
    got = paged_append(k, v, *batch.args(), starts=batch.starts, q=q if turn else None, table=table,
                       interleaved=interleaved)
    assert _lib.load().sf_q4_check_device_error() == 0
    assert torch.equal(batch.ks.double(), kscale) and torch.equal(batch.vs.double(), vscale)
    assert same(batch.v.double(), vc)
    diff = batch.k.double() - kc
    if turn:
        assert (diff.nan_to_num().abs() <= 0.1251 * kc.nan_to_num().abs() + 2.0 ** -9).all()   # one step at most
        assert ((diff != 0) & ~diff.isnan()).float().mean() <= 1e-4
        check_rotary(got, *turned(q, pos, table, interleaved), dtype)
    else:
        assert same(batch.k.double(), kc) and got is None
    assert torch.equal(batch.k.double().isnan(), kc.isnan())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,D", [(14, 2, 64), (8, 8, 128), (6, 3, 96), (4, 1, 256)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_append(cuda, page, H, Hkv, D, dtype):
    lens = [1, page, page + 1, 2 * page - 1, 3 * page + 5, 1000]
    check_append(Batch(lens, [1] * 6, H, Hkv, D, page, dtype, ragged=False), dtype)
    check_append(Batch(lens, [1, 3, page, 0, 2 * page + 7, 1000], H, Hkv, D, page, dtype), dtype, turn=False)
    check_append(Batch(lens, [1, page, page + 1, 5, 2 * page, 900], H, Hkv, D, page, dtype), dtype, interleaved=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rot", [32, 48, 20, 2])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_partial_rotary_and_strides(cuda, rot, interleaved):
    for dtype in (torch.bfloat16, torch.float32):
        b = lambda: Batch([70, 9, 0, 130], [6, 9, 0, 1], 5, 2, 64, 32, dtype, seed=rot)
        check_append(b(), dtype, rot=rot, interleaved=interleaved)
        check_append(b(), dtype, rot=rot, interleaved=interleaved, strided=True)


@pytest.mark.gpu
def test_append_scales_grow_and_special_values(cuda):
    """Pages whose old scale is smaller, larger and equal; zero rows; infinities and NaN among the new values."""
    def values(k, v):
        v[0] = 0
        v[1] *= 1000
        v[2, 0, 3], v[2, 0, 4], v[2, 0, 5] = float("inf"), float("-inf"), float("nan")
        v[3] = 448.0
        v[4] = 449.0
        v[5] = float("nan")
        v[6] = 1e-30
        k[1] *= 1e-6
        k[2, 1, 0] = float("nan")
    for dtype in (torch.float32, torch.bfloat16):
        check_append(Batch([20, 20, 20, 20, 20, 33, 33], [1] * 7, 4, 2, 64, 32, dtype, ragged=False), dtype, turn=False,
                     values=values)
    # a page filled a token at a time ends like the page's largest scale
    from siliconfer_b200.paged_kv import PagedKVCache
    cache = PagedKVCache(2, 1, 64, page_size=16)
    x = torch.randn(16, 1, 64, device="cuda") * torch.linspace(0.01, 5, 16, device="cuda")[:, None, None]
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    for i in range(16):
        cache.append(x[i:i + 1], x[i:i + 1], table, torch.tensor([i + 1], dtype=torch.int32, device="cuda"))
    got = cache.v_codes[1, 0].double() * cache.v_scales[1, 0].double()
    step = 2.0 ** -4 * x[:, 0].double().abs() + 2.0 ** -10 * cache.v_scales[1, 0].double()
    # rounded once, and once more (half a subnormal step) for each of the scale's growths
    assert ((got - x[:, 0].double()).abs() <= step + 16 * 2.0 ** -10 * cache.v_scales[1, 0].double()).all()
    out = cache.attend(x[15:16], table, torch.tensor([16], dtype=torch.int32, device="cuda"))
    assert torch.isfinite(out).all()


@pytest.mark.gpu
def test_indices_outside_their_tensors_are_skipped_and_reported(cuda):
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv import paged_append, paged_attention
    from siliconfer_b200.rotary import rotary_table
    lib = _lib.load()
    mk = lambda: Batch([40, 50], [1, 1], 8, 2, 64, 16, torch.bfloat16, ragged=False)
    kv = torch.randn(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    # a page outside the pool: its keys are left out of the sums
    b = mk()
    b.table[0, 1], b.table[1, 3] = 10 ** 6, -5
    before = b.k.clone().view(torch.uint8)
    out = paged_attention(b.q, *b.args())
    assert lib.sf_q4_check_device_error() == 10 and torch.isfinite(out).all()
    paged_append(kv, kv, *b.args())
    assert lib.sf_q4_check_device_error() == 10
    changed = (b.k.view(torch.uint8) != before).any(-1).any(-1).any(-1).nonzero().flatten().tolist()
    assert changed == [int(b.table[0, 2])]
    # lengths beyond the block table, negative ones, more new rows than tokens
    for lens in ([10 ** 9, 50], [-3, 50]):
        b = mk()
        b.seq_lens.copy_(torch.tensor(lens))
        before = b.k.clone().view(torch.uint8)
        out = paged_attention(b.q, *b.args())
        assert lib.sf_q4_check_device_error() == 10 and torch.isfinite(out).all()
        paged_append(kv, kv, *b.args())
        assert lib.sf_q4_check_device_error() == 10
        changed = (b.k.view(torch.uint8) != before).any(-1).any(-1).any(-1).nonzero().flatten().tolist()
        assert changed == [int(b.table[1, 3])]
    # starts that leave the rows
    b = mk()
    starts = torch.tensor([0, 5000, 2], dtype=torch.int32, device="cuda")
    out = paged_attention(b.q, *b.args(), starts=starts)
    paged_append(kv, kv, *b.args(), starts=starts)
    assert lib.sf_q4_check_device_error() == 10
    # a rotary table that ends before the position
    b = mk()
    paged_append(kv, kv, *b.args(), q=b.q, table=rotary_table(45, 64))
    assert lib.sf_q4_check_device_error() == 10
    assert (b.k[b.table[1, 3].long(), :, 1].float()).isnan().all()
    assert lib.sf_q4_check_device_error() == 0


@pytest.mark.gpu
def test_refusals(cuda):
    from siliconfer_b200.paged_kv import paged_append, paged_attention
    b = Batch([40, 50], [1, 1], 8, 2, 64, 16, torch.bfloat16, ragged=False)
    k, ks, v, vs, table, lens = b.args()
    x = torch.randn(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(100, 64, device="cuda")
    att = lambda q=b.q, k=k, ks=ks, v=v, vs=vs, table=table, lens=lens, **kw: paged_attention(q, k, ks, v, vs, table, lens, **kw)
    app = lambda a=x, c=x, k=k, ks=ks, table=table, lens=lens, **kw: paged_append(a, c, k, ks, v, vs, table, lens, **kw)
    for bad in (lambda: att(q=b.q.cpu()), lambda: att(q=b.q.double()), lambda: att(q=b.q[:, :7]), lambda: att(q=b.q[:, :, :32]),
                lambda: att(q=b.q[:1]), lambda: att(q=b.q[0]), lambda: att(k=k.float()), lambda: att(k=k[:, :1]),
                lambda: att(k=k.transpose(1, 2)), lambda: att(ks=ks[:1]), lambda: att(ks=ks.half()), lambda: att(vs=vs.cpu()),
                lambda: att(table=table.long()), lambda: att(table=table[0]), lambda: att(lens=lens.long()),
                lambda: att(lens=lens[:1]), lambda: att(starts=lens), lambda: att(starts=torch.zeros(3, device="cuda")),
                lambda: att(out_dtype=torch.int32), lambda: att(k=k[:, :, :8].contiguous(), v=v[:, :, :8].contiguous()),
                lambda: att(table=table[:, :0]), lambda: app(a=x.cpu()), lambda: app(a=x[:1]), lambda: app(c=x.float()),
                lambda: app(a=x[:, :1], c=x[:, :1]), lambda: app(q=b.q), lambda: app(q=b.q[:1], table=t),
                lambda: app(q=b.q.float(), table=t), lambda: app(table=t.half()), lambda: app(table=t[:, :63]),
                lambda: app(a=x.double(), c=x.double()), lambda: app(lens=lens.float())):
        with pytest.raises(RuntimeError):
            bad()
    odd = torch.zeros(4, 2, 24, 64, dtype=torch.uint8, device="cuda")
    with pytest.raises(RuntimeError, match="page_size"):
        att(k=odd, v=odd, ks=torch.ones(4, 2, device="cuda"), vs=torch.ones(4, 2, device="cuda"))


def test_validation_without_gpu():
    import ctypes

    from siliconfer_b200 import _lib
    lib, F = _lib.load(), 0x1000

    def cache(**k):
        return ctypes.byref(_lib.PagedCache(**{**dict(k_codes=F, k_scales=F, v_codes=F, v_scales=F, block_table=F, seq_lens=F,
                                                      starts=None, num_pages=4, n_kv_heads=2, page_size=16, head_dim=64,
                                                      batch=1, pages_per_seq=4), **k}))

    big = 1 << 30
    att = lambda c=None, **k: lib.sf_paged_attention(c or cache(), *{**dict(q=F, qd=0, ts=512, hs=64, o=F, od=0, lse=None, H=8,
                                                                          T=1, s=1.0, w=0, ws=F, wb=big, st=None), **k}.values())
    app = lambda c=None, **k: lib.sf_paged_append(c or cache(), *{**dict(k=F, a=128, b=64, v=F, c=128, d=64, q=None, e=0, f=0,
                                                                       qo=None, dt=0, H=0, T=1, t=None, mp=0, rot=0, il=0,
                                                                       st=None), **k}.values())
    for call in (att, app):
        assert call(cache(page_size=24)) == 6 and call(cache(head_dim=80)) == 6 and call(cache(batch=5000)) == 6
        assert call(cache(batch=0)) == 2 and call(cache(num_pages=0)) == 2 and call(cache(batch=2)) == 2 and call(T=-1) == 2
        assert call(cache(pages_per_seq=1 << 28)) == 2
        assert call(cache(k_codes=None)) == 1 and call(cache(seq_lens=None)) == 1 and call(cache(v_codes=0x1008)) == 4
        assert call(T=0) == 0
    assert att(H=7) == 2 and att(H=0) == 2 and att(qd=3) == 3 and att(od=9) == 3 and att(q=None) == 1 and att(ws=None) == 1
    assert att(wb=0) == 2 and b"workspace" in lib.sf_last_error()
    assert app(dt=5) == 3 and app(k=None) == 1 and app(q=F) == 1 and app(q=F, qo=F) == 2
    assert app(t=F, mp=8, rot=65) == 2 and app(t=F, mp=0, rot=64) == 2
    assert lib.sf_paged_attention(None, F, 0, 512, 64, F, 0, None, 8, 1, 1.0, 0, F, big, None) == 1
    assert lib.sf_paged_attention_workspace_bytes(128) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,page,rot,D", [(1, 16, 64, 64), (3, 64, 64, 64), (70, 64, 128, 128), (300, 256, 48, 96), (20, 32, 20, 64)])
def test_append_infinite_keys(cuda, n, page, rot, D, dtype, interleaved):
    """A turned infinity is infinite (NaN against another one), saturates, and does not set the page's scale."""
    from siliconfer_b200.paged_kv import paged_append
    from siliconfer_b200.rotary import rotary_table
    b = Batch([n + 5, n + 40], [n, n], 2, 2, D, page, dtype, seed=n)
    k = torch.randn(b.T, 2, D, generator=b.g, device="cuda").to(dtype)
    k[0, 0, 3], k[n, 1, 1], k[n, 1, 0] = float("inf"), float("-inf"), float("nan")
    k[b.T - 1, 0, 0] = k[b.T - 1, 0, rot // 2] = k[b.T - 1, 0, 1] = float("inf")
    pos = torch.cat([torch.arange(l - c, l, device="cuda") for _, l, c, _ in b.rows()])
    table = rotary_table(1000, rot)
    c, s = (x[:, None] for x in table.double()[pos].split(rot // 2, 1))
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y = k.double()
    x0, x1 = y[..., i].clone(), y[..., j].clone()
    y[..., i], y[..., j] = x0 * c - x1 * s, x0 * s + x1 * c
    kc, kscale = append_ref(b.k, b.ks, b, y)
    paged_append(k, torch.zeros_like(k), *b.args(), starts=b.starts, table=table, interleaved=interleaved)
    assert torch.equal(b.ks.double(), kscale)
    got = b.k.double()
    assert torch.equal(got.isnan(), kc.isnan()) and kc.isnan().any() and (kc.abs() == 448).any()
    diff = (got - kc).nan_to_num()
    assert (diff.abs() <= 0.1251 * kc.nan_to_num().abs() + 2.0 ** -9).all() and (diff != 0).double().mean() <= 1e-4


# Long runs of bf16 queries take tiles of 256 rows.  The bounds are the same: weights in fp16, queries to 2^-17 of the
# row's largest element.
@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D,page", [(64, 8, 128, 64), (14, 2, 64, 16), (32, 32, 128, 256), (8, 8, 64, 128), (16, 1, 128, 32),
                                          (40, 8, 64, 64)])
def test_prompts(cuda, H, Hkv, D, page):
    """Whole prompts, later chunks, runs that end anywhere in a tile; empty sequences and single tokens between."""
    n = 256 * 40 * Hkv // (H * Hkv) + 900      # rows for a quarter of the SMs at least
    for lens, news in (([n], [n]), ([n + 500, 0, 300, 70, 1], [n, 0, 290, 1, 1]), ([n, n - 3], [n - 128, n - 130]),
                       ([2500, 2049], [n, 255])):
        check_attention(Batch(lens, [min(a, b) for a, b in zip(news, lens)], H, Hkv, D, page, torch.bfloat16, seed=n))
    check_attention(Batch([n + 40] * 3, [n // 2] * 3, H, Hkv, D, page, torch.bfloat16, ragged=False), out_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 40, 128, 300, 5000])
def test_prompts_with_a_window(cuda, window):
    check_attention(Batch([1500, 900], [1400, 300], 16, 8, 128, 64, torch.bfloat16), window=window, out_dtype=torch.float16)
    check_attention(Batch([700, 600], [700, 600], 28, 4, 64, 16, torch.bfloat16), window=window, scale=-0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [0x7f, 0xff, 0x7e])
def test_prompts_beyond_the_end(cuda, fill):
    check_attention(Batch([1001, 650, 0], [1001, 200, 0], 64, 8, 128, 64, torch.bfloat16, fill=fill))
    check_attention(Batch([1500], [1490], 14, 2, 64, 16, torch.bfloat16, fill=fill))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_rows_keep_to_themselves(cuda, D):
    """NaN and infinite queries, NaN keys and values that some rows see and others do not, with a window and without."""
    from siliconfer_b200.paged_kv import paged_attention
    for window in (0, 200):
        b = Batch([900], [800], 32, 8, D, 16, torch.bfloat16)
        ref, _, vmax = b.ref(window=window)
        k, v = b.k.view(torch.uint8), b.v.view(torch.uint8)
        marks = (40, 333, 640, 897)
        for at in marks:
            k[b.table[0, at // 16], 1, at % 16] = 0x7f
            v[b.table[0, at // 16], 1, at % 16, 3] = 0xff
            v[b.table[0, at // 16], 0, at % 16, D - 1] = 0x7f
        b.q[300, 20, 5], b.q[301, 21, 0] = float("nan"), float("inf")
        out = paged_attention(b.q, *b.args(), starts=b.starts, window=window)
        pos = torch.arange(100, 900, device="cuda")
        sees = torch.zeros(800, dtype=torch.bool, device="cuda")
        for at in marks:
            sees |= (pos >= at) & ((pos < at + window) if window else True)
        bad = torch.zeros_like(out, dtype=torch.bool)
        bad[sees, 4:8] = True
        bad[sees, :4, D - 1] = True
        bad[300, 20] = bad[301, 21] = True
        assert torch.equal(out.isnan(), bad)
        assert ((out.double() - ref).abs()[~bad] <= 2.0 ** -10 * vmax + 2.0 ** -8 * ref.abs()[~bad]).all()


@pytest.mark.gpu
def test_prompt_values_strides_and_padding(cuda):
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv import paged_attention
    b = Batch([700, 800], [650, 800], 32, 8, 64, 16, torch.bfloat16)
    first = check_attention(b)
    for _ in range(3):
        assert torch.equal(check_attention(b), first)
    wide = torch.zeros(b.T, 35 * 64 + 1, device="cuda", dtype=torch.bfloat16)
    q = b.q
    for off in (0, 1, 72):
        wide[:, off:off + 32 * 64] = q.reshape(b.T, -1)
        b.q = wide[:, off:off + 32 * 64].view(b.T, 32, 64)
        assert torch.equal(check_attention(b), first)
    b.q = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(check_attention(b), first)
    # scores of rising size, so that references move; scales far apart, zero; queries of one size and of others
    b.q = (q.float() * torch.linspace(0.01, 6, b.T, device="cuda")[:, None, None]).to(torch.bfloat16)
    check_attention(b)
    b.vs = torch.exp2(torch.randint(-40, 12, b.vs.shape, generator=b.g, device="cuda").float())
    check_attention(b)
    b.vs[::2] = 0
    check_attention(b)
    b.q = (q.float() * 2.0 ** 60).to(torch.bfloat16)
    check_attention(b, scale=2.0 ** -63)
    b.q = torch.zeros_like(q)
    check_attention(b)
    # fewer tokens than rows: padding rows in front give 0; a page number out of range is an error, its keys are not seen
    b = Batch([600, 800], [600, 800], 32, 8, 64, 16, torch.bfloat16)
    b.seq_lens[0] = 500
    out, lse = paged_attention(b.q, *b.args(), starts=b.starts, return_lse=True)
    assert (out[:100] == 0).all() and (lse[:100] == -math.inf).all() and torch.isfinite(lse[100:]).all()
    assert _lib.load().sf_q4_check_device_error() == 0
    b.seq_lens[0] = 600
    b.table[0] = b.P + 5
    out, lse = paged_attention(b.q, *b.args(), starts=b.starts, return_lse=True)
    torch.cuda.synchronize()
    assert _lib.load().sf_q4_check_device_error() != 0
    assert (out[:600] == 0).all() and (lse[:600] == -math.inf).all() and torch.isfinite(out[600:].float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("page", [-1, -2, -(2 ** 31), 2 ** 31 - 1])
@pytest.mark.parametrize("n", [1, 600])
def test_page_numbers_out_of_range_are_reported(cuda, n, page):
    """For single tokens and for prompts; the other sequence's rows are what they were."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv import paged_attention
    b = Batch([700, 800], [n, n], 32, 8, 64, 16, torch.bfloat16)
    good = check_attention(b)
    b.table[0, 3] = page
    out = paged_attention(b.q, *b.args(), starts=b.starts)
    torch.cuda.synchronize()
    assert _lib.load().sf_q4_check_device_error() != 0
    assert torch.equal(out[n:], good[n:]) and torch.isfinite(out.float()).all()
    assert _lib.load().sf_q4_check_device_error() == 0


def _mass(b, **kw):
    """sum_j p_j |v_j| of every output."""
    v, b.v = b.v, (b.v.view(torch.uint8) & 0x7f).view(torch.float8_e4m3fn)
    out = b.ref(**kw)[0]
    b.v = v
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                             (torch.bfloat16, torch.float16), (torch.float32, torch.float16)])
@pytest.mark.parametrize("H,Hkv,D,n", [(64, 8, 128, 1), (14, 2, 64, 1), (8, 8, 256, 1), (4, 4, 96, 3), (64, 8, 128, 300),
                                       (16, 16, 64, 600)])
def test_weights_are_as_fine_as_the_output(cuda, H, Hkv, D, n, dtype, out_dtype):
    """The finer of the queries' and the output's types.  Few keys and queries exact in their type, so that a weight's own
    rounding shows: fp32 within 2e-5 of itself, and its share of the sum, 5e-5 of sum p |v| in all; fp16 2^-11 more, and
    half a unit of the output."""
    from siliconfer_b200.paged_kv import paged_attention
    b = Batch([n + 1, n + 2, n + 5, n + 30], [n] * 4, H, Hkv, D, 16, dtype)
    out = paged_attention(b.q, *b.args(), starts=b.starts, out_dtype=out_dtype)
    ref, mass = b.ref()[0], _mass(b)
    bound = 5e-5 * mass
    if out_dtype == torch.float16:
        bound = bound + 2.0 ** -11 * mass + 2.0 ** -11 * ref.abs() + 2.0 ** -24
    assert ((out.double() - ref).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,dtype", [(2, torch.bfloat16), (2, torch.float16), (1, torch.float32), (1, torch.bfloat16)])
@pytest.mark.parametrize("n,interleaved", [(64, False), (61, True)])
def test_append_heads_of_more_items_than_threads(cuda, H, dtype, n, interleaved):
    """48 items a head and 32 threads a token: many tokens of few heads, among more sequences than a search probes at once."""
    lens = [n + 5 * b for b in range(40)]
    b = Batch(lens, [n] * 40, H, 1, 96, 32, dtype, seed=H)
    check_append(b, dtype, rot=20, interleaved=interleaved)
    b = Batch(lens, [n] * 40, H, 1, 96, 32, dtype, seed=H)
    check_append(b, dtype, rot=96, interleaved=interleaved, strided=True)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 30, 1024])
@pytest.mark.parametrize("n,D", [(4, 64), (400, 128)])
def test_windows_wider_than_the_sequences(cuda, n, D, window):
    """They hide nothing, from sequences with fewer tokens than rows either."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv import paged_attention
    b = Batch([n, n, n + 500, n], [n] * 4, 32, 8, D, 16, torch.bfloat16)
    b.seq_lens.copy_(torch.tensor([1, n // 2, n + 500, 0]))
    want, lse = paged_attention(b.q, *b.args(), starts=b.starts, return_lse=True)
    out, l2 = paged_attention(b.q, *b.args(), starts=b.starts, return_lse=True, window=window)
    assert torch.equal(out, want) and torch.equal(l2, lse)
    assert torch.isfinite(l2[n - 1]).all() and (out[:n - 1] == 0).all()
    assert _lib.load().sf_q4_check_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 600])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 32), (64, 128)])
def test_pages_that_a_window_has_given_up(cuda, D, page, n):
    """Page numbers before a sequence's first key in the window are not looked at, for single tokens and for prompts."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv import paged_attention
    b = Batch([1500, 905], [n, n], 32, 8, D, page, torch.bfloat16)
    good = check_attention(b, window=200)
    for s, l, _, _ in b.rows():
        b.table[s, :max(0, l - n + 1 - 200) // page] = -1
    out = paged_attention(b.q, *b.args(), starts=b.starts, window=200)
    torch.cuda.synchronize()
    assert _lib.load().sf_q4_check_device_error() == 0
    assert torch.equal(out, good)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 400])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_no_sequence(cuda, n, dtype):
    """Rows before the first sequence's and behind the last one's: turned as at position 0, not written, and they see nothing;
    starts that fall or leave the rows: an error, and 0 for all of them."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv import paged_append, paged_attention
    from siliconfer_b200.rotary import rotary_table
    H, Hkv, D, before, after = 32, 8, 64, 3, 5
    b = Batch([700, n, 30], [n, n, 3], H, Hkv, D, 16, dtype)
    q = torch.randn(before + b.T + after, H, D, device="cuda").to(dtype)
    inside = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    inside[before:before + b.T] = True
    q[inside] = b.q

    def attend(starts):
        junk = [torch.full(s, 7.0, device="cuda", dtype=d) for s, d in (((q.shape), dtype), ((q.shape[:2]), torch.float32)) * 4]
        del junk   # what the call's outputs may be made of
        return paged_attention(q, *b.args(), starts=starts, return_lse=True)

    def check(out, lse):
        ref, lref, vmax = b.ref()
        bound = 3e-5 * vmax if dtype == torch.float32 else 2.0 ** -10 * vmax + 2.0 ** -8 * ref.abs()
        assert ((out[inside].double() - ref).abs() <= bound).all()
        assert ((lse[inside].double() - lref).abs() <= 4e-5 + 2e-6 * lref.abs()).all()
        assert (out[~inside] == 0).all() and (lse[~inside] == -math.inf).all()

    starts = b.starts + before
    check(*attend(starts))
    # a captured step, replayed with fewer tokens
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, l2 = paged_attention(q, *b.args(), starts=starts, return_lse=True)
    graph.replay()
    starts[-1] -= 2
    b.seq_lens[-1] -= 2
    graph.replay()
    inside[before + b.T - 2:] = False
    b.lens, b.news, b.T, b.q = [700, n, 28], [n, n, 1], b.T - 2, b.q[:-2]
    check(out, l2)
    # the append: the same rows alone, into a copy of the cache
    kv = torch.randn(q.shape[0], Hkv, D, device="cuda").to(dtype)
    table = rotary_table(701, D)
    caches = [t.clone() for t in (b.k, b.ks, b.v, b.vs)]
    want = paged_append(kv[inside], kv[inside], *caches, b.table, b.seq_lens, starts=starts - before, q=q[inside], table=table)
    turned = paged_append(kv, kv, *b.args(), starts=starts, q=q, table=table)
    assert torch.equal(turned[inside], want) and torch.equal(turned[~inside], q[~inside])
    for a, c in zip(b.args(), caches):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
    assert _lib.load().sf_q4_check_device_error() == 0
    for bad in ([0, 5, 4, 9], [0, 5, 6, q.shape[0] + 1], [-1, 5, 6, 9]):
        out, l2 = attend(torch.tensor(bad, dtype=torch.int32, device="cuda"))
        assert (out == 0).all() and (l2 == -math.inf).all()
        assert _lib.load().sf_q4_check_device_error() == 10


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_the_largest_batch(cuda, D):
    """4096 sequences, as single tokens and as short runs: nothing is refused, and the last ones' rows are their own."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv import paged_attention
    for H, n in ((2, 1), (16, 8)):
        b = Batch([n + k % 40 for k in range(4096)], [n] * 4096, H, 1, D, 16, torch.bfloat16, ragged=False)
        out = paged_attention(b.q, *b.args())
        ref, _, vmax = b.ref()
        assert ((out.double() - ref).abs() <= 2.0 ** -10 * vmax + 2.0 ** -8 * ref.abs()).all()
        assert _lib.load().sf_q4_check_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 64])
def test_batches_of_different_sizes_from_two_threads(cuda, n):
    """A launch's shared memory hangs on its batch; the calls of one thread leave the other's alone."""
    import ctypes
    import threading

    from siliconfer_b200 import _lib
    lib, refused = _lib.load(), []
    H, Hkv, D = 8, 8, 64

    def work(batch):
        b = Batch([n] * batch, [n] * batch, H, Hkv, D, 16, torch.bfloat16, ragged=False, seed=batch)
        cache = _lib.PagedCache(k_codes=b.k.data_ptr(), k_scales=b.ks.data_ptr(), v_codes=b.v.data_ptr(), v_scales=b.vs.data_ptr(),
                                block_table=b.table.data_ptr(), seq_lens=b.seq_lens.data_ptr(), starts=None, num_pages=b.P,
                                n_kv_heads=Hkv, page_size=16, head_dim=D, batch=batch, pages_per_seq=b.table.shape[1])
        size = lib.sf_paged_attention_workspace_bytes(D)
        ws, stream = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.cuda.Stream()
        ref = torch.empty(b.T, H, D, dtype=torch.bfloat16, device="cuda")
        out = torch.zeros_like(ref)
        torch.cuda.synchronize()
        for y, times in ((ref, 1), (out, 2000)):
            for _ in range(times):
                rc = lib.sf_paged_attention(ctypes.byref(cache), b.q.data_ptr(), 2, H * D, D, y.data_ptr(), 2, None, H, b.T, 0.125, 0,
                                            ws.data_ptr(), size, stream.cuda_stream)
                if rc:
                    refused.append((batch, rc))
                    return
            stream.synchronize()
        if not torch.equal(out, ref):
            refused.append((batch, "result"))

    threads = [threading.Thread(target=work, args=(k,)) for k in (20, 300)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not refused


def test_sequences_near_31_bits_are_refused_without_gpu():
    """Positions are 32-bit and tiles of keys are looked at ahead: the last 1023 positions are not for use."""
    import ctypes

    from siliconfer_b200 import _lib
    lib, F = _lib.load(), 0x1000
    for page in (16, 64, 256):
        for pages, want in ((2 ** 31 // page - 1024 // page, 0), (2 ** 31 // page - 1024 // page + 1, 2), (2 ** 31 // page - 1, 2),
                            (2 ** 31 // page, 2)):
            c = ctypes.byref(_lib.PagedCache(k_codes=F, k_scales=F, v_codes=F, v_scales=F, block_table=F, seq_lens=F, starts=None,
                                             num_pages=4, n_kv_heads=2, page_size=page, head_dim=64, batch=1, pages_per_seq=pages))
            # no rows: validated, not launched
            assert lib.sf_paged_attention(c, F, 0, 512, 64, F, 0, None, 8, 0, 1.0, 0, F, 1 << 30, None) == want
            assert lib.sf_paged_append(c, F, 128, 64, F, 128, 64, None, 0, 0, None, 0, 0, 0, None, 0, 0, 0, None) == want


@pytest.mark.gpu
@pytest.mark.parametrize("B,n,H,Hkv,length,launches", [
    (18, 1, 64, 1, 32768, 2), (3, 8, 64, 8, 32768, 2), (18, 1, 64, 1, 2048, 2), (8, 8, 64, 8, 32768, 2), (2, 32, 64, 8, 32768, 2),
    (16, 8, 64, 8, 2048, 1), (16, 8, 64, 8, 32768, 1), (1, 256, 64, 8, 32768, 1), (2, 32, 64, 8, 256, 1), (64, 4, 64, 4, 2048, 1)])
def test_few_rows_share_the_keys_of_long_sequences(cuda, B, n, H, Hkv, length, launches):
    """A kernel with a CTA for 256 rows (one launch) where a round of such tiles has rows enough, else keys are shared by all
    SMs (two launches), whichever was measured to be faster."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv import paged_attention
    b = Batch([length] + [n + 40] * (B - 1), [n] * B, H, Hkv, 128, 64, torch.bfloat16, ragged=False)
    before = _lib.launch_count()
    paged_attention(b.q, *b.args())
    assert _lib.launch_count() - before == launches
    check_attention(b)
