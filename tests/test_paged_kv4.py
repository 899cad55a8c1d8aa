"""The paged 4-bit cache and attention over it, against plain 64-bit arithmetic over the pages.

Bounds.
  * append: scales and codes are defined by one rounding each of 64-bit values, so they are compared bit for bit.
  * attention.  Queries and codes enter the first product exactly (fp32 queries as two fp16 numbers, 2^-22 of the row's
    largest element), so a score of magnitude up to about 40 is off by its fp32 sums, as in the e4m3 cache's tests: a weight
    by some 2e-5 of itself, the output by 3e-5 max|v|.  Weights of 16-bit queries and outputs are fp16 numbers, 2^-11 of
    each at most: 2^-11 max|v|.  With fp32 among the types: two fp16 parts, 2^-22.  The output's rounding: 2^-8 (bf16) or 2^-11 (fp16) of
    itself.  The log-sum keeps fp32: 4e-5.
  * long runs of 16-bit queries (one launch instead of two): keys and values are fp16 numbers there, 2^-11 of each element
    at most.  A score is off by 2^-11 sum |q k|, so the output by 2^-11 of E_p[sum |q k| (|v| + |out|)], p the softmax's
    weights, with 2 % for the second order, and by 2^-11 E_p|v| for the values; the log-sum by 2^-11 E_p[sum |q k|].
"""
import math
import random

import pytest
import torch

from test_paged_kv import Batch
from test_qk_norm_rotary import near, reference

NAN_BITS = (0x7fc0, 0x7f80, 0xffff, 0x7f00)   # NaN, infinity, another NaN, 1.7e38


class Batch4(Batch):
    def __init__(self, lens, news, H, Hkv, D, page, dtype, seed=0, ragged=True, spare=3, fill=None):
        super().__init__(lens, news, H, Hkv, D, page, dtype, seed=seed, ragged=ragged, spare=spare)
        shape = (self.P, Hkv, page)
        mk = lambda: torch.randint(0, 256, (*shape, D // 2), generator=self.g, device="cuda", dtype=torch.uint8)
        sc = lambda: (0.3 * torch.exp2(2 * torch.rand((*shape, 4), generator=self.g, device="cuda") - 1)).bfloat16()
        self.k, self.v, self.ks, self.vs = mk(), mk(), sc(), sc()
        if fill is not None:
            for b, l in enumerate(lens):
                for j in range(self.table.shape[1]):
                    at = (self.table[b, j], slice(None), slice(max(0, min(page, l - j * page)), None))
                    for t in (self.ks, self.vs):
                        t.view(torch.int16)[at] = fill - 65536 if fill > 32767 else fill

    def values(self, codes, scales, b, l):
        p = self.table[b, :-(-l // self.page)].long()
        return value_of(codes[p], scales[p]).permute(1, 0, 2, 3).reshape(self.Hkv, -1, self.D)[:, :l]


def value_of(codes, scales):
    """Element e of D: quarter c = e // (D / 4), place r: bits 4c .. 4c + 3 of the 16-bit word r."""
    word = codes.int()
    word = word[..., 0::2] + 256 * word[..., 1::2]
    return torch.cat([((word >> 4 * c) % 16 - 8).double() * scales[..., c:c + 1].double() for c in range(4)], -1)


OUT = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def bound_of(batch, out_dtype, ref, vmax, prompt=None):
    coarse = batch.dtype != torch.float32 and out_dtype != torch.float32
    bound = 3e-5 * vmax + (2.0 ** -11 * vmax if coarse else 0.0) + OUT[out_dtype] * ref.abs() + 2.0 ** -25
    return bound if prompt is None else bound + 1.02 * 2.0 ** -11 * prompt[0]


def spread(batch, scale=None, window=0):
    """(E_p[A (|v| + |out|)] + E_p|v|, E_p[A]) with A = scale * sum |q k|."""
    moved = torch.zeros(batch.T, batch.H, batch.D, dtype=torch.float64, device="cuda")
    size = torch.zeros(batch.T, batch.H, dtype=torch.float64, device="cuda")
    scale = batch.D ** -0.5 if scale is None else scale
    for b, l, n, at in batch.rows():
        if not n or not l:
            continue
        k, v = batch.values(batch.k, batch.ks, b, l), batch.values(batch.v, batch.vs, b, l)
        q = batch.q[at:at + n].double().view(n, batch.Hkv, batch.H // batch.Hkv, batch.D)
        far = torch.arange(l - n, l, device="cuda")[:, None] - torch.arange(l, device="cuda")
        hidden = (far < 0) | ((far >= window) if window else False)
        p = (torch.einsum("nhgd,hjd->nhgj", q, k) * scale).masked_fill(hidden[:, None, None], -math.inf).softmax(-1).nan_to_num()
        pa = p * torch.einsum("nhgd,hjd->nhgj", q.abs(), k.abs()) * abs(scale)
        out = torch.einsum("nhgj,hjd->nhgd", p, v)
        moved[at:at + n] = (torch.einsum("nhgj,hjd->nhgd", pa + p, v.abs()) + pa.sum(-1, keepdim=True) * out.abs()).reshape(n, batch.H, -1)
        size[at:at + n] = pa.sum(-1).reshape(n, batch.H)
    return moved, size


def check_attention(batch, out_dtype=None, **kw):
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv4 import paged4_attention
    before = _lib.launch_count()
    out, lse = paged4_attention(batch.q, *batch.args(), starts=batch.starts, out_dtype=out_dtype, return_lse=True, **kw)
    prompt = spread(batch, **kw) if _lib.launch_count() - before == 1 else None
    ref, lref, vmax = batch.ref(**kw)
    dtype = out_dtype or batch.dtype
    assert out.dtype == dtype and out.shape == ref.shape and lse.dtype == torch.float32
    assert ((out.double() - ref).abs() <= bound_of(batch, dtype, ref, vmax, prompt)).all()
    if prompt is not None:   # roundings of either sign: far below their sum
        assert (out.double() - ref).norm() <= 2.0 ** -8 * ref.norm()
    empty = lref == -math.inf
    assert torch.equal(empty, lse == -math.inf)
    off = 4e-5 + 2e-6 * lref.abs() + (0.0 if prompt is None else 2.0 ** -11 * prompt[1])
    assert ((lse.double() - lref).abs() <= off)[~empty].all()
    assert _lib.load().sf_q4_check_device_error() == 0
    return out


HEADS = [(1, 1), (8, 8), (14, 2), (8, 1), (12, 4), (64, 8), (16, 1), (40, 2), (9, 3)]
LENS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 500, 1000, 2049]
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("H,Hkv", HEADS)
def test_single_tokens(cuda, H, Hkv, D, dtype):
    """One new token each, a batch of every length, each page size."""
    for i, page in enumerate((16, 32, 64, 128, 256)):
        lens = LENS[i::2] if Hkv == 8 else LENS[i::3]
        check_attention(Batch4(lens, [1] * len(lens), H, Hkv, D, page, dtype, seed=page, ragged=False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", [(14, 2, 64), (8, 8, 128), (64, 8, 128), (8, 1, 256), (20, 4, 96)])
def test_several_tokens(cuda, H, Hkv, D, dtype):
    """Ragged counts of new tokens from none to whole prompts, with empty sequences between."""
    check_attention(Batch4([70, 5, 0, 300, 129, 64], [7, 5, 0, 1, 40, 64], H, Hkv, D, 32, dtype))
    check_attention(Batch4([33, 257], [33, 200], H, Hkv, D, 64, dtype))
    check_attention(Batch4([100, 100, 100], [4, 4, 4], H, Hkv, D, 16, dtype, ragged=False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [1, 7, 16, 33, 100, 5000])
def test_window(cuda, window, dtype):
    check_attention(Batch4([1, 40, 500, 130], [1, 9, 3, 130], 8, 2, 64, 32, dtype), window=window)
    check_attention(Batch4([700] * 3, [1] * 3, 16, 2, 128, 64, dtype, ragged=False), window=window, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_sequences_and_uneven_batches(cuda, dtype):
    check_attention(Batch4([40000], [1], 8, 1, 128, 64, dtype, ragged=False))
    check_attention(Batch4([9000, 1, 0, 17, 3001], [1, 1, 0, 1, 1], 64, 8, 128, 64, dtype))
    rng = random.Random(4)
    lens = [rng.randint(1, 400) for _ in range(200)]
    check_attention(Batch4(lens, [1] * 200, 4, 2, 64, 16, dtype, ragged=False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_rows_empty_and_no_rows(cuda, dtype):
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([5, 6], [1, 1], 8, 2, 64, 16, dtype, ragged=False)
    b.seq_lens.zero_()
    out, lse = paged4_attention(b.q, *b.args(), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out = paged4_attention(b.q[:0], *b.args(), starts=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 8, 64)
    b = Batch4([3, 40], [5, 2], 8, 2, 64, 16, dtype)     # two of the five rows lie before their sequence
    out, lse = paged4_attention(b.q, *b.args(), starts=b.starts, return_lse=True)
    assert (out[:2] == 0).all() and (lse[:2] == -math.inf).all() and torch.isfinite(lse[2:]).all()
    c = Batch4([3, 40], [3, 2], 8, 2, 64, 16, dtype)
    c.q, c.k, c.v, c.ks, c.vs, c.table = b.q[2:], b.k, b.v, b.ks, b.vs, b.table
    ref, _, vmax = c.ref()
    assert ((out[2:].double() - ref).abs() <= bound_of(c, dtype, ref, vmax)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fill", NAN_BITS)
def test_contents_beyond_the_end_do_not_matter(cuda, fill):
    """NaN, infinite and large scales in every slot past a sequence's end."""
    for dtype in TYPES:
        check_attention(Batch4([1, 20, 100, 130], [1, 1, 1, 1], 14, 2, 64, 64, dtype, ragged=False, fill=fill))
        check_attention(Batch4([9, 33, 65], [9, 2, 33], 8, 8, 128, 16, dtype, fill=fill))
        check_attention(Batch4([19, 250], [1, 3], 8, 1, 256, 256, dtype, fill=fill))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_small_values(cuda, dtype):
    """Scores that would overflow e^s, value scales far apart between tokens, zero scales, queries near their type's ends."""
    b = Batch4([200, 300], [1, 1], 8, 2, 64, 16, dtype, ragged=False)
    check_attention(b, scale=3.0 / 8)
    b.vs = torch.exp2(torch.randint(-20, 6, b.vs.shape[:3] + (1,), generator=b.g, device="cuda").float()).expand(-1, -1, -1, 4).bfloat16().contiguous()
    check_attention(b)
    b.vs[:, :, ::2] = 0
    check_attention(b)
    b.vs.fill_(2.0 ** 90)
    if dtype == torch.float32:
        check_attention(b)
    b.vs.fill_(2.0 ** -100)
    check_attention(b)
    b.vs.fill_(0)
    assert (check_attention(b) == 0).all()
    b.vs.fill_(0.5)
    b.q = (b.q.float() * (2.0 ** -12)).to(dtype)
    check_attention(b, scale=512.0)
    if dtype != torch.float16:
        b.q = (b.q.float() * 2.0 ** 60).to(dtype)
        check_attention(b, scale=2.0 ** -54)
    b.q.zero_()
    check_attention(b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_non_finite_values_stay_in_their_rows(cuda, dtype):
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([50, 60], [2, 2], 8, 2, 64, 16, dtype, ragged=False)
    b.q[0, 3, 5], b.q[1, 7, 0] = float("nan"), float("inf")
    b.vs[b.table[1, 0], 1, 3] = float("nan")      # sequence 1, kv head 1, a token that both rows see
    b.ks[b.table[0, 3], 0, 1] = float("nan")      # sequence 0, kv head 0, its last token: the second row sees it
    out = paged4_attention(b.q, *b.args())
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 3] = bad[1, 7] = True
    bad[2:, 4:] = True
    bad[1, :4] = True
    assert torch.equal(out.isnan(), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_values_that_a_row_does_not_see_cannot_reach_it(cuda, D, dtype):
    """NaN keys and values of later tokens of the same call, and of tokens before a row's window."""
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([90], [60], 8, 2, D, 16, dtype)
    ref, _, vmax = b.ref(window=10)
    pos = torch.arange(30, 90, device="cuda")
    sees = torch.zeros(60, dtype=torch.bool, device="cuda")
    for i, at in enumerate((40, 47, 70)):
        (b.ks if i else b.vs)[b.table[0, at // 16], 1, at % 16] = float("nan")
        b.vs[b.table[0, at // 16], 1, at % 16] = float("nan")
        sees |= (pos >= at) & (pos < at + 10)
    out = paged4_attention(b.q, *b.args(), starts=b.starts, window=10)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[sees, 4:] = True
    assert torch.equal(out.isnan(), bad) and (~sees).sum() > 5
    assert ((out.double() - ref).abs()[~bad] <= bound_of(b, dtype, ref, vmax)[~bad]).all()


def _mass(b):
    """sum p |v| of each element."""
    out = torch.zeros(b.T, b.H, b.D, dtype=torch.float64, device="cuda")
    for s, l, n, at in b.rows():
        k, v = b.values(b.k, b.ks, s, l), b.values(b.v, b.vs, s, l)
        q = b.q[at:at + n].double().view(n, b.Hkv, b.H // b.Hkv, b.D)
        w = torch.einsum("nhgd,hjd->nhgj", q, k) * b.D ** -0.5
        far = torch.arange(l - n, l, device="cuda")[:, None] - torch.arange(l, device="cuda")
        w = w.masked_fill((far < 0)[:, None, None], -math.inf).softmax(-1)
        out[at:at + n] = torch.einsum("nhgj,hjd->nhgd", w, v.abs()).reshape(n, b.H, b.D)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                             (torch.bfloat16, torch.float16), (torch.float32, torch.float16),
                                             (torch.float32, torch.bfloat16), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("H,Hkv,D,n", [(64, 8, 128, 1), (14, 2, 64, 1), (8, 8, 256, 1), (4, 4, 96, 3), (64, 8, 128, 300),
                                       (16, 16, 64, 600)])
def test_weights_are_as_fine_as_the_finer_type(cuda, H, Hkv, D, n, dtype, out_dtype):
    """fp32 among the types: within 5e-5 of sum p |v|, scores' roundings included, and half a step of the output.  Else a
    weight is an fp16 number: 2^-11 more."""
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([n + 1, n + 2, n + 5, n + 30], [n] * 4, H, Hkv, D, 16, dtype)
    out = paged4_attention(b.q, *b.args(), starts=b.starts, out_dtype=out_dtype)
    ref = b.ref()[0]
    bound = 5e-5 * _mass(b) + OUT[out_dtype] * ref.abs() + 2.0 ** -24
    if torch.float32 not in (dtype, out_dtype):   # and in a prompt's tiles fp16 keys and values
        bound = bound + 2.0 ** -11 * _mass(b) + 1.02 * 2.0 ** -11 * spread(b)[0]
    assert ((out.double() - ref).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv", [(8, 2), (32, 4)])
def test_strided_queries_types_and_repeats(cuda, H, Hkv):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        b = Batch4([300, 1000, 90], [1, 4, 2], H, Hkv, 128, 64, dtype)
        first = check_attention(b, out_dtype=torch.float32)
        wide = torch.zeros(b.T, (H + 3) * 128 + 1, device="cuda", dtype=dtype)
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
    from siliconfer_b200.paged_kv4 import paged4_attention
    a = Batch4([3000, 10], [1, 1], 32, 4, 128, 64, torch.bfloat16, ragged=False)
    b = Batch4([100, 2000, 77], [1, 1, 1], 32, 4, 128, 64, torch.bfloat16, ragged=False, seed=9)
    ra, rb = paged4_attention(a.q, *a.args()), paged4_attention(b.q, *b.args())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(20):
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(paged4_attention(x.q, *x.args()))
    torch.cuda.synchronize()
    assert all(torch.equal(y, r) for y, r in zip(got, [ra, rb] * 20))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = paged4_attention(a.q, *a.args())
    for lens in ([3000, 10], [17, 2]):       # lengths are read when the graph runs
        a.lens = lens
        a.seq_lens.copy_(torch.tensor(lens))
        graph.replay()
        torch.cuda.synchronize()
        ref, _, vmax = a.ref()
        assert ((y.double() - ref).abs() <= bound_of(a, torch.bfloat16, ref, vmax)).all()


@pytest.mark.gpu
def test_pages_past_31_bits(cuda):
    """A pool of more than 2^31 bytes and 2^32 elements: the pages at its end are read and written like the first ones."""
    from siliconfer_b200.paged_kv4 import paged4_append, quantize_kv4
    b = Batch4([40, 90], [1, 1], 8, 2, 128, 64, torch.bfloat16, ragged=False)
    P = 2 ** 31 // (2 * 64 * 64) + 40
    far = P - b.P
    big = []
    for src in (b.k, b.ks, b.v, b.vs):
        big.append(torch.zeros((P,) + src.shape[1:], dtype=src.dtype, device="cuda"))
        big[-1][far:] = src
    b.k, b.ks, b.v, b.vs = big
    b.table = b.table + far
    check_attention(b)
    x = torch.randn(2, 2, 128, device="cuda", dtype=torch.bfloat16)
    paged4_append(x, -x, *b.args())
    p = int(b.table[1, 1])
    for codes, scales, y in ((b.k, b.ks, x), (b.v, b.vs, -x)):
        c, s = quantize_kv4(y[1])
        assert torch.equal(codes[p, :, 89 - 64], c) and torch.equal(scales[p, :, 89 - 64], s)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [-1, -2, -(2 ** 31), 2 ** 31 - 1])
@pytest.mark.parametrize("n", [1, 600])
def test_page_numbers_out_of_range_are_reported(cuda, n, page):
    """For single tokens and for prompts; the other sequence's rows are what they were."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([700, 800], [n, n], 32, 8, 64, 16, torch.bfloat16)
    good = paged4_attention(b.q, *b.args(), starts=b.starts)
    b.table[0, 3] = page
    out = paged4_attention(b.q, *b.args(), starts=b.starts)
    torch.cuda.synchronize()
    assert _lib.load().sf_q4_check_device_error() == 10
    assert torch.equal(out[n:], good[n:]) and torch.isfinite(out.float()).all()
    assert _lib.load().sf_q4_check_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 600])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 32), (64, 128)])
def test_pages_that_a_window_has_given_up(cuda, D, page, n):
    """Page numbers before a sequence's first key in the window are not looked at, for single tokens and for prompts."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([1500, 905], [n, n], 32, 8, D, page, torch.bfloat16)
    good = paged4_attention(b.q, *b.args(), starts=b.starts, window=200)
    for s, l, _, _ in b.rows():
        b.table[s, :max(0, l - n + 1 - 200) // page] = -1
    out = paged4_attention(b.q, *b.args(), starts=b.starts, window=200)
    torch.cuda.synchronize()
    assert _lib.load().sf_q4_check_device_error() == 0
    assert torch.equal(out, good)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 30, 1024])
@pytest.mark.parametrize("n,D", [(4, 64), (400, 128)])
def test_windows_wider_than_the_sequences(cuda, n, D, window):
    """They hide nothing, from sequences with fewer tokens than rows either."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([n, n, n + 500, n], [n] * 4, 32, 8, D, 16, torch.bfloat16)
    b.seq_lens.copy_(torch.tensor([1, n // 2, n + 500, 0]))
    want, lse = paged4_attention(b.q, *b.args(), starts=b.starts, return_lse=True)
    out, l2 = paged4_attention(b.q, *b.args(), starts=b.starts, return_lse=True, window=window)
    assert torch.equal(out, want) and torch.equal(l2, lse)
    assert torch.isfinite(l2[n - 1]).all() and (out[:n - 1] == 0).all()
    assert _lib.load().sf_q4_check_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 400])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_no_sequence(cuda, n, dtype):
    """Rows before the first sequence's and behind the last one's: turned as at position 0 whatever their positions say, not
    written, and they see nothing; starts that fall or leave the rows: an error, and 0 for all of them."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv4 import paged4_append, paged4_attention
    from siliconfer_b200.rotary import rotary_axes, rotary_table
    H, Hkv, D, before, after = 32, 8, 64, 3, 5
    lib = _lib.load()
    b = Batch4([700, n, 30], [n, n, 3], H, Hkv, D, 16, dtype)
    T = before + b.T + after
    q = torch.randn(T, H, D, device="cuda").to(dtype)
    inside = torch.zeros(T, dtype=torch.bool, device="cuda")
    inside[before:before + b.T] = True
    q[inside] = b.q
    starts = b.starts + before
    out, lse = paged4_attention(q, *b.args(), starts=starts, return_lse=True)
    check_attention(b)   # the other call's parts of the keys may be others: alike within the bound
    ref, _, vmax = b.ref()
    assert ((out[inside].double() - ref).abs() <= bound_of(b, dtype, ref, vmax, None if dtype == torch.float32 else spread(b))).all()
    assert (out[~inside] == 0).all() and (lse[~inside] == -math.inf).all()
    kv = torch.randn(T, Hkv, D, device="cuda").to(dtype)
    table = rotary_table(1000, D)
    pos = torch.randint(0, 1000, (T, 2), device="cuda")
    pos[~inside] = -7
    held = [x.clone() for x in (b.k, b.ks, b.v, b.vs)]
    got = paged4_append(kv, kv, *b.args(), starts=starts, q=q, table=table, positions=pos, axes=rotary_axes((16, 16)), eps=1e-6)
    assert lib.sf_q4_check_device_error() == 0
    want, mass = reference(q[~inside], None, 1e-6, torch.zeros(before + after, device="cuda"), table, False, None)
    assert near(got[~inside], want, mass, dtype)
    written = torch.zeros(b.P, 16, dtype=torch.bool, device="cuda")
    for s, l, c, _ in b.rows():
        for p in range(l - c, l):
            written[b.table[s, p // 16], p % 16] = True
    for now, old in zip((b.k, b.ks, b.v, b.vs), held):
        assert torch.equal(now.transpose(1, 2)[~written], old.transpose(1, 2)[~written])
    for wrong in (starts.flip(0), starts + after + 1, starts - before - 1):
        out = paged4_attention(q, *b.args(), starts=wrong.contiguous())
        torch.cuda.synchronize()
        assert lib.sf_q4_check_device_error() == 10 and (out == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_the_largest_batch(cuda, D):
    """4096 sequences, as single tokens and as short runs: nothing is refused, and the last ones' rows are their own."""
    for H, n in ((2, 1), (16, 8)):
        check_attention(Batch4([n + k % 40 for k in range(4096)], [n] * 4096, H, 1, D, 16, torch.bfloat16, ragged=False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hkv,D,page", [(64, 8, 128, 64), (14, 2, 64, 16), (32, 32, 128, 256), (8, 8, 64, 128), (16, 1, 128, 32),
                                          (40, 8, 64, 64)])
def test_prompts(cuda, H, Hkv, D, page, dtype):
    """Whole prompts, later chunks, runs that end anywhere in a tile; empty sequences and single tokens between."""
    n = 256 * 40 * Hkv // (H * Hkv) + 900      # rows for a quarter of the SMs at least
    for lens, news in (([n], [n]), ([n + 500, 0, 300, 70, 1], [n, 0, 290, 1, 1]), ([n, n - 3], [n - 128, n - 130]),
                       ([2500, 2049], [n, 255])):
        check_attention(Batch4(lens, [min(a, b) for a, b in zip(news, lens)], H, Hkv, D, page, dtype, seed=n))
    check_attention(Batch4([n + 40] * 3, [n // 2] * 3, H, Hkv, D, page, dtype, ragged=False), out_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 40, 128, 300, 5000])
def test_prompts_with_a_window(cuda, window):
    check_attention(Batch4([1500, 900], [1400, 300], 16, 8, 128, 64, torch.bfloat16), window=window, out_dtype=torch.float16)
    check_attention(Batch4([700, 600], [700, 600], 28, 4, 64, 16, torch.bfloat16), window=window, scale=-0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("fill", NAN_BITS)
def test_prompts_beyond_the_end(cuda, fill):
    check_attention(Batch4([1001, 650, 0], [1001, 200, 0], 64, 8, 128, 64, torch.bfloat16, fill=fill))
    check_attention(Batch4([1500], [1490], 14, 2, 64, 16, torch.bfloat16, fill=fill))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_rows_keep_to_themselves(cuda, D):
    """NaN and infinite queries, NaN keys and values that some rows see and others do not, with a window and without."""
    from siliconfer_b200.paged_kv4 import paged4_attention
    for window in (0, 200):
        b = Batch4([900], [800], 32, 8, D, 16, torch.bfloat16)
        ref, _, vmax = b.ref(window=window)
        bound = bound_of(b, torch.bfloat16, ref, vmax, spread(b, window=window))
        marks = (40, 333, 640, 897)
        for i, at in enumerate(marks):
            (b.ks if i % 2 else b.vs)[b.table[0, at // 16], 1, at % 16] = float("nan")
        b.q[300, 20, 5], b.q[301, 21, 0] = float("nan"), float("inf")
        out = paged4_attention(b.q, *b.args(), starts=b.starts, window=window)
        pos = torch.arange(100, 900, device="cuda")
        bad = torch.zeros_like(out, dtype=torch.bool)
        for at in marks:
            bad[(pos >= at) & ((pos < at + window) if window else True), 4:8] = True
        bad[300, 20] = bad[301, 21] = True
        assert torch.equal(out.isnan(), bad) and (~bad).any()
        assert ((out.double() - ref).abs() <= bound)[~bad].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_values_strides_and_padding(cuda, dtype):
    """Repeats, strides, queries near their type's ends, no scale, value and key scales apart, padding rows, a captured call."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([700, 800], [650, 800], 32, 8, 64, 16, dtype)
    first = check_attention(b)
    for _ in range(3):
        assert torch.equal(check_attention(b), first)
    wide = torch.zeros(b.T, 35 * 64 + 1, device="cuda", dtype=dtype)
    q = b.q
    for off in (0, 1, 72):
        wide[:, off:off + 32 * 64] = q.reshape(b.T, -1)
        b.q = wide[:, off:off + 32 * 64].view(b.T, 32, 64)
        assert torch.equal(check_attention(b), first)
    b.q = q
    check_attention(b, scale=0.0)
    b.q = q * 2.0 ** -10
    check_attention(b, scale=100.0)
    if dtype == torch.bfloat16:
        b.q = q * 2.0 ** 100
        check_attention(b, scale=2.0 ** -103)
        b.q = q * 2.0 ** -110
        check_attention(b, scale=2.0 ** 100)
    b.q = q
    b.vs = (b.vs.float() * torch.exp2(torch.randint(-8, 3, b.vs.shape[:3] + (1,), generator=b.g, device="cuda"))).bfloat16()
    b.ks = (b.ks.float() * torch.exp2(torch.randint(-6, 1, b.ks.shape[:3] + (1,), generator=b.g, device="cuda"))).bfloat16()
    check_attention(b)
    b.vs[:, :, ::3] = 0
    b.ks[:, :, ::5] = 0
    check_attention(b)
    b.q = torch.zeros_like(q)
    check_attention(b)
    b.q = q
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = paged4_attention(b.q, *b.args(), starts=b.starts)
    for lens in ([700, 800], [651, 799], [20, 100]):      # fewer tokens than rows: padding rows in front
        b.seq_lens.copy_(torch.tensor(lens))
        graph.replay()
        torch.cuda.synchronize()
        assert _lib.load().sf_q4_check_device_error() == 0
        c = Batch4(lens, [min(650, lens[0]), min(800, lens[1])], 32, 8, 64, 16, dtype)
        keep = torch.cat([torch.arange(650 - c.news[0], 650), torch.arange(1450 - c.news[1], 1450)]).cuda()
        c.q, c.k, c.v, c.ks, c.vs, c.table = q[keep], b.k, b.v, b.ks, b.vs, b.table
        ref, _, vmax = c.ref()
        assert ((y[keep].double() - ref).abs() <= bound_of(c, dtype, ref, vmax, spread(c))).all()
        rest = torch.ones(1450, dtype=torch.bool, device="cuda")
        rest[keep] = False
        assert (y[rest] == 0).all()


@pytest.mark.gpu
def test_two_threads(cuda):
    """Calls of different batches from two threads, each on a stream of its own."""
    import threading

    from siliconfer_b200.paged_kv4 import paged4_attention
    wrong = []

    def work(batch, n):
        try:
            b = Batch4([n + k % 7 for k in range(batch)], [n] * batch, 16, 2, 128, 64, torch.bfloat16, ragged=False, seed=batch)
            ref, _, vmax = b.ref()
            torch.cuda.synchronize()
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(40):
                    out = paged4_attention(b.q, *b.args())
                    if not ((out.double() - ref).abs() <= bound_of(b, torch.bfloat16, ref, vmax)).all():
                        wrong.append(batch)
                torch.cuda.current_stream().synchronize()
        except RuntimeError as e:
            wrong.append(str(e))

    threads = [threading.Thread(target=work, args=a) for a in ((2, 40), (600, 1))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------
def codes_of(y):
    """y [..., D] in 64 bits -> (codes, scales): scales by one rounding to fp32 and one to bf16."""
    Q = y.shape[-1] // 4
    finite = torch.isfinite(y).all(-1)
    word, scales = torch.zeros(y.shape[:-1] + (Q,), dtype=torch.int32, device=y.device), []
    for c in range(4):
        part = y[..., c * Q:(c + 1) * Q]
        s = torch.clamp(torch.div(part.abs().amax(-1), torch.tensor(7.5, dtype=torch.float64, device=y.device)).float().bfloat16(), min=2.0 ** -126)
        n = torch.where(finite[..., None], torch.round(part / s.double()[..., None]).clamp(-8, 7), torch.zeros_like(part)).int() + 8
        word += n * 16 ** c
        scales.append(torch.where(finite, s, torch.full_like(s, float("nan"))))
    return torch.stack([word % 256, word // 256], -1).flatten(-2).to(torch.uint8), torch.stack(scales, -1)


def same_scales(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=1.0), b.nan_to_num(nan=1.0))


def check_append(batch, dtype, rot=None, interleaved=False, turn=True, eps=None, axes=1, values=None, strided=False, with_q=True,
                 weights=torch.float32):
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv4 import paged4_append
    from siliconfer_b200.rotary import rotary_axes, rotary_table
    T, H, Hkv, D = batch.T, batch.H, batch.Hkv, batch.D
    x = torch.randn(T, H + 2 * Hkv, D, generator=batch.g, device="cuda").to(dtype)
    if strided:
        wide = torch.zeros(T, (H + 2 * Hkv) * D + 5, device="cuda", dtype=dtype)
        wide[:, 3:3 + (H + 2 * Hkv) * D] = x.reshape(T, -1)
        x = wide[:, 3:3 + (H + 2 * Hkv) * D].view(T, H + 2 * Hkv, D)
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    if values:
        values(k, v)
    rot = D if rot is None else rot
    pos = torch.cat([torch.arange(l - n, l, device="cuda") for _, l, n, _ in batch.rows()])
    table = rotary_table(max(2000, int(pos.max()) + 1), rot) if turn else None
    positions = ax = None
    if turn and axes > 1:
        positions = torch.randint(0, 2000, (T, axes), generator=batch.g, device="cuda", dtype=torch.int32)
        ax = rotary_axes([rot // 2 - (axes - 1) * (rot // 2 // axes)] + [rot // 2 // axes] * (axes - 1), interleaved=True)
    w = [None, None] if eps is None else [(1 + 0.2 * torch.randn(D, generator=batch.g, device="cuda")).to(weights) for _ in range(2)]
    held = [t.clone() for t in (batch.k, batch.ks, batch.v, batch.vs)]
    q_in = q if with_q and (turn or eps is not None) else None
    got = paged4_append(k, v, *batch.args(), starts=batch.starts, q=q_in, table=table, interleaved=interleaved, positions=positions,
                        axes=ax, q_weight=w[0] if q_in is not None else None, k_weight=w[1], eps=eps)
    at = pos if positions is None else positions
    key, _ = reference(k, w[1], eps, at, table, interleaved, ax)
    slots = [(int(batch.table[b, p // batch.page]), p % batch.page) for b, l, n, _ in batch.rows() for p in range(l - n, l)]
    page_of, slot = torch.tensor(slots, device="cuda").T
    for i, y in ((0, key), (2, v.double())):
        codes, scales = codes_of(y)
        held[i][page_of, :, slot], held[i + 1][page_of, :, slot] = codes, scales
    assert torch.equal(batch.k, held[0]) and same_scales(batch.ks, held[1])
    assert torch.equal(batch.v, held[2]) and same_scales(batch.vs, held[3])
    if q_in is None:
        assert got is None
    else:
        want, mass = reference(q, w[0], eps, at, table, interleaved, ax)
        assert got.dtype == dtype and near(got, want, mass, dtype)
    assert _lib.load().sf_q4_check_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", [(14, 2, 64), (8, 8, 128), (6, 3, 96), (4, 1, 256)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_append(cuda, page, H, Hkv, D, dtype):
    lens = [1, page, page + 1, 2 * page - 1, 3 * page + 5, 1000]
    check_append(Batch4(lens, [1] * 6, H, Hkv, D, page, dtype, ragged=False), dtype, eps=1e-6)
    check_append(Batch4(lens, [1, 3, page, 0, 2 * page + 7, 1000], H, Hkv, D, page, dtype), dtype, turn=False)
    check_append(Batch4(lens, [1, page, page + 1, 5, 2 * page, 900], H, Hkv, D, page, dtype), dtype, interleaved=True, axes=3)
    check_append(Batch4(lens, [1, 3, page, 0, 7, 400], H, Hkv, D, page, dtype), dtype, eps=1e-5, turn=False, weights=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rot", [64, 32, 48, 20, 2])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_partial_rotary_and_strides(cuda, rot, interleaved):
    for dtype in (torch.bfloat16, torch.float32):
        b = lambda: Batch4([70, 9, 0, 130], [6, 9, 0, 1], 5, 2, 64, 32, dtype, seed=rot)
        check_append(b(), dtype, rot=rot, interleaved=interleaved)
        check_append(b(), dtype, rot=rot, interleaved=interleaved, eps=1e-6, strided=True, axes=2 if rot > 2 else 1)
        check_append(b(), dtype, rot=rot, interleaved=interleaved, with_q=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_append_special_values(cuda, dtype):
    """Zero vectors and quarters, tiny and large ones, ties, infinities and NaN, which keep to their vectors."""
    def values(k, v):
        for x in (k, v):
            x[0] = 0
            x[1, 0, 16:32] = 0
            x[2] = (x[2].float() * 1e-4).to(dtype)
            x[3] = (x[3].float() * 1e4).clamp(-6e4, 6e4).to(dtype)
            x[4, 0] = torch.arange(64, device="cuda").sub(32).to(dtype) / 2      # scale 2.125 = 16 / 7.5 rounded
            x[4, 1] = 7.5 * torch.arange(64, device="cuda").remainder(2).to(dtype)
            x[5, 0, :] = torch.tensor([7.5, 0.5, 1.5, -0.5, -1.5, 2.5, -2.5, -7.5], device="cuda").repeat(8).to(dtype)  # scale 1: ties
            x[6, 0, 9], x[7, 1, 63], x[8, 0, 0] = float("inf"), float("nan"), float("-inf")
            if dtype != torch.float16:
                x[9] = (x[9].float() * 1e-37).to(dtype)
                x[10, 0] = (x[10, 0].float() * 1e30).to(dtype)
            x[11] = 2.0 ** -24
    for turn, eps in ((False, None), (False, 1e-6)):
        check_append(Batch4([40, 30], [20, 5], 4, 2, 64, 16, dtype), dtype, turn=turn, eps=eps, values=values)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_append_many_tokens(cuda, dtype):
    """Millions of elements, of which some lie as near to a tie as 64 bits tell apart."""
    check_append(Batch4([3000, 900], [3000, 800], 8, 8, 128, 64, dtype), dtype, eps=1e-6)
    check_append(Batch4([1900], [1900], 3, 8, 128, 64, dtype, seed=5), dtype, interleaved=True, axes=3)


@pytest.mark.gpu
def test_append_more_sequences_than_a_search_probes_at_once(cuda):
    lens = [61 + 5 * b for b in range(140)]
    check_append(Batch4(lens, [b % 9 for b in range(140)], 2, 1, 96, 32, torch.bfloat16), torch.bfloat16, eps=1e-6)


@pytest.mark.gpu
def test_append_indices_outside_are_skipped_and_reported(cuda):
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv4 import paged4_append, paged4_attention
    from siliconfer_b200.rotary import rotary_table
    lib = _lib.load()
    mk = lambda: Batch4([40, 50], [1, 1], 8, 2, 64, 16, torch.bfloat16, ragged=False)
    kv = torch.randn(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    for page in (10 ** 6, -5):
        b = mk()
        b.table[0, 2] = page
        k0, v0 = b.k.clone(), b.v.clone()
        paged4_append(kv, kv, *b.args())
        torch.cuda.synchronize()
        assert lib.sf_q4_check_device_error() == 10
        p = int(b.table[1, 3])
        k0[p, :, 1], v0[p, :, 1] = b.k[p, :, 1], b.v[p, :, 1]
        assert torch.equal(b.k, k0) and torch.equal(b.v, v0)
    for lens in ([1000, 50], [-1, 50], [40, 65]):
        b = mk()
        b.seq_lens.copy_(torch.tensor(lens))
        paged4_append(kv, kv, *b.args())
        torch.cuda.synchronize()
        assert lib.sf_q4_check_device_error() == 10
        out = paged4_attention(b.q, *b.args())
        torch.cuda.synchronize()
        assert lib.sf_q4_check_device_error() == 10 and torch.isfinite(out).all()
    b = mk()
    paged4_append(kv, kv, *b.args(), table=rotary_table(45, 64), q=b.q)     # position 49 is past the table's end
    torch.cuda.synchronize()
    assert lib.sf_q4_check_device_error() == 10
    assert b.ks[b.table[1, 3], :, 1].isnan().all() and torch.isfinite(b.ks[b.table[0, 2], :, 7]).all()


@pytest.mark.gpu
def test_append_then_attend_captured(cuda):
    """A decode step (norm, turn, append, attend) in one graph, replayed as the sequences grow, and with fewer tokens."""
    from siliconfer_b200.paged_kv4 import Paged4KVCache, dequantize_kv4, quantize_kv4
    from siliconfer_b200.rotary import rotary_table
    H, Hkv, D, B, page = 8, 2, 64, 3, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = Paged4KVCache(20, Hkv, D, page)
    pages = torch.randperm(20, generator=g, device="cuda")[:18].view(B, 6).to(torch.int32)
    table, w = rotary_table(96, D), torch.randn(D, generator=g, device="cuda")
    lens = torch.tensor([0, 20, 31], dtype=torch.int32, device="cuda")
    x = torch.randn(B, H + 2 * Hkv, D, generator=g, device="cuda").bfloat16()
    hist = [[], [], []]
    y0 = torch.randn(51, 2 * Hkv, D, generator=g, device="cuda").bfloat16()
    starts = torch.tensor([0, 0, 20, 51], dtype=torch.int32, device="cuda")
    cache.append(y0[:, :Hkv], y0[:, Hkv:], pages, lens, starts, table=table, k_weight=w, eps=1e-6)
    for b, (lo, hi) in enumerate(((0, 0), (0, 20), (20, 51))):
        hist[b] += [(y0[i, :Hkv], y0[i, Hkv:], i - lo) for i in range(lo, hi)]

    def step():
        q = cache.append(x[:, H:H + Hkv], x[:, H + Hkv:], pages, lens, q=x[:, :H], table=table, q_weight=w, k_weight=w, eps=1e-6)
        return q, cache.attend(q, pages, lens, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        lens.add_(1)
        step()          # writes what the first replay writes again
        lens.sub_(1)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        lens.add_(1)
        q, (out, lse) = step()
    for _ in range(20):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            hist[b].append((x[b, H:H + Hkv].clone(), x[b, H + Hkv:].clone(), len(hist[b])))
            key, _ = reference(torch.stack([k for k, _, _ in hist[b]]), w, 1e-6, torch.tensor([p for _, _, p in hist[b]], device="cuda"), table, False, None)
            k = dequantize_kv4(*quantize_kv4(key)).double().repeat_interleave(H // Hkv, 1)
            v = dequantize_kv4(*quantize_kv4(torch.stack([v for _, v, _ in hist[b]]))).double().repeat_interleave(H // Hkv, 1)
            s = torch.einsum("hd,khd->hk", q[b].double(), k) * D ** -0.5
            ref = torch.einsum("hk,khd->hd", s.softmax(-1), v)
            assert ((out[b].double() - ref).abs() <= (3e-5 + 2.0 ** -11) * v.abs().max() + 2.0 ** -8 * ref.abs()).all()
            assert (lse[b].double() - s.logsumexp(-1)).abs().max() <= 4e-5 + 2e-6 * s.abs().max()
    assert lens.tolist() == [20, 40, 51]


@pytest.mark.gpu
def test_quantizer_in_torch(cuda):
    from siliconfer_b200.paged_kv4 import dequantize_kv4, quantize_kv4
    x = torch.randn(50, 3, 96, device="cuda")
    x[3, 1, 5], x[4] = float("inf"), 0
    codes, scales = quantize_kv4(x)
    want, ws = codes_of(x.double())
    assert torch.equal(codes, want) and same_scales(scales, ws)
    y, finite = dequantize_kv4(codes, scales), torch.isfinite(x).all(-1)
    assert torch.equal(y.isnan().any(-1), ~finite) and torch.equal(y[finite].double(), value_of(codes, scales)[finite])
    step = scales.float().repeat_interleave(24, -1)
    # 7.5 (1 + 2^-8) at most: half a step, and what the scale's rounding takes from the largest
    assert ((y - x).abs()[finite] <= (0.5 + 7.5 * 2.0 ** -8) * step[finite]).all()


@pytest.mark.gpu
def test_refusals(cuda):
    from siliconfer_b200.paged_kv4 import paged4_append, paged4_attention
    b = Batch4([40, 50], [1, 1], 8, 2, 64, 16, torch.bfloat16, ragged=False)
    k, ks, v, vs, table, lens = b.args()
    x = torch.randn(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    t, w = torch.zeros(100, 64, device="cuda"), torch.ones(64, device="cuda")
    pos = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    ax = torch.zeros(32, dtype=torch.uint8, device="cuda")
    att = lambda q=b.q, k=k, ks=ks, v=v, vs=vs, table=table, lens=lens, **kw: paged4_attention(q, k, ks, v, vs, table, lens, **kw)
    app = lambda a=x, c=x, k=k, ks=ks, vs=vs, table=table, lens=lens, **kw: paged4_append(a, c, k, ks, v, vs, table, lens, **kw)
    for bad in (lambda: att(q=b.q.cpu()), lambda: att(q=b.q.double()), lambda: att(q=b.q[:, :7]), lambda: att(q=b.q[:, :, :32]),
                lambda: att(q=b.q[:1]), lambda: att(q=b.q[0]), lambda: att(k=k.view(torch.int8)), lambda: att(k=k[:, :1]),
                lambda: att(k=k.transpose(1, 2)), lambda: att(ks=ks[:1]), lambda: att(ks=ks.half()), lambda: att(vs=vs.cpu()),
                lambda: att(ks=ks[..., :2]), lambda: att(vs=vs[..., 0]), lambda: att(table=table.long()), lambda: att(table=table[0]),
                lambda: att(lens=lens.long()), lambda: att(lens=lens[:1]), lambda: att(starts=lens),
                lambda: att(starts=torch.zeros(3, device="cuda")), lambda: att(window=2 ** 31), lambda: att(out_dtype=torch.float64),
                lambda: att(k=k[..., :16].contiguous(), v=v[..., :16].contiguous()),
                lambda: app(a=x.cpu()), lambda: app(c=x.float()), lambda: app(a=x[:, :1]), lambda: app(a=x[..., :32]),
                lambda: app(a=x[:1], c=x[:1]), lambda: app(a=x.double(), c=x.double()), lambda: app(ks=ks.float()),
                lambda: app(q=b.q), lambda: app(q=b.q[:1], table=t), lambda: app(q=b.q.float(), table=t), lambda: app(table=t.half()),
                lambda: app(table=t[:, :63]), lambda: app(table=torch.zeros(9, 66, device="cuda")), lambda: app(positions=pos[:, 0]),
                lambda: app(table=t, positions=pos), lambda: app(table=t, positions=pos, axes=ax[:5]), lambda: app(table=t, axes=ax),
                lambda: app(k_weight=w), lambda: app(k_weight=w[:5], eps=1e-6), lambda: app(q_weight=w, eps=1e-6), lambda: app(eps=-1.0),
                lambda: app(table=t, positions=pos[:1], axes=ax)):
        with pytest.raises(RuntimeError):
            bad()
    torch.cuda.synchronize()


def test_validation_without_gpu():
    import ctypes

    from siliconfer_b200 import _lib
    lib, F = _lib.load(), 0x1000

    def cache(**k):
        return ctypes.byref(_lib.Paged4Cache(**{**dict(k_codes=F, k_scales=F, v_codes=F, v_scales=F, block_table=F, seq_lens=F,
                                                       starts=None, num_pages=4, n_kv_heads=2, page_size=16, head_dim=64,
                                                       batch=1, pages_per_seq=4), **k}))

    big = 1 << 30
    att = lambda c=None, **k: lib.sf_paged4_attention(c or cache(), *{**dict(q=F, qd=0, ts=512, hs=64, o=F, od=0, lse=None, H=8, T=1,
                                                                            s=1.0, w=0, ws=F, n=big, st=None), **k}.values())
    app = lambda c=None, **k: lib.sf_paged4_append(c or cache(), *{**dict(
        k=F, kt=128, kh=64, v=F, vt=128, vh=64, q=F, qt=512, qh=64, qo=F, dt=0, H=8, T=1, wq=None, wk=None, wt=0, eps=-1.0, pos=None,
        p64=0, an=1, ax=None, tb=F, mp=9, rot=64, inter=0, st=None), **k}.values())
    for call in (att, app):
        for c, want in ((dict(page_size=8), 6), (dict(page_size=48), 6), (dict(page_size=512), 6), (dict(head_dim=80), 6),
                        (dict(head_dim=32), 6), (dict(batch=0), 2), (dict(batch=5000), 6), (dict(num_pages=0), 2), (dict(n_kv_heads=0), 2),
                        (dict(pages_per_seq=0), 2), (dict(pages_per_seq=2 ** 27), 2), (dict(k_codes=F + 8), 4), (dict(k_scales=F + 8), 4),
                        (dict(v_scales=F + 2), 4), (dict(k_codes=None), 1), (dict(v_scales=None), 1), (dict(block_table=None), 1),
                        (dict(batch=2), 2)):
            assert call(cache(**c)) == want, c
        assert call(T=-1) == 2 and call(T=0) == 0
    for kw, want in ((dict(qd=5), 3), (dict(od=3), 3), (dict(H=7), 2), (dict(H=0), 2), (dict(q=None), 1), (dict(o=None), 1),
                     (dict(ws=None), 1), (dict(n=16), 2), (dict(ws=F + 4), 4)):
        assert att(**kw) == want, kw
    for kw, want in ((dict(dt=4), 3), (dict(wt=3), 3), (dict(rot=63), 2), (dict(rot=66), 2), (dict(mp=0), 2), (dict(k=None), 1),
                     (dict(qo=None), 1), (dict(H=0), 2), (dict(pos=F, an=0), 2), (dict(pos=F, an=2), 2), (dict(pos=F, an=9, ax=F), 2),
                     (dict(H=1 << 16), 6)):
        assert app(**kw) == want, kw


def test_sequences_near_31_bits_are_refused_without_gpu():
    import ctypes

    from siliconfer_b200 import _lib
    lib, F = _lib.load(), 0x1000
    for page in (16, 64, 256):
        for pages, want in ((2 ** 31 // page - 1024 // page, 0), (2 ** 31 // page - 1024 // page + 1, 2), (2 ** 31 // page, 2)):
            c = ctypes.byref(_lib.Paged4Cache(k_codes=F, k_scales=F, v_codes=F, v_scales=F, block_table=F, seq_lens=F, starts=None,
                                              num_pages=4, n_kv_heads=2, page_size=page, head_dim=64, batch=1, pages_per_seq=pages))
            assert lib.sf_paged4_attention(c, F, 0, 512, 64, F, 0, None, 8, 0, 1.0, 0, F, 1 << 30, None) == want


def test_cache_and_quantizer_without_gpu():
    from siliconfer_b200.paged_kv4 import Paged4KVCache, dequantize_kv4, quantize_kv4
    c = Paged4KVCache(3, 2, 64, 16, device="cpu")
    assert c.k_codes.shape == (3, 2, 16, 32) and c.v_scales.shape == (3, 2, 16, 4)
    assert (dequantize_kv4(c.k_codes, c.k_scales) == 0).all()
    x = torch.arange(-32, 32).double().view(1, 64)
    codes, scales = quantize_kv4(x)
    assert (dequantize_kv4(codes, scales).double() - x).abs().max() <= float(scales.max()) * (0.5 + 7.5 * 2.0 ** -8)
    assert torch.equal(dequantize_kv4(codes, scales).double(), value_of(codes, scales))
    with pytest.raises(RuntimeError):
        Paged4KVCache(3, 2, 66, 16, device="cpu")
    with pytest.raises(RuntimeError):
        quantize_kv4(torch.zeros(2, 6))


NEAR_TIE = (-6, 104, -45, -122, 125, 78, -4, 40, -38, 30, 92, 120, -12, 69, 5, 77, -20, 112, -24, 34, 34, -45, -36, -120, 16, 69,
            82, -86, -37, 64, 57, 23, -63, -106, 110, -98, -50, -109, -74, 79, -68, -102, -68, 38, 82, 35, -109, -100, -19, 36,
            -22, 86, 106, -122, 55, -120, -12, -58, -66, 115, 27, -126, -28, -22)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_append_eps_64_bits(cuda, dtype):
    """With eps of 1 + 2^-24, which fp32 rounds to 1, element 61 is -7.4999999 scales and its code 1; with 1 -7.5000001 and 0."""
    from siliconfer_b200.paged_kv4 import Paged4KVCache, quantize_kv4
    x = torch.tensor(NEAR_TIE, dtype=torch.float64) * 2.0 ** -9
    got = []
    for eps in (1 + 2.0 ** -24, 1.0):
        codes, scales = quantize_kv4(x / ((x * x).mean() + eps).sqrt())
        cache = Paged4KVCache(1, 1, 64, 16, device="cuda")
        k = x.to("cuda", dtype).view(1, 1, 64)
        cache.append(k, k, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                     torch.ones(1, dtype=torch.int32, device="cuda"), eps=eps)
        assert torch.equal(cache.k_scales[0, 0, 0].cpu().view(torch.int16), scales.view(torch.int16))
        assert torch.equal(cache.k_codes[0, 0, 0].cpu(), codes)
        got.append(codes)
    assert not torch.equal(*got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_append_eps_below_fp32(cuda, dtype):
    """Heads of zeros stay zeros with any positive eps, queries that are returned and keys that are cut to codes alike."""
    from siliconfer_b200.paged_kv4 import Paged4KVCache
    x = torch.zeros(3, 2, 64, device="cuda", dtype=dtype)
    pages = torch.arange(3, dtype=torch.int32, device="cuda").view(3, 1)
    for eps in (1e-40, 1e-60, 1e-300):
        cache = Paged4KVCache(3, 2, 64, 16, device="cuda")
        q = cache.append(x, x, pages, torch.ones(3, dtype=torch.int32, device="cuda"), q=x, eps=eps)
        assert not q.any() and (cache.k_codes == 0x88).all() and (cache.k_scales[:, :, 0] == 2.0 ** -126).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 800])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [18, 20, 22, 23, 24, 25, 26, 27, 30, 36, 44, 60])
def test_scores_whose_last_place_is_above_one(cuda, power, D, n):
    """Scores of 2^power and more, which fp32 holds to 2^-24: whichever keys a row picks, its weights add up to one.  All values
    are one vector, so that the result is it, off by 2^-11 of its fp16 form in prompts, as much of a weight and half a step."""
    from siliconfer_b200.paged_kv4 import paged4_attention
    for v_power in (0, -30, 40):
        b = Batch4([900, 130], [n, min(n, 100)], 32, 8, D, 16, torch.bfloat16)
        b.v[:] = b.v[0, 0, 0]
        b.vs[:] = b.vs[0, 0, 0] * 2.0 ** v_power
        for scale in (2.0 ** (power - 5), -(2.0 ** (power - 5))):
            out, lse = paged4_attention(b.q, *b.args(), starts=b.starts, scale=scale, return_lse=True)
            want = value_of(b.v[0, 0, 0], b.vs[0, 0, 0])
            assert ((out.double() - want).abs() <= (2 * 2.0 ** -11 + 3e-5 + 2.0 ** -8) * want.abs()).all()
            ref = b.ref(scale=scale)[1]
            # fp32's rounding of the sum and of its parts, and in prompts of the keys
            assert ((lse.double() - ref).abs() <= 4e-5 + 2e-6 * ref.abs() + 2.0 ** -11 * spread(b, scale=scale)[1]).all()


def check_elements(b, launches, window=0):
    """Each element against what its own row sees.  Scores are off by 2^-11 sum |q k| in prompts and weights and values by 2^-11
    of themselves (the head), fp32 sums by 6e-5 of the same; a weight below fp16's normal numbers by 2^-25, where the largest
    stands at 2^13 and a value at 2^15 at most, its vector's largest at 2^11 at least: 2^-34 for each of up to 900 keys."""
    from siliconfer_b200 import _lib
    from siliconfer_b200.paged_kv4 import paged4_attention
    before = _lib.launch_count()
    out, lse = paged4_attention(b.q, *b.args(), starts=b.starts, window=window, return_lse=True)
    assert _lib.launch_count() - before == launches
    ref, lref, _ = b.ref(window=window)
    moved, size = spread(b, window=window)
    bound = (1.02 * 2.0 ** -11 + 6e-5) * moved + 2.0 ** -24 * moved.amax(-1, keepdim=True) + OUT[b.dtype] * ref.abs() + 2.0 ** -25
    assert ((out.double() - ref).abs() <= bound).all()
    assert ((lse.double() - lref).abs() <= 4e-5 + 2e-6 * lref.abs() + 2.0 ** -11 * size).all()
    assert _lib.load().sf_q4_check_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 800])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 150])
@pytest.mark.parametrize("dtype,gap", [(torch.bfloat16, 16), (torch.bfloat16, 24), (torch.bfloat16, 40), (torch.bfloat16, 90),
                                       (torch.float16, 16)])
def test_large_scales_that_a_row_does_not_see_cannot_reach_it(cuda, dtype, gap, window, D, n):
    """Values or keys 2^gap above the others, of later tokens of the same call and of tokens before a row's window: whether a
    row's tokens share a tile with them does not matter."""
    for keys in (False, True):
        b = Batch4([900], [n], 32, 8, D, 16, dtype)
        s = b.ks if keys else b.vs
        if dtype == torch.float16:
            s *= 2.0 ** -8
        for at in (40, 190, 333, 640, 897):
            s[b.table[0, at // 16], :, at % 16] *= 2.0 ** gap
        check_elements(b, 1 if n == 800 else 2, window)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 800])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("apart", [12, 25, 40, 60])
def test_scales_far_apart(cuda, apart, D, n):
    """Between tokens, values and keys, zeros among them; up to 2^12 between the quarters of a vector, too."""
    b = Batch4([900, 700], [n, n // 2], 32, 8, D, 16, torch.bfloat16)
    power = lambda s, last: torch.exp2(torch.randint(-apart, 1, s.shape[:3] + (last,), generator=b.g, device="cuda")).bfloat16()
    vs, ks = b.vs.clone(), b.ks.clone()
    b.vs = vs * power(vs, 1)
    check_elements(b, 1 if n == 800 else 2)
    b.ks = ks * power(ks, 1)
    check_elements(b, 1 if n == 800 else 2)
    b.vs[:, :, ::5] = 0
    b.ks[:, :, ::7] = 0
    check_elements(b, 1 if n == 800 else 2)
    if apart == 12:
        b.vs, b.ks = vs * power(vs, 4), ks * power(ks, 4)
        check_elements(b, 1 if n == 800 else 2)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n", [20, 800])
@pytest.mark.parametrize("window", [0, 100])
def test_padding_rows_whose_queries_are_not_finite(cuda, window, n, bad):
    """Nine rows in front of their sequence's first token, in a tile with rows of tokens: they see nothing and are 0."""
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([n - 9, 700], [n, 100], 32, 8, 64, 16, torch.bfloat16)
    good, lse = paged4_attention(b.q, *b.args(), starts=b.starts, window=window, return_lse=True)
    b.q[:9, :, 3] = bad
    b.q[:9, 5] = bad
    out, l2 = paged4_attention(b.q, *b.args(), starts=b.starts, window=window, return_lse=True)
    assert (out[:9] == 0).all() and (l2[:9] == -math.inf).all()
    assert torch.equal(out, good) and torch.equal(l2, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 64), (64, 8, 128), (8, 8, 256), (4, 4, 96)])
def test_queries_with_two_large_elements(cuda, H, Hkv, D, dtype):
    """A hundred and fifty times the others, in each quarter.  A score's fp32 sums, some 32 of 2^-24 of sum |q k| each: 2^-19 of
    it; a weight's and the log-sum's error is the scores'."""
    from siliconfer_b200.paged_kv4 import paged4_attention
    for at in (3, D // 4 + 1, D // 2 + 5, 3 * D // 4 + 7):
        b = Batch4([700, 30, 1000], [1, 2, 1], H, Hkv, D, 16, dtype)
        b.q[..., at] *= 100
        b.q[..., at + 2] *= 50
        out, lse = paged4_attention(b.q, *b.args(), starts=b.starts, return_lse=True)
        ref, lref, _ = b.ref()
        moved, size = spread(b)
        off = 4e-5 + 2e-6 * lref.abs() + 2.0 ** -19 * size
        assert ((lse.double() - lref).abs() <= off).all()
        assert ((out.double() - ref).abs() <= (2 * off[..., None] + 2.0 ** -11) * moved + OUT[dtype] * ref.abs() + 2.0 ** -25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_keys_that_a_turn_takes_past_fp32(cuda, dtype):
    """3.3e38 (cos + sin) is a number in 64 bits and its scale one in bf16; an infinity beside such numbers stays one."""
    def values(k, v):
        for x in (k, v):
            x[:9] = (3.3e38 * x[:9].sign().float()).to(dtype)
            x[9] = (x[9].float() * 1.2e38).clamp(-3.3e38, 3.3e38).to(dtype)
            x[10, 0, 3:30] = 3.3e38
            x[13], x[13, 0, 1], x[13, 0, -3] = 0, 3.3e38, -3.3e38
            x[11, 1, 40], x[12, 0, 7] = float("inf"), float("nan")
            x[11, 1, 41:], x[12, 0, :5] = -3.3e38, 3.3e38
    for D in (64, 96, 128, 256):
        for kw in (dict(), dict(interleaved=True), dict(rot=D // 2), dict(rot=20)):
            check_append(Batch4([40, 30], [20, 5], 4, 2, D, 16, dtype), dtype, values=values, with_q=False, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 800])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [-57, -30, 60, 99])
def test_value_scales_at_the_ends_of_their_range(cuda, power, D, n):
    """From 2^-60 to 2^100, each element relative to its own row's values."""
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([900, 40], [n, 2], 32, 8, D, 16, torch.bfloat16)
    b.vs *= 2.0 ** power
    out, lse = paged4_attention(b.q, *b.args(), starts=b.starts, return_lse=True)
    ref, lref, _ = b.ref()
    moved, size = spread(b)
    bound = (1.02 * 2.0 ** -11 + 6e-5) * moved + 2.0 ** -24 * moved.amax(-1, keepdim=True) + 2.0 ** -8 * ref.abs()
    assert ((out.double() - ref).abs() <= bound).all()
    assert ((lse.double() - lref).abs() <= 4e-5 + 2e-6 * lref.abs() + 2.0 ** -11 * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 800])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_past_fp32_are_not_taken_for_numbers(cuda, D, n):
    """A key whose score passes fp32's range in the middle of a sequence: rows that it would win are NaN, the others hold."""
    from siliconfer_b200.paged_kv4 import paged4_attention
    b = Batch4([900], [n], 32, 8, D, 16, torch.bfloat16)
    b.q *= 2.0 ** 32
    good = paged4_attention(b.q, *b.args(), starts=b.starts)
    b.ks[b.table[0, 20], :, 13] = 2.0 ** 100          # token 333
    key = value_of(b.k[b.table[0, 20], :, 13], b.ks[b.table[0, 20], :, 13]).repeat_interleave(4, 0)
    score = torch.einsum("thd,hd->th", b.q.double(), key) * D ** -0.5
    sees = (torch.arange(900 - n, 900, device="cuda") >= 333)[:, None]
    out = paged4_attention(b.q, *b.args(), starts=b.starts)
    wins, others = sees & (score > 2.0 ** 129), ~sees | (score < -(2.0 ** 129))
    assert wins.any() and out[wins].isnan().all()
    assert others.any() and torch.isfinite(out[others]).all() and out[others].abs().max() <= 1.01 * good.abs().max()
