"""Norms and rotary positions of query and key heads, against the formulas in 64 bits.

Bound.  An element's fp32 path, in units of 2^-24: a lane adds 16 squares and five sums over lanes follow, at most 21 of the
sum, which the root halves; the division by D and eps add 1 after it, the reciprocal root 4 (2 last places of 2^-23), two
products 2; a turn's product and sum 2 of |a cos| + |b sin|: 20 in all, 24 asked.  A 16-bit output adds half a step: 2^-8
(bf16) or 2^-11 (fp16) of itself, and half an fp16 subnormal step, 2^-25.
"""
import pytest
import torch

from siliconfer_b200.rotary import qk_norm_rotary

STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(x, weight, eps, positions, table, interleaved, axes):
    """(the result, |a cos| + |b sin|) in 64 bits; x [T, heads, D]."""
    y = x.double()
    if eps is not None:
        y = y / ((y * y).mean(-1, keepdim=True) + eps).sqrt()
        y = y if weight is None else y * weight.double()
    mass = y.abs()
    if table is not None:
        half = table.shape[1] // 2
        at = positions.long().view(len(x), -1)
        at = at[:, axes.long()] if axes is not None else at.expand(-1, half)
        j = torch.arange(half, device=x.device)
        c, s = table.double()[at, j][:, None], table.double()[at, half + j][:, None]
        lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
        a, b = y[..., lo], y[..., hi]
        z, m = y.clone(), mass.clone()
        z[..., lo], z[..., hi] = a * c - b * s, a * s + b * c
        m[..., lo], m[..., hi] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
        y, mass = z, m
    return y, mass


def near(got, want, mass, dtype):
    bound = 24 * 2.0 ** -24 * mass
    if dtype != torch.float32:
        bound = bound + STEP[dtype] * (want.abs() + bound) + 2.0 ** -25
    return ((got.double() - want).abs() <= bound + 1e-37).all()


def case(T, H, Hkv, D, dtype, axes=1, seed=0, max_pos=500, rot=None, pos64=False, weights=torch.float32):
    from siliconfer_b200.rotary import rotary_axes, rotary_table
    g = torch.Generator(device="cuda").manual_seed(seed + T + D)
    x = torch.randn(T, H + 2 * Hkv, D, generator=g, device="cuda").to(dtype)
    rot = D if rot is None else rot
    pos = torch.randint(0, max_pos, (T, axes), generator=g, device="cuda", dtype=torch.int64 if pos64 else torch.int32)
    sections = [rot // 2 - (axes - 1) * (rot // 2 // axes)] + [rot // 2 // axes] * (axes - 1)
    w = [(1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(weights) for _ in range(2)]
    return dict(q=x[:, :H], k=x[:, H:H + Hkv], positions=pos if axes > 1 else pos[:, 0], table=rotary_table(max_pos, rot),
                q_weight=w[0], k_weight=w[1]), rotary_axes(sections, interleaved=True) if axes > 1 else None


def check(c, axes, eps=1e-6, interleaved=False):
    from siliconfer_b200 import _lib
    from siliconfer_b200.rotary import qk_norm_rotary
    if eps is None:
        c = {**c, "q_weight": None, "k_weight": None}
    q, k = qk_norm_rotary(**c, eps=eps, interleaved=interleaved, axes=axes)
    dtype = c["q"].dtype
    for got, x, w in ((q, c["q"], c["q_weight"]), (k, c["k"], c["k_weight"])):
        if x is None:
            assert got is None
            continue
        assert got.dtype == dtype and got.shape == x.shape and got.is_contiguous()
        want, mass = reference(x, w, eps, c["positions"], c["table"], interleaved, axes)
        assert near(got, want, mass, dtype)
    assert _lib.load().sf_q4_check_device_error() == 0
    return q, k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,D", [(14, 2, 64), (1, 1, 128), (64, 8, 128), (3, 5, 96), (8, 1, 256), (16, 16, 80), (5, 2, 72),
                                     (2, 1, 36), (7, 3, 4), (4, 2, 512), (33, 1, 112), (2, 2, 248)])
def test_heads(cuda, H, Hkv, D, dtype):
    for T, axes, inter, eps in ((1, 1, False, 1e-6), (5, 3, False, 1e-5), (2, 1, True, None), (130, 2, True, 1e-6), (3, 1, False, None)):
        c, ax = case(T, H, Hkv, D, dtype, min(axes, D // 2), pos64=T == 5, weights=dtype if T == 1 else torch.float32)
        check(c, ax, eps, inter)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 32), (128, 64), (128, 32), (128, 2), (96, 72), (96, 20), (80, 40), (72, 36), (256, 64), (36, 10)])
def test_part_of_a_head(cuda, D, rot, interleaved):
    for dtype in (torch.bfloat16, torch.float32):
        for axes in (1, min(3, rot // 2)):
            c, ax = case(37, 6, 2, D, dtype, axes, rot=rot)
            check(c, ax, interleaved=interleaved)
            check(c, ax, eps=None, interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 7, 300, 2500])
def test_many_tokens_and_head_counts(cuda, T):
    for H, Hkv in ((1, 0), (0, 3), (128, 8), (200, 1), (20, 20)):
        c, ax = case(T, H, max(Hkv, 1), 128, torch.bfloat16, 3)
        if Hkv == 0:
            c["k"], c["k_weight"] = None, None
        check(c, ax)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_offsets_and_place(cuda, dtype):
    """Rows of any stride, starts that are no multiple of a wide load, heads of transposed tensors, and x as its own output."""
    from siliconfer_b200.rotary import apply_rotary
    c, ax = case(9, 6, 2, 64, dtype, 3)
    first = check(c, ax)
    for off in (0, 1, 2, 3, 65):
        wide = torch.zeros(9, 8 * 64 + 67, device="cuda", dtype=dtype)
        wide[:, off:off + 8 * 64] = torch.cat([c["q"], c["k"]], 1).reshape(9, -1)
        x = wide[:, off:off + 8 * 64].view(9, 8, 64)
        got = check({**c, "q": x[:, :6], "k": x[:, 6:]}, ax)
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    flipped = {**c, "q": c["q"].transpose(0, 1).contiguous().transpose(0, 1), "k": c["k"].transpose(1, 2).contiguous().transpose(1, 2)}
    assert all(torch.equal(a, b) for a, b in zip(check(flipped, ax), first))
    for inter in (False, True):
        for table in (c["table"], c["table"][:, :20].contiguous()):
            x, axes = c["q"].clone(), ax[:table.shape[1] // 2]
            want = apply_rotary(x, c["positions"], table, inter, axes=axes)
            ref, mass = reference(x, None, None, c["positions"], table, inter, axes)
            assert near(want, ref, mass, dtype)
            y = apply_rotary(x, c["positions"], table, inter, out=x, axes=axes)
            assert y.data_ptr() == x.data_ptr() and torch.equal(x, want)


@pytest.mark.gpu
def test_one_axis_is_the_rotary_of_before(cuda):
    """Alike within the roundings of two ways to the same products."""
    from siliconfer_b200.rotary import apply_rotary, rotary_axes
    c, _ = case(40, 6, 2, 128, torch.float32)
    axes = rotary_axes([64])
    for inter in (False, True):
        a = apply_rotary(c["q"], c["positions"], c["table"], inter)
        b = apply_rotary(c["q"], c["positions"], c["table"], inter, axes=axes)
        assert (a - b).abs().max() <= 4 * 2.0 ** -24 * c["q"].abs().max() * 2


@pytest.mark.gpu
def test_values_at_the_ends(cuda):
    """Zero heads, heads of tiny and of large values, infinities and NaN keep to their heads."""
    from siliconfer_b200.rotary import qk_norm_rotary
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        c, ax = case(6, 4, 2, 64, dtype, 2)
        q = c["q"] = c["q"].clone()
        q[0, 0] = 0
        q[1, 1] *= 1e-3
        q[2, 2] = (q[2, 2].float() * 3e4).clamp(-6e4, 6e4).to(dtype)
        q[3, 3, 5] = 1000
        check(c, ax)
        q[4, 0, 3], q[5, 1, 60], q[5, 2, 0] = float("nan"), float("inf"), float("-inf")
        got, k = qk_norm_rotary(**c, axes=ax)
        bad = torch.zeros(6, 4, dtype=torch.bool, device="cuda")
        bad[4, 0] = bad[5, 1] = bad[5, 2] = True
        assert torch.isfinite(got[~bad]).all() and torch.isfinite(k).all()
        assert got.isnan().any(-1).eq(bad).all()


@pytest.mark.gpu
def test_positions_and_axes_outside_are_reported(cuda):
    from siliconfer_b200 import _lib
    from siliconfer_b200.rotary import qk_norm_rotary
    lib = _lib.load()
    c, ax = case(5, 4, 2, 64, torch.bfloat16, 2, pos64=True)
    good = check(c, ax)
    for bad in (500, -1, 2 ** 40):
        pos = c["positions"].clone()
        pos[2, 1] = bad
        got = qk_norm_rotary(**{**c, "positions": pos}, axes=ax)
        torch.cuda.synchronize()
        assert lib.sf_q4_check_device_error() == 10 and lib.sf_q4_check_device_error() == 0
        rows = torch.arange(5, device="cuda") != 2
        hit = torch.cat([ax == 1, ax == 1])
        for a, b in zip(got, good):
            assert torch.equal(a[rows], b[rows]) and a[2][:, hit].isnan().all() and torch.equal(a[2][:, ~hit], b[2][:, ~hit])
    axes = ax.clone()
    axes[3] = 2
    got = qk_norm_rotary(**c, axes=axes)
    torch.cuda.synchronize()
    assert lib.sf_q4_check_device_error() == 10
    assert got[0][:, :, 3].isnan().all() and got[0][:, :, 35].isnan().all() and torch.equal(got[0][:, :, 4:32], good[0][:, :, 4:32])


@pytest.mark.gpu
def test_streams_and_capture(cuda):
    from siliconfer_b200.rotary import qk_norm_rotary
    c, ax = case(50, 14, 2, 64, torch.bfloat16, 3)
    want = check(c, ax)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(qk_norm_rotary(**c, axes=ax))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qk_norm_rotary(**c, axes=ax)
    for seed in (1, 2):
        new, _ = case(50, 14, 2, 64, torch.bfloat16, 3, seed=seed)
        c["q"].copy_(new["q"]), c["k"].copy_(new["k"]), c["positions"].copy_(new["positions"])
        graph.replay()
        torch.cuda.synchronize()
        for got, x, w in zip(out, (c["q"], c["k"]), (c["q_weight"], c["k_weight"])):
            ref, mass = reference(x, w, 1e-6, c["positions"], c["table"], False, ax)
            assert near(got, ref, mass, torch.bfloat16)


@pytest.mark.gpu
def test_no_rows_no_gradient(cuda):
    from siliconfer_b200 import _lib
    from siliconfer_b200.rotary import qk_norm_rotary
    c, ax = case(4, 3, 2, 64, torch.float32, 2)
    before = _lib.launch_count()
    q, k = qk_norm_rotary(c["q"][:0], c["k"][:0], c["positions"][:0], c["table"], axes=ax)
    assert q.shape == (0, 3, 64) and k.shape == (0, 2, 64) and _lib.launch_count() == before
    q, _ = qk_norm_rotary(c["q"].clone().requires_grad_(), None, c["positions"], c["table"], axes=ax)
    assert not q.requires_grad


@pytest.mark.gpu
def test_refusals(cuda):
    from siliconfer_b200.rotary import apply_rotary, qk_norm_rotary
    c, ax = case(4, 3, 2, 64, torch.float32, 2)
    run = lambda **kw: qk_norm_rotary(**{**c, "axes": ax, **kw})
    for bad in (dict(q=c["q"].cpu()), dict(q=c["q"][0]), dict(q=c["q"].double()), dict(k=c["k"].half()), dict(k=c["k"][:3]),
                dict(k=c["k"][..., :32]), dict(positions=c["positions"][:3]), dict(positions=c["positions"].float()),
                dict(positions=None), dict(axes=None), dict(axes=ax[:5]), dict(axes=ax.int()), dict(axes=ax.cpu()),
                dict(table=c["table"].half()), dict(table=torch.zeros(10, 66, device="cuda")), dict(table=c["table"][:0]),
                dict(table=None), dict(q_weight=c["q_weight"][:3]), dict(k_weight=c["k_weight"].bfloat16()), dict(eps=-1.0),
                dict(eps=float("nan")), dict(eps=None), dict(positions=torch.zeros(4, 9, device="cuda", dtype=torch.int32)),
                dict(q=torch.zeros(4, 3, 66, device="cuda"), k=None, q_weight=None, k_weight=None)):
        with pytest.raises(RuntimeError):
            run(**bad)
    with pytest.raises(RuntimeError):
        apply_rotary(c["q"], c["positions"], c["table"], out=c["q"][:, :2], axes=ax)


def test_axes_of_sections():
    from siliconfer_b200.rotary import rotary_axes
    assert rotary_axes((2, 3, 1)).tolist() == [0, 0, 1, 1, 1, 2]
    assert rotary_axes((4, 2, 2), interleaved=True).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert rotary_axes((0, 2), interleaved=True).tolist() == [1, 1]
    assert rotary_axes((16, 24, 24)).dtype == torch.uint8
    for bad in ((), (0,), (-1, 2), (1,) * 9):
        with pytest.raises(RuntimeError):
            rotary_axes(bad)


def test_validation_without_gpu():
    from siliconfer_b200 import _lib
    lib, F = _lib.load(), 0x1000
    base = dict(q=F, qts=64, qhs=64, qo=F, qots=64, qohs=64, H=1, k=F, kts=64, khs=64, ko=F, kots=64, kohs=64, Hkv=1, dt=0, wq=None,
                wk=None, wt=0, eps=1e-6, pos=F, p64=0, an=1, ax=None, table=F, mp=8, rot=64, inter=0, T=1, D=64, st=None)
    call = lambda **k: lib.sf_qk_norm_rotary(*{**base, **k}.values())
    for kw, want in ((dict(T=-1), 2), (dict(H=-1), 2), (dict(D=66), 6), (dict(D=132), 6), (dict(D=528), 6), (dict(D=264), 6), (dict(D=0), 6),
                     (dict(dt=3), 3), (dict(wt=7), 3), (dict(rot=65), 2), (dict(rot=66), 2), (dict(table=None), 2), (dict(mp=0), 2),
                     (dict(an=9), 2), (dict(an=0), 2), (dict(an=2), 2), (dict(q=None), 1), (dict(ko=None), 1), (dict(pos=None), 1),
                     (dict(H=1 << 17), 6), (dict(T=0), 0), (dict(H=0, Hkv=0), 0)):
        assert call(**kw) == want, kw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_eps_below_fp32(cuda, dtype):
    """A vector of zeros stays one with any positive eps, those that fp32 has no number for among them."""
    x = torch.zeros(3, 2, 64, device="cuda", dtype=dtype)
    for eps in (1e-40, 1e-60, 1e-300):
        q, k = qk_norm_rotary(x, x[:, :1], eps=eps)
        assert not q.any() and not k.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_sequences(cuda, dtype):
    """With the sequences' lengths: tokens as without them, rows that hold none as at position 0, packed rows or not."""
    from siliconfer_b200 import _lib
    lib = _lib.load()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for axes, lens, starts, real in ((1, ints(9, 0, 2), ints(3, 7, 9, 12), [*range(3, 7), 10, 11]), (3, ints(9, 1, 2, 40, 5), None, [*range(0, 3), 5, 7, 8, *range(9, 15)]),
                                     (2, torch.full((15,), 7, dtype=torch.int32, device="cuda"), None, list(range(15)))):
        c, ax = case(15, 6, 2, 64, dtype, axes)
        want = check(c, ax)
        zero = qk_norm_rotary(**{**c, "positions": torch.zeros_like(c["positions"])}, axes=ax)
        rest = torch.ones(15, dtype=torch.bool, device="cuda")
        rest[real] = False
        c["positions"][rest] = 10 ** 6
        got = qk_norm_rotary(**c, axes=ax, seq_lens=lens, starts=starts)
        assert lib.sf_q4_check_device_error() == 0
        for a, b, z in zip(got, want, zero):
            assert torch.equal(a[~rest], b[~rest]) and torch.equal(a[rest], z[rest])
        if starts is None:
            lens[0] = -1
        else:
            starts[0] = 20
        got = qk_norm_rotary(**{**c, "positions": torch.zeros_like(c["positions"])}, axes=ax, seq_lens=lens, starts=starts)
        torch.cuda.synchronize()
        assert lib.sf_q4_check_device_error() == 10 and all(torch.equal(a, z) for a, z in zip(got, zero))
    run = lambda **kw: qk_norm_rotary(**{**c, **kw}, axes=ax)
    for bad in (dict(starts=ints(0, 15)), dict(seq_lens=ints(1, 2)), dict(seq_lens=ints(5).long()), dict(seq_lens=ints(5).cpu()),
                dict(seq_lens=ints(5).view(1, 1)), dict(seq_lens=ints(5), starts=ints(0, 5, 15)), dict(seq_lens=ints()),
                dict(seq_lens=ints(5), starts=ints(0, 15).long())):
        with pytest.raises(RuntimeError):
            run(**bad)


def test_validation_of_rows_without_gpu():
    from siliconfer_b200 import _lib
    lib, F = _lib.load(), 0x1000
    base = dict(q=F, qts=64, qhs=64, qo=F, qots=64, qohs=64, H=1, k=F, kts=64, khs=64, ko=F, kots=64, kohs=64, Hkv=1, dt=0, wq=None,
                wk=None, wt=0, eps=1e-6, pos=F, p64=0, an=1, ax=None, table=F, mp=8, rot=64, inter=0, T=3, D=64, lens=F, starts=None, n=1,
                st=None)
    call = lambda **k: lib.sf_qk_norm_rotary_rows(*{**base, **k}.values())
    for kw, want in ((dict(n=0), 2), (dict(n=2), 2), (dict(lens=None, starts=F), 1), (dict(T=-1), 2), (dict(pos=None), 1), (dict(T=0), 0)):
        assert call(**kw) == want, kw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_head_of_any_stride(cuda, dtype):
    """Where there is one head nothing steps from it to the next."""
    from siliconfer_b200.paged_kv4 import Paged4KVCache
    x = torch.randn(4, 1, 64, device="cuda").to(dtype)
    far = x.as_strided((4, 1, 64), (64, 2 ** 31 + 67, 1))
    assert far.stride(1) > 2 ** 31
    for a, b in zip(qk_norm_rotary(x, x), qk_norm_rotary(far, far)):
        assert torch.equal(a, b)
    held = []
    for y in (x, far):
        cache = Paged4KVCache(4, 1, 64, 16)
        q = cache.append(y, y, torch.arange(4, dtype=torch.int32, device="cuda").view(4, 1),
                         torch.ones(4, dtype=torch.int32, device="cuda"), q=y, eps=1e-6)
        held.append((q, cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales))
    assert all(torch.equal(a, b) for a, b in zip(*held))


def test_head_strides_past_31_bits_are_refused_without_gpu():
    from siliconfer_b200 import _lib
    lib, F, far = _lib.load(), 0x1000, 1 << 31
    base = dict(q=F, qts=64, qhs=64, qo=F, qots=64, qohs=64, H=2, k=F, kts=64, khs=64, ko=F, kots=64, kohs=64, Hkv=2, dt=0, wq=None,
                wk=None, wt=0, eps=1e-6, pos=F, p64=0, an=1, ax=None, table=F, mp=8, rot=64, inter=0, T=1, D=64, st=None)
    for kw in (dict(qhs=far), dict(qohs=far), dict(khs=far), dict(kohs=far)):
        assert lib.sf_qk_norm_rotary(*{**base, **kw}.values()) == 6, kw
