"""RMS norm with the residual's addition, and e4m3 rows with a scale for every 128 columns, against 64-bit arithmetic.

Bounds.  fp32: the mean of K squares is off by a few 2^-24 (pairwise sums in
lanes and warps), the root, the product and the weight add one rounding each:
2e-6 of |y| leaves room for K in the tens of thousands.  A 16-bit output adds
half a unit in its last place: 2^-9 (bf16) or 2^-12 (fp16) of |y|, or 2^-25
below fp16's normal range.  e4m3: half a step is 2^-4 of the value, or
2^-10 of the scale below the smallest normal code.
"""
import numpy as np
import pytest
import torch

HALF_ULP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _inputs(T, K, dtype, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed + T * 31 + K)
    x = (torch.randn(T, K, generator=g) * torch.where(torch.rand(K, generator=g) < 0.02, 20.0, 1.0)).to(dtype).cuda()
    r = torch.randn(T, K, generator=g).to(dtype).cuda() if residual else None
    return x, r, (1 + 0.1 * torch.randn(K, generator=g)).to(dtype).cuda()


def _ref(x, r, w, eps=1e-6):
    h = x.double() + (0 if r is None else r.double())
    y = h / ((h ** 2).mean(-1, keepdim=True) + eps).sqrt()
    return h, y if w is None else y * w.double()


def _check_float(y, ref, dtype):
    bound = (2e-6 + HALF_ULP[dtype]) * ref.abs() + (2.0 ** -24 if dtype == torch.float16 else 1e-30)
    assert y.dtype == dtype
    assert (y.double() - ref).abs().le(bound).all()


def _check_codes(codes, scales, ref):
    T, K = ref.shape
    G = -(-K // 128)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == ref.shape and scales.shape == (T, G)
    amax = torch.nn.functional.pad(ref.abs(), (0, G * 128 - K)).view(T, G, 128).amax(2)
    want = torch.where(amax == 0, torch.ones_like(amax), amax / 448)
    assert ((scales.double() - want).abs() <= 4e-6 * want).all()
    s = scales.double().repeat_interleave(128, 1)[:, :K]
    err = (codes.double() * s - ref).abs()
    assert (err <= 2.0 ** -4 * 1.0001 * ref.abs() + 2.0 ** -10 * 1.0001 * s).all()


SHAPES = [(1, 1), (1, 7), (3, 127), (2, 128), (5, 129), (1, 896), (33, 896), (2, 1000), (4, 1024), (1, 4096), (7, 4097),
          (3, 4864), (65, 8192), (2, 8200), (1, 11008), (2, 28672), (1, 40001)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,K", SHAPES)
def test_norm_matches_fp64(cuda, T, K, dtype):
    from siliconfer_b200.norm import rms_norm, rms_norm_e4m3
    x, r, w = _inputs(T, K, dtype)
    for res in (None, r):
        h, ref = _ref(x, res, w)
        y = rms_norm(x, w, residual=res)
        if res is not None:
            y, h_out = y
            _check_float(h_out, h, dtype)
        _check_float(y, ref, dtype)
        out = rms_norm_e4m3(x, w, residual=res)
        _check_codes(out[0], out[1], ref)
        if res is not None:
            _check_float(out[2], h, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("x_dtype,w_dtype,out", [(torch.bfloat16, torch.float32, torch.float32),
                                                 (torch.float32, torch.bfloat16, torch.float16),
                                                 (torch.float16, torch.float16, torch.bfloat16)])
def test_norm_mixed_types_and_no_weight(cuda, x_dtype, w_dtype, out):
    from siliconfer_b200.norm import rms_norm
    x, _, w = _inputs(9, 1040, x_dtype, residual=False)
    _check_float(rms_norm(x, w.to(w_dtype), out_dtype=out), _ref(x, None, w.to(w_dtype))[1], out)
    _check_float(rms_norm(x, out_dtype=out), _ref(x, None, None)[1], out)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [896, 901])
def test_norm_strides_and_shapes(cuda, K):
    """Rows of a wider tensor, rows at odd offsets, a broadcast row, a transposed tensor and leading dimensions."""
    from siliconfer_b200.norm import quantize_e4m3, rms_norm, rms_norm_e4m3
    wide = torch.randn(6, 2 * K + 3, device="cuda", dtype=torch.bfloat16)
    w = torch.rand(K, device="cuda", dtype=torch.bfloat16) + 0.5
    views = [wide[:, :K], wide[:, 3:3 + K], wide[::2, 1:1 + K], wide[:1, :K].expand(4, K),
             torch.randn(K, 5, device="cuda", dtype=torch.bfloat16).t()]
    for x in views:
        r = torch.randn(x.shape, device="cuda", dtype=torch.bfloat16)
        h, ref = _ref(x, r, w)
        y, h_out = rms_norm(x, w, residual=r)
        _check_float(y, ref, torch.bfloat16)
        _check_float(h_out, h, torch.bfloat16)
        y, h_out = rms_norm(r, w, residual=x)
        _check_float(y, ref, torch.bfloat16)
        codes, scales = quantize_e4m3(x)
        _check_codes(codes, scales, x.double())
    x = torch.randn(2, 3, 4, K, device="cuda")
    codes, scales, h = rms_norm_e4m3(x, residual=x)
    assert codes.shape == x.shape and scales.shape == (2, 3, 4, -(-K // 128)) and h.shape == x.shape
    _check_codes(codes.reshape(24, K), scales.view(24, -1), _ref(x.view(24, K), x.view(24, K), None)[1])
    y, h = rms_norm(x[0, 0, 0], residual=x[0, 0, 1])
    _check_float(y, _ref(x[0, 0, 0], x[0, 0, 1], None)[1], torch.float32)


@pytest.mark.gpu
def test_norm_special_values(cuda):
    from siliconfer_b200.norm import quantize_e4m3, rms_norm, rms_norm_e4m3
    x = torch.randn(4, 300, device="cuda")
    x[0] = 0                      # a row of zeros: y = 0, scale 1
    x[1, 5] = float("nan")        # spoils its row
    codes, scales = rms_norm_e4m3(x)
    assert (codes[0].float() == 0).all() and (scales[0] == 1).all()
    assert rms_norm(x)[1].isnan().all() and (codes[1].float() * scales[1].repeat_interleave(128)[:300]).isnan().all()
    _check_codes(codes[2:], scales[2:], _ref(x[2:], None, None)[1])
    x[1] = torch.randn(300, device="cuda")
    x[1, 130] = float("inf")      # quantize: spoils its group of 128 only
    x[2, :128] = 1e-41            # subnormal group: the scale stays a normal number
    x[3, :128] = 3e38
    codes, scales = quantize_e4m3(x)
    value = codes.float() * scales.repeat_interleave(128, 1)[:, :300]
    assert value[1, 128:256].isnan().all()
    _check_codes(codes[1:2, :128], scales[1:2, :1], x[1:2, :128].double())
    _check_codes(codes[1:2, 256:], scales[1:2, 2:], x[1:2, 256:].double())
    assert (scales >= 2.0 ** -126).all() and (value[2, :128].abs() <= 2.0 ** -126 * 2.0 ** -9).all()
    assert ((value[3, :128] / 3e38 - 1).abs() < 1e-5).all()


@pytest.mark.gpu
def test_norm_empty_in_place_residual_and_streams(cuda):
    from siliconfer_b200 import _lib
    from siliconfer_b200.norm import quantize_e4m3, rms_norm
    n0 = _lib.launch_count()
    y, h = rms_norm(torch.empty(0, 64, device="cuda"), residual=torch.empty(0, 64, device="cuda"))
    assert y.shape == h.shape == (0, 64) and quantize_e4m3(torch.empty(0, 64, device="cuda"))[0].shape == (0, 64)
    assert _lib.launch_count() == n0
    # the C entry may write h over the residual
    x, r, w = _inputs(5, 512, torch.bfloat16)
    h_ref, ref = _ref(x, r, w)
    y = torch.empty_like(x)
    _lib.check(_lib.load().sf_rms_norm(x.data_ptr(), 2, 512, r.data_ptr(), 512, r.data_ptr(), w.data_ptr(), 2, 1e-6,
                                       y.data_ptr(), 2, 512, None, 5, 512, torch.cuda.current_stream().cuda_stream))
    _check_float(r, h_ref, torch.bfloat16)
    _check_float(y, ref, torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = rms_norm(x, w)
    s.synchronize()
    _check_float(y, _ref(x, None, w)[1], torch.bfloat16)


@pytest.mark.gpu
def test_norm_refusals(cuda):
    from siliconfer_b200.norm import quantize_e4m3, rms_norm
    x = torch.zeros(2, 64, device="cuda")
    for bad in (lambda: rms_norm(x.cpu()), lambda: rms_norm(x.double()), lambda: rms_norm(x, torch.ones(63, device="cuda")),
                lambda: rms_norm(x, torch.ones(64)), lambda: rms_norm(x, residual=x[:1]),
                lambda: rms_norm(x, residual=x.half()), lambda: rms_norm(x[:, :0]), lambda: quantize_e4m3(x.cpu()),
                lambda: rms_norm(x, torch.ones(64, device="cuda", dtype=torch.int32)),
                lambda: rms_norm(x, out_dtype=torch.float64)):
        with pytest.raises(RuntimeError):
            bad()


def test_norm_validation_without_gpu():
    from siliconfer_b200 import _lib
    lib, F = _lib.load(), 0x1000
    call = lambda **k: lib.sf_rms_norm(*{**dict(x=F, xdt=0, ldx=64, r=None, ldr=64, h=None, w=None, wdt=0, eps=1e-6, y=F,
                                                ydt=0, ldy=64, s=None, T=1, K=64, st=None), **k}.values())
    assert call(T=-1) == 2 and call(K=0) == 2 and call(ldx=63) == 2 and call(ldy=63) == 2 and call(r=F, h=F, ldr=3) == 2
    assert call(xdt=3) == 3 and call(ydt=4) == 3 and call(w=F, wdt=9) == 3
    assert call(x=None) == 1 and call(r=F) == 1 and call(h=F) == 1 and call(ydt=3) == 1
    assert call(T=0, x=None) == 0
    q = lambda **k: lib.sf_quantize_e4m3(*{**dict(x=F, xdt=0, ldx=64, y=F, ldy=64, s=F, T=1, K=64, st=None), **k}.values())
    assert q(K=0) == 2 and q(xdt=3) == 3 and q(s=None) == 1 and q(ldy=1) == 2 and q(T=0) == 0


def _check_quotients(codes, scales, y):
    """Scales that are max|y| / 448 rounded once, and codes that are y / scale rounded to fp32 and to e4m3: no bound."""
    T, K = y.shape
    G = -(-K // 128)
    amax = torch.nn.functional.pad(y.abs(), (0, G * 128 - K)).view(T, G, 128).amax(2)
    want = torch.where(amax == 0, torch.ones_like(amax), (amax.double() / 448).float().clamp_min(2.0 ** -126))
    assert torch.equal(scales, want)
    q = (y.double() / scales.double().repeat_interleave(128, 1)[:, :K]).float()
    assert torch.equal(codes.float(), q.clamp(-448, 448).to(torch.float8_e4m3fn).float())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,K", [(1, 4096), (600, 1024), (333, 901), (40, 20000)])
def test_scales_and_codes_are_rounded_quotients(cuda, T, K, dtype):
    from siliconfer_b200.norm import quantize_e4m3, rms_norm, rms_norm_e4m3
    x, r, w = _inputs(T, K, dtype, seed=5)
    _check_quotients(*quantize_e4m3(x), x.float())
    for res in (None, r):
        y = rms_norm(x, w, residual=res, out_dtype=torch.float32)
        _check_quotients(*rms_norm_e4m3(x, w, residual=res)[:2], y if res is None else y[0])


@pytest.mark.gpu
def test_codes_at_ties(cuda):
    """All midpoints of two codes and their neighbours in fp32, under scales that divide them exactly and that do not."""
    from siliconfer_b200.norm import quantize_e4m3
    codes = torch.arange(0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = torch.nn.functional.pad((codes[1:] + codes[:-1]) / 2, (0, 1), value=448.0)    # 126 of them, and 448
    rows = torch.stack([torch.nextafter(mid, mid * 0 + d) for d in (0.0, 1e9)] + [mid, -mid])
    rows[:, -1] = 448
    rows = torch.cat([rows * f for f in (1.0, 3.0, 7.0, 1.1, 0.3, 2.0 ** -100, 2.0 ** 100)]).cuda()
    _check_quotients(*quantize_e4m3(rows), rows)
