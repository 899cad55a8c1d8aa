"""Linear layers over e4m3 rows and weights, against the same product in 64 bits.

Bound.  Codes multiply exactly; a sum of 128 products of magnitude at most m
loses at most some 64 units of 2^-23 m in the tensor core's aligned adds, and
each of the K / 128 scaled partial sums adds one rounding:
|error| <= (64 + K / 32) 2^-23 sum |x w|, to which a 16-bit output adds half a
unit in its last place.
"""
import pytest
import torch

HALF_ULP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _codes(rows, K, g, pad=0):
    pitch = (K + 15) // 16 * 16 + pad
    store = torch.zeros(rows, pitch, dtype=torch.uint8, device="cuda")
    store[:, :K] = (torch.randn(rows, K, generator=g, device="cuda") * 80).clamp(-448, 448).to(torch.float8_e4m3fn).view(
        torch.uint8)
    # what a row's padding holds must not matter
    store[:, K:] = 0x7f
    return store.view(torch.float8_e4m3fn)[:, :K]


def _case(T, N, K, seed=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed + T + 7 * N + 31 * K)
    kb, nb = -(-K // 128), -(-N // 128)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")
    return (_codes(T, K, g, pad), rand(T, kb) * 0.02 + 1e-3, _codes(N, K, g, pad), rand(nb, kb) * 1e-3 + 1e-5,
            torch.randn(N, generator=g, device="cuda"))


def _ref(x, xs, w, ws, bias=None):
    K, N = x.shape[1], w.shape[0]
    xd = x.double() * xs.double().repeat_interleave(128, 1)[:, :K]
    wd = w.double() * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = xd @ wd.t()
    return (y if bias is None else y + bias.double()), xd.abs() @ wd.abs().t()


def _check(y, ref, mass, K, dtype, bias=None):
    bound = (64 + K / 32) * 2.0 ** -23 * mass + (HALF_ULP[dtype] + 2.0 ** -23) * ref.abs() + 1e-7
    if bias is not None:
        bound = bound + 2.0 ** -23 * bias.double().abs()
    assert y.dtype == dtype and y.shape == ref.shape
    assert ((y.double() - ref).abs() <= bound).all()


SHAPES = [(1, 128, 128), (1, 1, 1), (1, 4096, 4096), (2, 130, 16), (3, 896, 896), (5, 100, 100), (8, 128, 896),
          (16, 4864, 896), (17, 896, 4864), (31, 300, 1000), (33, 256, 257), (48, 1024, 1024), (64, 129, 4096),
          (65, 4096, 512), (100, 999, 1111), (128, 896, 896), (130, 11008, 640), (200, 896, 1408), (256, 4096, 4096),
          (257, 385, 2049), (511, 1000, 896), (1000, 4864, 896), (2048, 1024, 4096), (1, 28672, 1024), (1, 128, 28672)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", SHAPES)
def test_matches_fp64(cuda, T, N, K):
    from siliconfer_b200 import _lib
    from siliconfer_b200.fp8_linear import fp8_linear
    x, xs, w, ws, bias = _case(T, N, K)
    ref, mass = _ref(x, xs, w, ws)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        _check(fp8_linear(x, xs, w, ws, out_dtype=dtype), ref, mass, K, dtype)
    _check(fp8_linear(x, xs, w, ws, bias=bias), ref + bias.double(), mass, K, torch.float32, bias)
    assert _lib.load().sf_q4_check_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", [(1, 4096, 4096), (7, 300, 11008), (40, 640, 2048)])
def test_repeats_bit_for_bit(cuda, T, N, K):
    from siliconfer_b200.fp8_linear import fp8_linear
    x, xs, w, ws, _ = _case(T, N, K)
    first = fp8_linear(x, xs, w, ws)
    for _ in range(3):
        assert torch.equal(fp8_linear(x, xs, w, ws), first)


@pytest.mark.gpu
def test_strides_layouts_and_types(cuda):
    from siliconfer_b200.fp8_linear import fp8_linear
    x, xs, w, ws, _ = _case(40, 200, 300, pad=32)
    ref, mass = _ref(x, xs, w, ws)
    _check(fp8_linear(x, xs, w, ws), ref, mass, 300, torch.float32)
    # uint8 codes, leading dimensions, scales as a transposed view, every other row of a larger tensor
    u = x.as_strided(x.shape, x.stride()).view(torch.uint8)
    _check(fp8_linear(u, xs.t().contiguous().t(), w.view(torch.uint8), ws), ref, mass, 300, torch.float32)
    x3, s3 = x.contiguous()[:, :288].contiguous().view(4, 10, 288), xs.view(4, 10, -1)
    y = fp8_linear(x3, s3, w.contiguous()[:, :288].contiguous(), ws)
    r3, m3 = _ref(x3.reshape(40, 288), xs, w.contiguous()[:, :288], ws)
    assert y.shape == (4, 10, 200)
    _check(y.view(40, 200), r3, m3, 288, torch.float32)
    r2, m2 = _ref(x[::2], xs[::2], w, ws)
    _check(fp8_linear(x[::2], xs[::2], w, ws), r2, m2, 300, torch.float32)
    # a single row of any stride
    _check(fp8_linear(x[3:4], xs[3:4], w[:1], ws[:1]), ref[3:4, :1], mass[3:4, :1], 300, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20, 200])
def test_special_values_stay_in_their_row(cuda, T):
    """A NaN code or scale spoils its own token or output column only; zero scales give zeros."""
    from siliconfer_b200.fp8_linear import fp8_linear
    x, xs, w, ws, _ = _case(T, 300, 512)
    x = x.clone()
    w = w.clone()
    x.view(torch.uint8)[T // 2, 77] = 0x7f
    w.view(torch.uint8)[130, 5] = 0xff
    y = fp8_linear(x, xs, w, ws)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[T // 2] = True
    bad[:, 130] = True
    assert torch.equal(y.isnan(), bad)
    xs = xs.clone()
    xs[0] = 0
    y = fp8_linear(x, xs, w, ws)
    if T > 1:
        assert (y[0][torch.arange(300, device="cuda") != 130] == 0).all()


@pytest.mark.gpu
def test_module_with_norm_in_front(cuda):
    """rms_norm_e4m3 -> Fp8Linear gives the float path's result up to the two quantizations, whose steps are 2^-4."""
    from siliconfer_b200.fp8_linear import Fp8Linear, quantize_weight_e4m3
    from siliconfer_b200.norm import rms_norm, rms_norm_e4m3
    g = torch.Generator().manual_seed(5)
    w = torch.randn(300, 901, generator=g) * 0.02
    x = torch.randn(6, 901, generator=g).cuda().bfloat16()
    layer = Fp8Linear(w, bias=torch.ones(300), out_dtype=torch.float32)
    codes, scales = quantize_weight_e4m3(w)
    step = 2.0 ** -4 * w.abs() + 2.0 ** -10 * scales.repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :901]
    assert ((codes.float() * scales.repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :901] - w).abs()
            <= step * 1.0001).all()
    pair = rms_norm_e4m3(x)
    y = layer(pair)
    ref, mass = _ref(pair[0], pair[1], layer.codes[:, :901], layer.scales)
    _check(y, ref + 1, mass, 901, torch.float32, torch.ones(1, device="cuda"))
    normed = rms_norm(x, out_dtype=torch.float32)
    plain = layer(normed)
    assert torch.equal(plain, y)
    whole = normed.double() @ w.double().cuda().t() + 1
    assert (y.double() - whole).norm() <= 2 * 2.0 ** -4 * whole.norm()
    assert torch.equal(layer.to("cpu").to("cuda")(pair), y)


@pytest.mark.gpu
def test_empty_and_capture(cuda):
    from siliconfer_b200 import _lib
    from siliconfer_b200.fp8_linear import fp8_linear
    x, xs, w, ws, _ = _case(4, 256, 256)
    n0 = _lib.launch_count()
    assert fp8_linear(x[:0], xs[:0], w, ws).shape == (0, 256)
    assert fp8_linear(x, xs, w[:0], ws[:0]).shape == (4, 0)
    assert _lib.launch_count() == n0
    ref = fp8_linear(x, xs, w, ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fp8_linear(x, xs, w, ws)
    graph.replay()
    assert torch.equal(y, ref)


@pytest.mark.gpu
def test_refusals(cuda):
    from siliconfer_b200.fp8_linear import Fp8Linear, fp8_linear, quantize_weight_e4m3
    x, xs, w, ws, b = _case(4, 256, 256)
    for bad in (lambda: fp8_linear(x.cpu(), xs, w, ws), lambda: fp8_linear(x, xs.cpu(), w, ws),
                lambda: fp8_linear(x.float(), xs, w, ws), lambda: fp8_linear(x, xs.half(), w, ws),
                lambda: fp8_linear(x, xs[:, :1], w, ws), lambda: fp8_linear(x, xs, w, ws[:1]),
                lambda: fp8_linear(x, xs, w[:, :128], ws), lambda: fp8_linear(x, xs, w, ws, bias=b[:3]),
                lambda: fp8_linear(x, xs, w, ws, bias=b.half()), lambda: fp8_linear(x, xs, w, ws, out_dtype=torch.int32),
                lambda: fp8_linear(x, xs, w.t(), ws), lambda: quantize_weight_e4m3(torch.zeros(0, 4)),
                lambda: Fp8Linear(torch.zeros(4, 32))(torch.zeros(1, 31, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()
    odd = torch.zeros(4, 257, dtype=torch.uint8, device="cuda")
    with pytest.raises(RuntimeError, match="multiples of 16"):
        fp8_linear(odd, torch.ones(4, 3, device="cuda"), odd, torch.ones(1, 3, device="cuda"))
    with pytest.raises(RuntimeError, match="multiples of 16"):
        fp8_linear(odd[:, 1:], torch.ones(4, 2, device="cuda"), odd[:, 1:], torch.ones(1, 2, device="cuda"))


def test_validation_without_gpu():
    from siliconfer_b200 import _lib
    lib, F = _lib.load(), 0x1000
    call = lambda **k: lib.sf_fp8_linear(*{**dict(X=F, ldx=256, xs=F, W=F, ldw=256, ws=F, b=None, Y=F, ydt=0, T=1, N=8,
                                                  K=256, st=None), **k}.values())
    assert call(T=-1) == 2 and call(K=0) == 2 and call(ldx=240) == 2 and call(ldw=128) == 2
    assert call(ydt=3) == 3 and call(X=None) == 1 and call(ws=None) == 1
    assert call(X=0x1001) == 4 and call(ldx=257) == 4 and call(W=0x1008) == 4
    assert call(T=0) == 0 and call(N=0) == 0


def test_weight_quantizer_on_cpu():
    from siliconfer_b200.fp8_linear import quantize_weight_e4m3
    w = torch.randn(130, 257)
    w[:128, :128] = 0
    codes, scales = quantize_weight_e4m3(w)
    assert codes.shape == w.shape and codes.stride(0) % 16 == 0 and scales.shape == (2, 3)
    assert scales[0, 0] == 1 and (codes[:128, :128].float() == 0).all()
    assert torch.allclose(scales[1, 2], w[128:, 256:].abs().max() / 448)


@pytest.mark.gpu
def test_calls_of_different_sizes_from_two_threads(cuda):
    """A launch's shared memory hangs on its tokens; the calls of one thread leave the other's alone."""
    import threading

    from siliconfer_b200 import _lib
    lib, refused = _lib.load(), []

    def work(T):
        x, xs, w, ws, _ = _case(T, 256, 512, seed=T)
        ref = torch.empty(T, 256, device="cuda")
        y, stream = torch.zeros_like(ref), torch.cuda.Stream()
        torch.cuda.synchronize()
        for out, n in ((ref, 1), (y, 4000)):
            for _ in range(n):
                rc = lib.sf_fp8_linear(x.data_ptr(), x.stride(0), xs.data_ptr(), w.data_ptr(), w.stride(0), ws.data_ptr(), None,
                                       out.data_ptr(), 0, T, 256, 512, stream.cuda_stream)
                if rc:
                    refused.append((T, rc))
                    return
            stream.synchronize()
        if not torch.equal(y, ref):
            refused.append((T, "result"))

    threads = [threading.Thread(target=work, args=(T,)) for T in (16, 100)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not refused
