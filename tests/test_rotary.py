"""Rotary positions against complex products in 64 bits, from the same 32-bit table.

Bound: two products and a sum in fp32, |error| <= 2^-22 (|a| + |b|) of the pair times the table's largest value, to
which a 16-bit output adds half a unit in its last place.
"""
import math

import numpy as np
import pytest
import torch

HALF_ULP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def turned(x, pos, table, interleaved):
    """x [T, H, D] in 64 bits, and the bound's |a| + |b|."""
    x = x.double()
    rot = table.shape[1]
    half = rot // 2
    z = torch.complex(*table.double()[pos.long()].split(half, 1))[:, None]
    y, mass = x.clone(), x.abs()
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, half), slice(half, rot))
    v = torch.complex(x[..., i].contiguous(), x[..., j].contiguous()) * z
    y[..., i], y[..., j] = v.real, v.imag
    both = mass[..., i] + mass[..., j]
    mass[..., i], mass[..., j] = both, both
    return y, mass * max(1.0, float(table.abs().max()))


def check(y, ref, mass, dtype):
    assert y.dtype == dtype
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-30
    assert ((y.double() - ref).abs() <= 2.0 ** -22 * mass + HALF_ULP[dtype] * ref.abs() + tiny).all()


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 2, 2), (1, 32, 128, 128), (5, 14, 64, 64), (3, 8, 256, 64), (7, 3, 96, 48),
                                       (4, 5, 80, 20), (2, 3, 65, 64), (130, 64, 128, 128), (6, 2, 64, 8), (3, 2, 64, 0)])
def test_matches_fp64(cuda, T, H, D, rot, dtype, interleaved):
    from siliconfer_b200.rotary import apply_rotary, rotary_table
    g = torch.Generator().manual_seed(T + H + D + rot)
    x = torch.randn(T, H, D, generator=g).to(dtype).cuda()
    table = rotary_table(5000, rot) if rot else torch.empty(5000, 0, device="cuda")
    for pdt in (torch.int32, torch.int64):
        pos = torch.randint(0, 5000, (T,), generator=g).to(pdt).cuda()
        ref, mass = turned(x, pos, table, interleaved) if rot else (x.double(), x.double().abs())
        check(apply_rotary(x, pos, table, interleaved), ref, mass, dtype)
        y = x.clone()
        assert apply_rotary(y, pos, table, interleaved, out=y) is not None
        check(y, ref, mass, dtype)


@pytest.mark.gpu
def test_strides(cuda):
    """Slices of a fused projection, heads that do not start at 16 bytes, a transposed layout, one row for all."""
    from siliconfer_b200.rotary import apply_rotary, rotary_table
    table = rotary_table(100, 64)
    pos = torch.tensor([99, 0, 7, 50], device="cuda")
    wide = torch.randn(4, 1000, device="cuda", dtype=torch.bfloat16)
    for x in (wide[:, :640].view(4, 10, 64), wide[:, 3:643].view(4, 10, 64),
              torch.randn(10, 4, 64, device="cuda", dtype=torch.bfloat16).transpose(0, 1),
              torch.randn(4, 64, 10, device="cuda", dtype=torch.bfloat16).transpose(1, 2),
              torch.randn(1, 10, 64, device="cuda", dtype=torch.bfloat16).expand(4, 10, 64)):
        ref, mass = turned(x, pos, table, False)
        check(apply_rotary(x, pos, table), ref, mass, torch.bfloat16)
    out = torch.zeros(4, 1000, device="cuda", dtype=torch.bfloat16)
    ref, mass = turned(wide[:, :640].view(4, 10, 64), pos, table, True)
    apply_rotary(wide[:, :640].view(4, 10, 64), pos, table, True, out=out[:, 200:840].view(4, 10, 64))
    check(out[:, 200:840].view(4, 10, 64), ref, mass, torch.bfloat16)
    assert (out[:, :200] == 0).all() and (out[:, 840:] == 0).all()


@pytest.mark.gpu
def test_position_outside_the_table_is_reported(cuda):
    from siliconfer_b200 import _lib
    from siliconfer_b200.rotary import apply_rotary, rotary_table
    table = rotary_table(10, 32)
    x = torch.randn(3, 2, 64, device="cuda")
    y = apply_rotary(x, torch.tensor([0, 10, -1], device="cuda"), table)
    assert _lib.load().sf_q4_check_device_error() == 10
    assert _lib.load().sf_q4_check_device_error() == 0
    assert torch.isfinite(y[0]).all() and y[1:, :, :32].isnan().all() and torch.equal(y[1:, :, 32:], x[1:, :, 32:])


@pytest.mark.gpu
def test_refusals_and_empty(cuda):
    from siliconfer_b200.rotary import apply_rotary, rotary_table
    x, t, p = torch.randn(2, 3, 64, device="cuda"), rotary_table(10, 64), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: apply_rotary(x.cpu(), p, t), lambda: apply_rotary(x, p.cpu(), t), lambda: apply_rotary(x, p[:1], t),
                lambda: apply_rotary(x, p.float(), t), lambda: apply_rotary(x, p, t.half()),
                lambda: apply_rotary(x, p, rotary_table(10, 66)), lambda: apply_rotary(x[0], p, t),
                lambda: apply_rotary(x, p, t[:0]), lambda: apply_rotary(x, p, t, out=x[:1]),
                lambda: apply_rotary(x.expand(2, 3, 64)[:, :, :63], p, torch.zeros(10, 63, device="cuda")),
                lambda: apply_rotary(x, p, t, out=torch.empty(2, 64, 3, device="cuda").transpose(1, 2)),
                lambda: apply_rotary(x.double(), p, t)):
        with pytest.raises(RuntimeError):
            bad()
    assert apply_rotary(x[:0], p[:0], t).shape == (0, 3, 64)


def test_tables():
    from siliconfer_b200.rotary import rotary_frequencies, rotary_table
    t = rotary_table(1 << 17, 4, device="cpu")
    assert t.shape == (1 << 17, 4) and t.dtype == torch.float32
    p = (1 << 17) - 1
    want = [math.cos(p), math.cos(p * 0.01), math.sin(p), math.sin(p * 0.01)]
    assert np.allclose(t[p].numpy(), want, atol=1e-7, rtol=0)
    base, gain = rotary_frequencies(128)
    assert gain == 1 and np.allclose(base, 10000.0 ** (-np.arange(64) / 64))
    assert np.allclose(rotary_frequencies(128, scaling="linear", factor=4.0)[0], base / 4)
    ntk = rotary_frequencies(128, scaling="ntk", factor=4.0)[0]
    assert np.isclose(ntk[0], base[0]) and np.isclose(ntk[-1], base[-1] / 4)
    yarn, gain = rotary_frequencies(128, scaling="yarn", factor=8.0, original_max=4096)
    turns = 4096 * base / (2 * math.pi)
    assert np.isclose(gain, 0.1 * math.log(8) + 1)
    assert np.allclose(yarn[turns > 33], base[turns > 33]) and np.allclose(yarn[turns < 0.9], base[turns < 0.9] / 8)
    assert (yarn <= base * 1.0000001).all() and (yarn >= base / 8 * 0.9999999).all()
    assert np.allclose(rotary_table(3, 8, scaling="yarn", factor=2.0, device="cpu")[0, :4], 0.1 * math.log(2) + 1)
    for bad in (dict(rot=3), dict(rot=0), dict(rot=8, scaling="other"), dict(rot=8, scaling="linear", factor=0.5)):
        with pytest.raises(RuntimeError):
            rotary_frequencies(**bad)
    with pytest.raises(RuntimeError):
        rotary_table(0, 8)


def test_validation_without_gpu():
    from siliconfer_b200 import _lib
    lib, F = _lib.load(), 0x1000
    call = lambda **k: lib.sf_rotary(*{**dict(x=F, dt=0, xts=64, xhs=64, o=F, ots=64, ohs=64, p=F, p64=0, t=F, mp=8, rot=64,
                                              il=0, T=1, H=1, D=64, st=None), **k}.values())
    assert call(T=-1) == 2 and call(rot=63) == 2 and call(rot=66) == 2 and call(mp=0) == 2 and call(t=None) == 2
    assert call(dt=3) == 3 and call(x=None) == 1 and call(p=None) == 1 and call(T=0) == 0 and call(H=0) == 0
