"""Rotary positions: refusals of the C entry on CPU, values on the GPU against 64-bit rotations.

Tolerance: sine and cosine of a reduced angle (fp32 fraction of a turn: 2 pi 2^-25; sincospif 2
steps; the factor 1 step) <= 2^-21 absolute for factors up to 2, two products and a sum 2 u each,
so 2^-20 (|a| + |b|) on either element of a pair, and half a step of the output type.
"""

import ctypes
import math

import pytest
import torch

import memt_b200 as M
from memt_b200 import _lib

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _args(**over):
    f = dict(num_heads=2, num_key_heads=1, head_dim=64, rotary_dim=32, dtype=_lib.MEMT_BF16, total_tokens=0, q=16,
             q_stride=128, k=16, k_stride=64, q_out=16, q_out_stride=128, k_out=16, k_out_stride=64, positions=16,
             inv_freq=16, attention_scale=1.0)
    f.update(over)
    return _lib.RotaryArgs(**f)


@pytest.mark.parametrize("over", [
    dict(struct_size=4), dict(num_heads=0), dict(num_key_heads=-1), dict(rotary_dim=0), dict(rotary_dim=31),
    dict(rotary_dim=66), dict(dtype=3), dict(total_tokens=-1), dict(q=None), dict(q_out=None), dict(positions=None),
    dict(inv_freq=None), dict(q_stride=100), dict(k_stride=32), dict(k_out=None), dict(k_out_stride=1)])
def test_rotary_refuses(over):
    a = _args(**over)
    assert _lib.load().memt_rotary(ctypes.byref(a), None) == _lib.MEMT_ERR_INVALID_ARGUMENT


def test_empty_rotary_launches_nothing():
    lib = _lib.load()
    assert lib.memt_rotary(None, None) == _lib.MEMT_ERR_INVALID_ARGUMENT
    assert lib.memt_rotary(ctypes.byref(_args()), None) == _lib.MEMT_OK
    assert lib.memt_rotary(ctypes.byref(_args(num_key_heads=0, k=None, k_out=None)), None) == _lib.MEMT_OK


def test_frequencies():
    inv, scale = M.rotary_frequencies(8, 100.0, device="cpu")
    assert inv.dtype == torch.float64 and scale == 1.0
    assert torch.allclose(inv, torch.tensor([100.0 ** (-i / 4) for i in range(4)], dtype=torch.float64), rtol=1e-14)
    linear, _ = M.rotary_frequencies(8, 100.0, scaling="linear", factor=4.0, device="cpu")
    assert torch.allclose(linear, inv / 4, rtol=1e-14)
    ntk, _ = M.rotary_frequencies(8, 100.0, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(inv[-1]) / 4, rel_tol=1e-12)
    yarn, att = M.rotary_frequencies(64, scaling="yarn", factor=8.0, trained_tokens=4096, device="cpu")
    plain, _ = M.rotary_frequencies(64, device="cpu")
    assert yarn[0] == plain[0] and math.isclose(float(yarn[-1]), float(plain[-1]) / 8, rel_tol=1e-12)
    assert math.isclose(att, 0.1 * math.log(8) + 1) and bool((yarn <= plain).all())
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, base=0.5), dict(rotary_dim=8, factor=0.5),
                dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, scaling="yarn")):
        with pytest.raises(ValueError):
            M.rotary_frequencies(**bad, device="cpu")


def test_rotary_refuses_host_tensors():
    x = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError):
        M.rotary(x, x, torch.arange(3), torch.ones(4, dtype=torch.float64))


def _reference(x, pos, inv, interleaved, inverse, scale):
    """fp64 rotation and the elementwise |a| + |b| of each pair (the bound's scale)."""
    n = inv.numel()
    x = x.double().cpu()
    ang = pos.double().cpu()[:, None] * inv.cpu() * (-1 if inverse else 1)
    c, s = (scale * ang.cos())[:, None], (scale * ang.sin())[:, None]
    y, m = x.clone(), torch.zeros_like(x)
    ia, ib = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    m[..., ia] = m[..., ib] = a.abs() + b.abs()
    return y, m


def _check(got, x, pos, inv, interleaved, inverse, scale, dtype):
    y, m = _reference(x, pos, inv, interleaved, inverse, scale)
    err = (got.double().cpu() - y).abs()
    tol = 2.0 ** -20 * m + HALF[dtype] * y.abs() * 1.001 * (m > 0)
    assert bool((err <= tol).all()), f"worst {float((err - tol).max()):.3g} over its bound"


SHAPES = [  # tokens, heads, key heads, head dim, rotary dim
    (1, 1, 1, 2, 2), (3, 2, 1, 64, 64), (37, 4, 2, 128, 64), (5, 3, 3, 96, 32), (130, 1, 1, 80, 20), (65, 16, 2, 256, 64),
    (7, 2, 2, 68, 68), (700, 16, 16, 128, 128)]


@gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_values(cuda, shape, dtype, interleaved, inverse):
    L, H, Hk, D, R = shape
    gen = torch.Generator().manual_seed(L)
    q, k = (torch.randn(L, h, D, generator=gen).to(dtype).cuda() for h in (H, Hk))
    pos = torch.randint(-50, 2_000_000, (L,), generator=gen).cuda()
    inv, _ = M.rotary_frequencies(R, scaling="linear", factor=1.5)
    qo, ko = M.rotary(q, k, pos, inv, interleaved=interleaved, inverse=inverse, attention_scale=1.25)
    for got, x in ((qo, q), (ko, k)):
        assert got.shape == x.shape and got.dtype == dtype
        _check(got, x, pos, inv, interleaved, inverse, 1.25, dtype)
    # in place and int32 positions: the same bits
    q2, k2 = q.clone(), k.clone()
    M.rotary(q2, k2, pos.int(), inv, interleaved=interleaved, inverse=inverse, attention_scale=1.25, q_out=q2, k_out=k2)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)
    only, none = M.rotary(q, None, pos, inv, interleaved=interleaved, inverse=inverse, attention_scale=1.25)
    assert none is None and torch.equal(only, qo)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_split_views_in_place(cuda, dtype):
    """q and k as columns of one projection, rotated in place; the other columns stay."""
    L, H, Hk, D = 33, 4, 2, 64
    wide = torch.randn(L, (H + Hk) * D + 24, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    for at in (8, 3):  # aligned and unaligned columns
        buf = wide.clone()
        q = buf[:, at:at + H * D].view(L, H, D)
        k = buf[:, at + H * D:at + (H + Hk) * D].view(L, Hk, D)
        q0, k0 = q.clone(), k.clone()
        pos = torch.arange(L, device="cuda")
        inv, _ = M.rotary_frequencies(32)
        M.rotary(q, k, pos, inv, q_out=q, k_out=k)
        _check(q, q0, pos, inv, False, False, 1.0, dtype)
        _check(k, k0, pos, inv, False, False, 1.0, dtype)
        assert torch.equal(buf[:, :at], wide[:, :at])
        assert torch.equal(buf[:, at + (H + Hk) * D:], wide[:, at + (H + Hk) * D:])


@gpu
def test_rows_beyond_32_bits(cuda):
    """More than 2^31 elements: the last rows equal those of a call of their own."""
    L, H, D = 262200, 64, 128
    q = torch.randn(L, H, D, device="cuda", dtype=torch.bfloat16)
    pos, (inv, _) = torch.arange(L, device="cuda"), M.rotary_frequencies(64)
    last, _ = M.rotary(q[-100:].clone(), None, pos[-100:], inv)
    M.rotary(q, None, pos, inv, q_out=q)
    assert torch.equal(q[-100:], last)


@gpu
def test_inverse_undoes_and_is_the_gradient(cuda):
    """<rotary(x), y> = <x, inverse(y)>: the inverse is the transpose, up to fp32 rounding."""
    gen = torch.Generator().manual_seed(2)
    x, y = (torch.randn(20, 2, 64, generator=gen).cuda() for _ in range(2))
    pos = torch.arange(20, device="cuda") * 977
    inv, att = M.rotary_frequencies(48, scaling="yarn", factor=2.0, trained_tokens=512)
    f, _ = M.rotary(x, None, pos, inv, attention_scale=att)
    b, _ = M.rotary(y, None, pos, inv, attention_scale=att, inverse=True)
    # each product is off by 2^-20 (|a| + |b|) |y| at most, on both sides
    bound = 2 * 2.0 ** -20 * 2 * float(x.double().abs().sum()) * float(y.abs().max())
    assert abs(float((f.double() * y.double()).sum() - (x.double() * b.double()).sum())) <= bound
    back, _ = M.rotary(M.rotary(x, None, pos, inv)[0], None, pos, inv, inverse=True)
    assert float((back - x).abs().max()) <= 2.0 ** -18 * float(x.abs().max()) * 2


@gpu
def test_rotary_refuses_arguments(cuda):
    q, k = torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, 1, 64, device="cuda")
    pos, (inv, _) = torch.arange(4, device="cuda"), M.rotary_frequencies(16)
    f = M.rotary
    buf = torch.zeros(5, 2, 64, device="cuda")
    bad = [
        lambda: f(q.half(), None, pos, inv), lambda: f(q, k.bfloat16(), pos, inv), lambda: f(q, k[:3], pos, inv),
        lambda: f(q, k, pos[:3], inv), lambda: f(q, k, pos.float(), inv), lambda: f(q, k, pos.cpu(), inv),
        lambda: f(q, k, pos, inv.float()), lambda: f(q, k, pos, torch.ones(33, dtype=torch.float64, device="cuda")),
        lambda: f(q, k, pos, inv, q_out=q[:3]), lambda: f(q, k, pos, inv, q_out=q.bfloat16()),
        lambda: f(q[:, :0], k, pos, inv), lambda: f(q, None, pos, inv, k_out=k), lambda: f(buf[:4], None, pos, inv, q_out=buf[1:]),
        lambda: f(q, k, pos, inv, k_out=q[:, :1]), lambda: f(q, k, pos, inv, q_out=q, k_out=q[:, 1:]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
