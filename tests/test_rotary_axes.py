"""Rotary positions with several axes: refusals of the C entry on CPU, values on the GPU against 64-bit rotations.

Tolerance: sine and cosine of a reduced angle (fp32 fraction of a turn: 2 pi 2^-25; sincospif 2 steps; the factor
1 step) <= 2^-21 absolute for factors up to 2, two products and a sum 2 u each, so 2^-20 (|a| + |b|) on either
element of a pair, and half a step of the output type.
"""

import ctypes

import pytest
import torch

import memt_b200 as M
from memt_b200 import _lib

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _args(**over):
    mb = 1 << 20
    f = dict(num_heads=2, num_key_heads=1, head_dim=64, rotary_dim=32, dtype=_lib.MEMT_BF16, total_tokens=8, q=mb,
             q_stride=128, k=2 * mb, k_stride=64, q_out=3 * mb, q_out_stride=128, k_out=4 * mb, k_out_stride=64,
             positions=5 * mb, position_stride=8, positions_int64=1, num_axes=3, pair_axes=6 * mb, inv_freq=7 * mb,
             attention_scale=1.0)
    f.update(over)
    return _lib.RotaryAxesArgs(**f)


@pytest.mark.parametrize("over", [
    dict(struct_size=4), dict(num_heads=0), dict(num_key_heads=-1), dict(rotary_dim=0), dict(rotary_dim=31),
    dict(rotary_dim=66), dict(dtype=3), dict(total_tokens=-1), dict(q=None), dict(q_out=None), dict(positions=None),
    dict(inv_freq=None), dict(q_stride=100), dict(k_stride=32), dict(k_out=None), dict(k_out_stride=1),
    dict(num_axes=0), dict(pair_axes=None), dict(position_stride=7),
    # outputs over what every thread reads; the last of three rows of positions
    dict(q_out=6 << 20), dict(k_out=(6 << 20) + 48), dict(q_out=(7 << 20) + 64), dict(q_out=(5 << 20) + 128),
    dict(k_out=(5 << 20) + 160, position_stride=16)])
def test_rotary_axes_refuses(over):
    a = _args(**over)
    assert _lib.load().memt_rotary_axes(ctypes.byref(a), None) == _lib.MEMT_ERR_INVALID_ARGUMENT


def test_empty_rotary_axes_launches_nothing():
    lib = _lib.load()
    assert lib.memt_rotary_axes(None, None) == _lib.MEMT_ERR_INVALID_ARGUMENT
    assert lib.memt_rotary_axes(ctypes.byref(_args(total_tokens=0)), None) == _lib.MEMT_OK
    assert lib.memt_rotary_axes(ctypes.byref(_args(total_tokens=0, num_key_heads=0, k=None, k_out=None)), None) \
        == _lib.MEMT_OK


def test_sections():
    runs = M.rotary_sections([2, 3, 0, 1], device="cpu")
    assert runs.dtype == torch.int32 and runs.tolist() == [0, 0, 1, 1, 1, 3]
    assert M.rotary_sections((4, 2, 2), cycled=True, device="cpu").tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert M.rotary_sections([5], device="cpu").tolist() == [0] * 5
    for bad in ([], [0], [0, 0], [3, -1]):
        with pytest.raises(ValueError):
            M.rotary_sections(bad, device="cpu")


def test_rotary_axes_refuses_host_tensors():
    x = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError):
        M.rotary_axes(x, x, torch.zeros(3, 3, dtype=torch.int64), torch.ones(4, dtype=torch.float64),
                      torch.zeros(4, dtype=torch.int32))


def _reference(x, pos, axes, inv, interleaved, inverse, scale):
    """fp64 rotation and the elementwise |a| + |b| of each pair (the bound's scale)."""
    n = inv.numel()
    x, pos, axes = x.double().cpu(), pos.double().cpu(), axes.cpu()
    at = torch.stack([pos[a] if 0 <= a < len(pos) else torch.zeros(pos.shape[1], dtype=torch.float64)
                      for a in axes.tolist()], 1)
    ang = at * inv.cpu() * (-1 if inverse else 1)
    c, s = (scale * ang.cos())[:, None], (scale * ang.sin())[:, None]
    y, m = x.clone(), torch.zeros_like(x)
    ia, ib = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    m[..., ia] = m[..., ib] = a.abs() + b.abs()
    return y, m


def _check(got, x, pos, axes, inv, interleaved, inverse, scale, dtype):
    y, m = _reference(x, pos, axes, inv, interleaved, inverse, scale)
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
@pytest.mark.parametrize("cycled", [False, True])
def test_rotary_axes_values(cuda, shape, dtype, interleaved, cycled):
    L, H, Hk, D, R = shape
    gen = torch.Generator().manual_seed(L)
    q, k = (torch.randn(L, h, D, generator=gen).to(dtype).cuda() for h in (H, Hk))
    counts = [R // 2 - 2 * (R // 6), R // 6, R // 6]
    axes = M.rotary_sections(counts, cycled=cycled)
    pos = torch.randint(-50, 2_000_000, (3, L), generator=gen).cuda()
    inv, _ = M.rotary_frequencies(R, scaling="linear", factor=1.5)
    for inverse in (False, True):
        kinds = dict(interleaved=interleaved, inverse=inverse, attention_scale=1.25)
        qo, ko = M.rotary_axes(q, k, pos, inv, axes, **kinds)
        for got, x in ((qo, q), (ko, k)):
            assert got.shape == x.shape and got.dtype == dtype
            _check(got, x, pos, axes, inv, interleaved, inverse, 1.25, dtype)
        # in place, int32 positions in a slice of a longer buffer: the same bits
        q2, k2 = q.clone(), k.clone()
        buf = torch.full((3, L + 5), -7, dtype=torch.int32, device="cuda")
        buf[:, :L] = pos
        M.rotary_axes(q2, k2, buf[:, :L], inv, axes, q_out=q2, k_out=k2, **kinds)
        assert torch.equal(q2, qo) and torch.equal(k2, ko)
        only, none = M.rotary_axes(q, None, pos[:, None], inv, axes, **kinds)
        assert none is None and torch.equal(only, qo)
        # the same position on every axis: what rotary makes of it
        qa, ka = M.rotary_axes(q, k, pos[:1].expand(3, L), inv, axes, **kinds)
        qb, kb = M.rotary(q, k, pos[0], inv, **kinds)
        assert torch.equal(qa, qb) and torch.equal(ka, kb)
        # one axis
        qa, ka = M.rotary_axes(q, k, pos[:1], inv, torch.zeros_like(axes), **kinds)
        assert torch.equal(qa, qb) and torch.equal(ka, kb)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_axes_outside_turn_nothing(cuda, dtype):
    L, H, D, R = 9, 3, 64, 48
    q = torch.randn(L, H, D, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    axes = torch.tensor([0, 1, 2, -1, 3, 2 ** 31 - 1, -2 ** 31, 1] * 3, dtype=torch.int32, device="cuda")
    pos = torch.randint(0, 10_000, (3, L), generator=torch.Generator().manual_seed(2)).cuda()
    inv, _ = M.rotary_frequencies(R)
    qo, _ = M.rotary_axes(q, None, pos, inv, axes)
    _check(qo, q, pos, axes, inv, False, False, 1.0, dtype)
    assert torch.equal(qo[..., 3], q[..., 3]) and torch.equal(qo[..., 24 + 4], q[..., 24 + 4])


@gpu
def test_inverse_is_the_transpose(cuda):
    """<rotary_axes(x), y> = <x, rotary_axes(y, inverse)>, and its differences along a direction."""
    L, H, D, R = 21, 2, 64, 32
    gen = torch.Generator().manual_seed(4)
    x, y, d = (torch.randn(L, H, D, generator=gen).cuda() for _ in range(3))
    pos = torch.randint(0, 5000, (2, L), generator=gen).cuda()
    inv, _ = M.rotary_frequencies(R)
    axes = M.rotary_sections([9, 7], cycled=True)
    turn = lambda z, **kw: M.rotary_axes(z, None, pos, inv, axes, attention_scale=1.5, **kw)[0].double()  # noqa: E731
    back = turn(y, inverse=True)
    left, right = float((turn(x) * y.double()).sum()), float((x.double() * back).sum())
    slack = 2.0 ** -19 * 2 * float((x.double().abs().sum() * y.double().abs().max()))
    assert abs(left - right) <= slack
    change = float(((turn(x + d) - turn(x - d)) / 2 * y.double()).sum())
    assert abs(change - float((d.double() * back).sum())) <= 4 * slack


@gpu
def test_refused_arguments_and_overlaps(cuda):
    L, H, D = 6, 2, 64
    q, k = torch.randn(L, H, D, device="cuda"), torch.randn(L, 1, D, device="cuda")
    inv, _ = M.rotary_frequencies(32)
    axes = M.rotary_sections([6, 5, 5])
    pos = torch.zeros(3, L, dtype=torch.int64, device="cuda")
    M.rotary_axes(q, k, pos, inv, axes)
    for bad in (dict(pair_axes=axes.long()), dict(pair_axes=axes[:15]), dict(pair_axes=axes.cpu()),
                dict(positions=pos[0]), dict(positions=pos[:, :5]), dict(positions=pos[:0]), dict(positions=pos.float()),
                dict(positions=pos.cpu()), dict(positions=pos[:, None].expand(3, 2, L)), dict(inv_freq=inv.float()),
                dict(k=k[:5]), dict(k=k.bfloat16()), dict(q=q.half()), dict(k_out=q), dict(q_out=q[:5]),
                dict(q_out=pos.view(torch.float32).view(-1)[:0].view(0, H, D))):
        with pytest.raises(ValueError):
            M.rotary_axes(**{**dict(q=q, k=k, positions=pos, inv_freq=inv, pair_axes=axes), **bad})
    buf = torch.zeros(L * H * D + 64, device="cuda")
    inside = buf[L * H * D - 32:L * H * D - 16].view(torch.int32)
    inside.copy_(axes)
    with pytest.raises(ValueError):  # an output over the pairs' axes
        M.rotary_axes(q, None, pos, inv, inside, q_out=buf[:L * H * D].view(L, H, D))


@gpu
def test_captured_and_on_another_stream(cuda):
    L, H, D = 33, 4, 128
    q, k = torch.randn(L, H, D, device="cuda").bfloat16(), torch.randn(L, 2, D, device="cuda").bfloat16()
    inv, _ = M.rotary_frequencies(128)
    axes = M.rotary_sections([16, 24, 24])
    pos = torch.randint(0, 5000, (3, L), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = M.rotary_axes(q, k, pos, inv, axes)
    for _ in range(2):
        pos.add_(77)
        want = M.rotary_axes(q, k, pos, inv, axes)
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
