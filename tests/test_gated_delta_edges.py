"""The gated delta rule's calls that are allowed and rare: offsets that overlap, packs of more CTAs than multiprocessors,
rows and states behind 2^31 elements, samples at the bounds between the forms. Bounds as in test_gated_delta."""

import ctypes

import pytest
import torch

import memt_b200 as M
from memt_b200 import _lib
from test_gated_delta import _args, _check, _chunk_bounds, _inputs, _recurrence

gpu = pytest.mark.gpu


def test_status_needs_a_place():
    assert _lib.load().memt_gated_delta_status(None, None) == _lib.MEMT_ERR_INVALID_ARGUMENT


def test_workspace_is_refused_before_anything_runs():
    lib, mb = _lib.load(), 1 << 20
    far = dict(q=mb << 4, k=mb << 5, v=mb << 6, out=mb << 7, g=mb << 8, beta=mb << 9, cu_seqlens=mb << 10,
               final_state=mb << 11)
    for n, tokens in ((1, 1000), (3, 100), (1, 4096)):  # in chunks, with both forms, in segments
        need = lib.memt_gated_delta_workspace_size(n, tokens, 4, 64, _lib.MEMT_BF16)
        assert need > 256
        a = _args(num_samples=n, total_tokens=tokens, **far)
        call = lambda ws, size: lib.memt_gated_delta(ctypes.byref(a), ws, size, None)  # noqa: E731
        assert call(None, need) == _lib.MEMT_ERR_WORKSPACE
        assert call(mb << 12, need - 1) == _lib.MEMT_ERR_WORKSPACE
        assert call((mb << 12) + 128, need) == _lib.MEMT_ERR_WORKSPACE
        for there in ("q", "v", "out", "g", "beta", "final_state", "cu_seqlens"):
            assert call(far[there], need) == _lib.MEMT_ERR_INVALID_ARGUMENT, there


def test_workspace_grows_with_the_call():
    """More samples or tokens never take less room within one form, and sizes at the limits do not wrap."""
    f = _lib.load().memt_gated_delta_workspace_size
    for D in (64, 128, 256):
        sizes = [f(200, t, 16, D, _lib.MEMT_BF16) for t in range(100, 40000, 321)]
        assert sizes == sorted(sizes)
        assert f(1, 2 ** 31 - 1, 1, D, _lib.MEMT_BF16) >= (2 ** 31 // 64) * 20480
        assert f(2 ** 30, 2 ** 31 - 2, 64, D, _lib.MEMT_BF16) == 0 and f(2 ** 30, 1, 4, D, _lib.MEMT_F32) == 0
        for n, tokens, heads in ((2 ** 30, 2 ** 31 - 2, 4), (2 ** 30, 1, 4), (1, 2 ** 31 - 2, 2 ** 20)):
            far = [(i + 1) << 52 for i in range(8)]  # (nothing reads them: more CTAs than a grid holds)
            a = _args(num_samples=n, total_tokens=tokens, num_heads=heads, num_key_heads=1, head_dim=D,
                      q_stride=D, k_stride=D, v_stride=heads * D, out_stride=heads * D,
                      **dict(zip(("q", "k", "v", "out", "g", "beta", "cu_seqlens", "final_state"), far)))
            assert _lib.load().memt_gated_delta(ctypes.byref(a), 1 << 60, 2 ** 60, None) == _lib.MEMT_ERR_UNSUPPORTED


@gpu
def test_status_after_calls_of_every_kind(cuda):
    lib, status = _lib.load(), ctypes.c_int32(-1)
    stream = torch.cuda.current_stream().cuda_stream
    for lengths in ([5], [300, 70], [2900], [3, 200, 1, 2]):
        M.gated_delta(*_inputs(3, lengths, 1, 2, 64, torch.bfloat16))
        assert lib.memt_gated_delta_status(stream, ctypes.byref(status)) == _lib.MEMT_OK and status.value == 0


@gpu
@pytest.mark.parametrize("D,L,times", [(64, 500, 3), (128, 300, 2), (256, 200, 2), (64, 16000, 2), (128, 12000, 2)])
def test_samples_that_share_their_rows(cuda, D, L, times):
    """Offsets that go back: each sample is the recurrence over its rows, whatever form is left for it."""
    H = 1
    q, k, v, g, b, h0, _ = _inputs(31, [L], 1, H, D, torch.bfloat16)
    offsets = [0] + [L, 0] * times
    N = len(offsets) - 1
    h = torch.randn(N, H, D, D, device="cuda") * 0.5
    o, final = M.gated_delta(q, k, v, g, b, h, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    for n in range(N):
        if n % 2:
            assert torch.equal(final[n], h[n])  # empty
            continue
        x = (q, k, v, g, b, h[n:n + 1], torch.tensor([0, L]))
        _, ref, _, E = _recurrence(*x, D ** -0.5)
        _, Ec = _chunk_bounds(*x, D ** -0.5, D if L > 2000 else 0)
        err = (final[n:n + 1].double() - ref).norm(dim=2)
        assert bool((err <= torch.maximum(E, Ec) * 1.01).all()), n


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_more_long_samples_than_the_tokens_allow(cuda, D):
    """Both forms in one call, and more samples of many tokens than any offsets in order could have."""
    L, N, H = 200, 101, 2
    q, k, v, g, b, _, _ = _inputs(32, [L], 1, H, D, torch.bfloat16)
    h = torch.randn(N, H, D, D, device="cuda") * 0.5
    offsets = torch.tensor([0] + [L, 0] * (N // 2) + [3], dtype=torch.int32, device="cuda")
    _, final = M.gated_delta(q, k, v, g, b, h, offsets)
    for n in (0, 2, 6, 8, 50, 98):
        x = (q, k, v, g, b, h[n:n + 1], torch.tensor([0, L]))
        _, ref, _, E = _recurrence(*x, D ** -0.5)
        _, Ec = _chunk_bounds(*x, D ** -0.5)
        assert bool(((final[n:n + 1].double() - ref).norm(dim=2) <= torch.maximum(E, Ec) * 1.01).all()), n
    assert torch.equal(final[1], h[1])


@gpu
@pytest.mark.parametrize("D,few", [(64, 40), (128, 20), (256, 14)])
def test_samples_at_the_bound_between_the_forms(cuda, D, few):
    lengths = [few, few + 1, 1, 0, few - 1, 64, 65]
    x = _inputs(33, lengths, 1, 2, D, torch.bfloat16)
    o, final = M.gated_delta(*x)
    _check(o, final, x, torch.bfloat16, D ** -0.5)


@gpu
def test_many_samples_the_longest_first(cuda):
    """More CTAs than multiprocessors: in order of length. Each sample's results are those of calls of fewer."""
    H, D = 8, 64
    lengths = [700 + 173 * (i * 7 % 20) for i in range(20)]
    q, k, v, g, b, h0, cu = _inputs(34, lengths, 4, H, D, torch.bfloat16)
    o, final = M.gated_delta(q, k, v, g, b, h0, cu)
    for n0 in (0, 10):
        a, e = int(cu[n0]), int(cu[n0 + 10])
        on, fn = M.gated_delta(q[a:e], k[a:e], v[a:e], g[a:e], b[a:e], h0[n0:n0 + 10], cu[n0:n0 + 11] - a)
        assert torch.equal(o[a:e], on) and torch.equal(final[n0:n0 + 10], fn)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_and_states_behind_31_bits(cuda, dtype):
    """Strides and slots whose offsets pass 2^31 elements."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    D, H, L = 256, 16, 150
    q, k, v, g, b, h0, cu = _inputs(35, [L], 2, H, D, dtype)
    step = (1 << 24) + 64
    rows = lambda x: torch.as_strided(torch.empty(L * step, device="cuda", dtype=dtype), x.shape, (step, D, 1))  # noqa: E731
    far = []
    for x in (q, k, v):
        far.append(rows(x))
        far[-1].copy_(x)
    out = rows(v)
    want = M.gated_delta(q, k, v, g, b, h0, cu)
    got = M.gated_delta(*far, g, b, h0, cu, out=out)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    del far, out, got
    pool = torch.empty(2100, H, D, D, device="cuda")  # 2^20 elements a slot
    pool[2099] = h0[0]
    slot = torch.tensor([2099], dtype=torch.int32, device="cuda")
    o, _ = M.gated_delta(q, k, v, g, b, pool, cu, initial_slots=slot, final_state=pool, final_slots=slot)
    assert torch.equal(o, want[0]) and torch.equal(pool[2099], want[1][0])
    pool[2099] = h0[0]
    o1 = M.gated_delta_step(q[:1], k[:1], v[:1], g[:1], b[:1], pool, slots=slot)
    small = h0.clone()
    o2 = M.gated_delta_step(q[:1], k[:1], v[:1], g[:1], b[:1], small)
    assert torch.equal(o1, o2) and torch.equal(pool[2099], small[0])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_step_with_a_value_that_is_not_finite(cuda, dtype, value):
    """It stays in its session, head and column."""
    N, H, D = 3, 2, 64
    q, k, v, g, b, h0, _ = _inputs(36, [1] * N, 1, H, D, dtype)
    clean = h0.clone()
    o = M.gated_delta_step(q, k, v, g, b, clean)
    v = v.clone()
    v[1, 1, 7] = value
    states = h0.clone()
    o2 = M.gated_delta_step(q, k, v, g, b, states)
    assert not bool(torch.isfinite(o2[1, 1, 7])) and not bool(torch.isfinite(states[1, 1, :, 7]).any())
    o2[1, 1, 7] = o[1, 1, 7]
    states[1, 1, :, 7] = clean[1, 1, :, 7]
    assert torch.equal(o2, o) and torch.equal(states, clean)


@gpu
@pytest.mark.parametrize("N,most", [(1500, 12), (1030, 67), (33, 200)])
def test_many_samples(cuda, N, most):
    """Calls whose chunks are listed before (more than 32 samples, and more than one round of a CTA): few tokens each
    with longer ones among them, all in chunks, and empty ones."""
    gen = torch.Generator().manual_seed(N)
    lengths = torch.randint(0 if most == 12 else most - 3, most + 1, (N,), generator=gen)
    if most == 12:
        longer = torch.randperm(N, generator=gen)[:40]
        lengths[longer] = torch.randint(41, 300, (40,), generator=gen)
    lengths[-1], lengths[5] = 0, 0
    x = _inputs(37, lengths.tolist(), 1, 1, 64, torch.bfloat16)
    o, final = M.gated_delta(*x)
    _check(o, final, x, torch.bfloat16, 64 ** -0.5)
    other = M.gated_delta(*x[:6], x[6].cuda())
    assert torch.equal(o, other[0]) and torch.equal(final, other[1])


@gpu
@pytest.mark.parametrize("first,second", [([7, 60, 0, 130] * 10, [0, 41, 150, 6] * 10), ([5000, 1000], [900, 5100]),
                                          ([9, 2, 33, 5] * 12, [1, 45, 0, 3] * 12)])
def test_offsets_change_between_replays(cuda, first, second):
    """The lengths are the device's: a captured call follows them."""
    assert sum(first) == sum(second)
    x = _inputs(38, first, 1, 1, 64, torch.bfloat16)
    cu = x[6].cuda()
    other = torch.tensor([0] + second).cumsum(0).to(torch.int32).cuda()
    want = [M.gated_delta(*x[:6], c.clone()) for c in (cu, other)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = M.gated_delta(*x[:6], cu)
    for offsets, (o, final) in ((other, want[1]), (x[6].cuda(), want[0]), (other, want[1])):
        cu.copy_(offsets)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], o) and torch.equal(got[1], final)
