"""Causal linear attention with a decay for each head and the single-token steps.

CPU: refusals of the C entry points. GPU: every operator against the recurrence in 64 bits on the
same (rounded) inputs.

Tolerances are elementwise bounds. With u = 2^-24 (half an fp32 step) and A the same recurrence
over absolute values (an upper bound of every partial sum):
  * one recurrence step rounds the decay (expf: 2 steps), a product, a sum: <= 8 u of A a token;
    a sum over D rows <= D u of A; hence (8 T + D + 8) u A for T tokens of the fp32 kernels;
  * the chunked bf16 kernel keeps the state in fp32: weights exp(R) carry the rounding of the
    exponent sum R (7 additions, |R| <= r: 7 r u) and of exp2 (4 u), the three-term split of k
    leaves 2 u, 3 x 64 truncating additions of a chunk <= 2 u each, the carry 4 u a chunk:
    (7 r + 6 + 384 + 4 chunks) u A;
  * its output rounds scores, state copy and result to bf16 (half a step: 2^-8 each):
    2^-8 (1 + 2^-7) (A_o + |o|) plus the fp32 share above.
"""

import ctypes

import numpy as np
import pytest
import torch

import memt_b200 as M
from memt_b200 import _lib

gpu = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}


# ---------------------------------------------------------------------------
# refusals of the C entry points (nothing is launched)
# ---------------------------------------------------------------------------

def _linear_args(**over):
    f = dict(num_samples=1, num_heads=4, num_key_heads=2, head_dim=64, dtype=_lib.MEMT_BF16, total_tokens=8,
             cu_seqlens=16, q=16, q_stride=128, k=16, k_stride=128, v=16, v_stride=256, g=16,
             g_layout=_lib.GATE_PER_HEAD, scale=1.0, out=16, out_stride=256, final_state=16)
    f.update(over)
    return _lib.LinearAttentionArgs(**f)


BAD_LINEAR = [
    (dict(struct_size=8), "INVALID_ARGUMENT"), (dict(num_samples=0), "INVALID_ARGUMENT"),
    (dict(num_heads=3), "INVALID_ARGUMENT"), (dict(num_key_heads=0), "INVALID_ARGUMENT"),
    (dict(total_tokens=-1), "INVALID_ARGUMENT"), (dict(total_tokens=2 ** 31), "INVALID_ARGUMENT"),
    (dict(dtype=5), "INVALID_ARGUMENT"), (dict(head_dim=96), "UNSUPPORTED"), (dict(q=None), "INVALID_ARGUMENT"),
    (dict(final_state=None), "INVALID_ARGUMENT"), (dict(g=None), "INVALID_ARGUMENT"),
    (dict(g_layout=_lib.GATE_NONE), "INVALID_ARGUMENT"), (dict(g_layout=_lib.GATE_PER_CHANNEL), "INVALID_ARGUMENT"),
    (dict(q_stride=120), "INVALID_ARGUMENT"), (dict(v_stride=128), "INVALID_ARGUMENT"),
    (dict(out_stride=128), "INVALID_ARGUMENT"), (dict(k_stride=132), "MISALIGNED"), (dict(v=24), "MISALIGNED"),
    (dict(initial_slots=16, num_initial_slots=1), "INVALID_ARGUMENT"),
    (dict(final_slots=16, num_final_slots=0), "INVALID_ARGUMENT"),
    # states of two samples (64 KB each) that overlap by one
    (dict(num_samples=2, initial_state=16 + 65536), "INVALID_ARGUMENT"),
    (dict(num_samples=2, initial_state=16, final_state=16 + 65536), "INVALID_ARGUMENT"),
]


@pytest.mark.parametrize("over,error", BAD_LINEAR)
def test_linear_attention_refuses(over, error):
    a = _linear_args(**over)
    assert _lib.load().memt_linear_attention(ctypes.byref(a), 256, 1 << 40, None) == getattr(_lib, "MEMT_ERR_" + error)


def test_linear_attention_refuses_workspace():
    # one long sample of few heads: its segments' states need memory
    lib, a = _lib.load(), _linear_args(total_tokens=1 << 20)
    assert lib.memt_linear_attention(None, 256, 1 << 40, None) == _lib.MEMT_ERR_INVALID_ARGUMENT
    assert lib.memt_linear_attention(ctypes.byref(a), None, 1 << 40, None) == _lib.MEMT_ERR_WORKSPACE
    assert lib.memt_linear_attention(ctypes.byref(a), 256, 0, None) == _lib.MEMT_ERR_WORKSPACE
    assert lib.memt_linear_attention(ctypes.byref(a), 264, 1 << 40, None) == _lib.MEMT_ERR_WORKSPACE
    f = lib.memt_linear_attention_workspace_size
    assert f(8, 65536, 16, 128, _lib.MEMT_BF16) == 256  # enough samples and heads: no segments
    assert f(1, 65536, 16, 128, _lib.MEMT_BF16) >= 9 * 16 * 128 * 128 * 4
    assert f(1, 65536, 16, 128, _lib.MEMT_F32) == 256
    assert f(1, 0, 1, 64, _lib.MEMT_BF16) >= 256 and f(1, 100, 1, 96, _lib.MEMT_BF16) == 0
    assert f(0, 100, 1, 64, _lib.MEMT_BF16) == 0 and f(1, 100, 1, 64, 9) == 0


def _step_args(**over):
    f = dict(rule=_lib.RULE_GDN2, num_samples=0, num_heads=4, num_key_heads=2, head_dim=64, dtype=_lib.MEMT_BF16,
             q=16, q_stride=128, k=16, k_stride=128, v=16, v_stride=256, g=16, g_layout=_lib.GATE_PER_HEAD,
             states=16, scale=1.0, out=16, out_stride=256)
    f.update(over)
    return _lib.RecurrentStepArgs(**f)


BAD_STEP = [
    (dict(struct_size=8), "INVALID_ARGUMENT"), (dict(rule=2), "INVALID_ARGUMENT"),
    (dict(num_samples=-1), "INVALID_ARGUMENT"), (dict(num_heads=5), "INVALID_ARGUMENT"),
    (dict(dtype=2), "INVALID_ARGUMENT"), (dict(head_dim=32), "UNSUPPORTED"), (dict(states=None), "INVALID_ARGUMENT"),
    (dict(states=20), "MISALIGNED"), (dict(g=None), "INVALID_ARGUMENT"), (dict(g_layout=4), "INVALID_ARGUMENT"),
    (dict(beta=16), "INVALID_ARGUMENT"), (dict(beta_layout=1), "INVALID_ARGUMENT"),
    (dict(q_stride=64), "INVALID_ARGUMENT"), (dict(out_stride=8), "INVALID_ARGUMENT"),
    (dict(slots=16, num_slots=0), "INVALID_ARGUMENT"),
    (dict(rule=_lib.RULE_LINEAR, write=16), "UNSUPPORTED"), (dict(rule=_lib.RULE_LINEAR, read_incoming=1), "UNSUPPORTED"),
    (dict(rule=_lib.RULE_LINEAR, g_layout=_lib.GATE_PER_CHANNEL), "UNSUPPORTED"),
]


@pytest.mark.parametrize("over,error", BAD_STEP)
def test_step_refuses(over, error):
    a = _step_args(**over)
    assert _lib.load().memt_recurrent_step(ctypes.byref(a), None) == getattr(_lib, "MEMT_ERR_" + error)


def test_empty_step_launches_nothing():
    assert _lib.load().memt_recurrent_step(ctypes.byref(_step_args()), None) == _lib.MEMT_OK
    assert _lib.load().memt_recurrent_step(None, None) == _lib.MEMT_ERR_INVALID_ARGUMENT


def test_operators_refuse_host_tensors():
    x, s = torch.zeros(3, 2, 64), torch.zeros(3, 2, 64, 64)
    with pytest.raises(ValueError):
        M.linear_attention(x, x, x, None, s, torch.tensor([0, 1, 2, 3]))
    with pytest.raises(ValueError):
        M.linear_attention_step(x, x, x, None, s)
    with pytest.raises(ValueError):
        M.gdn2_step(x, x, x, None, s)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _recurrence(q, k, v, g, h0, cu, scale):
    """fp64 (o, final) and the same recurrence over absolute values (A_o, A_final). CPU tensors."""
    L, H, D = v.shape
    rep = H // q.shape[1]
    q, k, v = (x.double() for x in (q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1), v))
    a = torch.ones(L, H, dtype=torch.float64) if g is None else torch.exp(g.double()).expand(L, H)
    S, B = h0.double().clone(), h0.double().abs()
    o, A = torch.zeros(L, H, D, dtype=torch.float64), torch.zeros(L, H, D, dtype=torch.float64)
    for n in range(len(cu) - 1):
        for t in range(int(cu[n]), int(cu[n + 1])):
            S[n] = a[t][:, None, None] * S[n] + k[t][:, :, None] * v[t][:, None, :]
            B[n] = a[t][:, None, None] * B[n] + (k[t][:, :, None] * v[t][:, None, :]).abs()
            o[t] = scale * torch.einsum("hk,hkv->hv", q[t], S[n])
            A[t] = abs(scale) * torch.einsum("hk,hkv->hv", q[t].abs(), B[n])
    return o, S, A, B


def _inputs(seed, lengths, Hk, H, D, dtype, decay, gscale=1.0):
    gen = torch.Generator().manual_seed(seed)
    L, N = sum(lengths), len(lengths)
    unit = lambda x: x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    q = unit(torch.randn(L, Hk, D, generator=gen)).to(dtype)
    k = unit(torch.randn(L, Hk, D, generator=gen)).to(dtype)
    v = torch.randn(L, H, D, generator=gen).to(dtype)
    g = {"none": None, "head": -torch.exp2(-8.0 * torch.arange(1, H + 1) / H),
         "token": torch.nn.functional.logsigmoid(2 + 0.5 * torch.randn(L, H, generator=gen))}[decay]
    g = None if g is None else g * gscale
    h0 = 0.5 * torch.randn(N, H, D, D, generator=gen)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32)
    return q, k, v, g, h0, cu


def _dev(*xs):
    return tuple(None if x is None else x.cuda() for x in xs)


def _check(got, ref, tol, what):
    err = (got.double().cpu() - ref).abs()
    bad = err > tol
    assert not bool(bad.any()) and not bool(torch.isnan(err).any()), \
        f"{what}: worst {float((err / (tol + 1e-300)).max()):.3g} of its bound"


def _tolerances(ref, lengths, D, dtype, g, H):
    o, S, A, B = ref
    T = max(lengths)
    if dtype == torch.float32:
        return (8 * T + D + 8) * U * A + U * o.abs() + 1e-40, (8 * T + 8) * U * B + 1e-40
    r = 0.0 if g is None else 64 * float(g.abs().max()) * 1.4427
    share = (7 * r + 390 + 4 * (T / 64 + 1)) * U
    return HALF[dtype] * (1 + 2.0 ** -7) * (A + o.abs()) + (share + D * U) * A + 1e-40, share * B + 1e-40


def _run_and_check(lengths, Hk, H, D, dtype, decay, seed=0, gscale=1.0):
    q, k, v, g, h0, cu = _inputs(seed, lengths, Hk, H, D, dtype, decay, gscale)
    scale = D ** -0.5
    ref = _recurrence(q, k, v, g, h0, cu, scale)
    dq, dk, dv, dg, dh, dcu = _dev(q, k, v, g, h0, cu)
    before = dh.clone()
    o, final = M.linear_attention(dq, dk, dv, dg, dh, dcu)
    torch.cuda.synchronize()
    to, ts = _tolerances(ref, lengths, D, dtype, g, H)
    _check(final, ref[1], ts, "state")
    _check(o, ref[0], to, "output")
    assert torch.equal(dh, before)
    return o, final


# ---------------------------------------------------------------------------
# linear_attention
# ---------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lengths", [[1], [8], [13], [33], [63], [64], [65], [128, 1, 0, 200], [0, 3, 130],
                                     [5, 0, 40, 12, 1, 9, 33, 2], [1] * 70 + [40, 0, 30] + [2] * 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_attention_lengths(cuda, D, lengths, dtype):
    _run_and_check(lengths, 2, 2, D, dtype, "token", seed=D + len(lengths))


@gpu
@pytest.mark.parametrize("decay", ["token", "head", "none"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_few_tokens_beside_prompts(cuda, D, decay):
    """Short samples and prompts in one call, with shared key heads, in place in a pool: both kernels
    write their own samples' slots and rows, and nothing else."""
    lengths, Hk, H = [1, 4, 0, 5, 90, 2, 1, 33, 6, 3], 2, 4
    q, k, v, g, h0, cu = _inputs(3, lengths, Hk, H, D, torch.bfloat16, decay)
    at, others = torch.tensor([7, 2, 11, 0, 5, 9, 3, 1, 10, 4]), torch.tensor([6, 8])
    ref = _recurrence(q, k, v, g, h0, cu, D ** -0.5)
    pool = torch.full((12, H, D, D), 3.0)
    pool[at] = h0
    dq, dk, dv, dg, dpool, dcu, slots = _dev(q, k, v, g, pool, cu, at.int())
    out = torch.full((q.shape[0] + 2, H, D), 5.0, dtype=torch.bfloat16, device="cuda")
    M.linear_attention(dq, dk, dv, dg, dpool, dcu, out=out[1:-1], final_state=dpool, initial_slots=slots,
                       final_slots=slots)
    torch.cuda.synchronize()
    to, ts = _tolerances(ref, lengths, D, torch.bfloat16, g, H)
    _check(out[1:-1], ref[0], to, "output")
    _check(dpool[at.cuda()], ref[1], ts, "state")
    assert bool((out[0] == 5).all()) and bool((out[-1] == 5).all()) and bool((dpool[others.cuda()] == 3).all())


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_graph_replays_with_other_lengths(cuda, D):
    """A captured call replayed with other offsets and tokens: short samples turn long and back."""
    N, H, L = 40, 2, 200
    packs = ([5] * N, [1] * 38 + [100, 62], [0] * 39 + [L], [L - 39] + [1] * 39, [0, 25, 9, 7] * 4 + [1] * 24)
    q, k, v, g, h0, cu = _dev(*_inputs(23, packs[0], H, H, D, torch.bfloat16, "token"))
    o, final = torch.zeros_like(v), torch.zeros_like(h0)
    run = lambda: M.linear_attention(q, k, v, g, h0, cu, out=o, final_state=final)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed, lengths in enumerate(packs):
        new = _inputs(seed, [L], H, H, D, torch.bfloat16, "token")
        for x, y in zip((q, k, v, g), new):
            x.copy_(y)
        cu.copy_(torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32))
        o.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        ref = _recurrence(*new[:4], h0.cpu(), cu.cpu(), D ** -0.5)
        to, ts = _tolerances(ref, lengths, D, torch.bfloat16, new[3], H)
        used = sum(lengths)
        _check(final, ref[1], ts, f"state of pack {seed}")
        _check(o[:used], ref[0][:used], to[:used], f"output of pack {seed}")
        assert bool((o[used:] == 3).all())


@gpu
@pytest.mark.parametrize("decay", ["none", "head", "token"])
@pytest.mark.parametrize("Hk,H", [(1, 3), (2, 4), (3, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_attention_heads_and_decays(cuda, decay, Hk, H, dtype):
    _run_and_check([150, 70], Hk, H, 64, dtype, decay, seed=H)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_linear_attention_many_chunks(cuda, D):
    _run_and_check([1100], 1, 2, D, torch.bfloat16, "head", seed=3)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lengths", [[2500], [4000, 0, 2500, 3], [64 * 40, 64 * 20 + 1]])
@pytest.mark.parametrize("decay", ["head", "token"])
def test_few_long_samples_in_segments(cuda, D, lengths, decay):
    """Few (sample, head) pairs: the tokens are split over segments. Every segment adds one join of its
    state (4 u) to the chunks' own; states start in a pool, one tensor for both, shared key heads."""
    Hk, H, N = 1, 2, len(lengths)
    q, k, v, g, h0, cu = _inputs(D, lengths, Hk, H, D, torch.bfloat16, decay, 0.05)
    ref = _recurrence(q, k, v, g, h0, cu, D ** -0.5)
    pool = torch.full((N + 2, H, D, D), 3.0)
    slots = list(range(N + 1, 1, -1))
    pool[slots] = h0
    dq, dk, dv, dg, dpool, dcu = _dev(q, k, v, g, pool, cu)
    ds = torch.tensor(slots, dtype=torch.int32, device="cuda")
    o, final = M.linear_attention(dq, dk, dv, dg, dpool, dcu, initial_slots=ds, final_state=dpool, final_slots=ds)
    torch.cuda.synchronize()
    to, ts = _tolerances(ref, [2 * n for n in lengths], D, torch.bfloat16, g, H)
    _check(final[slots], ref[1], ts, "state")
    _check(o, ref[0], to, "output")
    assert bool((final[:2] == 3.0).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strong_decays_and_resets(cuda, dtype):
    """Decays from none to a full reset (g = -inf forgets everything before the token)."""
    lengths, H, D = [200, 90], 2, 64
    q, k, v, g, h0, cu = _inputs(5, lengths, H, H, D, dtype, "token")
    g[::7] = -40.0
    g[::31] = 0.0
    g[50] = -float("inf")
    g[64] = -float("inf")
    g[127:131] = -float("inf")
    g[230] = -1e4
    ref = _recurrence(q, k, v, g, h0, cu, D ** -0.5)
    dq, dk, dv, dg, dh, dcu = _dev(q, k, v, g, h0, cu)
    o, final = M.linear_attention(dq, dk, dv, dg, dh, dcu)
    torch.cuda.synchronize()
    # exponents: sums between two tokens that still see each other stay below 60 in magnitude
    # where the weight is above 2^-86; smaller weights are below every bound here
    to, ts = _tolerances(ref, lengths, D, dtype, torch.tensor([1.0]), H)
    _check(final, ref[1], ts + 1e-20, "state")
    _check(o, ref[0], to + 1e-20, "output")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_places_do_not_leak(cuda, dtype):
    """NaN and infinities in rows behind a sample's end, in other samples and in other heads stay
    there; rows of out that belong to no sample are left as they were."""
    lengths, H, D = [70, 33, 65], 2, 64
    q, k, v, g, h0, cu = _inputs(6, lengths, H, H, D, dtype, "token")
    pad = 40
    rows = sum(lengths)

    def padded(x, value):
        return torch.cat([x, torch.full((pad, *x.shape[1:]), value, dtype=x.dtype)])

    q, k, v, g = padded(q, float("nan")), padded(k, float("inf")), padded(v, float("nan")), padded(g, float("nan"))
    bad = slice(70, 103)  # the middle sample
    k[bad, 0], v[bad, 0] = float("nan"), float("inf")
    ref = _recurrence(q[:rows], k[:rows], v[:rows], g[:rows], h0, cu, D ** -0.5)
    out = torch.full((rows + pad, H, D), 7.0, dtype=dtype, device="cuda")
    dq, dk, dv, dg, dh, dcu = _dev(q, k, v, g, h0, cu)
    o, final = M.linear_attention(dq, dk, dv, dg, dh, dcu, out=out)
    torch.cuda.synchronize()
    assert bool((o[rows:] == 7.0).all())
    to, ts = _tolerances(ref, lengths, D, dtype, g[:rows], H)
    clean = [r for r in range(rows) if not 70 <= r < 103]
    _check(o[clean], ref[0][clean], to[clean], "output")
    _check(o[bad, 1], ref[0][bad, 1], to[bad, 1], "other head")
    for n in (0, 2):
        _check(final[n], ref[1][n], ts[n], "state")
    _check(final[1, 1], ref[1][1, 1], ts[1, 1], "other head's state")
    assert bool(torch.isnan(final[1, 0]).all()) and bool(torch.isnan(o[bad, 0].float()).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_pools_and_in_place(cuda, dtype):
    """Split views of one projection, an output inside a wider buffer, pools updated in place, an
    input slot outside the pool (zeros), an output slot outside it and one named twice."""
    lengths, Hk, H, D = [40, 77, 5, 64], 1, 2, 64
    q, k, v, g, h0, cu = _inputs(8, lengths, Hk, H, D, dtype, "head")
    L = sum(lengths)
    wide = torch.zeros(L, (2 * Hk + H) * D + 64, dtype=dtype)
    wide[:, :D], wide[:, D:2 * D], wide[:, 2 * D:4 * D] = q[:, 0], k[:, 0], v.reshape(L, H * D)
    wide = wide.cuda()
    q2, k2, v2 = wide[:, :D].view(L, 1, D), wide[:, D:2 * D].view(L, 1, D), wide[:, 2 * D:4 * D].view(L, H, D)
    pool = torch.randn(7, H, D, D, generator=torch.Generator().manual_seed(1))
    ins, outs = [3, 9, 0, 5], [3, 1, -1, 3]
    start = torch.stack([pool[s] if 0 <= s < 7 else torch.zeros_like(pool[0]) for s in ins])
    ref = _recurrence(q, k, v, g, start, cu, 0.3)
    dpool, dg, dcu = _dev(pool, g, cu)
    slots = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    buffer = torch.full((L, H * D + 128), -3.0, dtype=dtype, device="cuda")
    o, final = M.linear_attention(q2, k2, v2, dg, dpool, dcu, scale=0.3, initial_slots=slots(ins),
                                  final_state=dpool, final_slots=slots(outs),
                                  out=buffer[:, 64:64 + H * D].view(L, H, D))
    torch.cuda.synchronize()
    assert final.data_ptr() == dpool.data_ptr() and o.data_ptr() == buffer[:, 64:].data_ptr()
    assert bool((buffer[:, :64] == -3).all()) and bool((buffer[:, 64 + H * D:] == -3).all())
    to, ts = _tolerances(ref, lengths, D, dtype, g, H)
    _check(o, ref[0], to, "output")
    _check(final[3], ref[1][0], ts[0], "slot 3 (first of two)")
    _check(final[1], ref[1][1], ts[1], "slot 1")
    for s in (0, 2, 4, 5, 6):
        assert torch.equal(final[s].cpu(), pool[s])


@gpu
def test_no_initial_state_is_zeros_and_host_offsets(cuda):
    q, k, v, g, h0, cu = _inputs(9, [50, 90], 2, 2, 64, torch.bfloat16, "token")
    dq, dk, dv, dg, dh, dcu = _dev(q, k, v, g, torch.zeros_like(h0), cu)
    a = M.linear_attention(dq, dk, dv, dg, dh, dcu)
    b = M.linear_attention(dq[None], dk[None], dv[None], dg[None], None, cu.long())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_tokens_at_all(cuda, dtype):
    """Only empty samples: the states are copied, in place or not; no decay, no output rows."""
    h0 = torch.randn(3, 2, 64, 64, device="cuda")
    x = torch.empty(0, 2, 64, dtype=dtype, device="cuda")
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    for g in (None, torch.empty(0, 2, device="cuda"), torch.zeros(2, device="cuda")):
        o, final = M.linear_attention(x, x, x, g, h0, cu)
        assert o.shape == (0, 2, 64) and torch.equal(final, h0)
    _, final = M.linear_attention(x, x, x, None, None, cu)
    assert bool((final == 0).all())


@gpu
def test_pools_and_rows_beyond_32_bits(cuda):
    """State pools of more than 2^32 bytes and 2^31 elements, and token rows of more than 2^31 elements."""
    H, D = 16, 128
    pool = torch.empty(8300, H, D, D, device="cuda")  # 2.18e9 elements
    slots = torch.tensor([8299, 1], dtype=torch.int32, device="cuda")
    gen, q, k, v, _ = _step_inputs(3, 2, H, H, D, torch.bfloat16)
    S = torch.randn(2, H, D, D, generator=gen).cuda()
    dq, dk, dv, dg = _dev(q, k, v, -torch.rand(2, H, generator=gen))
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for run in (lambda s, sl: M.linear_attention_step(dq, dk, dv, dg, s, slots=sl),
                lambda s, sl: M.gdn2_step(dq, dk, dv, dg, s, slots=sl),
                lambda s, sl: M.linear_attention(dq, dk, dv, dg, s, cu, initial_slots=sl, final_state=s,
                                                 final_slots=sl)[0]):
        pool[slots.long()] = S
        small = S.clone()
        o, want = run(pool, slots), run(small, torch.arange(2, dtype=torch.int32, device="cuda"))
        assert torch.equal(o, want) and torch.equal(pool[slots.long()], small)
    del pool
    # strong decays: a row depends on the last tokens alone, so a short run gives the last rows
    L, H = 270000, 64
    v = torch.randn(L, H, D, device="cuda", dtype=torch.bfloat16)
    q, k = (torch.nn.functional.normalize(torch.randn(L, 1, D, device="cuda"), dim=-1).bfloat16() for _ in range(2))
    g = torch.full((H,), -1.0, device="cuda")
    o, final = M.linear_attention(q, k, v, g, None, torch.tensor([0, L]))
    t = slice(L - 240 - L % 64, L)  # whole chunks behind its start
    t = slice((t.start // 64) * 64, L)
    o1, final1 = M.linear_attention(q[t], k[t], v[t], g, None, torch.tensor([0, L - t.start]))
    torch.cuda.synchronize()
    # what came before the short run has decayed to e^-200
    assert torch.equal(o[-64:], o1[-64:])
    assert float((final - final1).abs().max()) <= 1e-6 * float(final1.abs().max())


@gpu
@pytest.mark.parametrize("D,lengths", [(128, [130, 64, 300]), (64, [3, 70, 0, 32, 33, 1]), (128, [12, 90, 13, 1, 2]),
                                       (256, [8, 9, 100, 1, 30]), (64, [1] * 70 + [40, 0, 30, 2]),
                                       (256, [1] * 70 + [40, 0, 30, 2])])
def test_samples_are_independent_of_the_pack(cuda, D, lengths):
    """A sample's result does not depend on what it is packed with, bit for bit, while the mean length
    is at most 64 tokens (short samples run token by token, longer ones in chunks, each by its own
    length) or no sample is short."""
    q, k, v, g, h0, cu = _dev(*_inputs(10, lengths, 2, 2, D, torch.bfloat16, "token"))
    o, final = M.linear_attention(q, k, v, g, h0, cu)
    at = 0
    for n, T in enumerate(lengths):
        s = slice(at, at + T)
        o1, f1 = M.linear_attention(q[s], k[s], v[s], g[s], h0[n:n + 1], torch.tensor([0, T]))
        assert torch.equal(o[s], o1) and torch.equal(final[n], f1[0])
        at += T


@gpu
def test_bad_offsets_are_clamped(cuda):
    """Device offsets outside the rows or decreasing never reach outside the tensors."""
    q, k, v, g, h0, _ = _dev(*_inputs(11, [64, 64], 1, 1, 64, torch.bfloat16, "token"))
    for bad in ([0, 200, 128], [-5, 64, 1 << 30], [100, 20, 128]):
        o, final = M.linear_attention(q, k, v, g, h0, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert bool(torch.isfinite(final).all())
    # in segments: samples that overlap add up to more tokens than there are
    q, k, v, g, h0, _ = _dev(*_inputs(11, [3000, 2000, 10], 1, 1, 64, torch.bfloat16, "token"))
    for bad in ([0, 5010, 0, 5010], [0, 5010, -1, 1 << 30]):
        M.linear_attention(q, k, v, g, h0, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cu,L", [([0, 100] * 12, 100), ([0, 90, 40, 60, 60, 61] * 5, 90),   # chunks beside tokens
                                  ([0, 5010, 0, 5010], 5010), ([0, 4000, 1, 3000, 0, 9], 4000)])  # segments
def test_overlapping_samples_are_whole(cuda, D, cu, L):
    """Samples whose offsets overlap add up to more tokens than there are; each still ends in the state
    of its own tokens (rows of the output that two of them share belong to either)."""
    q, k, v, g, _, _ = _inputs(17, [L], 1, 1, D, torch.bfloat16, "token")
    h0 = 0.5 * torch.randn(len(cu) - 1, 1, D, D, generator=torch.Generator().manual_seed(2))
    ranges = [(a, max(a, b)) for a, b in zip(cu[:-1], cu[1:])]
    refs = []
    for n, (a, b) in enumerate(ranges):
        ref = _recurrence(q[a:b], k[a:b], v[a:b], g[a:b], h0[n:n + 1], torch.tensor([0, b - a]), 1.0)
        refs.append((ref, _tolerances(ref, [max(b - a, 1)], D, torch.bfloat16, g, 1)[1]))
    dq, dk, dv, dg, dh = _dev(q, k, v, g, h0)
    final = torch.full_like(dh, float("nan"))
    M.linear_attention(dq, dk, dv, dg, dh, torch.tensor(cu, dtype=torch.int32, device="cuda"), final_state=final)
    torch.cuda.synchronize()
    for n, (ref, tol) in enumerate(refs):
        _check(final[n:n + 1], ref[1], tol, f"state {n}")


@gpu
def test_linear_attention_refuses_arguments(cuda):
    q, k, v, g, h0, cu = _dev(*_inputs(12, [20, 12], 2, 2, 64, torch.bfloat16, "token"))
    f = M.linear_attention
    slots = torch.zeros(2, dtype=torch.int32, device="cuda")
    bad = [
        lambda: f(q.half(), k.half(), v.half(), g, h0, cu), lambda: f(q.float(), k, v, g, h0, cu),
        lambda: f(q[:, :, :32], k[:, :, :32], v[:, :, :32], g, h0, cu), lambda: f(q[:10], k, v, g, h0, cu),
        lambda: f(q.repeat(1, 2, 1)[:, :3], k.repeat(1, 2, 1)[:, :3], v, g, h0, cu),
        lambda: f(q, k, v, g.double(), h0, cu), lambda: f(q, k, v, g[:5], h0, cu),
        lambda: f(q, k, v, g, h0[:1], cu), lambda: f(q, k, v, g, h0.half(), cu),
        lambda: f(q, k, v, g, h0, cu[:1]), lambda: f(q, k, v, g, h0, cu.float()),
        lambda: f(q, k, v, g, h0, torch.tensor([0, 40, 32])), lambda: f(q, k, v, g, h0, torch.tensor([0, 20, 33])),
        lambda: f(q, k, v, g, None, cu, initial_slots=slots), lambda: f(q, k, v, g, h0, cu, final_slots=slots),
        lambda: f(q, k, v, g, h0, cu, initial_slots=slots.long()), lambda: f(q, k, v, g, h0, cu, out=v),
        lambda: f(q, k, v, g, h0, cu, out=torch.empty_like(v).float()),
        lambda: f(q, k, v, g, h0, cu, final_state=torch.empty(2, 2, 64, 128, device="cuda")[..., :64]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")


@gpu
@pytest.mark.parametrize("lengths", [[700, 300], [3000]])
def test_graphs_streams_and_replays(cuda, lengths):
    """Two captured graphs of one stream, replayed together on two streams, and an eager call give
    the same results: no scratch is shared (one long sample: with segments' states in a workspace)."""
    cases = [_dev(*_inputs(20 + i, lengths, 2, 4, 128, torch.bfloat16, "token")) for i in range(2)]
    eager = [M.linear_attention(*c) for c in cases]
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    for c in cases:
        with torch.cuda.stream(stream):
            M.linear_attention(*c)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(M.linear_attention(*c))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (o, f), (eo, ef) in zip(outs, eager):
        assert torch.equal(o, eo) and torch.equal(f, ef)
    again = [M.linear_attention(*c) for c in cases]
    for (o, f), (eo, ef) in zip(again, eager):
        assert torch.equal(o, eo) and torch.equal(f, ef)


# ---------------------------------------------------------------------------
# single-token steps
# ---------------------------------------------------------------------------

def _step_inputs(seed, N, Hk, H, D, dtype):
    gen = torch.Generator().manual_seed(seed)
    unit = lambda x: x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    q, k = (unit(torch.randn(N, Hk, D, generator=gen)).to(dtype) for _ in range(2))
    v = torch.randn(N, H, D, generator=gen).to(dtype)
    sig = lambda *s: torch.sigmoid(torch.randn(*s, generator=gen)).to(dtype)  # noqa: E731
    return gen, q, k, v, sig


def _step_reference(q, k, v, g, S, beta=None, erase=None, write=None, delta=False, incoming=False, scale=1.0):
    """fp64 (o, S_new, A_o, A_S)"""
    rep = v.shape[1] // q.shape[1]
    up = lambda x: x.double().repeat_interleave(rep, 1)  # noqa: E731
    q, k, v, S = up(q), up(k), v.double(), S.double()
    a = torch.ones((), dtype=torch.float64) if g is None else torch.exp(g.double())
    if g is not None:
        a = a[:, :, :, None] if a.dim() == 3 else (a[None, :] if a.dim() == 1 else a)[:, :, None, None]
    new, mag = a * S, a * S.abs()
    if delta:
        if beta is not None:
            b = beta.double().sqrt()
            k = k * up(b if b.dim() == 3 else b[:, :, None])
        kb = k if erase is None else k * up(erase)
        v = v if write is None else v * write.double()
        vm = v.abs() + torch.einsum("nhk,nhkv->nhv", kb.abs(), mag)
        v = v - torch.einsum("nhk,nhkv->nhv", kb, new)
    else:
        vm = v.abs()
    new = new + k[..., :, None] * v[..., None, :]
    mag = mag + k.abs()[..., :, None] * vm[..., None, :]
    src, smag = (S, S.abs()) if incoming else (new, mag)
    return (scale * torch.einsum("nhk,nhkv->nhv", q, src), new,
            scale * torch.einsum("nhk,nhkv->nhv", q.abs(), smag), mag)


def _check_step(o, states, ref, D, dtype):
    # the delta rule's extra sum over D rows enters the state too: (D + 16) u
    _check(states, ref[1], (D + 16) * U * ref[3] + 1e-40, "state")
    _check(o, ref[0], (2 * D + 24) * U * ref[2] + HALF[dtype] * ref[0].abs() * 1.01 + 1e-40, "output")


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("N,Hk,H", [(1, 1, 1), (3, 2, 4), (5, 3, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("decay", ["none", "head", "token"])
def test_linear_attention_step(cuda, D, N, Hk, H, dtype, decay):
    gen, q, k, v, _ = _step_inputs(D + N, N, Hk, H, D, dtype)
    g = {"none": None, "head": -torch.rand(H, generator=gen), "token": -torch.rand(N, H, generator=gen)}[decay]
    S = torch.randn(N, H, D, D, generator=gen)
    ref = _step_reference(q, k, v, g, S, scale=D ** -0.5)
    dq, dk, dv, dg, dS = _dev(q, k, v, g, S)
    o = M.linear_attention_step(dq, dk, dv, dg, dS)
    torch.cuda.synchronize()
    _check_step(o, dS, ref, D, dtype)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gates", ["none", "head", "channel", "erase", "constant"])
@pytest.mark.parametrize("incoming", [False, True])
def test_gdn2_step(cuda, D, dtype, gates, incoming):
    N, Hk, H = 4, 2, 4
    gen, q, k, v, sig = _step_inputs(D, N, Hk, H, D, dtype)
    g = {"none": None, "constant": -torch.rand(H, generator=gen)}.get(
        gates, -torch.rand(*((N, H) if gates == "head" else (N, H, D)), generator=gen))
    beta = {"head": sig(N, Hk), "channel": sig(N, Hk, D), "constant": sig(N, Hk)}.get(gates)
    erase = sig(N, Hk, D) if gates == "erase" else None
    write = sig(N, H, D) if gates in ("channel", "erase") else None
    S = torch.randn(N, H, D, D, generator=gen)
    ref = _step_reference(q, k, v, g, S, beta, erase, write, True, incoming, 0.25)
    dq, dk, dv, dg, dS, db, de, dw = _dev(q, k, v, g, S, beta, erase, write)
    o = M.gdn2_step(dq, dk, dv, dg, dS, beta=db, erase=de, write=dw, scale=0.25, read_incoming=incoming)
    torch.cuda.synchronize()
    _check_step(o, dS, ref, D, dtype)


@gpu
@pytest.mark.parametrize("D,N,H", [(64, 120, 16), (64, 201, 9), (128, 47, 13), (128, 150, 8), (256, 37, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gates", ["head", "channel"])
@pytest.mark.parametrize("incoming", [False, True])
def test_gdn2_step_of_many_sessions(cuda, D, N, H, dtype, gates, incoming):
    """Many sessions, odd counts among them, in a pool with skipped and repeated slots."""
    Hk = H if H % 2 else H // 2
    gen, q, k, v, sig = _step_inputs(N, N, Hk, H, D, dtype)
    g = -torch.rand(*((N, H) if gates == "head" else (N, H, D)), generator=gen)
    beta = sig(N, Hk) if gates == "head" else sig(N, Hk, D)
    erase, write = (None, None) if gates == "head" else (sig(N, Hk, D), sig(N, H, D))
    pool = torch.randn(N + 3, H, D, D, generator=gen)
    slots = torch.randperm(N + 3, generator=gen)[:N].to(torch.int32)
    slots[5], slots[9], slots[20] = -1, N + 3, slots[2]
    live = [i for i in range(N) if i not in (5, 9, 20)]
    at = slots[live].long()
    pick = lambda x: None if x is None else x[live]  # noqa: E731
    ref = _step_reference(q[live], k[live], v[live], g[live], pool[at], pick(beta), pick(erase), pick(write), True,
                          incoming, 0.25)
    dq, dk, dv, dg, dp, ds, db, de, dw = _dev(q, k, v, g, pool, slots, beta, erase, write)
    out = torch.full((N, H, D), 5.0, dtype=dtype, device="cuda")
    o = M.gdn2_step(dq, dk, dv, dg, dp, beta=db, erase=de, write=dw, scale=0.25, slots=ds, read_incoming=incoming, out=out)
    torch.cuda.synchronize()
    _check_step(o[live], dp[at.cuda()], ref, D, dtype)
    assert bool((o[[5, 9, 20]] == 5.0).all())
    untouched = sorted(set(range(N + 3)) - set(at.tolist()))
    assert torch.equal(dp[untouched].cpu(), pool[untouched])


@gpu
@pytest.mark.parametrize("rule", ["linear", "gdn2"])
def test_step_pools_views_and_skipped_rows(cuda, rule):
    """Slots of a pool; a slot outside it and a slot named twice are skipped, with their rows of o;
    q, k, v as split views, o inside a wider buffer."""
    N, H, D = 6, 2, 128
    gen, q, k, v, _ = _step_inputs(1, N, H, H, D, torch.bfloat16)
    g = -torch.rand(N, H, generator=gen)
    pool = torch.randn(9, H, D, D, generator=gen)
    slots = [8, -1, 2, 9, 8, 0]
    live = [0, 2, 5]
    at = [slots[i] for i in live]
    ref = _step_reference(q[live], k[live], v[live], g[live], pool[at], delta=rule == "gdn2", scale=0.5)
    wide = torch.cat([q.reshape(N, -1), k.reshape(N, -1), v.reshape(N, -1)], 1).cuda()
    qv, kv, vv = (wide[:, i * H * D:(i + 1) * H * D].view(N, H, D) for i in range(3))
    dpool, dg = _dev(pool, g)
    buffer = torch.full((N, H * D + 64), 5.0, dtype=torch.bfloat16, device="cuda")
    step = M.gdn2_step if rule == "gdn2" else M.linear_attention_step
    o = step(qv, kv, vv, dg, dpool, scale=0.5, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"),
             out=buffer[:, 64:].view(N, H, D))
    torch.cuda.synchronize()
    _check_step(o[live], dpool[at], ref, D, torch.bfloat16)
    assert bool((o[[1, 3, 4]] == 5.0).all()) and bool((buffer[:, :64] == 5.0).all())
    for s in (1, 3, 4, 5, 6, 7):
        assert torch.equal(dpool[s].cpu(), pool[s])


@gpu
def test_empty_batch_and_refused_steps(cuda):
    _, q, k, v, sig = _step_inputs(2, 3, 2, 2, 64, torch.bfloat16)
    dq, dk, dv = _dev(q, k, v)
    S = torch.zeros(3, 2, 64, 64, device="cuda")
    assert M.linear_attention_step(dq[:0], dk[:0], dv[:0], None, S[:0]).shape == (0, 2, 64)
    g3 = torch.zeros(3, 2, 64, device="cuda")
    b = sig(3, 2).cuda()
    bad = [
        lambda: M.linear_attention_step(dq, dk, dv, g3, S), lambda: M.linear_attention_step(dq, dk, dv, None, S[:2]),
        lambda: M.linear_attention_step(dq, dk, dv, None, S.half()),
        lambda: M.linear_attention_step(dq, dk, dv, None, S.transpose(0, 1)),
        lambda: M.linear_attention_step(dq, dk, dv, None, S, slots=torch.zeros(3, device="cuda", dtype=torch.int64)),
        lambda: M.linear_attention_step(dq, dk, dv, None, S, out=dv), lambda: M.gdn2_step(dq, dk, dv, None, S, beta=b.float()),
        lambda: M.gdn2_step(dq, dk, dv, None, S, beta=b[:, :1]), lambda: M.gdn2_step(dq, dk, dv, None, S, erase=b),
        lambda: M.gdn2_step(dq, dk, dv, None, S, write=dv.float()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")


@gpu
def test_step_matches_the_update_it_stands_beside(cuda):
    """gdn2_step in fp32 is gdn2_update's fp32 recurrence on one-token samples: fp32 rounding of
    two orders of the same sums ((D + 16) u each)."""
    N, H, D = 5, 3, 64
    gen, q, k, v, sig = _step_inputs(4, N, H, H, D, torch.float32)
    g, S = -torch.rand(N, H, generator=gen), torch.randn(N, H, D, D, generator=gen)
    beta, write = sig(N, H), sig(N, H, D)
    ref = _step_reference(q, k, v, g, S, beta, None, write, True)
    dq, dk, dv, dg, dS, db, dw = _dev(q, k, v, g, S, beta, write)
    final = M.gdn2_update(dk, dv, dg, dS, torch.arange(N + 1, dtype=torch.int32, device="cuda"), num_samples=N,
                          total_tokens=N, beta=db, write=dw)
    M.gdn2_step(dq, dk, dv, dg, dS, beta=db, write=dw)
    torch.cuda.synchronize()
    _check(final, dS.double().cpu(), 2 * (D + 16) * U * ref[3], "state")


@gpu
def test_step_in_a_graph_advances_the_states(cuda):
    N, H, D = 3, 2, 128
    gen, q, k, v, _ = _step_inputs(6, N, H, H, D, torch.bfloat16)
    dq, dk, dv, dg, S = _dev(q, k, v, -torch.rand(N, H, generator=gen), torch.randn(N, H, D, D, generator=gen))
    eager = S.clone()
    for _ in range(4):
        want = M.linear_attention_step(dq, dk, dv, dg, eager)
    out = torch.empty_like(dv)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    keep = S.clone()
    with torch.cuda.stream(stream):
        M.linear_attention_step(dq, dk, dv, dg, S, out=out)
    stream.synchronize()
    S.copy_(keep)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        M.linear_attention_step(dq, dk, dv, dg, S, out=out)
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(S, eager) and torch.equal(out, want)


# ---------------------------------------------------------------------------
# a serving run: rotary, prompts, then decode steps
# ---------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_steps_equal_one_long_prompt(cuda, dtype):
    """Rotated prompts through linear_attention into a pool, then six decode tokens through rotary
    and linear_attention_step, against the 64-bit recurrence over the whole sequences."""
    prompts, extra, Hk, H, D = [90, 17], 6, 2, 4, 64
    full = [p + extra for p in prompts]
    q, k, v, g, h0, cu = _inputs(30, full, Hk, H, D, dtype, "token")
    inv, att = M.rotary_frequencies(32, scaling="yarn", factor=4.0, trained_tokens=64)
    pos = torch.cat([torch.arange(n) for n in full]) + 1000
    dq, dk, dv, dg, dpos = _dev(q, k, v, g, pos)
    rq, rk = M.rotary(dq, dk, dpos, inv, attention_scale=att)
    scale = D ** -0.5
    ref = _recurrence(rq.cpu(), rk.cpu(), v, g, h0, cu, scale)
    pool = torch.zeros(4, H, D, D, device="cuda")
    slots = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    pool[slots.long()] = h0.cuda()
    start = [0, full[0]]
    rows = torch.cat([torch.arange(s, s + p) for s, p in zip(start, prompts)]).cuda()
    pq, pk = M.rotary(dq[rows], dk[rows], dpos[rows], inv, attention_scale=att)
    cu_p = torch.tensor([0, prompts[0], sum(prompts)], dtype=torch.int32, device="cuda")
    o, _ = M.linear_attention(pq, pk, dv[rows], dg[rows], pool, cu_p, initial_slots=slots, final_state=pool,
                              final_slots=slots)
    to, ts = _tolerances(ref, full, D, dtype, g, H)
    got = torch.zeros(sum(full), H, D, device="cuda", dtype=dtype)
    got[rows] = o
    for i in range(extra):
        at = torch.tensor([s + p + i for s, p in zip(start, prompts)], device="cuda")
        sq, sk = M.rotary(dq[at], dk[at], dpos[at], inv, attention_scale=att)
        got[at] = M.linear_attention_step(sq, sk, dv[at], dg[at], pool, slots=slots)
    torch.cuda.synchronize()
    _check(got, ref[0], to, "outputs")
    _check(pool[[2, 0]], ref[1], ts + (8 * extra + 8) * U * ref[3], "states")
    assert bool((pool[[1, 3]] == 0).all())
