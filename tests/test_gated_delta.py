"""The gated delta rule over prompts: refusals of the C entry on CPU, values on the GPU against the recurrence
in 64 bits on the same (rounded) inputs.

Tolerances. Every value column s of a state goes its own way, s' = (I - beta k k^T) a s + beta k v, and for
beta |k|^2 <= 2 that map does not lengthen a difference. So an error grows by no more than what each step adds, and
the bounds are bounds of columns in the 2-norm (and of single outputs). With u = 2^-24 (half an fp32 step):
  * token by token, both sums over D rows are at most D / 32 packed additions of two rows on each of 32 / 4
    (D = 256: 32 / 2) lanes and an exchange between them: <= 14 roundings; the decay (expf: 2 u), products and sums of
    the correction and the update are 8 more. One token adds at most u (24 |a s| + 10 |v|) for |k|, beta <= 1 (2^-7 of
    slack for rounded keys is in the constants), its output u 24 scale |q| |s|.
  * in chunks of 64 tokens, with T = (I + A)^-1, r = beta (v - f K s), U = T r, s' = a s + (w K)^T U: each of s, T, r and
    w U enters its product as two bf16 terms (2^-16 relative is left out; the product of two remainders too), which
    add truncating to an fp32 sum: 2 u for each of the D, 64 or 64 terms, two or three times. Norms of K, T and w K are
    those of the chunk in hand. T is inverted in fp32: 64 u |T| (1 + |A|) of itself, and A carries 2 D + 20 + 7 r
    roundings for decays that sum to r in log2 (beyond r = 30 the weight itself is below u). The carried
    state: 4 u.
  * over segments a sample's state is M s + H with a matrix M and sums H that walks of their own have made. A column's
    error in such a walk is a linear map's of that column; over the columns of M it adds up in the Frobenius norm, which for
    columns of length <= 1 is sqrt(D) times the bound of one, against |s| then. Sums and matrix do not share r and u:
    norms of their parts stand for those of the whole. The product itself: D additions on |M| |s| <= sqrt(D) |s|.
  * its outputs round the state's copy, the scores and U to bf16 (half a step: 2^-8 each, elementwise in the sums
    over absolute values) on top of the state's own error times |q|.
Each output is rounded once more to its type.
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
# refusals of the C entry point (nothing is launched)
# ---------------------------------------------------------------------------

def _args(**over):
    """Arguments apart from one another, at addresses that nothing reads."""
    mb = 1 << 20
    f = dict(num_samples=1, num_heads=4, num_key_heads=2, head_dim=64, dtype=_lib.MEMT_BF16, total_tokens=8,
             cu_seqlens=mb, q=2 * mb, q_stride=128, k=3 * mb, k_stride=128, v=4 * mb, v_stride=256, g=5 * mb,
             g_layout=_lib.GATE_PER_HEAD, beta=6 * mb, beta_layout=_lib.GATE_PER_VALUE_HEAD, scale=1.0, out=7 * mb,
             out_stride=256, final_state=8 * mb)
    f.update(over)
    return _lib.GatedDeltaArgs(**f)


BAD = [
    (dict(struct_size=8), "INVALID_ARGUMENT"), (dict(num_samples=0), "INVALID_ARGUMENT"),
    (dict(num_heads=3), "INVALID_ARGUMENT"), (dict(num_key_heads=0), "INVALID_ARGUMENT"),
    (dict(total_tokens=-1), "INVALID_ARGUMENT"), (dict(total_tokens=2 ** 31), "INVALID_ARGUMENT"),
    (dict(dtype=5), "INVALID_ARGUMENT"), (dict(head_dim=96), "UNSUPPORTED"), (dict(q=None), "INVALID_ARGUMENT"),
    (dict(out=None), "INVALID_ARGUMENT"), (dict(cu_seqlens=None), "INVALID_ARGUMENT"),
    (dict(final_state=None), "INVALID_ARGUMENT"), (dict(g=None), "INVALID_ARGUMENT"),
    (dict(g_layout=_lib.GATE_NONE), "INVALID_ARGUMENT"), (dict(g_layout=_lib.GATE_PER_CHANNEL), "INVALID_ARGUMENT"),
    (dict(g_layout=_lib.GATE_PER_VALUE_HEAD), "INVALID_ARGUMENT"),
    (dict(beta=None), "INVALID_ARGUMENT"), (dict(beta_layout=_lib.GATE_NONE), "INVALID_ARGUMENT"),
    (dict(beta_layout=_lib.GATE_PER_CHANNEL), "INVALID_ARGUMENT"),
    (dict(beta_layout=_lib.GATE_CONSTANT), "INVALID_ARGUMENT"), (dict(beta_layout=-1), "INVALID_ARGUMENT"),
    (dict(q_stride=120), "INVALID_ARGUMENT"), (dict(v_stride=128), "INVALID_ARGUMENT"),
    (dict(out_stride=128), "INVALID_ARGUMENT"), (dict(k_stride=132), "MISALIGNED"),
    (dict(v=(4 << 20) + 8), "MISALIGNED"), (dict(final_state=(8 << 20) + 4), "MISALIGNED"),
    (dict(initial_slots=16, num_initial_slots=1), "INVALID_ARGUMENT"),
    (dict(final_slots=16, num_final_slots=0), "INVALID_ARGUMENT"),
    # states of two samples (64 KB each) that overlap by one
    (dict(num_samples=2, initial_state=(8 << 20) + 65536), "INVALID_ARGUMENT"),
    # what is written over what is read
    (dict(out=(6 << 20) + 32), "INVALID_ARGUMENT"), (dict(out=5 << 20), "INVALID_ARGUMENT"),
    (dict(out=4 << 20), "INVALID_ARGUMENT"), (dict(out=(8 << 20) + 1024), "INVALID_ARGUMENT"),
    (dict(beta=(8 << 20) + 256), "INVALID_ARGUMENT"), (dict(cu_seqlens=(8 << 20) + 256), "INVALID_ARGUMENT"),
]


@pytest.mark.parametrize("over,error", BAD)
def test_gated_delta_refuses(over, error):
    a = _args(**over)
    need = _lib.load().memt_gated_delta_workspace_size(1, 8, 4, 64, _lib.MEMT_BF16)
    assert need == 256
    assert _lib.load().memt_gated_delta(ctypes.byref(a), None, 0, None) == getattr(_lib, "MEMT_ERR_" + error)


def _step_args(**over):
    f = dict(rule=_lib.RULE_GATED_DELTA, num_samples=0, num_heads=4, num_key_heads=2, head_dim=64, dtype=_lib.MEMT_BF16,
             q=16, q_stride=128, k=16, k_stride=128, v=16, v_stride=256, g=16, g_layout=_lib.GATE_PER_HEAD, beta=16,
             beta_layout=_lib.GATE_PER_VALUE_HEAD, states=16, scale=1.0, out=16, out_stride=256)
    f.update(over)
    return _lib.RecurrentStepArgs(**f)


def test_step_refuses_what_other_rules_have():
    call = lambda **over: _lib.load().memt_recurrent_step(ctypes.byref(_step_args(**over)), None)  # noqa: E731
    assert call() == _lib.MEMT_OK and call(beta_layout=_lib.GATE_PER_HEAD) == _lib.MEMT_OK
    for over in (dict(g_layout=_lib.GATE_PER_CHANNEL), dict(beta_layout=_lib.GATE_PER_CHANNEL), dict(erase=16),
                 dict(write=16), dict(read_incoming=1), dict(rule=_lib.RULE_GDN2)):
        assert call(**over) == _lib.MEMT_ERR_UNSUPPORTED
    for over in (dict(beta=None), dict(beta_layout=_lib.GATE_CONSTANT), dict(beta_layout=5), dict(rule=4)):
        assert call(**over) == _lib.MEMT_ERR_INVALID_ARGUMENT


def test_gated_delta_refuses_nothing_at_all_and_sizes():
    lib = _lib.load()
    assert lib.memt_gated_delta(None, None, 0, None) == _lib.MEMT_ERR_INVALID_ARGUMENT
    f = lib.memt_gated_delta_workspace_size
    assert f(0, 100, 1, 64, _lib.MEMT_BF16) == 0 and f(1, 100, 1, 96, _lib.MEMT_BF16) == 0
    assert f(1, -1, 1, 64, _lib.MEMT_BF16) == 0 and f(1, 100, 1, 64, 9) == 0
    assert f(1, 0, 1, 64, _lib.MEMT_BF16) >= 256 and f(1, 65536, 16, 128, _lib.MEMT_F32) == 256


def test_gated_delta_refuses_host_tensors():
    x, b = torch.zeros(3, 2, 64), torch.zeros(3, 2)
    with pytest.raises(ValueError):
        M.gated_delta(x, x, x, None, b, torch.zeros(3, 2, 64, 64), torch.tensor([0, 1, 2, 3]))


# ---------------------------------------------------------------------------
# the definition in 64 bits, and bounds of what the kernels may add
# ---------------------------------------------------------------------------

def _wide(q, k, v, g, beta):
    """fp64 q, k [L, H, D], v, decays [L, H], beta [L, H]."""
    L, H, _ = v.shape
    rep = H // q.shape[1]
    q, k = (x.double().repeat_interleave(rep, 1) for x in (q, k))
    a = torch.ones(L, H, dtype=torch.float64, device=v.device) if g is None else g.double().exp().expand(L, H)
    b = torch.ones_like(a) if beta is None else beta.double()
    return q, k, v.double(), a, b if b.shape[1] == H else b.repeat_interleave(rep, 1)


def _recurrence(q, k, v, g, beta, h0, cu, scale):
    """fp64 (o, final), and bounds of the token-by-token form's errors: of o, and of the columns of final [N, H, D]."""
    L, H, D = v.shape
    q, k, v, a, b = _wide(q, k, v, g, beta)
    S = h0.double().clone()
    E = torch.zeros(S.shape[0], H, D, dtype=torch.float64, device=v.device)
    o, A = torch.zeros_like(v), torch.zeros_like(v)
    for n in range(len(cu) - 1):
        for t in range(int(cu[n]), int(cu[n + 1])):
            at = a[t][:, None, None] * S[n]
            d = b[t][:, None] * (v[t] - torch.einsum("hk,hkv->hv", k[t], at))
            S[n] = at + k[t][:, :, None] * d[:, None, :]
            o[t] = scale * torch.einsum("hk,hkv->hv", q[t], S[n])
            E[n] = a[t][:, None] * E[n] + U * (24 * at.norm(dim=1) + 10 * v[t].abs())
            A[t] = abs(scale) * q[t].norm(dim=1)[:, None] * (E[n] + 24 * U * (at.norm(dim=1) + S[n].norm(dim=1)))
    return o, S, A, E


def _chunk_bounds(q, k, v, g, beta, h0, cu, scale, joined=0):
    """The same of the chunked form: (bound of o, of the columns of final); joined: D, with segments."""
    L, H, D = v.shape
    q, k, v, a, b = _wide(q, k, v, g, beta)
    S = h0.double().clone()
    E = torch.zeros(S.shape[0], H, D, dtype=torch.float64, device=v.device)
    A = torch.zeros_like(v)
    two, bf = lambda x: torch.linalg.matrix_norm(x, 2), 2.0 ** -8  # noqa: E731
    for n in range(len(cu) - 1):
        for t0 in range(int(cu[n]), int(cu[n + 1]), 64):
            t1 = min(t0 + 64, int(cu[n + 1]))
            kc, qc, vc = (x[t0:t1].transpose(0, 1) for x in (k, q, v))           # [H, C, D]
            G = a[t0:t1].clamp(min=1e-300).log().cumsum(0).T                     # [H, C]
            f, w, bc = G.exp()[..., None], (G[:, -1:] - G).exp()[..., None], b[t0:t1].T[..., None]
            i = torch.arange(t1 - t0, device=v.device)
            causal = i[:, None] >= i
            weight = torch.where(causal, G[:, :, None] - G[:, None, :], -torch.inf).exp()
            low = (kc @ kc.transpose(1, 2)) * weight * bc * (i[:, None] > i)
            T = torch.linalg.inv(torch.eye(t1 - t0, dtype=torch.float64, device=v.device) + low)
            r = bc * (vc - f * (kc @ S[n]))
            u = T @ r
            nk, nT, nA, nw = two(kc)[:, None], two(T)[:, None], two(low)[:, None], two(w * kc)[:, None]
            total = min(float(G.abs().max()) * 1.4427, 30.0)
            cols = lambda x: x.norm(dim=1)                                       # noqa: E731  [H, C, D] -> [H, D]
            s, rn, un = cols(S[n]), cols(r), cols(u)
            dr = nk * (2.0 ** -16 + 4 * D * U) * s * (1 + joined ** 0.5) + 4 * U * cols(vc) + (2.0 ** -16 + 4 * U) * rn
            dT = (2.0 ** -15 + 384 * U) * T.flatten(1).norm(dim=1)[:, None] + 64 * U * nT * (1 + nA) \
                + (2 * D + 20 + 7 * total) * U * nT ** 2 * low.flatten(1).norm(dim=1)[:, None]
            du = nT * dr + dT * rn + nk * nT * E[n]
            ru, uu = rn, un
            if joined:  # the segment's own sums and the matrix on s apart
                ru = (1 + joined ** 0.5) * (cols(bc * vc) + nk * s)
                uu = nT * ru
            step = nw * (nT * dr + dT * ru + (2.0 ** -16 + 256 * U + 7 * total * U) * uu)
            inter = f * (qc.abs() @ S[n].abs())
            scores = (qc @ kc.transpose(1, 2)).abs() * weight
            A[t0:t1] = abs(scale) * ((3 * bf * (inter + scores @ u.abs()) + 2 * bf * bf * inter)
                                     + f * qc.norm(dim=2, keepdim=True) * E[n][:, None]
                                     + scores.norm(dim=2, keepdim=True) * du[:, None]).transpose(0, 1)
            keep = G[:, -1].exp()[:, None]
            S[n] = keep[..., None] * S[n] + (w * kc).transpose(1, 2) @ u
            E[n] = keep * E[n] + step + (4 + 3 * joined) * U * cols(S[n])
            if joined:  # (a product with each segment's matrix at most a chunk, |M| <= 1)
                E[n] += joined ** 1.5 * U * s
    return A, E


def _inputs(seed, lengths, Hk, H, D, dtype, decay="token", gscale=1.0, beta="value", alike=0.0):
    gen = torch.Generator().manual_seed(seed)
    L, N = sum(lengths), len(lengths)
    unit = lambda x: x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    q = unit(torch.randn(L, Hk, D, generator=gen)).to(dtype)
    k = unit(torch.randn(L, Hk, D, generator=gen) + alike * torch.randn(1, Hk, D, generator=gen)).to(dtype)
    v = torch.randn(L, H, D, generator=gen).to(dtype)
    g = {"none": None, "head": -torch.exp2(-8.0 * torch.arange(1, H + 1) / H),
         "token": torch.nn.functional.logsigmoid(2 + 0.5 * torch.randn(L, H, generator=gen))}[decay]
    g = None if g is None else g * gscale
    b = {"none": None, "key": torch.rand(L, Hk, generator=gen).to(dtype),
         "value": torch.rand(L, H, generator=gen).to(dtype)}[beta]
    h0 = 0.5 * torch.randn(N, H, D, D, generator=gen)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32)
    return tuple(None if x is None else x.cuda() for x in (q, k, v, g, b, h0)) + (cu,)


def _check(o, final, x, dtype, scale, joined=False):
    """Outputs and final states against the definition; `x` as from _inputs. joined: samples walked in segments."""
    q, k, v, g, b, h0, cu = x
    ref_o, ref_s, A, E = _recurrence(q, k, v, g, b, h0, cu, scale)
    if dtype is torch.bfloat16:  # either form
        Ac, Ec = _chunk_bounds(q, k, v, g, b, h0, cu, scale, v.shape[2] if joined else 0)
        A, E = torch.maximum(A, Ac), torch.maximum(E, Ec)
    eo, es = (o.double() - ref_o).abs(), (final.double() - ref_s).norm(dim=2)
    to = A * 1.01 + HALF[dtype] * (ref_o.abs() + A) + 1e-40
    assert not bool(torch.isnan(eo).any()) and not bool(torch.isnan(es).any())
    assert bool((es <= E * 1.01 + 1e-40).all()), f"state: worst {float((es / (E + 1e-40)).max()):.3g} of its bound"
    assert bool((eo <= to).all()), f"output: worst {float((eo / to).max()):.3g} of its bound"


def _run_and_check(lengths, Hk, H, D, dtype, seed=0, **kinds):
    x = _inputs(seed, lengths, Hk, H, D, dtype, **kinds)
    before = x[5].clone()
    o, final = M.gated_delta(*x)
    torch.cuda.synchronize()
    assert o.dtype == dtype and torch.equal(x[5], before)
    _check(o, final, x, dtype, D ** -0.5)
    return o, final


def test_bounds_and_chunks_are_of_the_same_recurrence():
    """On the CPU: the chunk quantities that the bounds use give the recurrence's states, and the states' derivative
    along a difference is no longer than the difference (what the bounds rest on)."""
    gen = torch.Generator().manual_seed(3)
    L, H, D = 100, 2, 16
    k = torch.nn.functional.normalize(torch.randn(L, H, D, generator=gen).double(), dim=-1)
    q, v = torch.randn(L, H, D, generator=gen).double(), torch.randn(L, H, D, generator=gen).double()
    g, b = -torch.rand(L, H, generator=gen), torch.rand(L, H, generator=gen).double()
    h0, h1 = torch.randn(1, H, D, D, generator=gen), torch.randn(1, H, D, D, generator=gen)
    cu = torch.tensor([0, L])
    o, S, _, E = _recurrence(q, k, v, g, b, h0, cu, 1.0)
    _, S1, _, _ = _recurrence(q, k, v, g, b, h1, cu, 1.0)
    assert bool(((S1 - S).norm(dim=2) <= (h1 - h0).double().norm(dim=2)).all()) and bool((E > 0).all())
    s = h0.double()[0]
    for t0 in (0, 64):
        t1 = min(t0 + 64, L)
        G = g[t0:t1].double().cumsum(0).T
        kc, vc, bc = k[t0:t1].transpose(0, 1), v[t0:t1].transpose(0, 1), b[t0:t1].T[..., None]
        i = torch.arange(t1 - t0)
        weight = torch.where(i[:, None] >= i, G[:, :, None] - G[:, None, :], -torch.inf).exp()
        low = (kc @ kc.transpose(1, 2)) * weight * bc * (i[:, None] > i)
        u = torch.linalg.solve(torch.eye(t1 - t0).double() + low, bc * (vc - G.exp()[..., None] * (kc @ s)))
        scores = (q[t0:t1].transpose(0, 1) @ kc.transpose(1, 2)) * weight
        oc = G.exp()[..., None] * (q[t0:t1].transpose(0, 1) @ s) + scores @ u
        assert torch.allclose(oc.transpose(0, 1), o[t0:t1], atol=1e-11)
        s = G[:, -1].exp()[:, None, None] * s + ((G[:, -1:] - G).exp()[..., None] * kc).transpose(1, 2) @ u
    assert torch.allclose(s, S[0], atol=1e-11)


# ---------------------------------------------------------------------------
# values
# ---------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lengths", [[1], [8], [13], [33], [63], [64], [65], [128, 1, 0, 200], [0, 3, 130], [25, 1, 9]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths(cuda, D, lengths, dtype):
    _run_and_check(lengths, 1, 2, D, dtype)


@gpu
@pytest.mark.parametrize("decay", ["none", "head", "token"])
@pytest.mark.parametrize("beta", ["none", "key", "value"])
@pytest.mark.parametrize("Hk,H", [(1, 3), (2, 4), (3, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_heads_and_gates(cuda, decay, beta, Hk, H, dtype):
    _run_and_check([70, 130], Hk, H, 64, dtype, decay=decay, beta=beta)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("decay", ["none", "head", "token"])
def test_many_chunks(cuda, D, decay):
    _run_and_check([64 * 9 + 5, 64 * 6], 2, 2, D, torch.bfloat16, decay=decay)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lengths,decay", [([2900], "token"), ([2200], "none"), ([64 * 60, 7, 5000, 0], "head")])
def test_segments(cuda, D, lengths, decay):
    """Few long samples: walked in segments, each twice."""
    Hk, H = (1, 2) if len(lengths) == 1 else (1, 1)
    x = _inputs(4, lengths, Hk, H, D, torch.bfloat16, decay=decay)
    need = _lib.load().memt_gated_delta_workspace_size
    chunked = (sum(lengths) // 64 + len(lengths)) * H * 20480 + 256
    assert need(len(lengths), sum(lengths), H, D, _lib.MEMT_BF16) > chunked  # (holds states of segments)
    o, final = M.gated_delta(*x)
    _check(o, final, x, torch.bfloat16, D ** -0.5, joined=True)
    # without a first state, and in place
    zero = torch.zeros_like(x[5])
    ref = M.gated_delta(*x[:5], zero, x[6])
    got = M.gated_delta(*x[:5], None, x[6])
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
    states = x[5].clone()
    o2, _ = M.gated_delta(*x[:5], states, x[6], final_state=states)
    assert torch.equal(o, o2) and torch.equal(states, final)


@gpu
@pytest.mark.parametrize("what", ["v", "k"])
def test_segments_with_a_token_that_is_not_finite(cuda, what):
    L, H, D, t = 2500, 1, 64, 1301
    x = list(_inputs(6, [L], 1, H, D, torch.bfloat16))
    o, final = M.gated_delta(*x)
    x["k v".split().index(what) + 1][t, 0, 5] = float("inf")
    o2, f2 = M.gated_delta(*x)
    others = torch.arange(D, device="cuda") != 5
    cols = others if what == "v" else torch.zeros_like(others)
    near = 0.06 * float(o.float().abs().max())  # the column and its neighbours are made again, in the other form
    assert bool(((o2[:t].float() - o[:t].float()).abs() <= near).all())
    assert bool(((o2[:, :, cols].float() - o[:, :, cols].float()).abs() <= near).all())
    assert bool(((f2[..., cols] - final[..., cols]).abs() <= 1e-3).all())
    assert not bool(torch.isfinite(o2[t:, :, ~cols]).any()) and not bool(torch.isfinite(f2[..., ~cols]).any())


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_keys_that_are_alike(cuda, D, dtype):
    """Tokens that overwrite one another: the triangular system is far from the identity."""
    _run_and_check([200, 64], 1, 2, D, dtype, decay="head", beta="none", alike=8.0)
    _run_and_check([150], 1, 2, D, dtype, decay="token", beta="value", alike=3.0)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("decay", ["none", "head", "token"])
def test_few_tokens_beside_prompts(cuda, D, decay):
    _run_and_check([1, 90, 3, 0, 8, 70, 12, 30, 2], 1, 2, D, torch.bfloat16, decay=decay)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_strong_decays_and_resets(cuda, dtype, D):
    """Decays that leave nothing, also several in a block of tokens, and -inf: the state restarts there."""
    x = list(_inputs(5, [150, 70], 1, 2, D, dtype, decay="token", gscale=20.0))
    for t in (0, 17, 18, 63, 64, 100, 149, 160):
        x[3][t, 0] = -1e4
    o, final = M.gated_delta(*x)
    _check(o, final, x, dtype, D ** -0.5)
    x[3][30] = -float("inf")
    x[3][31, 1] = -float("inf")
    x[3][130:140] = -float("inf")
    y = list(x)
    y[3] = x[3].clamp(min=-2e3)  # e^-2000 is zero in 64 bits as well
    o, final = M.gated_delta(*x)
    _check(o, final, y, dtype, D ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_pools_and_in_place(cuda, dtype):
    lengths, Hk, H, D = [70, 0, 5, 130], 2, 4, 64
    x = _inputs(7, lengths, Hk, H, D, dtype)
    q, k, v, g, b, h0, cu = x
    scale, L = 0.3, sum(lengths)
    wide = torch.full((L, (2 * Hk + H) * D + 16), 7.0, device="cuda", dtype=dtype)
    views = []
    for at, y in ((0, q), (Hk * D, k), (2 * Hk * D, v)):
        n = y.shape[1] * D
        wide[:, at:at + n] = y.reshape(L, n)
        views.append(wide[:, at:at + n].view(L, y.shape[1], D))
    pool = torch.full((7, H, D, D), 3.0, device="cuda")
    slots = torch.tensor([5, 0, 2, 6], dtype=torch.int32, device="cuda")
    pool[slots.long()] = h0
    buf = torch.full((L + 5, H * D + 8), -3.0, device="cuda", dtype=dtype)
    out = buf[:L, :H * D].view(L, H, D)
    o, final = M.gated_delta(*views, g, b, pool, cu.cuda(), scale=scale, out=out, initial_slots=slots, final_state=pool,
                             final_slots=slots)
    assert final is pool and o.data_ptr() == out.data_ptr()
    _check(o, pool[slots.long()], x, dtype, scale)
    assert bool((buf[L:] == -3.0).all()) and bool((buf[:, H * D:] == -3.0).all())
    assert bool((pool[[1, 3, 4]] == 3.0).all()) and bool((wide[:, -16:] == 7.0).all())
    # without slots, in place; without a state; a leading 1
    s = h0.clone()
    o2, f2 = M.gated_delta(q[None], k[None], v[None], g[None], b[None], s, cu, scale=scale, final_state=s)
    assert f2 is s and torch.equal(o2, o) and torch.equal(s, pool[slots.long()])
    zero = _inputs(7, lengths, Hk, H, D, dtype)[:5] + (torch.zeros_like(h0), cu)
    o3, f3 = M.gated_delta(q, k, v, g, b, None, cu.cuda().long(), scale=scale)
    _check(o3, f3, zero, dtype, scale)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[3, 1, 2, 5], [90, 70, 100, 3]])
def test_slots_outside_the_pool_and_named_twice(cuda, dtype, lengths):
    H, D = 2, 128
    x = _inputs(9, lengths, 1, H, D, dtype)
    q, k, v, g, b, h0, cu = x
    pool = torch.zeros(3, H, D, D, device="cuda")
    pool[:] = h0[:3]
    first = torch.tensor([1, -1, 3, 0], dtype=torch.int32, device="cuda")     # two of them outside
    last = torch.tensor([2, 2, -1, 1], dtype=torch.int32, device="cuda")      # slot 2 twice, one outside
    final = torch.full((3, H, D, D), 9.0, device="cuda")
    o, _ = M.gated_delta(q, k, v, g, b, pool, cu, initial_slots=first, final_state=final, final_slots=last)
    start = torch.stack([h0[1], torch.zeros_like(h0[0]), torch.zeros_like(h0[0]), h0[0]])
    plain = torch.empty(4, H, D, D, device="cuda")
    o2, _ = M.gated_delta(q, k, v, g, b, start, cu, final_state=plain)
    assert torch.equal(o, o2)
    _check(o2, plain, (q, k, v, g, b, start, cu), dtype, D ** -0.5)
    assert torch.equal(final[2], plain[0]) and torch.equal(final[1], plain[3]) and bool((final[0] == 9.0).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_behind_the_last_sample_and_clamped_offsets(cuda, dtype):
    """Rows that no sample has keep what they held, whatever stands in the inputs there; bad offsets are clamped."""
    H, D, L = 2, 64, 90
    x = _inputs(11, [40, L - 40], 1, H, D, dtype)
    q, k, v, g, b, h0, _ = x
    for y in (q, k, v):
        y[70:] = float("nan")
    g[70:], b[70:] = float("nan"), float("nan")
    out = torch.full((L, H, D), 5.0, device="cuda", dtype=dtype)
    o, final = M.gated_delta(q, k, v, g, b, h0, torch.tensor([3, 40, 70], device="cuda", dtype=torch.int32), out=out)
    assert bool((o[:3] == 5.0).all()) and bool((o[70:] == 5.0).all())
    y = tuple(z[3:70].contiguous() for z in (q, k, v, g, b)) + (h0, torch.tensor([0, 37, 67]))
    _check(o[3:70], final, y, dtype, D ** -0.5)
    for bad, good in (([-5, 30, 60], [0, 30, 60]), ([0, 50, 20], [0, 50, 50]), ([0, 30, 2 ** 31 + 5], [0, 30, L])):
        states = []
        for offsets in (bad, good):
            h = h0.clone()
            kind = torch.int64 if max(offsets) > L else torch.int32
            M.gated_delta(q, k, v, g, b, h, torch.tensor(offsets, device="cuda", dtype=kind), final_state=h)
            states.append(h)
        assert torch.equal(torch.nan_to_num(states[0]), torch.nan_to_num(states[1]))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_tokens_at_all(cuda, dtype):
    H, D = 2, 64
    e, h0 = torch.empty(0, H, D, device="cuda", dtype=dtype), torch.randn(2, H, D, D, device="cuda")
    o, final = M.gated_delta(e, e, e, torch.empty(0, H, device="cuda"), e[..., 0], h0,
                             torch.zeros(3, device="cuda", dtype=torch.int32))
    assert o.shape == (0, H, D) and torch.equal(final, h0)


@gpu
@pytest.mark.parametrize("D,lengths", [(128, [130, 64, 300]), (64, [3, 70, 0, 32, 33, 1]), (256, [90, 13, 100])])
def test_samples_are_independent_of_the_pack(cuda, D, lengths):
    """Bit for bit; in bf16 for samples that go in the same form alone."""
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, g, b, h0, cu = _inputs(2, lengths, 2, 2, D, dtype)
        o, final = M.gated_delta(q, k, v, g, b, h0, cu)
        for n in range(len(lengths)):
            a, e = int(cu[n]), int(cu[n + 1])
            if dtype is torch.bfloat16 and (e - a <= 64 or sum(lengths) <= 64 * len(lengths)):
                continue
            on, fn = M.gated_delta(q[a:e], k[a:e], v[a:e], g[a:e], b[a:e], h0[n:n + 1], torch.tensor([0, e - a]))
            assert torch.equal(o[a:e], on) and torch.equal(final[n], fn[0])


@gpu
def test_refused_arguments(cuda):
    q, k, v, g, b, h0, cu = _inputs(1, [5, 4], 2, 4, 64, torch.bfloat16)
    ok = dict(q=q, k=k, v=v, g=g, beta=b, initial_state=h0, cu_seqlens=cu)
    M.gated_delta(**ok)
    wide = torch.zeros(9, 4 * 64 * 2, device="cuda", dtype=torch.bfloat16)
    for bad in (dict(q=q[:, :1]), dict(k=k.float()), dict(v=v[:, :3]), dict(q=q[..., :32]), dict(v=v.half()),
                dict(beta=b.float()), dict(beta=b[:, :3]), dict(beta=b[:5]), dict(beta=b.cpu()), dict(g=g.double()),
                dict(g=g[:, :2]), dict(g=g[..., None].expand(9, 4, 64)), dict(initial_state=h0[:1]),
                dict(initial_state=h0.double()), dict(cu_seqlens=torch.tensor([0, 5, 10])),
                dict(cu_seqlens=torch.tensor([0, 6, 5])), dict(cu_seqlens=torch.tensor([0.0, 5.0, 9.0])),
                dict(out=v), dict(out=v[:4]), dict(out=torch.empty_like(v, dtype=torch.float32)),
                dict(final_state=h0[:1].expand(2, 4, 64, 64)), dict(final_slots=torch.zeros(2, dtype=torch.int32, device="cuda")),
                dict(initial_slots=torch.zeros(3, dtype=torch.int32, device="cuda")),
                dict(initial_state=None, initial_slots=torch.zeros(2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            M.gated_delta(**{**ok, **bad})
    # an output over beta's rows, and beside them
    beta = wide[:, 256:260]
    beta.copy_(b)
    with pytest.raises(ValueError):
        M.gated_delta(**{**ok, "beta": wide.view(-1)[:36].view(9, 4), "out": wide[:, :256].view(9, 4, 64)})


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_then_steps_equal_one_long_prompt(cuda, dtype, D):
    """A rotated prompt, then single tokens, over one pool: what one prompt of all
    of them gives, within both forms' bounds."""
    Hk, H, T, more = 2, 4, 130, 6
    q, k, v, g, b, h0, _ = _inputs(13, [T + more], Hk, H, D, dtype)
    inv, att = M.rotary_frequencies(32)
    axes = M.rotary_sections([6, 5, 5])
    pos = torch.stack([torch.arange(T + more, device="cuda") // 20 + 9, torch.arange(T + more, device="cuda") % 4,
                       torch.arange(T + more, device="cuda") % 5])
    qr, kr = M.rotary_axes(q, k, pos, inv, axes)
    whole = (qr, kr, v, g, b, h0, torch.tensor([0, T + more]))
    pool = torch.zeros(3, H, D, D, device="cuda")
    pool[2] = h0[0]
    slot = torch.tensor([2], dtype=torch.int32, device="cuda")
    o1, _ = M.gated_delta(qr[:T], kr[:T], v[:T], g[:T], b[:T], pool, torch.tensor([0, T]), initial_slots=slot,
                          final_state=pool, final_slots=slot)
    rows = [o1]
    for t in range(T, T + more):
        qt, kt = M.rotary_axes(q[t:t + 1], k[t:t + 1], pos[:, t:t + 1], inv, axes)
        assert torch.equal(qt, qr[t:t + 1]) and torch.equal(kt, kr[t:t + 1])
        rows.append(M.gated_delta_step(qt, kt, v[t:t + 1], g[t:t + 1], b[t:t + 1], pool, slots=slot))
    _check(torch.cat(rows), pool[2:], whole, dtype, D ** -0.5)
    o2, f2 = M.gated_delta(*whole)
    _check(o2, f2, whole, dtype, D ** -0.5)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("N,Hk,H", [(1, 1, 1), (3, 2, 6), (5, 3, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("decay,beta", [("none", "value"), ("head", "key"), ("token", "value"), ("token", "none")])
def test_step(cuda, D, N, Hk, H, dtype, decay, beta):
    x = _inputs(17, [1] * N, Hk, H, D, dtype, decay=decay, beta=beta)
    q, k, v, g, b, h0, cu = x
    s = h0.clone()
    o = M.gated_delta_step(q, k, v, g, b, s)
    _check(o, s, x, dtype, D ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_pools_views_and_skipped_rows(cuda, dtype):
    N, Hk, H, D = 5, 2, 4, 64
    q, k, v, g, b, h0, _ = _inputs(21, [1] * N, Hk, H, D, dtype)
    wide = torch.zeros(N, (2 * Hk + H) * D + 8, device="cuda", dtype=dtype)
    views = []
    for at, y in ((0, q), (Hk * D, k), (2 * Hk * D, v)):
        wide[:, at:at + y.shape[1] * D] = y.reshape(N, -1)
        views.append(wide[:, at:at + y.shape[1] * D].view(N, y.shape[1], D))
    slots = torch.tensor([3, -1, 0, 3, 9], dtype=torch.int32, device="cuda")  # padded, named twice, outside
    pool = torch.full((6, H, D, D), 2.0, device="cuda")
    pool[3], pool[0] = h0[0], h0[2]
    out = torch.full((N, H, D), 7.0, device="cuda", dtype=dtype)
    o = M.gated_delta_step(*views, g, b, pool, slots=slots, out=out, scale=0.7)
    pick = torch.tensor([0, 2], device="cuda")
    x = tuple(y[pick] for y in (q, k, v, g, b, h0)) + (torch.tensor([0, 1, 2]),)
    _check(o[pick], pool[[3, 0]], x, dtype, 0.7)
    assert bool((o[[1, 3, 4]] == 7.0).all()) and bool((pool[[1, 2, 4, 5]] == 2.0).all())
    assert M.gated_delta_step(q[:0], k[:0], v[:0], g[:0], b[:0], h0[:0]).shape == (0, H, D)
    for bad in (dict(beta=b[:, :3]), dict(beta=b.double()), dict(g=g[..., None].expand(N, H, D)),
                dict(states=h0[:2]), dict(out=v)):
        with pytest.raises(ValueError):
            M.gated_delta_step(**{**dict(q=q, k=k, v=v, g=g, beta=b, states=h0), **bad})


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", ["v", "k", "q", "g", "beta"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("lengths", [[12, 3], [150, 70]])
def test_a_token_that_is_not_finite_leaves_earlier_ones(cuda, D, dtype, what, value, lengths):
    """Causal for values that are not finite: tokens before one, the other samples and (for v) the other columns keep
    their results; from it on they are what the definition makes of it."""
    H, t = 2, lengths[0] - 3
    x = _inputs(19, lengths, 1, H, D, dtype)
    q, k, v, g, b, h0, cu = x
    o, final = M.gated_delta(*x)
    ref = list(y.clone() for y in x)
    bad = list(y.clone() for y in x)
    at = {"q": 0, "k": 1, "v": 2, "g": 3, "beta": 4}[what]
    bad[at][(t, 0, 5) if what in "qkv" else (t, 1)] = value if what != "g" else float("nan")
    o2, f2 = M.gated_delta(*bad)
    r_o, r_s, A, E = _recurrence(*bad, D ** -0.5)
    assert torch.equal(torch.isfinite(o2), torch.isfinite(r_o)), "outputs"
    assert torch.equal(torch.isfinite(f2), torch.isfinite(r_s)), "states"
    assert torch.equal(f2[1], final[1])
    _check_finite(o2, o, r_o, dtype)
    if what == "q":
        assert torch.equal(f2, final)


def _check_finite(o2, o, r_o, dtype):
    """Where the definition is finite, the result stays near it (what was finite before within two roundings of what
    it was, the form may have changed)."""
    fine = torch.isfinite(r_o)
    err = (o2.double() - r_o)[fine].abs()
    scale = r_o[fine].abs().max()
    assert bool((err <= 8 * HALF[dtype] * scale + (3e-5 if dtype is torch.float32 else 0.05) * scale).all())


@gpu
@pytest.mark.parametrize("lengths", [[700, 300], [3000], [2, 1, 3]])
def test_graphs_streams_and_replays(cuda, lengths):
    """Captured calls replay with other inputs; two captured graphs and another stream share nothing."""
    D, H = 64, 2
    x = _inputs(23, lengths, 1, H, D, torch.bfloat16)
    y = _inputs(24, lengths, 1, H, D, torch.bfloat16)
    cu = x[6].cuda()
    want = [M.gated_delta(*z[:6], cu) for z in (x, y)]
    torch.cuda.synchronize()
    static = [z.clone() for z in x[:6]]
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(M.gated_delta(*static, cu))
        graphs.append(graph)
    with pytest.raises(ValueError):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            M.gated_delta(*static, x[6])
    other = torch.cuda.Stream()
    for z, (o, f) in zip((x, y), want):
        for s, r in zip(static, z):
            s.copy_(r)
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            eager = M.gated_delta(*z[:6], cu)
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for got in (*outs, eager):
            assert torch.equal(got[0], o) and torch.equal(got[1], f)
