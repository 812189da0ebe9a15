"""The gated delta rule's bf16 forms, each held to its own bounds (those of test_gated_delta, which allows a sample either
form's): samples of few tokens to the token-by-token form's, segments of several samples with values that are not
finite to the segments'. And what a serving host packs: one prompt beside many single tokens."""

import pytest
import torch

import memt_b200 as M
from test_gated_delta import HALF, _chunk_bounds, _inputs, _recurrence

gpu = pytest.mark.gpu
BF = torch.bfloat16


def _bounds(x, D, joined=False):
    """(outputs, states, their bounds) of the token-by-token form, and the bounds of the chunked one."""
    ref_o, ref_s, A, E = _recurrence(*x, D ** -0.5)
    Ac, Ec = _chunk_bounds(*x, D ** -0.5, D if joined else 0)
    out = lambda a: a * 1.01 + HALF[BF] * (ref_o.abs() + a) + 1e-40  # noqa: E731
    return ref_o, ref_s, out(A), E * 1.01 + 1e-40, out(torch.maximum(A, Ac)), torch.maximum(E, Ec) * 1.01 + 1e-40


@gpu
@pytest.mark.parametrize("D,few", [(64, 40), (128, 20), (256, 14)])
@pytest.mark.parametrize("decay", ["none", "head", "token"])
def test_few_tokens_to_their_own_bounds(cuda, D, few, decay):
    """In a call of both forms: states to fp32's roundings, a hundred times closer than in chunks."""
    lengths = [few, 90, 1, 0, few - 1, 70, 2, few + 1, 9]
    x = _inputs(61, lengths, 1, 2, D, BF, decay=decay)
    assert sum(lengths) <= 64 * len(lengths)
    o, final = M.gated_delta(*x)
    ref_o, ref_s, to, ts, tco, tcs = _bounds(x, D)
    for n, length in enumerate(lengths):
        rows = slice(int(x[6][n]), int(x[6][n + 1]))
        small = length <= few
        assert bool(((o[rows].double() - ref_o[rows]).abs() <= (to if small else tco)[rows]).all()), n
        assert bool(((final[n].double() - ref_s[n]).norm(dim=1) <= (ts if small else tcs)[n]).all()), n


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_one_call_of_few_tokens_to_its_own_bounds(cuda, D):
    x = _inputs(62, [{64: 40, 128: 20, 256: 14}[D]], 1, 2, D, BF)
    o, final = M.gated_delta(*x)
    ref_o, ref_s, to, ts, _, _ = _bounds(x, D)
    assert bool(((o.double() - ref_o).abs() <= to).all()) and bool(((final.double() - ref_s).norm(dim=2) <= ts).all())


@gpu
@pytest.mark.parametrize("D,lengths", [(64, [2500, 1900]), (128, [2300, 2600]), (256, [2400])])
@pytest.mark.parametrize("what", ["v", "k", "g", "beta"])
def test_segments_with_a_token_that_is_not_finite(cuda, D, lengths, what):
    """In the last sample: the others keep their bits, tokens before it and (for v) the other columns their bounds."""
    n = len(lengths) - 1
    t0, t = sum(lengths[:n]), sum(lengths[:n]) + 1301
    x = _inputs(63, lengths, 1, 1, D, BF)
    o, final = M.gated_delta(*x)
    bad = [y.clone() if y is not None else None for y in x]
    at = {"k": 1, "v": 2, "g": 3, "beta": 4}[what]
    bad[at][(t, 0, 5) if what in "kv" else (t, 0)] = float("nan")
    o2, f2 = M.gated_delta(*bad)
    assert torch.equal(o2[:t0], o[:t0]) and torch.equal(f2[:n], final[:n])
    ref_o, ref_s, _, _, to, ts = _bounds(tuple(y[t0:] for y in x[:5]) + (x[5][n:], x[6][n:] - t0), D, joined=True)
    err = (o2[t0:].double() - ref_o).abs()
    assert bool((err[:t - t0] <= to[:t - t0]).all())
    others = torch.arange(D, device="cuda") != 5 if what == "v" else torch.zeros(D, dtype=torch.bool, device="cuda")
    assert bool((err <= to)[..., others].all())
    assert bool(((f2[n].double() - ref_s[0]).norm(dim=1) <= ts[0])[:, others].all())
    assert not bool(torch.isfinite(o2[t:][..., ~others]).any()) and not bool(torch.isfinite(f2[n][..., ~others]).any())


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_a_prompt_beside_many_single_tokens(cuda, D):
    """A mean above 64 tokens a sample: all in chunks, most of them of one token."""
    lengths = [1] * 40 + [4000] + [1] * 20
    x = _inputs(64, lengths, 1, 1, D, BF)
    o, final = M.gated_delta(*x)
    ref_o, ref_s, _, _, to, ts = _bounds(x, D)
    assert bool(((o.double() - ref_o).abs() <= to).all())
    assert bool(((final.double() - ref_s).norm(dim=2) <= ts).all())


@gpu
@pytest.mark.parametrize("lengths", [[700, 300], [3000], [2, 1, 3], [90, 3, 0, 150] * 10])
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_the_same_call_twice_is_the_same(cuda, lengths, dtype):
    x = _inputs(65, lengths, 1, 2, 128, dtype)
    first = [y.clone() for y in M.gated_delta(*x)]
    for _ in range(5):
        again = M.gated_delta(*x)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def _two_terms(q, k, v, g, beta, h0, cu, scale):
    """(outputs, a bound of their error before they are rounded) of the chunked form, in which every factor of an output, the
    state and U and the scores, is two bf16 terms: 2^-16 of each value is left out at most (two half steps of 2^-8), so
    is the product of two remainders; sums are fp32, truncating: 2 u an addition. To it the errors of the state before the
    chunk and of U, as test_gated_delta has them for the columns (there 2^-8 stands for these 2^-16)."""
    L, H, D = v.shape
    rep = H // q.shape[1]
    u24, two = 2.0 ** -24, 2.0 ** -16
    q, k = (x.double().repeat_interleave(rep, 1) for x in (q, k))
    v = v.double()
    a = torch.ones(L, H, dtype=torch.float64, device=v.device) if g is None else g.double().exp().expand(L, H)
    b = beta.double()
    S = h0.double().clone()
    E = torch.zeros(S.shape[0], H, D, dtype=torch.float64, device=v.device)
    o, A = torch.zeros_like(v), torch.zeros_like(v)
    norm = lambda x: torch.linalg.matrix_norm(x, 2)[:, None]  # noqa: E731
    cols = lambda x: x.norm(dim=1)  # noqa: E731
    for n in range(len(cu) - 1):
        for t0 in range(int(cu[n]), int(cu[n + 1]), 64):
            t1 = min(t0 + 64, int(cu[n + 1]))
            kc, qc, vc = (x[t0:t1].transpose(0, 1) for x in (k, q, v))
            G = a[t0:t1].log().cumsum(0).T
            f, w, bc = G.exp()[..., None], (G[:, -1:] - G).exp()[..., None], b[t0:t1].T[..., None]
            i = torch.arange(t1 - t0, device=v.device)
            weight = torch.where(i[:, None] >= i, G[:, :, None] - G[:, None, :], -torch.inf).exp()
            low = (kc @ kc.transpose(1, 2)) * weight * bc * (i[:, None] > i)
            T = torch.linalg.inv(torch.eye(t1 - t0, dtype=torch.float64, device=v.device) + low)
            r = bc * (vc - f * (kc @ S[n]))
            u = T @ r
            scores = (qc @ kc.transpose(1, 2)) * weight
            o[t0:t1] = scale * (f * (qc @ S[n]) + scores @ u).transpose(0, 1)
            turns = min(float(G.abs().max()) * 1.4427, 30.0)
            nk, nT = norm(kc), norm(T)
            dr = nk * (two + 4 * D * u24) * cols(S[n]) + 4 * u24 * cols(vc) + (two + 4 * u24) * cols(r)
            dT = (2 * two + 384 * u24) * T.flatten(1).norm(dim=1)[:, None] + 64 * u24 * nT * (1 + norm(low)) \
                + (2 * D + 20 + 7 * turns) * u24 * nT ** 2 * low.flatten(1).norm(dim=1)[:, None]
            du = nT * dr + dT * cols(r) + nk * nT * E[n]
            inter, sums = f * (qc.abs() @ S[n].abs()), scores.abs() @ u.abs()
            A[t0:t1] = abs(scale) * ((two + (4 * D + 16 + 7 * turns) * u24) * inter
                                     + (3 * two + (384 + 2 * D + 20 + 7 * turns) * u24) * sums
                                     + f * qc.norm(dim=2, keepdim=True) * E[n][:, None]
                                     + scores.norm(dim=2, keepdim=True) * du[:, None]).transpose(0, 1)
            keep = G[:, -1].exp()[:, None]
            E[n] = keep * E[n] + norm(w * kc) * (nT * dr + dT * cols(r) + (two + (256 + 7 * turns) * u24) * cols(u)) \
                + 4 * u24 * cols(S[n])
            S[n] = keep[..., None] * S[n] + (w * kc).transpose(1, 2) @ u
    return o, A


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("decay", ["none", "head", "token"])
@pytest.mark.parametrize("lengths", [[300, 64, 70, 130], [800]])
def test_outputs_in_chunks_are_rounded_once(cuda, D, decay, lengths):
    """What an output loses besides its own rounding is some 2^-16 of its terms."""
    x = _inputs(66, lengths, 1, 2, D, BF, decay=decay)
    o, _ = M.gated_delta(*x)
    ref, A = _two_terms(*x, D ** -0.5)
    assert torch.allclose(ref, _recurrence(*x, D ** -0.5)[0], atol=1e-10)
    err = (o.double() - ref).abs()
    bound = A * 1.01 + HALF[BF] * (ref.abs() + A) + 1e-40
    assert bool((err <= bound).all()), f"worst {float((err / bound).max()):.3g} of its bound"
    rounding = (ref.bfloat16().double() - ref).norm()  # of the exact outputs alone
    assert float(err.norm()) <= 1.02 * float(rounding) + float(A.norm())
