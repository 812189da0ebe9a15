"""Queries of the gated delta rule that are not finite: what the definition makes of them, infinities with their signs, in
every form, and nothing else changes. Bounds as in test_gated_delta."""

import pytest
import torch

import memt_b200 as M
from test_gated_delta import _inputs, _recurrence

gpu = pytest.mark.gpu


def _kinds(x):
    """0 finite, 1 and 2 the infinities, 3 NaN."""
    return torch.isposinf(x) + 2 * torch.isneginf(x) + 3 * torch.isnan(x)


def _state_after(x, t):
    """The states [H, D, D] that token t of the first sample reads, in 64 bits."""
    q, k, v, g, b, h0, _ = x
    return _recurrence(q[:t + 1], k[:t + 1], v[:t + 1], g[:t + 1], b[:t + 1], h0[:1], torch.tensor([0, t + 1]), 1.0)[1][0]


def _check(o, clean, bad, t, scale):
    """Row t is the definition's; the other rows keep their bits."""
    S = _state_after(bad, t)                                                # [H, D, D]
    q = bad[0][t].double().repeat_interleave(S.shape[0] // bad[0].shape[1], 0)
    want = scale * torch.einsum("hk,hkv->hv", q, S)
    sure = (torch.where(torch.isinf(q)[..., None], S.abs(), 1.0) > 1e-3).all(1)  # signs beyond any rounding
    assert float(sure.double().mean()) > 0.9
    assert torch.equal(_kinds(o[t])[sure], _kinds(want)[sure])
    assert not bool(torch.isfinite(o[t]).any())
    rest = torch.arange(o.shape[0], device=o.device) != t
    assert torch.equal(o[rest], clean[rest])


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,t", [([12, 3], 9), ([1, 1], 0), ([150, 70], 0), ([150, 70], 40), ([150, 70], 63),
                                       ([150, 70], 64), ([150, 70], 149), ([128, 64], 127)])
@pytest.mark.parametrize("places", [{5: 1}, {5: -1}, {5: 1, 40: -1}, {5: 1, 6: float("nan")}])
def test_a_query_that_is_not_finite(cuda, D, dtype, lengths, t, places):
    x = _inputs(51, lengths, 1, 2, D, dtype)
    o, final = M.gated_delta(*x)
    bad = list(x)
    bad[0] = x[0].clone()
    for i, sign in places.items():
        bad[0][t, 0, i] = sign * float("inf")
    o2, f2 = M.gated_delta(*bad)
    assert torch.equal(f2, final)
    _check(o2, o, bad, t, D ** -0.5)


@gpu
@pytest.mark.parametrize("D,L", [(64, 2900), (128, 2600), (256, 2400)])
@pytest.mark.parametrize("t", [3, 1301, -1])
def test_in_segments(cuda, D, L, t):
    x = _inputs(52, [L], 1, 1, D, torch.bfloat16, decay="head")
    o, final = M.gated_delta(*x)
    bad = list(x)
    bad[0] = x[0].clone()
    bad[0][t, 0, 7] = -float("inf")
    o2, f2 = M.gated_delta(*bad)
    assert torch.equal(f2, final)
    _check(o2, o, bad, t % L, D ** -0.5)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_states_in_place(cuda, D):
    """The first state is read again for the outputs, the last one waits: in a pool and without, beside a column of v that
    is made again altogether, and with a query of NaN alone, for which nothing is."""
    lengths, H = [200, 0, 90], 2
    x = _inputs(53, lengths, 1, H, D, torch.bfloat16)
    o, final = M.gated_delta(*x)
    bad = list(x)
    bad[0], bad[2] = x[0].clone(), x[2].clone()
    bad[0][70, 0, 3], bad[0][130, 0, 9] = float("inf"), float("nan")
    bad[2][100, 1, 60] = float("nan")  # a head and a column that the columns below do not hold
    fresh = M.gated_delta(*bad)
    pool = torch.zeros(5, H, D, D, device="cuda")
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    pool[slots.long()] = x[5]
    o2, _ = M.gated_delta(*bad[:5], pool, x[6], initial_slots=slots, final_state=pool, final_slots=slots)
    states = x[5].clone()
    o3, _ = M.gated_delta(*bad[:5], states, x[6], final_state=states)
    for got, s in ((fresh[0], fresh[1]), (o2, pool[slots.long()]), (o3, states)):
        assert torch.equal(torch.nan_to_num(got, 7.0, 8.0, 9.0), torch.nan_to_num(fresh[0], 7.0, 8.0, 9.0))
        assert torch.equal(torch.nan_to_num(s, 7.0), torch.nan_to_num(fresh[1], 7.0))
    keep = torch.arange(D, device="cuda") // 16 != 60 // 16
    assert torch.equal(fresh[1][1:], final[1:]) and torch.equal(fresh[1][0, 0], final[0, 0])
    assert torch.equal(fresh[1][0, 1][:, keep], final[0, 1][:, keep])
    assert bool(torch.isnan(fresh[1][0, 1, :, 60]).all())
    rows = torch.ones(sum(lengths), dtype=torch.bool, device="cuda")
    rows[70] = rows[130] = False
    assert torch.equal(fresh[0][rows][:, 0], o[rows][:, 0])
    assert torch.equal(fresh[0][rows][:, 1, keep], o[rows][:, 1, keep])
    assert bool(torch.isnan(fresh[0][130]).all())
    bad[2] = x[2]
    _check_rows(fresh[0], bad, 70, D, keep)


def _check_rows(o, bad, t, D, keep):
    S = _state_after(bad, t)
    want = torch.einsum("k,hkv->hv", bad[0][t, 0].double(), S)
    sure = (S[:, 3].abs() > 1e-3) & keep
    assert torch.equal(_kinds(o[t])[sure], _kinds(want)[sure])


@gpu
def test_rows_of_the_next_sample_are_not_looked_at(cuda):
    """A chunk that ends inside: the tile holds the next sample's rows, whose queries are not this sample's."""
    x = _inputs(54, [100, 130], 1, 2, 64, torch.bfloat16)
    o, final = M.gated_delta(*x)
    bad = list(x)
    bad[0] = x[0].clone()
    bad[0][100:128] = float("inf")
    o2, f2 = M.gated_delta(*bad)
    assert torch.equal(f2, final) and torch.equal(o2[:100], o[:100]) and torch.equal(o2[128:], o[128:])


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("decay", ["none", "head", "token"])
@pytest.mark.parametrize("first", [[150], [3]])
def test_an_infinite_state(cuda, D, dtype, decay, first):
    """One infinite element of the state that a sample of one token starts from: the correction is infinite, the other
    rows become infinities and its own NaN, whichever form the sample goes in."""
    H, r, c = 2, 9, 21
    x = _inputs(55, first + [1], 1, H, D, dtype, decay=decay)
    x[5][1, 1, r, c] = float("inf")
    o, final = M.gated_delta(*x)
    q, k, v, g, b, h0, cu = x
    clean = h0.clone()
    clean[1, 1, r, c] = 0.0
    o2, f2 = M.gated_delta(q, k, v, g, b, clean, cu)
    ref_o, ref, _, _ = _recurrence(*x, D ** -0.5)
    assert int(torch.isinf(ref[1, 1, :, c]).sum()) == D - 1
    assert torch.equal(_kinds(final), _kinds(ref)) and torch.equal(_kinds(o), _kinds(ref_o))
    cols = torch.arange(D, device="cuda") // 16 != c // 16
    assert torch.equal(final[1, 0], f2[1, 0]) and torch.equal(final[1, 1][:, cols], f2[1, 1][:, cols])
    assert torch.equal(final[0], f2[0]) and torch.equal(o[:-1], o2[:-1])


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what,place", [("v", 1), ("v", -1), ("q", 1), ("q", -1), ("k", 1), ("state", 1), ("q", float("nan"))])
def test_the_step(cuda, D, dtype, what, place):
    """One session's output and state are the definition's, the other sessions keep their bits."""
    N, H, c = 3, 2, 11
    x = _inputs(56, [1] * N, 1, H, D, dtype)
    clean = x[5].clone()
    o = M.gated_delta_step(*x[:5], clean)
    bad = [y.clone() if y is not None else None for y in x]
    inf = place * float("inf")
    if what == "v":
        bad[2][1, 1, c] = inf
    elif what == "state":
        bad[5][1, 1, 9, c] = inf
    else:
        bad["qk".index(what)][1, 0, 9] = inf
    states = bad[5].clone()
    o2 = M.gated_delta_step(*bad[:5], states)
    ref_o, ref, _, _ = _recurrence(*bad, D ** -0.5)
    assert not bool(torch.isfinite(ref_o[1, 1, c])) and torch.equal(_kinds(states), _kinds(ref))
    sure = torch.ones(N, H, D, dtype=torch.bool, device="cuda")
    if what == "q":
        sure[1] = ref[1, :, 9].abs() > 1e-3
        assert float(sure[1].double().mean()) > 0.9
    assert torch.equal(_kinds(o2)[sure], _kinds(ref_o)[sure])
    keep = torch.isfinite(ref_o)
    assert torch.equal(o2[keep], o[keep]) and torch.equal(states[torch.isfinite(ref)], clean[torch.isfinite(ref)])
    # the same token as a prompt
    o3, f3 = M.gated_delta(*bad)
    assert torch.equal(_kinds(o3)[sure], _kinds(o2)[sure]) and torch.equal(_kinds(f3), _kinds(states))
