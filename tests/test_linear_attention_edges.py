"""Edges of linear attention and the single-token steps, beside tests/test_linear_attention.py, whose
recurrence in 64 bits and elementwise bounds are used here.
"""

import ctypes

import pytest
import torch

import memt_b200 as M
from memt_b200 import _lib
from test_linear_attention import (HALF, U, _check, _dev, _inputs, _recurrence, _run_and_check, _step_inputs,
                                   _step_reference, _tolerances)

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pool", [False, True])
def test_in_place_samples_of_one_chunk(cuda, dtype, pool):
    """States updated in place at D = 64 by samples of one chunk each: every warp loads its share of a
    state before another one stores its own. Outputs as well as states, and repeats bit for bit."""
    lengths, H, D = [25 + i % 40 for i in range(96)], 8, 64
    N = len(lengths)
    q, k, v, g, h0, cu = _inputs(41, lengths, 4, H, D, dtype, "token")
    ref = _recurrence(q, k, v, g, h0, cu, D ** -0.5)
    to, ts = _tolerances(ref, lengths, D, dtype, g, H)
    dq, dk, dv, dg, dcu = _dev(q, k, v, g, cu)
    slots = torch.arange(N, dtype=torch.int32, device="cuda").flip(0) if pool else None
    places = {"initial_slots": slots, "final_slots": slots} if pool else {}
    start = (h0.flip(0) if pool else h0).cuda()
    apart = M.linear_attention(dq, dk, dv, dg, start, dcu, final_state=torch.zeros_like(start), **places)
    _check(apart[0], ref[0], to, "output")
    for _ in range(20):
        states = start.clone()
        o, final = M.linear_attention(dq, dk, dv, dg, states, dcu, final_state=states, **places)
        torch.cuda.synchronize()
        assert final is states and torch.equal(states, apart[1]) and torch.equal(o, apart[0])
    _check(final.flip(0) if pool else final, ref[1], ts, "state")


# ---------------------------------------------------------------------------
# outputs and states that overlap other arguments (refused before any launch)
# ---------------------------------------------------------------------------

P = 1 << 20  # addresses a MB apart: nothing is read there


def _linear(**over):
    """A valid call of 8 tokens, 4 heads on 2 key heads, D = 64, bf16; every argument apart."""
    f = dict(num_samples=2, num_heads=4, num_key_heads=2, head_dim=64, dtype=_lib.MEMT_BF16, total_tokens=8,
             cu_seqlens=P, q=2 * P, q_stride=128, k=3 * P, k_stride=128, v=4 * P, v_stride=256, g=5 * P,
             g_layout=_lib.GATE_PER_HEAD, scale=1.0, out=6 * P, out_stride=256, initial_state=7 * P,
             final_state=8 * P)
    f.update(over)
    a = _lib.LinearAttentionArgs(**f)
    return _lib.load().memt_linear_attention(ctypes.byref(a), None, 0, None)


def _step(**over):
    """A valid step of 2 sessions with every gate, 2 heads, D = 128, bf16; every argument apart."""
    f = dict(rule=_lib.RULE_GDN2, num_samples=2, num_heads=2, num_key_heads=2, head_dim=128, dtype=_lib.MEMT_BF16,
             q=P, q_stride=256, k=2 * P, k_stride=256, v=3 * P, v_stride=256, g=4 * P,
             g_layout=_lib.GATE_PER_CHANNEL, beta=5 * P, beta_layout=_lib.GATE_PER_CHANNEL, erase=6 * P, write=7 * P,
             states=8 * P, scale=1.0, out=9 * P, out_stride=256)
    f.update(over)
    a = _lib.RecurrentStepArgs(**f)
    return _lib.load().memt_recurrent_step(ctypes.byref(a), None)


def _rotary(**over):
    f = dict(num_heads=2, num_key_heads=1, head_dim=64, rotary_dim=32, dtype=_lib.MEMT_BF16, total_tokens=4, q=P,
             q_stride=128, k=2 * P, k_stride=64, q_out=3 * P, q_out_stride=128, k_out=4 * P, k_out_stride=64,
             positions=5 * P, positions_int64=1, inv_freq=6 * P, attention_scale=1.0)
    f.update(over)
    a = _lib.RotaryArgs(**f)
    return _lib.load().memt_rotary(ctypes.byref(a), None)


STATE64, STATE128 = 4 * 64 * 64 * 4, 2 * 128 * 128 * 4  # bytes of a sample's states above


@pytest.mark.parametrize("over", [
    dict(out=2 * P), dict(out=3 * P + 7 * 256 + 240), dict(out=4 * P - 7 * 512 - 16), dict(out=5 * P),
    dict(out=5 * P + 8 * 16 - 16), dict(out=P), dict(out=7 * P), dict(out=7 * P + 2 * STATE64 - 16),
    dict(out=8 * P + 16), dict(out=5 * P, g_layout=_lib.GATE_CONSTANT),
    dict(dtype=_lib.MEMT_F32, q_stride=128, out=5 * P),
    dict(final_state=2 * P), dict(final_state=4 * P + 8 * 512 - 16), dict(final_state=5 * P), dict(final_state=P),
    dict(initial_slots=9 * P, num_initial_slots=3, out=9 * P), dict(final_slots=9 * P, num_final_slots=5, out=9 * P),
    dict(final_slots=9 * P, num_final_slots=5, out=8 * P + 5 * STATE64 - 16),
    dict(final_slots=8 * P, num_final_slots=5),
    # columns of one wide buffer that share one element vector
    dict(q=2 * P, q_stride=512, out=2 * P + 240, out_stride=512),
    dict(v=4 * P, v_stride=640, out=4 * P + 1280 - 496, out_stride=640),
    dict(v=4 * P, v_stride=640, out=4 * P - 1280 - 496, out_stride=640)])
def test_linear_attention_refuses_overlaps(over):
    assert _linear(**over) == _lib.MEMT_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("over", [
    dict(out=P), dict(out=2 * P), dict(out=3 * P), dict(out=4 * P), dict(out=5 * P), dict(out=6 * P),
    dict(out=7 * P), dict(out=7 * P + 256), dict(out=7 * P - 1008), dict(out=6 * P + 1008), dict(out=8 * P),
    dict(out=8 * P + 2 * STATE128 - 16), dict(out=4 * P + 2 * 1024 - 16),
    dict(out=5 * P, beta_layout=_lib.GATE_PER_HEAD), dict(out=4 * P, g_layout=_lib.GATE_CONSTANT),
    dict(slots=10 * P, num_slots=4, out=10 * P), dict(slots=10 * P, num_slots=4, out=8 * P + 4 * STATE128 - 16),
    dict(slots=8 * P, num_slots=4), dict(states=P), dict(states=4 * P), dict(states=5 * P), dict(states=6 * P),
    dict(states=7 * P), dict(states=3 * P - 2 * STATE128 + 16)])
def test_step_refuses_overlaps(over):
    assert _step(**over) == _lib.MEMT_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("over", [
    dict(q_out=5 * P), dict(k_out=5 * P + 16), dict(q_out=6 * P), dict(k_out=6 * P + 112),
    dict(q_out=5 * P - 3 * 512 - 240, q_out_stride=256), dict(k_out=6 * P - 16)])
def test_rotary_refuses_overlaps(over):
    assert _rotary(**over) == _lib.MEMT_ERR_INVALID_ARGUMENT


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_outputs_over_gates_are_refused_and_beside_them_are_not(cuda, D, dtype):
    """Through the Python layer: out as one of the gates raises; gates, inputs and output as columns of one
    wide buffer, the output between them, are apart and give what separate tensors give."""
    N, H = 3, 2
    gen = torch.Generator().manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k, v = (0.1 * r(N, H, D) for _ in range(3))
    erase, write, beta = (torch.sigmoid(r(N, H, D)) for _ in range(3))
    S = r(N, H, D, D).cuda()
    g = -torch.rand(N, H, D, generator=gen).cuda()
    args = [x.to(dtype).cuda() for x in (q, k, v, erase, write, beta)]
    q, k, v, erase, write, beta = args
    kept = S.clone()
    states = [S.view(-1)[-N * H * D:].view(N, H, D)] if dtype == torch.float32 else []
    for out in [erase, write, beta, q, k, v] + ([g] if states else []) + states:
        with pytest.raises(ValueError):
            M.gdn2_step(q, k, v, g, S, beta=beta, erase=erase, write=write, out=out)
    for out in [q, v] + states:
        with pytest.raises(ValueError):
            M.linear_attention_step(q, k, v, None, S, out=out)
    torch.cuda.synchronize()
    assert torch.equal(S, kept)
    want = M.gdn2_step(q, k, v, g, S, beta=beta, erase=erase, write=write)
    wide = torch.zeros(N, 4 * H * D, dtype=dtype, device="cuda")
    cols = [wide[:, i * H * D:(i + 1) * H * D].view(N, H, D) for i in range(4)]
    for c, x in zip(cols, (q, k, v)):
        c.copy_(x)
    got = M.gdn2_step(cols[0], cols[1], cols[2], g, kept, beta=beta, erase=erase, write=write, out=cols[3])
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(kept, S)


@gpu
def test_linear_attention_refuses_an_output_over_its_decay(cuda):
    """fp32: the output over the states, and decays that lie inside the output's last row."""
    q, k, v, g, h0, cu = _dev(*_inputs(3, [20, 12], 2, 2, 64, torch.float32, "token"))
    buf = torch.zeros(v.numel(), device="cuda")
    inside = buf[-g.numel():].view_as(g)
    for decay, places in ((inside, dict(out=buf.view_as(v))), (g, dict(out=h0.view(-1)[:v.numel()].view_as(v))),
                          (g, dict(out=h0.view(-1)[-v.numel():].view_as(v), final_state=h0))):
        with pytest.raises(ValueError):
            M.linear_attention(q, k, v, decay, h0, cu, **places)


@pytest.mark.parametrize("tokens", [0, 8])
@pytest.mark.parametrize("dtype", [_lib.MEMT_BF16, _lib.MEMT_F32])
def test_linear_attention_refuses_a_missing_constant_decay(tokens, dtype):
    """The [H] decays are read whatever the number of tokens."""
    over = dict(g=None, g_layout=_lib.GATE_CONSTANT, dtype=dtype, total_tokens=tokens)
    assert _linear(**over) == _lib.MEMT_ERR_INVALID_ARGUMENT


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_incoming_read_does_not_know_the_token(cuda, D, dtype, value):
    """read_incoming: a value of the token that is not finite enters the new state's column and leaves the
    output, which reads the state before it, as it is."""
    N, H = 3, 2
    gen, q, k, v, _ = _step_inputs(7, N, H, H, D, dtype)
    g, S = -torch.rand(N, H, generator=gen), torch.randn(N, H, D, D, generator=gen)
    v[1, 0, 5] = value
    ref = _step_reference(q, k, v, g, S, delta=True, incoming=True)
    dq, dk, dv, dg, dS = _dev(q, k, v, g, S)
    o = M.gdn2_step(dq, dk, dv, dg, dS, scale=1.0, read_incoming=True)
    torch.cuda.synchronize()
    clean = torch.ones(N, H, D, dtype=torch.bool)
    clean[1, 0, 5] = False
    at = clean[:, :, None, :].expand_as(S)
    _check(o, ref[0], (2 * D + 24) * U * ref[2] + HALF[dtype] * ref[0].abs() * 1.01 + 1e-40, "output")
    _check(dS.cpu()[at], ref[1][at], (D + 16) * U * ref[3][at] + 1e-40, "state")
    assert not bool(torch.isfinite(dS[1, 0, :, 5]).any())


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [2, 32])
@pytest.mark.parametrize("what", ["v", "k", "q", "g"])
def test_a_token_that_is_not_finite_leaves_earlier_ones(cuda, D, dtype, heads, what):
    """NaN or infinity in one token of a sample: outputs of earlier tokens of every 16-token block, of other
    columns (v), heads and samples stay within their bounds; its own column is spoiled from it on."""
    lengths, Hk, H = [5, 320, 64, 200], heads // 2, heads
    q, k, v, g, h0, cu = _inputs(D + heads, lengths, Hk, H, D, dtype, "token")
    clean = _recurrence(q, k, v, g, h0, cu, D ** -0.5)
    to, ts = _tolerances(clean, lengths, D, dtype, g, H)
    values = [float("nan"), float("inf"), -float("inf")]
    # row, value head, column (of v): first and last tokens of blocks and chunks, two in a column of one chunk
    marks = [(5 + 17, 0, 3), (5 + 31, 1, 40), (5 + 64, 0, 63), (5 + 50, 0, 9), (5 + 20, 0, 9), (5 + 255, 1, D - 1),
             (325, 1, 0), (325 + 63, 0, 33), (389 + 199, 0, 1), (389 + 128 + 7, 1, D // 2)]
    spoiled = torch.zeros(v.shape, dtype=torch.bool)
    ends = {n: (int(cu[n]), int(cu[n + 1])) for n in range(4)}
    for i, (t, h, c) in enumerate(marks):
        end = next(e for s, e in ends.values() if s <= t < e)
        value = values[i % 3]
        if what == "v":
            v[t, h, c] = value
            spoiled[t:end, h, c] = True
        elif what == "k":
            k[t, 0, c] = value
            spoiled[t:end, :2] = True  # both value heads of key head 0
        elif what == "q":
            q[t, 0, c] = value
            spoiled[t, :2] = True
        else:
            g[t, h] = float("nan")
            spoiled[t:end, h] = True
    o, final = M.linear_attention(*_dev(q, k, v, g, h0, cu))
    torch.cuda.synchronize()
    o, final = o.float().cpu(), final.cpu()
    _check(o[~spoiled], clean[0][~spoiled], to[~spoiled], "output")
    assert not bool(torch.isfinite(o[spoiled]).any())
    last = torch.stack([spoiled[e - 1] for _, e in ends.values()])  # [N, H, D]: columns of the final states
    if what == "q":
        last.zero_()
    at = last[:, :, None, :].expand_as(final)
    _check(final[~at], clean[1][~at], ts[~at], "state")
    if what in ("v", "g"):
        assert not bool(torch.isfinite(final[at]).any())


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("in_place", [False, True])
def test_values_that_are_not_finite_in_segments(cuda, D, in_place):
    """The same where a sample is split: later segments start from a state that is not finite, the outputs of
    the token's block are made from its own segment's start."""
    L, H = 2500, 2
    q, k, v, g, h0, cu = _inputs(D, [L], 1, H, D, torch.bfloat16, "token", 0.05)
    assert _lib.load().memt_linear_attention_workspace_size(1, L, H, D, _lib.MEMT_BF16) > 256
    clean = _recurrence(q, k, v, g, h0, cu, D ** -0.5)
    to, ts = _tolerances(clean, [2 * L], D, torch.bfloat16, g, H)
    spoiled = torch.zeros(v.shape, dtype=torch.bool)
    for t, h, c, value in ((1003, 0, 5, "nan"), (2, 1, 6, "inf"), (L - 1, 0, D - 1, "nan"), (1500, 0, 5, "inf")):
        v[t, h, c] = float(value)
        spoiled[t:, h, c] = True
    dq, dk, dv, dg, dh, dcu = _dev(q, k, v, g, h0, cu)
    o, final = M.linear_attention(dq, dk, dv, dg, dh, dcu, final_state=dh if in_place else None)
    torch.cuda.synchronize()
    o, final = o.float().cpu(), final.cpu()
    _check(o[~spoiled], clean[0][~spoiled], to[~spoiled], "output")
    assert not bool(torch.isfinite(o[spoiled]).any())
    at = spoiled[-1][None, :, None, :].expand_as(final)
    _check(final[~at], clean[1][~at], ts[~at], "state")
    assert not bool(torch.isfinite(final[at]).any())


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("decay", ["none", "head", "token"])
@pytest.mark.parametrize("lengths,H", [([70, 3], 2), ([1500], 2), ([300, 200], 2)])
def test_infinite_states_stay_infinite(cuda, D, dtype, decay, lengths, H):
    """An infinite element of the initial state keeps its sign through any decay above zero, and the outputs
    of its column are infinite with q's sign; everything else is within its bound."""
    q, k, v, g, h0, cu = _inputs(D, lengths, H, H, D, dtype, decay, 0.05)
    clean = _recurrence(q, k, v, g, h0, cu, D ** -0.5)
    to, ts = _tolerances(clean, [2 * n for n in lengths], D, dtype, g, H)
    places = [(0, 0, 5, 7, 1.0), (0, 1, 0, D - 1, -1.0), (len(lengths) - 1, 1, D - 1, 40, 1.0)]
    at, spoiled = torch.zeros(h0.shape, dtype=torch.bool), torch.zeros(v.shape, dtype=torch.bool)
    for n, h, d, c, sign in places:
        h0[n, h, d, c] = sign * float("inf")
        at[n, h, d, c] = True
        spoiled[int(cu[n]):int(cu[n + 1]), h, c] = True
    o, final = M.linear_attention(*_dev(q, k, v, g, h0, cu))
    torch.cuda.synchronize()
    o, final = o.float().cpu(), final.cpu()
    assert torch.equal(final[at], h0[at])
    _check(final[~at], clean[1][~at], ts[~at], "state")
    _check(o[~spoiled], clean[0][~spoiled], to[~spoiled], "output")
    for n, h, d, c, sign in places:
        rows = slice(int(cu[n]), int(cu[n + 1]))
        assert torch.equal(o[rows, h, c], sign * torch.sign(q[rows, h, d].float()) * float("inf"))


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,H", [([70, 3], 2), ([1500], 2), ([300, 200], 2)])
def test_infinite_values_make_infinite_states(cuda, D, dtype, lengths, H):
    """An infinite v makes its column of the state infinite with k's signs, as k v^T is."""
    q, k, v, g, h0, cu = _inputs(D, lengths, H, H, D, dtype, "token", 0.05)
    clean = _recurrence(q, k, v, g, h0, cu, D ** -0.5)
    _, ts = _tolerances(clean, [2 * n for n in lengths], D, dtype, g, H)
    k[33, 0], k[lengths[0] - 1, 1] = (torch.where(k[t, h] == 0, 0.125, k[t, h].float()).to(dtype)
                                      for t, h in ((33, 0), (lengths[0] - 1, 1)))
    v[33, 0, 7], v[lengths[0] - 1, 1, 40] = float("inf"), -float("inf")
    o, final = M.linear_attention(*_dev(q, k, v, g, h0, cu))
    torch.cuda.synchronize()
    final = final.cpu()
    assert torch.equal(final[0, 0, :, 7], torch.sign(k[33, 0].float()) * float("inf"))
    assert torch.equal(final[0, 1, :, 40], -torch.sign(k[lengths[0] - 1, 1].float()) * float("inf"))
    at = torch.zeros(h0.shape, dtype=torch.bool)
    at[0, 0, :, 7] = at[0, 1, :, 40] = True
    _check(final[~at], clean[1][~at], ts[~at], "state")


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("L", [1, 5, 70])
def test_rows_at_any_address(cuda, dtype, L):
    """Inputs off the 16-byte grid, whole tensors and columns of a wider buffer: the same bits as aligned ones."""
    Hk, H, D = 1, 2, 64
    q, k, v, g, h0, cu = _dev(*_inputs(L, [L], Hk, H, D, dtype, "token"))
    want, state = M.linear_attention(q, k, v, g, h0, cu)
    s1 = h0.expand(L, H, D, D).clone()
    s2 = s1.clone()
    step = M.linear_attention_step(q, k, v, g, s1)

    def shifted(x):
        buf = torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")
        buf[1:] = x.reshape(-1)
        return buf[1:].view_as(x)

    wide = torch.zeros(L, (2 * Hk + H) * D + 8, dtype=dtype, device="cuda")
    cols = (wide[:, 3:3 + D].view(L, Hk, D), wide[:, 3 + D:3 + 2 * D].view(L, Hk, D),
            wide[:, 3 + 2 * D:3 + 4 * D].view(L, H, D))
    for c, x in zip(cols, (q, k, v)):
        c.copy_(x)
    for args in ((shifted(q), shifted(k), shifted(v)), cols):
        o, f = M.linear_attention(*args, shifted(g), h0, cu)
        assert torch.equal(o, want) and torch.equal(f, state)
    assert torch.equal(M.linear_attention_step(*cols, shifted(g), s2), step) and torch.equal(s1, s2)


@gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("pinned", [False, True])
def test_host_offsets_do_not_block_the_host(cuda, dtype, pinned):
    """Offsets on the host are copied in stream order: nothing synchronises, later changes of the host tensor
    are not seen, and a capture, which could only keep their address, refuses them."""
    q, k, v, g, h0, cu = _inputs(9, [50, 90], 2, 2, 64, torch.bfloat16, "token")
    dq, dk, dv, dg, dh, dcu = _dev(q, k, v, g, h0, cu)
    want = M.linear_attention(dq, dk, dv, dg, dh, dcu)
    busy = torch.randn(4096, 4096, device="cuda")
    host = cu.to(dtype)
    host = host.pin_memory() if pinned else host
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(20):
            busy = busy @ busy * 1e-4
        o, f = M.linear_attention(dq, dk, dv, dg, dh, host)
        host.zero_()
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    torch.cuda.synchronize()
    assert torch.equal(o, want[0]) and torch.equal(f, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError):
            M.linear_attention(dq, dk, dv, dg, dh, host)
        busy.add_(1)
    graph.replay()
    torch.cuda.synchronize()


@gpu
def test_offsets_beyond_32_bits_are_clamped(cuda):
    """int64 device offsets outside int32 are clamped to the rows like any other."""
    q, k, v, g, h0, _ = _dev(*_inputs(13, [40, 60], 2, 2, 64, torch.bfloat16, "token"))
    for wide, cu in (([0, 40, 2 ** 32 + 50], [0, 40, 100]), ([-2 ** 32 + 40, 40, 100], [0, 40, 100]),
                     ([0, 2 ** 33, 2 ** 40], [0, 100, 100])):
        o, f = M.linear_attention(q, k, v, g, h0, torch.tensor(wide, device="cuda"))
        want = M.linear_attention(q, k, v, g, h0, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        assert torch.equal(o, want[0]) and torch.equal(f, want[1])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_outputs_of_one_head(cuda, dtype):
    """With one head its stride says nothing: an output that is a transposed [1, L, D] buffer is rows."""
    q, k, v, g, h0, cu = _dev(*_inputs(14, [40, 60], 1, 1, 64, dtype, "token"))
    want, _ = M.linear_attention(q, k, v, g, h0, cu)
    out = torch.zeros(1, 100, 64, dtype=dtype, device="cuda").transpose(0, 1)
    o, _ = M.linear_attention(q, k, v, g, h0, cu, out=out)
    assert torch.equal(out, want) and o.data_ptr() == out.data_ptr()
    states = torch.zeros(100, 1, 64, 64, device="cuda")
    same = states.clone()
    want = M.linear_attention_step(q, k, v, g, states)
    assert torch.equal(M.linear_attention_step(q, k, v, g, same, out=out), want) and torch.equal(same, states)


def test_status_needs_a_place():
    assert _lib.load().memt_linear_attention_status(None, None) == _lib.MEMT_ERR_INVALID_ARGUMENT


@gpu
def test_status_after_calls_of_every_kind(cuda):
    """No wait of the chunked kernel runs out: whole samples, segments, empty ones, values that are not finite."""
    lib, status = _lib.load(), ctypes.c_int32(-1)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for D in (64, 128, 256):
        for lengths, H in (([100], 1), ([3000], 2), ([64, 0, 1, 300], 64)):
            args = _dev(*_inputs(D, lengths, 1, H, D, torch.bfloat16, "token"))
            M.linear_attention(*args)
            args[2][7, 0, 3] = float("nan")
            M.linear_attention(*args)
    for _ in range(2):
        assert lib.memt_linear_attention_status(stream, ctypes.byref(status)) == _lib.MEMT_OK and status.value == 0


# ---------------------------------------------------------------------------
# whole samples of many chunks
# ---------------------------------------------------------------------------

def _whole(N, L, H, D):
    """The call keeps no segments: a CTA walks a sample's chunks from the first to the last."""
    assert _lib.load().memt_linear_attention_workspace_size(N, L, H, D, _lib.MEMT_BF16) == 256


@gpu
@pytest.mark.parametrize("D,H", [(64, 32), (128, 32), (256, 16)])
@pytest.mark.parametrize("decay", ["head", "token"])
def test_chains_of_chunks(cuda, D, H, decay):
    """17 and 11 chunks a CTA: every stage of the tiles and every decay table is used several times."""
    lengths = [1100, 700]
    _whole(2, sum(lengths), H, D)
    _run_and_check(lengths, H // 2, H, D, torch.bfloat16, decay, seed=D, gscale=0.05)


RAGGED = [1500, 900, 0, 1500, 1280, 1, 2000, 900, 1700, 1300]  # more than 148 CTAs, above 1024 tokens in the mean


@gpu
def test_longest_samples_first(cuda):
    """The order by length, with equal lengths, an empty sample and one of one token, in place in a pool."""
    H, D, N = 16, 64, len(RAGGED)
    _whole(N, sum(RAGGED), H, D)
    q, k, v, g, h0, cu = _inputs(19, RAGGED, 4, H, D, torch.bfloat16, "token", 0.05)
    ref = _recurrence(q, k, v, g, h0, cu, D ** -0.5)
    to, ts = _tolerances(ref, RAGGED, D, torch.bfloat16, g, H)
    slots = torch.tensor([3, 11, 0, 7, 5, 2, 9, 1, 10, 4])
    pool = torch.full((12, H, D, D), 3.0)
    pool[slots] = h0
    dq, dk, dv, dg, dpool, dcu, ds = _dev(q, k, v, g, pool, cu, slots.int())
    o, _ = M.linear_attention(dq, dk, dv, dg, dpool, dcu, initial_slots=ds, final_state=dpool, final_slots=ds)
    torch.cuda.synchronize()
    _check(o, ref[0], to, "output")
    _check(dpool[slots.cuda()], ref[1], ts, "state")
    assert bool((dpool[[6, 8]] == 3.0).all())


@gpu
@pytest.mark.parametrize("D,H", [(128, 64), (256, 32)])
def test_longest_samples_first_equal_each_alone(cuda, D, H):
    """Bit for bit what each sample gives in a call of its own (whole as well)."""
    _whole(len(RAGGED), sum(RAGGED), H, D)
    gen = torch.Generator(device="cuda").manual_seed(D)
    L = sum(RAGGED)
    q, k = (torch.nn.functional.normalize(torch.randn(L, H // 4, D, generator=gen, device="cuda"), dim=-1).bfloat16()
            for _ in range(2))
    v = torch.randn(L, H, D, generator=gen, device="cuda").bfloat16()
    g = 0.05 * torch.nn.functional.logsigmoid(2 + torch.randn(L, H, generator=gen, device="cuda"))
    h0 = torch.randn(len(RAGGED), H, D, D, generator=gen, device="cuda")
    cu = [sum(RAGGED[:i]) for i in range(len(RAGGED) + 1)]
    o, final = M.linear_attention(q, k, v, g, h0, torch.tensor(cu))
    for n, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        if b - a > 24:  # (few tokens alone run token by token)
            _whole(1, b - a, H, D)
            o1, f1 = M.linear_attention(q[a:b], k[a:b], v[a:b], g[a:b], h0[n:n + 1], torch.tensor([0, b - a]))
            assert torch.equal(o[a:b], o1) and torch.equal(final[n], f1[0])
        elif a == b:
            assert torch.equal(final[n], h0[n])


@pytest.mark.parametrize("over", [
    dict(initial_slots=9 * P, num_initial_slots=4, initial_state=7 * P, final_state=7 * P + STATE64 // 4),
    dict(final_slots=9 * P, num_final_slots=4, initial_state=7 * P + 3 * STATE64 + 16, final_state=7 * P),
    dict(initial_slots=9 * P, num_initial_slots=4, final_slots=10 * P, num_final_slots=4, initial_state=7 * P,
         final_state=7 * P - STATE64 // 2)])
def test_linear_attention_refuses_pools_that_share_parts_of_states(over):
    assert _linear(**over) == _lib.MEMT_ERR_INVALID_ARGUMENT


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pools_that_share_whole_states(cuda, dtype):
    """Views of one pool, shifted by two states; slots keep the samples apart, or in place."""
    q, k, v, g, h0, cu = _dev(*_inputs(15, [40, 60], 2, 2, 64, dtype, "token"))
    want, state = M.linear_attention(q, k, v, g, h0, cu)
    pool = torch.full((6, 2, 64, 64), 3.0, device="cuda")
    pool[1], pool[4] = h0[0], h0[1]
    slots = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    o, _ = M.linear_attention(q, k, v, g, pool[:5], cu, initial_slots=slots(1, 4), final_state=pool[2:],
                              final_slots=slots(3, 2))  # states 5 and 4
    assert torch.equal(o, want) and torch.equal(pool[5], state[0]) and torch.equal(pool[4], state[1])
    assert bool((pool[[0, 2, 3]] == 3.0).all()) and torch.equal(pool[1], h0[0])
    with pytest.raises(ValueError):
        M.linear_attention(q, k, v, g, pool.view(-1)[64 * 64:64 * 64 + 4 * 2 * 64 * 64].view(4, 2, 64, 64), cu,
                           initial_slots=slots(0, 1), final_state=pool, final_slots=slots(2, 3))


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("L", [300, 2500])
def test_infinite_values_that_meet(cuda, D, dtype, L):
    """Infinite columns of the state under further infinities of either sign and full resets, element by element
    as the definition: the same infinities, NaN where two meet or a reset multiplies one by zero."""
    H = 2
    q, k, v, g, h0, cu = _inputs(D + L, [L], H, H, D, dtype, "token", 0.05)
    rows = [40, 41, 100, 170, 171, L - 2]
    for t in rows:
        k[t] = torch.where(k[t] == 0, torch.full_like(k[t], 0.125), k[t])
    inf = float("inf")
    v[40, 0, 1], v[170, 0, 1] = inf, inf                       # two that agree where k's signs do
    v[41, 0, 2], v[L - 2, 0, 2], k[L - 2, 0] = inf, inf, k[41, 0]  # two that agree everywhere
    v[100, 1, 3], v[171, 1, 4] = -inf, inf                     # one before a reset, one behind it
    v[40, 0, 5], v[100, 0, 5] = inf, float("nan")
    g[150, 1] = -inf
    ref = _recurrence(q, k, v, g, h0, cu, D ** -0.5)
    o, final = M.linear_attention(*_dev(q, k, v, g, h0, cu))
    torch.cuda.synchronize()
    final, want = final.cpu()[0], ref[1][0]
    for h, c in ((0, 1), (0, 2), (0, 5), (1, 3), (1, 4)):
        assert not bool(torch.isfinite(want[h, :, c]).any())
        assert torch.equal(final[h, :, c].double().nan_to_num(7.0), want[h, :, c].nan_to_num(7.0)), (h, c)
    _, ts = _tolerances(_recurrence(q, k, v.nan_to_num(0.0, 0.0, 0.0), g, h0, cu, D ** -0.5), [2 * L], D, dtype,
                        torch.tensor([1.0]), H)
    clean = torch.isfinite(want)
    _check(final[clean], want[clean], ts[0][clean] + 1e-20, "state")
