"""Edges of linear attention and the single-token steps, beside tests/test_linear_attention.py, whose
recurrence in 64 bits and elementwise bounds are used here.
"""

import ctypes

import pytest
import torch

import memt_b200 as M
from memt_b200 import _lib
from test_linear_attention import (_check, _dev, _inputs, _recurrence, _tolerances)

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
