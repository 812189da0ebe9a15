"""Rotary positions of queries and keys (``memt_rotary``), and the frequencies they turn by.

``rotary`` prepares q and k for ``linear_attention`` and its step; ``rotary_frequencies`` builds the
angles per position, also stretched for contexts longer than the trained one.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .linear import _call, _overlap, _ptr
from .ops import _DTYPE, _tokens_unchecked

__all__ = ["rotary", "rotary_frequencies"]

_rotary_args = _lib.Packed(_lib.RotaryArgs)


def rotary_frequencies(rotary_dim, base=10000.0, *, scaling=None, factor=1.0, trained_tokens=None, fast_turns=32.0,
                       slow_turns=1.0, device="cuda"):
    """(inv_freq fp64 [rotary_dim / 2] on ``device``, attention_scale) for ``rotary``.

    Pair i turns by base ** (-2 i / rotary_dim) a position. ``scaling`` stretches the context by
    ``factor``: "linear" divides every angle; "ntk" raises the base so that the slowest pair is
    divided by the factor and the fastest hardly at all; "yarn" divides the pairs that make fewer
    than ``slow_turns`` turns over ``trained_tokens``, keeps those of more than ``fast_turns``,
    blends in between, and scales the rotated values by 0.1 ln(factor) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError("rotary_dim must be even and at least 2")
    if base <= 1.0 or factor < 1.0:
        raise ValueError("base must be above 1 and factor at least 1")
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64)
    attention_scale = 1.0
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv = base ** (-2.0 * pair / rotary_dim)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        if trained_tokens is None or trained_tokens < 1:
            raise ValueError("yarn scaling needs trained_tokens")
        if not 0.0 < slow_turns <= fast_turns:
            raise ValueError("slow_turns must be above 0 and at most fast_turns")

        def pair_of(turns):  # the pair that makes this many turns over the trained context
            return rotary_dim * math.log(trained_tokens / (2 * math.pi * turns)) / (2 * math.log(base))

        low = max(math.floor(pair_of(fast_turns)), 0)
        high = min(math.ceil(pair_of(slow_turns)), rotary_dim - 1)
        ramp = ((pair - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        if pair_of(slow_turns) < 0:  # not even the first pair makes as many
            ramp = torch.ones_like(pair)
        inv = inv / factor * ramp + inv * (1.0 - ramp)
        attention_scale = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return inv.to(device), attention_scale


def _head_rows(x, name):
    """[1, L, H, D] or [L, H, D] with contiguous heads -> ([L, H, D], elements per token row)."""
    if x.dim() != 3 or not x.is_cuda:
        x = _tokens_unchecked(x, name)
    L, H, D = x.shape
    row, head, one = x.stride()
    if one == 1 and (head == D or H == 1):
        if L <= 1:
            return x, H * D
        if row >= H * D:
            return x, row
    return x.contiguous(), H * D


def rotary(q, k, positions, inv_freq, *, interleaved=False, inverse=False, attention_scale=1.0, q_out=None,
           k_out=None):
    """Rotary positions in one launch -> (q_out [L, H, D], k_out [L, Hk, D]), in the inputs' dtype.

    The first 2 * inv_freq.numel() elements of each head are turned, pair i by
    positions * inv_freq[i] (elements i and i + n of the first 2n, or 2i and 2i + 1 when
    ``interleaved``), and multiplied by ``attention_scale``; the rest is copied. ``inverse`` turns
    back: with the same scale it is the operator's backward pass. q, k: bf16 or fp32 [L, H, D]
    token rows (a leading 1 and split views are accepted); k may be None. positions: int32 or int64
    [L]. inv_freq: fp64 on the device (``rotary_frequencies``). ``q_out`` / ``k_out`` may be q / k
    themselves (in place); other overlaps of an output with an input or output are refused.
    """
    q, sq = _head_rows(q, "q")
    L, H, D = q.shape
    dev = q.device
    if q.dtype not in _DTYPE:
        raise ValueError(f"unsupported dtype {q.dtype}")
    Hk, sk = 0, 0
    if k is not None:
        k, sk = _head_rows(k, "k")
        Hk = k.shape[1]
        if H == 0 and Hk > 0:
            raise ValueError("k needs a q of at least one head")
        if k.shape[0] != L or k.shape[2] != D or k.dtype != q.dtype or k.device != dev:
            raise ValueError("k must be [L, key heads, D] in q's dtype and on its device")
    elif k_out is not None:
        raise ValueError("k_out needs k")
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in ((L,), (1, L)):
        raise ValueError(f"positions must be int32 or int64 [{L}]")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not 2 <= 2 * inv_freq.numel() <= D:
        raise ValueError(f"inv_freq must be fp64 with at most {D // 2} angles")
    if positions.device != dev or inv_freq.device != dev:
        raise ValueError(f"positions and inv_freq must be on {dev}")
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    qo, sqo = _output(q, sq, q_out, "q_out")
    ko, sko = (None, 0) if k is None else _output(k, sk, k_out, "k_out")
    if k is not None and (q_out is not None or k_out is not None):
        both = qo is q and ko is k  # in place: the outputs are the inputs
        if (_overlap(qo, sqo, ko, sko)
                or not both and (q_out is not None and _overlap(qo, sqo, k, sk)
                                 or k_out is not None and _overlap(ko, sko, q, sq))):
            raise ValueError("q_out and k_out must not overlap each other or the other input")
    if L == 0 or H == 0:
        return qo, ko
    args = _rotary_args(
        H, Hk, D, 2 * inv_freq.numel(), _DTYPE[q.dtype], L, q.data_ptr(), sq, _ptr(k), sk, qo.data_ptr(), sqo, _ptr(ko),
        sko, positions.data_ptr(), 1 if positions.dtype is torch.int64 else 0, 1 if interleaved else 0,
        inv_freq.data_ptr(), attention_scale, 1 if inverse else 0)
    _call("memt_rotary", dev, args)
    return qo, ko


def _output(x, stride, out, name):
    """A new tensor like x, or the given output's token rows (x itself, or rows apart from it)."""
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device), x.shape[1] * x.shape[2]
    if out is x:
        return x, stride
    o = _tokens_unchecked(out, name)
    L, H, D = x.shape
    if o.shape != x.shape or o.dtype != x.dtype or o.device != x.device:
        raise ValueError(f"{name}: expected {tuple(x.shape)} {x.dtype} on {x.device}")
    s = o.stride()
    if s[2] != 1 or (s[1] != D and H > 1) or (L > 1 and s[0] < H * D):
        raise ValueError(f"{name}: token rows must be contiguous heads")
    so = s[0] if L > 1 else H * D
    if not (o.data_ptr() == x.data_ptr() and so == stride) and _overlap(o, so, x, stride):
        raise ValueError(f"{name} must be the input itself or not overlap it")
    return o, so
