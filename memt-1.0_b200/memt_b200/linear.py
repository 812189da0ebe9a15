"""Causal linear attention with a decay for each head, and single-token recurrent steps.

* ``linear_attention``       S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t over packed
                             prompts (``memt_linear_attention``)
* ``linear_attention_step``  the same recurrence for one token of each session, in place
* ``gdn2_step``              one token of the stable GDN-2 rule (the recurrence of ``gdn2_update``)
                             for each session, in place (both ``memt_recurrent_step``)

States are the framework's fp32 [N, H, K, V] tensors or pools of them addressed by int32 slots, so
one pool serves ``gdn2_update``, the reads and these operators. Queries and keys may have fewer
heads than the values: value head h then uses key head h // (H // key heads).

Every operator runs on the current torch CUDA stream of its tensors' device (whichever device is
current), never synchronises the host and raises ``ValueError`` for invalid arguments before any
launch. They compute no gradients.
"""

from __future__ import annotations

from ctypes import c_size_t, c_void_p

import torch

from . import _lib
from .ops import _DTYPE, _pool, _states, _tokens_unchecked

__all__ = ["linear_attention", "linear_attention_step", "gdn2_step"]

_current_device = torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream
_entries: dict = {}


def _call(name, dev, *args):
    """The entry point ``name`` on ``dev``'s current stream, with ``dev`` current; args: its packed
    struct, then (pointer, size) of a workspace where it takes one."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = _lib.packed_entry(name, *((c_void_p, c_size_t) if len(args) == 3 else ()), c_void_p)
    stream = _raw_stream(dev.index)
    if _current_device() == dev.index:
        status = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            status = fn(*args, stream)
    if status != _lib.MEMT_OK:
        _lib.check(status, name)


def _ptr(x):
    return 0 if x is None else x.data_ptr()


_linear_args = _lib.Packed(_lib.LinearAttentionArgs)
_step_args = _lib.Packed(_lib.RecurrentStepArgs)


def _rows(x, name, vec):
    """[1, L, H, D] or [L, H, D] -> ([L, H, D], elements per token row). Token rows whose heads are
    contiguous and whose starts are 16-byte aligned (a split view of a wider projection) are used
    in place; anything else is copied."""
    if x.dim() != 3 or not x.is_cuda:
        x = _tokens_unchecked(x, name)
    L, H, D = x.shape
    row, head, one = x.stride()
    if one == 1 and (head == D or H == 1) and x.data_ptr() % 16 == 0:
        if L <= 1:
            return x, H * D
        if row >= H * D and row % vec == 0:
            return x, row
    x = x.contiguous()
    if x.data_ptr() % 16 != 0:  # a whole tensor at an odd address
        x = x.clone(memory_format=torch.contiguous_format)
    return x, H * D


def _overlap(a, sa, b, sb):
    """Whether two tensors of token rows (row strides sa, sb in elements) may share elements.
    Interleaved views of one buffer with equal row strides are told apart by their columns."""
    size = a.element_size()
    a0, b0 = a.data_ptr(), b.data_ptr()
    wa, wb = a.shape[1] * a.shape[2] * size, b.shape[1] * b.shape[2] * b.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    ea = a0 + (a.shape[0] - 1) * sa * size + wa
    eb = b0 + (b.shape[0] - 1) * sb * b.element_size() + wb
    if ea <= b0 or eb <= a0:
        return False
    row = sa * size
    if row != sb * b.element_size() or a.shape[0] == 1 or b.shape[0] == 1:
        return True
    off = (b0 - a0) % row
    return off < wa or off + wb > row


def _out_rows(out, like, inputs, vec, name="out"):
    """A given output [L, H, D] (or [1, L, H, D]) of ``like``'s shape and dtype, written in place."""
    o = _tokens_unchecked(out, name)
    L, H, D = like.shape
    if o.shape != like.shape or o.dtype != like.dtype or o.device != like.device:
        raise ValueError(f"{name}: expected {tuple(like.shape)} {like.dtype} on {like.device}")
    s = o.stride()
    if s[2] != 1 or (s[1] != D and H > 1) or o.data_ptr() % 16 != 0 or (L > 1 and (s[0] < H * D or s[0] % vec != 0)):
        raise ValueError(f"{name}: token rows must be contiguous heads on 16-byte boundaries")
    stride = s[0] if L > 1 else H * D
    for x, sx in inputs:
        if _overlap(o, stride, x, sx):
            raise ValueError(f"{name} must not overlap an input")
    return o, stride


def _qkv(q, k, v):
    """Checked token rows of q, k [L, Hk, D] and v [L, H, D]: ((q, stride), (k, ...), (v, ...), vec)."""
    dtype = v.dtype
    if dtype not in _DTYPE:
        raise ValueError(f"unsupported dtype {dtype}")
    vec = 8 if dtype is torch.bfloat16 else 4
    q, sq = _rows(q, "q", vec)
    k, sk = _rows(k, "k", vec)
    v, sv = _rows(v, "v", vec)
    dev = v.get_device()
    if q.dtype is not dtype or k.dtype is not dtype or q.get_device() != dev or k.get_device() != dev:
        raise ValueError("q, k and v must share dtype and device")
    L, H, D = v.shape
    Hk = q.shape[1]
    if q.shape != k.shape or q.shape[0] != L or q.shape[2] != D:
        raise ValueError("q and k must be [L, key heads, D] beside v [L, H, D]")
    if Hk < 1 or H % Hk != 0:
        raise ValueError(f"{H} value heads are no multiple of {Hk} key heads")
    if D not in (64, 128, 256):
        raise ValueError(f"head dim {D} is not 64, 128 or 256")
    return q, sq, k, sk, v, sv, vec


def _head_decay(g, L, H, dev, channels=None):
    """Log decay None, [H], [L, H] (or [L, H, channels]) -> (tensor, layout)."""
    if g is None:
        return None, _lib.GATE_NONE
    if g.dtype != torch.float32 or g.device != dev:
        raise ValueError(f"log-decay must be float32 on {dev}")
    shape = tuple(g.shape)
    if shape == (H,):
        return g.contiguous(), _lib.GATE_CONSTANT
    if shape[:1] == (1,) and len(shape) > 2 and shape[1] == L and shape != (L, H, channels):
        g, shape = g[0], shape[1:]
    if shape == (L, H) or shape == (L, H, 1):
        return g.contiguous(), _lib.GATE_PER_HEAD
    if channels is not None and shape == (L, H, channels):
        return g.contiguous(), _lib.GATE_PER_CHANNEL
    raise ValueError(f"g: expected [{H}], [{L}, {H}]" + (f" or [{L}, {H}, {channels}]" if channels else "")
                     + f", got {shape}")


def _offsets(cu_seqlens, L, dev):
    """Device int32 offsets. Host offsets are validated and copied in stream order, from memory of their own."""
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError("cu_seqlens must hold at least two integer offsets")
    if not cu_seqlens.is_cuda:
        cu = cu_seqlens.to(torch.int64)
        if int(cu[0]) < 0 or int(cu[-1]) > L or bool((cu[1:] < cu[:-1]).any()):
            raise ValueError("cu_seqlens must be nondecreasing offsets within the token rows")
        with torch.cuda.device(dev):
            if torch.cuda.is_current_stream_capturing():
                raise ValueError("cu_seqlens must be on the device while a graph is captured")
        cu_seqlens = cu_seqlens.to(torch.int32, copy=True).contiguous()
        return cu_seqlens.to(dev, non_blocking=True)  # pageable: staged before the call returns
    elif cu_seqlens.device != dev:
        raise ValueError(f"cu_seqlens must be on {dev}")
    if cu_seqlens.dtype is torch.int64:  # clamped as the kernels clamp, before 32 bits lose what is outside
        cu_seqlens = cu_seqlens.clamp(0, L).to(torch.int32)
    return cu_seqlens.contiguous()


def linear_attention(q, k, v, g, initial_state, cu_seqlens, *, scale=None, out=None, final_state=None,
                     initial_slots=None, final_slots=None):
    """Causal linear attention over packed samples -> (o [L, H, D] in v's dtype, final_state).

    Per sample: S_t = exp(g_t) S_{t-1} + k_t v_t^T from ``initial_state``, o_t = scale S_t^T q_t.
    q, k: [L, Hk, D]; v: [L, H, D], bf16 (tensor cores) or fp32 (exact token recurrence), D 64, 128 or
    256; a leading 1 and split views are accepted. g: fp32 natural-log decay <= 0, [L, H] for each
    token or [H] for all, or None (no decay). initial_state: fp32 [N, H, D, D], or None for zeros.
    cu_seqlens: N + 1 offsets, int32 on the device (int64 or host offsets are converted, host ones not
    while a graph is captured); rows of o outside every sample are left as they were. scale defaults to D ** -0.5.

    initial_slots / final_slots (int32 [N] on the device): initial_state / final_state are then pools
    [S, H, D, D], and sample n starts from initial_state[initial_slots[n]] and ends in
    final_state[final_slots[n]]. A slot outside its pool reads zeros, or is not written; of samples
    that name one final slot the first is written. The two pools may be one tensor if no sample starts
    from a slot that another one ends in. ``out`` must not overlap any other argument, nor the final
    states any but the initial ones.
    """
    q, sq, k, sk, v, sv, vec = _qkv(q, k, v)
    L, H, D = v.shape
    dev = v.device
    g, g_layout = _head_decay(g, L, H, dev)
    cu = _offsets(cu_seqlens, L, dev)
    N = cu.numel() - 1
    n_in = n_out = 0
    if initial_state is None:
        if initial_slots is not None:
            raise ValueError("initial_slots index into initial_state, which must then be given")
    else:
        initial_state, initial_slots, n_in = _pool(initial_state, initial_slots, N, H, D, D, dev, "initial_state")
    if final_state is None:
        if final_slots is not None:
            raise ValueError("final_slots index into final_state, which must then be given")
        final_state = torch.empty(N, H, D, D, device=dev, dtype=torch.float32)
    elif final_slots is not None:
        _, final_slots, n_out = _pool(final_state, final_slots, N, H, D, D, dev, "final_state")
    else:
        _states(final_state, N, H, D, D, dev, "final_state")
        if not final_state.is_contiguous():
            raise ValueError("final_state must be contiguous")
    if out is None:
        o, so = torch.empty(L, H, D, device=dev, dtype=v.dtype), H * D
    else:
        o, so = _out_rows(out, v, ((q, sq), (k, sk), (v, sv)), vec)
    lib = _lib.load()
    dtype = _DTYPE[v.dtype]
    need = lib.memt_linear_attention_workspace_size(N, L, H, D, dtype)
    # from the caching allocator, so that neither streams nor captured graphs share it
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 256 else None
    args = _linear_args(
        N, H, q.shape[1], D, dtype, L, cu.data_ptr(), q.data_ptr(), sq, k.data_ptr(), sk, v.data_ptr(), sv, _ptr(g),
        g_layout, D ** -0.5 if scale is None else scale, o.data_ptr(), so, _ptr(initial_state), final_state.data_ptr(),
        _ptr(initial_slots), n_in, _ptr(final_slots), n_out)
    _call("memt_linear_attention", dev, args, _ptr(ws), need)
    return o, final_state


def linear_attention_step(q, k, v, g, states, *, scale=None, slots=None, out=None):
    """One token of ``linear_attention`` for each of N sessions -> o [N, H, D]; states in place.

    q, k: [N, Hk, D]; v: [N, H, D], bf16 or fp32; g: fp32 [N, H], [H] or None. states: fp32
    [N, H, D, D], or with slots (int32 [N] on the device) a pool [S, H, D, D] of which session n
    updates states[slots[n]]. A session whose slot lies outside the pool, or is an earlier session's,
    is skipped: its state and its row of o are left as they were (pad a batch with slot -1). Neither
    ``out`` nor the states may overlap any other argument.
    """
    return _step(_lib.RULE_LINEAR, q, k, v, g, states, None, None, None, scale, slots, False, out)


def gdn2_step(q, k, v, g, states, *, beta=None, erase=None, write=None, scale=None, slots=None, read_incoming=False,
              out=None):
    """One token of the stable GDN-2 rule for each of N sessions -> o [N, H, D]; states in place.

    The recurrence of ``gdn2_update`` in fp32 arithmetic: k' = sqrt(beta) k, S~ = diag(exp(g)) S,
    S = S~ + k' (write v - S~^T (erase k'))^T. o = scale S^T q reads the new state, or with
    ``read_incoming`` the state before the update, as a commit does. g: fp32 [N, H], [N, H, D], [H]
    or None; beta: [N, Hk] or [N, Hk, D]; erase: [N, Hk, D]; write: [N, H, D], in q's dtype. States,
    slots, heads and overlaps as in ``linear_attention_step``.
    """
    return _step(_lib.RULE_GDN2, q, k, v, g, states, beta, erase, write, scale, slots, read_incoming, out)


def _gate_rows(x, shapes, like, name):
    if x.dtype != like.dtype or x.device != like.device:
        raise ValueError(f"{name}: expected {like.dtype} on {like.device}")
    shape = tuple(x.shape)
    if shape not in shapes:
        if shape[:1] == (1,) and shape[1:] in shapes:
            x = x[0]
        else:
            raise ValueError(f"{name}: expected {' or '.join(map(str, shapes))}, got {shape}")
    return x.contiguous()


def _step(rule, q, k, v, g, states, beta, erase, write, scale, slots, read_incoming, out):
    q, sq, k, sk, v, sv, vec = _qkv(q, k, v)
    N, H, D = v.shape
    Hk = q.shape[1]
    dev = v.device
    g, g_layout = _head_decay(g, N, H, dev, D if rule == _lib.RULE_GDN2 else None)
    beta_layout = _lib.GATE_NONE
    if beta is not None:
        beta = _gate_rows(beta, ((N, Hk), (N, Hk, D)), v, "beta")
        beta_layout = _lib.GATE_PER_HEAD if beta.dim() == 2 else _lib.GATE_PER_CHANNEL
    if erase is not None:
        erase = _gate_rows(erase, ((N, Hk, D),), v, "erase")
    if write is not None:
        write = _gate_rows(write, ((N, H, D),), v, "write")
    if not states.is_contiguous():
        raise ValueError("states are updated in place and must be contiguous")
    _, slots, num_slots = _pool(states, slots, N, H, D, D, dev, "states")
    if out is None:
        o, so = torch.empty(N, H, D, device=dev, dtype=v.dtype), H * D
    else:
        o, so = _out_rows(out, v, ((q, sq), (k, sk), (v, sv)), vec)
    if N == 0:
        return o
    args = _step_args(
        rule, N, H, Hk, D, _DTYPE[v.dtype], 1 if read_incoming else 0, q.data_ptr(), sq, k.data_ptr(), sk, v.data_ptr(),
        sv, _ptr(g), g_layout, beta_layout, _ptr(beta), _ptr(erase), _ptr(write), states.data_ptr(), _ptr(slots),
        num_slots, D ** -0.5 if scale is None else scale, o.data_ptr(), so)
    _call("memt_recurrent_step", dev, args)
    return o
