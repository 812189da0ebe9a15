"""The gated delta rule over prompts and single tokens, and rotary positions with several axes: what is timed.

Three operators, each beside its plain form in elementary torch operations:

* ``gated_delta``  packed prompts, S_t = a_t S_{t-1} + beta_t k_t (v_t - a_t S_{t-1}^T k_t)^T with a_t = exp(g_t),
                   o_t = scale S_t^T q_t: every token reads the state it has just written
* ``gated_delta_step``  one token of it for each session, the states updated in place
* ``rotary_axes``  rotary positions of queries and keys with several axes (time, height, width), each pair
                   of elements turned by the position on an axis of its own

Shapes: q, k [L, key_heads, dim]; v, o [L, heads, dim] (value head h uses key head
h // (heads // key_heads)); g fp32 [L, heads] or [heads]; beta [L, heads]; states fp32
[samples, heads, dim, dim] or a pool of such rows; positions [axes, L].
"""

import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda"
CHUNK = 64           # tokens per chunk of the plain form
_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_package = None


def _memt():
    global _package
    if _package is None:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "memt-1.0_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        import memt_b200

        _package = memt_b200
    return _package


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _prompts(name, sessions, tokens, key_heads, heads, dim, *, dtype="bf16", ragged=False, decay="token", pool=False):
    case = {"op": "gated_delta", "sessions": sessions, "tokens": tokens, "key_heads": key_heads, "heads": heads,
            "dim": dim, "dtype": dtype, "ragged": ragged, "decay": decay, "pool": pool}
    return {"name": name, **case} if name else case


def _step(name, sessions, key_heads, heads, dim, *, dtype="bf16", decay="token", pool=True):
    case = {"op": "gated_delta_step", "sessions": sessions, "tokens": 1, "key_heads": key_heads, "heads": heads,
            "dim": dim, "dtype": dtype, "ragged": False, "decay": decay, "pool": pool}
    return {"name": name, **case} if name else case


def _axes(name, tokens, heads, key_heads, dim, rotary_dim, axes, *, dtype="bf16", cycled=False, interleaved=False,
          inverse=False, in_place=False, first=0):
    case = {"op": "rotary_axes", "tokens": tokens, "heads": heads, "key_heads": key_heads, "dim": dim,
            "rotary_dim": rotary_dim, "axes": axes, "dtype": dtype, "cycled": cycled, "interleaved": interleaved,
            "inverse": inverse, "in_place": in_place, "first": first}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one short first message: latency
        _prompts("delta prompt short", 1, 100, 4, 4, 64, decay="head"),
        # eight sessions of one 8192-token segment each: the benchmark's update shape
        _prompts("delta prompts even", 8, 8192, 16, 16, 128),
        # a serving batch packed by cu_seqlens, an empty sample in it, shared key heads, states in a pool
        _prompts("delta prompts ragged pool", 16, 16384, 8, 16, 128, ragged=True, decay="head", pool=True),
        # one session's long history: few chains
        _prompts("delta prompt long", 1, 65536, 16, 16, 128),
        # a rank's heads of the wide layer
        _prompts("delta prompts wide heads", 4, 4096, 16, 16, 256),
        # a serving step in which each of many sessions brings a few tokens, states in a pool
        _prompts("delta sessions few tokens", 256, 16, 16, 16, 128, ragged=True, pool=True),
        # two sessions of a small layer in fp32
        _prompts("delta prompts fp32", 2, 1000, 2, 4, 64, dtype="fp32", ragged=True),
        # decode of 256 concurrent sessions, one layer
        _step("delta step 256 sessions", 256, 16, 16, 128),
        # decode of a single session of a small layer in fp32: latency
        _step("delta step one fp32", 1, 4, 8, 64, dtype="fp32", decay="head", pool=False),
        # queries and keys of packed video prompts, whole heads, far positions in time
        _axes("axes prompts", 65536, 16, 16, 128, 128, 3, first=1000000),
        # a part of wide heads, the axes in turn, interleaved pairs, backward direction, odd token count
        _axes("axes part inverse", 8191, 16, 2, 256, 64, 3, dtype="fp32", cycled=True, interleaved=True, inverse=True,
              first=30000),
        # decode of 256 sessions, in place
        _axes("axes decode", 256, 16, 2, 128, 128, 3, cycled=True, in_place=True, first=5),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["gated_delta", "gated_delta", "gated_delta", "gated_delta_step", "rotary_axes"])
    dim = rng.choice([64, 128, 128, 256])
    key_heads = _log_int(rng, 1, 16)
    heads = key_heads * rng.choice([1, 1, 2, 4])
    if op == "rotary_axes":
        most = min(65536, (1 << 28) // (dim * (heads + key_heads)))
        return _axes(None, _log_int(rng, 1, most), heads, key_heads, dim, rng.choice([dim, dim // 2, dim // 4]),
                     rng.choice([1, 2, 3, 3, 4]), dtype=rng.choice(["bf16", "fp32"]) if dim < 256 else "bf16",
                     cycled=rng.random() < 0.5, interleaved=rng.random() < 0.5, inverse=rng.random() < 0.5,
                     in_place=rng.random() < 0.5, first=_log_int(rng, 1, 1000000))
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op == "gated_delta_step":
        return _step(None, _log_int(rng, 1, max(1, min(256, (1 << 26) // (heads * dim * dim)))), key_heads, heads, dim,
                     dtype=rng.choice(["bf16", "fp32"]), decay=rng.choice(["head", "token"]), pool=rng.random() < 0.5)
    if rng.random() < 0.3:  # many sessions of few tokens
        sessions = _log_int(rng, 8, max(8, min(256, (1 << 26) // (heads * dim * dim))))
        tokens = _log_int(rng, 1, 64)
    else:
        sessions = _log_int(rng, 1, 32)
        room = (1 << 27 if dtype == "bf16" else 1 << 22) // (sessions * heads * dim)
        tokens = _log_int(rng, 1, max(1, min(65536 if dim < 256 else 16384, room)))
    return _prompts(None, sessions, tokens, key_heads, heads, dim, dtype=dtype, ragged=rng.random() < 0.5,
                    decay=rng.choice(["head", "token", "token"]), pool=rng.random() < 0.5)


def _lengths(case):
    """Tokens of each sample: equal, or spread from the longest down with one empty sample."""
    n, most = case["sessions"], case["tokens"]
    if not case["ragged"]:
        return [most] * n
    r = random.Random(1000 * n + most)
    lengths = [most] + [r.randint(1, most) for _ in range(n - 1)]
    if n > 3:
        lengths[2] = 0
    return lengths


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEVICE).to(dtype)


def _unit(gen, shape, dtype):
    x = torch.randn(shape, generator=gen, device=DEVICE)
    return (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dim, heads, kh, dtype = case["dim"], case["heads"], case["key_heads"], _TYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "rotary_axes":
        rows, axes, pairs = case["tokens"], case["axes"], case["rotary_dim"] // 2
        s["q"] = _normal(gen, (rows, heads, dim), dtype)
        s["k"] = _normal(gen, (rows, kh, dim), dtype)
        s["positions"] = _grid(gen, rows, axes, case["first"])
        s["inv_freq"] = torch.pow(torch.tensor(10000.0, device=DEVICE, dtype=torch.float64),
                                  -torch.arange(pairs, device=DEVICE, dtype=torch.float64) / pairs)
        s["pair_axes"] = _pair_axes(pairs, axes, case["cycled"])
        return s
    n, lengths = case["sessions"], _lengths(case)
    rows = sum(lengths)
    s["cu_seqlens"] = torch.cumsum(torch.tensor([0] + lengths, device=DEVICE, dtype=torch.int32), 0, dtype=torch.int32)
    s["longest"] = max(lengths)
    s["q"] = _unit(gen, (rows, kh, dim), dtype)
    s["k"] = _unit(gen, (rows, kh, dim), dtype)
    s["v"] = _normal(gen, (rows, heads, dim), dtype)
    if case["decay"] == "head":  # fixed slopes
        s["g"] = -torch.exp2(-8.0 * torch.arange(1, heads + 1, device=DEVICE, dtype=torch.float32) / heads)
    else:
        s["g"] = torch.nn.functional.logsigmoid(2.0 + 0.5 * _normal(gen, (rows, heads)))
    s["beta"] = torch.sigmoid(_normal(gen, (rows, heads))).to(dtype)
    s["scale"] = dim ** -0.5
    states, s["slots"] = n, None
    if case["pool"]:
        states = n + max(1, n // 8)
        s["slots"] = torch.randperm(states, generator=gen, device=DEVICE)[:n].to(torch.int32)
    s["states"] = 0.02 * _normal(gen, (states, heads, dim, dim))
    return s


def _grid(gen, rows, axes, first):
    """Positions of the patches of images in time order: frames of 24 x 32 patches (of 8 and 4 more on a fourth axis)."""
    t = torch.arange(rows, device=DEVICE)
    start = torch.randint(0, 1000, (1,), generator=gen, device=DEVICE) + first
    each = [start + t] if axes == 1 else [start + t // 768, start % 97 + t // 32 % 24, start % 89 + t % 32, t % 4]
    return torch.stack([x.expand(rows) for x in each[:axes]])


def _pair_axes(pairs, axes, cycled):
    """The axis of each pair: the axes in turn, or a run of pairs for each (the first gets what is left over)."""
    i = torch.arange(pairs, device=DEVICE)
    if cycled:
        return (i % axes).to(torch.int32)
    run = pairs // axes
    return ((i - (pairs - run * axes)).clamp(min=0) // max(run, 1)).clamp(max=axes - 1).to(torch.int32)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    return _RUN[s["op"]](s)


def _run_gated_delta(s):
    if own:
        if s["pool"]:
            return list(_memt().gated_delta(s["q"], s["k"], s["v"], s["g"], s["beta"], s["states"], s["cu_seqlens"],
                                            scale=s["scale"], initial_slots=s["slots"], final_state=s["states"],
                                            final_slots=s["slots"]))
        return list(_memt().gated_delta(s["q"], s["k"], s["v"], s["g"], s["beta"], s["states"], s["cu_seqlens"],
                                        scale=s["scale"]))
    o, final = _plain_gated_delta(s["q"], s["k"], s["v"], s["g"], s["beta"], s["states"], s["slots"], s["cu_seqlens"],
                                  s["longest"], s["scale"])
    if s["pool"]:
        s["states"][s["slots"].long()] = final
        final = s["states"]
    return [o, final]


def _plain_gated_delta(q, k, v, g, beta, states, slots, cu, longest, scale):
    """Chunked, fp32, the samples padded to the longest. Within a chunk the tokens' corrections are the solution
    of a unit triangular system, whose inverse (the product of I + (-A)^(2^i), exact after six factors) is formed
    in 64 bits; everything but the state's own chain of two products a chunk is done for all chunks at once."""
    rows, heads, dim = v.shape
    rep = heads // q.shape[1]
    n, chunks = cu.numel() - 1, -(-longest // CHUNK)
    at = torch.arange(chunks * CHUNK, device=q.device)
    length = (cu[1:] - cu[:-1]).long()
    live = at[None, :] < length[:, None]                                     # [n, T]
    index = (cu[:-1].long()[:, None] + at[None, :]).clamp(max=rows - 1)

    def tiles(x):  # [rows, h, d] -> fp32 [n, h, chunks, CHUNK, d], zero rows behind each sample
        x = torch.where(live[:, :, None, None], x[index].float(), 0.0)
        return x.view(n, chunks, CHUNK, x.shape[2], x.shape[3]).permute(0, 3, 1, 2, 4)

    qt, kt = tiles(q).repeat_interleave(rep, 1), tiles(k).repeat_interleave(rep, 1)
    vt, bt = tiles(v), tiles(beta[..., None])
    gt = (g.double().expand(rows, heads) if g.dim() == 1 else g.double())[index]
    gt = torch.where(live[:, :, None], gt, 0.0).view(n, chunks, CHUNK, heads).permute(0, 3, 1, 2)
    run_g = gt.cumsum(-1)                                                    # [n, h, chunks, CHUNK]
    grown = run_g.exp().float()[..., None]
    i = torch.arange(CHUNK, device=q.device)
    weight = torch.where(i[:, None] >= i, run_g[..., :, None] - run_g[..., None, :], -math.inf).exp()
    below = (kt @ kt.transpose(-1, -2)).double() * weight * bt * (i[:, None] > i)
    inverse = torch.eye(CHUNK, dtype=torch.float64, device=q.device) - below
    power = below
    for _ in range(5):
        power = power @ power
        inverse = inverse + inverse @ power
    inverse = inverse.float()
    written, known = inverse @ (bt * vt), inverse @ (bt * grown * kt)
    scores = (qt @ kt.transpose(-1, -2)) * weight.float()
    ahead = (kt * (run_g[..., -1:] - run_g).exp().float()[..., None]).transpose(-1, -2)
    kept = grown[..., -1:, :]
    s = (states if slots is None else states[slots.long()]).float()
    incoming, values = [], []
    for c in range(chunks):  # the chain: each chunk corrects what the state before it holds
        incoming.append(s)
        values.append(written[:, :, c] - known[:, :, c] @ s)
        s = kept[:, :, c] * s + ahead[:, :, c] @ values[c]
    incoming, values = torch.stack(incoming, 2), torch.stack(values, 2)
    o = (scale * ((qt * grown) @ incoming + scores @ values)).to(v.dtype)
    o = o.permute(0, 2, 3, 1, 4).reshape(n, chunks * CHUNK, heads, dim)
    token = torch.arange(rows, device=q.device)
    sample = torch.searchsorted(cu[1:].long(), token, right=True)
    return o[sample, token - cu.long()[sample]], s.contiguous()


def _run_gated_delta_step(s):
    if own:
        return [_memt().gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["states"], scale=s["scale"],
                                         slots=s["slots"]), s["states"]]
    rep = s["v"].shape[1] // s["q"].shape[1]
    q, k = s["q"].float().repeat_interleave(rep, 1), s["k"].float().repeat_interleave(rep, 1)
    at = slice(None) if s["slots"] is None else s["slots"].long()
    state = s["states"][at] * s["g"].exp()[..., None, None]
    delta = s["beta"].float()[..., None] * (s["v"].float() - (k[..., None, :] @ state).squeeze(-2))
    state = state + k[..., :, None] * delta[..., None, :]
    s["states"][at] = state
    return [(s["scale"] * (q[..., None, :] @ state).squeeze(-2)).to(s["v"].dtype), s["states"]]


def _run_rotary_axes(s):
    if own:
        place = {"q_out": s["q"], "k_out": s["k"]} if s["in_place"] else {}
        return list(_memt().rotary_axes(s["q"], s["k"], s["positions"], s["inv_freq"], s["pair_axes"],
                                        interleaved=s["interleaved"], inverse=s["inverse"], **place))
    angle = s["positions"].double()[s["pair_axes"].long()].transpose(0, 1) * s["inv_freq"]
    cos = angle.cos().float()[:, None]
    sin = (-angle.sin() if s["inverse"] else angle.sin()).float()[:, None]
    q = _plain_rotate(s["q"], cos, sin, s["interleaved"])
    k = _plain_rotate(s["k"], cos, sin, s["interleaved"])
    if s["in_place"]:
        q, k = s["q"].copy_(q), s["k"].copy_(k)
    return [q, k]


def _plain_rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    part, rest = x[..., :2 * half].float(), x[..., 2 * half:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., :half], part[..., half:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y.to(x.dtype), rest), -1)


_RUN = {"gated_delta": _run_gated_delta, "gated_delta_step": _run_gated_delta_step, "rotary_axes": _run_rotary_axes}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    dim, heads, kh = case["dim"], case["heads"], case["key_heads"]
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "rotary_axes":
        part = case["rotary_dim"] if case["in_place"] else dim
        rows = case["tokens"] * (heads + kh)
        return {"bytes": rows * part * 2 * size + case["tokens"] * case["axes"] * 8, "flops": rows * case["rotary_dim"] * 3}
    rows = sum(_lengths(case))
    state = case["sessions"] * heads * dim * dim
    gates = (heads * 4 if case["decay"] == "head" else rows * heads * 4) + rows * heads * size
    # The recurrence itself costs 7 dim^2 for each token and head (decay, prediction, rank-one update, read). In chunks
    # of C tokens: three products with the state, 6 dim^2, and the causal halves of four with C tokens, 4 C dim.
    return {"bytes": rows * dim * (2 * kh + 2 * heads) * size + gates + 8 * state,
            "flops": rows * heads * min(7 * dim * dim, 6 * dim * dim + 4 * CHUNK * dim)}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary_axes":
        return [_exact_rotary(s, s["q"]), _exact_rotary(s, s["k"])]
    lengths = _lengths(case)
    rows, heads, dim = s["v"].shape
    rep = heads // s["q"].shape[1]
    q, k = (x.double().repeat_interleave(rep, 1) * f for x, f in ((s["q"], s["scale"]), (s["k"], 1.0)))
    v, beta, a = s["v"].double(), s["beta"].double(), torch.exp(s["g"].double()).expand(rows, heads)
    states = s["states"].double()
    # token by token; the samples that still have tokens are the first ones when sorted by length
    order = sorted(range(len(lengths)), key=lambda j: -lengths[j])
    picked = torch.tensor(order, device=DEVICE)
    where = picked if s["slots"] is None else s["slots"].long()[picked]
    begin = s["cu_seqlens"].long()[picked]
    state = states[where]
    o = torch.zeros_like(v)
    alive = len(order)
    for t in range(max(lengths)):
        while alive and lengths[order[alive - 1]] <= t:
            alive -= 1
        at, S = begin[:alive] + t, state[:alive]
        S.mul_(a[at][..., None, None])
        known = torch.matmul(k[at][..., None, :], S)[..., 0, :]
        S.addcmul_(k[at][..., :, None], (beta[at][..., None] * (v[at] - known))[..., None, :])
        o[at] = torch.matmul(q[at][..., None, :], S)[..., 0, :]
    states[where] = state
    return [o, states]


def _exact_rotary(s, x):
    """Each pair as a complex number, turned by the angle of its axis's position."""
    pairs = s["rotary_dim"] // 2
    turn = torch.empty(s["tokens"], pairs, device=x.device, dtype=torch.float64)
    for i, axis in enumerate(s["pair_axes"].tolist()):
        turn[:, i] = s["positions"][axis].double() * s["inv_freq"][i]
    turn = torch.exp(torch.complex(torch.zeros_like(turn), -turn if s["inverse"] else turn))[:, None, :]
    y = x.double()
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if s["interleaved"] else \
        (slice(0, pairs), slice(pairs, 2 * pairs))
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y
