"""The per-head-decay linear attention, the single-token recurrences and the rotary positions: what is timed.

Four operators, each beside its plain form in elementary torch operations:

* ``linear_attention``       packed prompts, S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t
* ``linear_attention_step``  one token for each session, the states updated in place
* ``gdn2_step``              one token of the gated delta rule for each session, the states updated in place
* ``rotary``                 rotary positions of queries and keys, both layouts, whole heads or a part of them

Shapes: q, k [L, key_heads, dim]; v, o [L, heads, dim] (value head h reads key head
h // (heads // key_heads)); states fp32 [samples, heads, dim, dim] or a pool of such rows.
"""

import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda"
CHUNK = 128          # tokens per chunk of the plain form
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

def _prompts(name, sessions, tokens, key_heads, heads, dim, *, ragged=False, decay="token", pool=False):
    case = {"op": "linear_attention", "sessions": sessions, "tokens": tokens, "key_heads": key_heads, "heads": heads,
            "dim": dim, "ragged": ragged, "decay": decay, "pool": pool}
    return {"name": name, **case} if name else case


def _step(name, op, sessions, key_heads, heads, dim, *, dtype="bf16", decay="head", pool=True, incoming=False):
    case = {"op": op, "sessions": sessions, "key_heads": key_heads, "heads": heads, "dim": dim, "dtype": dtype,
            "decay": decay, "pool": pool}
    if op == "gdn2_step":
        case["incoming"] = incoming
    return {"name": name, **case} if name else case


def _rotary(name, tokens, heads, key_heads, dim, rotary_dim, *, dtype="bf16", interleaved=False, inverse=False,
            scaling="none", in_place=False, first=0):
    case = {"op": "rotary", "tokens": tokens, "heads": heads, "key_heads": key_heads, "dim": dim,
            "rotary_dim": rotary_dim, "dtype": dtype, "interleaved": interleaved, "inverse": inverse,
            "scaling": scaling, "in_place": in_place, "first": first}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one short first message: latency
        _prompts("prompt short", 1, 100, 4, 4, 64, decay="head"),
        # eight sessions of one 8192-token segment each: the benchmark's update shape
        _prompts("prompts even", 8, 8192, 16, 16, 128),
        # a serving batch packed by cu_seqlens, an empty sample in it, shared key heads, states in a pool
        _prompts("prompts ragged pool", 16, 16384, 8, 16, 128, ragged=True, decay="head", pool=True),
        # a rank's heads of the wide layer, long prompts
        _prompts("prompts wide heads", 4, 16384, 16, 16, 256),
        # one session's long history: few chains, so the tokens have to be split
        _prompts("prompt long", 1, 65536, 16, 16, 128, decay="head"),
        # decode of 256 concurrent sessions, one layer
        _step("step 256 sessions", "linear_attention_step", 256, 16, 16, 128),
        # decode of a single session: latency
        _step("step one session", "linear_attention_step", 1, 8, 16, 128, decay="token", pool=False),
        # one committed token in each of 256 sessions, channel-wise decay and write gate
        _step("delta step 256 sessions", "gdn2_step", 256, 16, 16, 128, decay="channel"),
        # a few sessions in fp32, reading the incoming snapshot
        _step("delta step few fp32", "gdn2_step", 3, 4, 4, 64, dtype="fp32", decay="token", pool=False, incoming=True),
        # queries and keys of a packed prompt batch, whole heads, far positions
        _rotary("rotary prompts", 65536, 16, 16, 128, 128, first=1000000),
        # a part of wide heads, interleaved pairs, stretched context, backward direction, odd token count
        _rotary("rotary part inverse", 8191, 16, 2, 256, 64, dtype="fp32", interleaved=True, inverse=True,
                scaling="yarn", first=30000),
        # decode of 256 sessions, in place
        _rotary("rotary decode", 256, 16, 2, 128, 128, in_place=True, scaling="linear", first=5),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["linear_attention", "linear_attention", "linear_attention_step", "gdn2_step", "rotary"])
    dim = rng.choice([64, 128, 128, 256])
    key_heads = _log_int(rng, 1, 16)
    heads = key_heads * rng.choice([1, 1, 2, 4])
    if kind == "linear_attention":
        sessions = _log_int(rng, 1, 32)
        most = min(65536, (1 << 27) // (sessions * heads * dim))
        tokens = _log_int(rng, 1, max(most, 1))
        return _prompts(None, sessions, tokens, key_heads, heads, dim, ragged=rng.random() < 0.5,
                        decay=rng.choice(["head", "token"]), pool=rng.random() < 0.5)
    if kind == "rotary":
        most = min(65536, (1 << 28) // (dim * (heads + key_heads)))
        return _rotary(None, _log_int(rng, 1, most), heads, key_heads, dim, rng.choice([dim, dim // 2, dim // 4]),
                       dtype=rng.choice(["bf16", "fp32"]) if dim < 256 else "bf16", interleaved=rng.random() < 0.5,
                       inverse=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "yarn"]),
                       in_place=rng.random() < 0.5, first=_log_int(rng, 1, 1000000))
    sessions = _log_int(rng, 1, max(1, min(256, (1 << 26) // (heads * dim * dim))))
    decay = rng.choice(["head", "token"] if kind == "linear_attention_step" else ["token", "channel"])
    return _step(None, kind, sessions, key_heads, heads, dim, dtype=rng.choice(["bf16", "fp32"]), decay=decay,
                 pool=rng.random() < 0.5, incoming=rng.random() < 0.5)


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


def _decay(gen, kind, rows, heads, dim):
    """Log decays: fixed slopes for each head, or logsigmoid(N(2, 0.5)) for each token (and channel)."""
    if kind == "head":
        return -torch.exp2(-8.0 * torch.arange(1, heads + 1, device=DEVICE, dtype=torch.float32) / heads)
    shape = (rows, heads, dim) if kind == "channel" else (rows, heads)
    return torch.nn.functional.logsigmoid(2.0 + 0.5 * _normal(gen, shape))


def _slots(gen, n):
    """(rows of the pool, a slot for each sample)"""
    rows = n + max(1, n // 8)
    return rows, torch.randperm(rows, generator=gen, device=DEVICE)[:n].to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    op, dim, heads, kh = case["op"], case["dim"], case["heads"], case["key_heads"]
    s = dict(case)
    if op == "rotary":
        dtype = _TYPES[case["dtype"]]
        s["q"] = _normal(gen, (case["tokens"], heads, dim), dtype)
        s["k"] = _normal(gen, (case["tokens"], kh, dim), dtype)
        first = torch.randint(0, 1000, (1,), generator=gen, device=DEVICE) + case["first"]
        s["positions"] = first + torch.arange(case["tokens"], device=DEVICE)
        s["inv_freq"], s["attention_scale"] = _frequencies(case["rotary_dim"], case["scaling"])
        return s
    n = case["sessions"]
    if op == "linear_attention":
        lengths = _lengths(case)
        rows = sum(lengths)
        dtype = torch.bfloat16
        cu = torch.tensor([0] + lengths, device=DEVICE, dtype=torch.int32)
        s["cu_seqlens"] = torch.cumsum(cu, 0, dtype=torch.int32)
        s["longest"] = max(lengths)
    else:
        rows, dtype = n, _TYPES[case["dtype"]]
    s["q"] = _unit(gen, (rows, kh, dim), dtype)
    s["k"] = _unit(gen, (rows, kh, dim), dtype)
    s["v"] = _normal(gen, (rows, heads, dim), dtype)
    s["g"] = _decay(gen, case["decay"], rows, heads, dim)
    s["scale"] = dim ** -0.5
    states, s["slots"] = n, None
    if case["pool"]:
        states, s["slots"] = _slots(gen, n)
    s["states"] = 0.02 * _normal(gen, (states, heads, dim, dim))
    if op == "gdn2_step":
        s["beta"] = torch.sigmoid(_normal(gen, (rows, kh))).to(dtype)
        s["write"] = torch.sigmoid(_normal(gen, (rows, heads, dim))).to(dtype) if case["decay"] == "channel" else None
    return s


def _frequencies(rotary_dim, scaling):
    """fp64 angle per position of each pair and the factor on the rotated values."""
    base, factor, trained = 10000.0, 8.0, 4096
    pair = torch.arange(rotary_dim // 2, device=DEVICE, dtype=torch.float64)
    inv = torch.pow(torch.tensor(base, device=DEVICE, dtype=torch.float64), -2.0 * pair / rotary_dim)
    if scaling == "linear":
        return inv / factor, 1.0
    if scaling == "yarn":
        turn = lambda t: rotary_dim * math.log(trained / (2 * math.pi * t)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), rotary_dim - 1)
        ramp = ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return inv, 1.0


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    return _RUN[s["op"]](s)


def _run_linear_attention(s):
    if own:
        if s["pool"]:
            return list(_memt().linear_attention(s["q"], s["k"], s["v"], s["g"], s["states"], s["cu_seqlens"],
                                                 scale=s["scale"], initial_slots=s["slots"], final_state=s["states"],
                                                 final_slots=s["slots"]))
        return list(_memt().linear_attention(s["q"], s["k"], s["v"], s["g"], s["states"], s["cu_seqlens"],
                                             scale=s["scale"]))
    o, final = _plain_linear_attention(s["q"], s["k"], s["v"], s["g"], s["states"], s["slots"], s["cu_seqlens"],
                                       s["longest"], s["scale"])
    if s["pool"]:
        s["states"][s["slots"].long()] = final
        final = s["states"]
    return [o, final]


def _plain_linear_attention(q, k, v, g, states, slots, cu, longest, scale):
    """Chunked, fp32, every chunk at once: the samples padded to the longest, the states before each
    chunk as one product of the chunks' own contributions with their decays."""
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

    qt = tiles(q).repeat_interleave(rep, 1)
    kt = tiles(k).repeat_interleave(rep, 1)
    vt = tiles(v)
    gt = (g.double().expand(rows, heads) if g.dim() == 1 else g.double())[index]
    gt = torch.where(live[:, :, None], gt, 0.0).view(n, chunks, CHUNK, heads).permute(0, 3, 1, 2)
    run_g = gt.cumsum(-1)                                                    # [n, h, chunks, CHUNK]
    causal = at[:CHUNK, None] >= at[None, :CHUNK]
    weight = torch.where(causal, run_g[..., :, None] - run_g[..., None, :], -math.inf).exp().float()
    intra = ((qt @ kt.transpose(-1, -2)) * weight) @ vt
    own_part = (kt * (run_g[..., -1:] - run_g).exp().float()[..., None]).transpose(-1, -2) @ vt
    total = torch.nn.functional.pad(run_g[..., -1].cumsum(-1), (1, 0))       # [n, h, chunks + 1]
    before = at[:chunks + 1, None] > at[None, :chunks]
    carry = torch.where(before, total[..., :, None] - total[..., None, 1:], -math.inf).exp().float()
    first = (states if slots is None else states[slots.long()]).float()
    s = (carry @ own_part.flatten(-2)).view(n, heads, chunks + 1, dim, dim)
    s = s + total.exp().float()[..., None, None] * first[:, :, None]
    inter = (qt * run_g.exp().float()[..., None]) @ s[:, :, :-1]
    o = (scale * (inter + intra)).to(v.dtype).permute(0, 2, 3, 1, 4).reshape(n, chunks * CHUNK, heads, dim)
    token = torch.arange(rows, device=q.device)
    sample = torch.searchsorted(cu[1:].long(), token, right=True)
    return o[sample, token - cu.long()[sample]], s[:, :, -1].contiguous()


def _run_linear_attention_step(s):
    if own:
        return [_memt().linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["states"], scale=s["scale"],
                                              slots=s["slots"]), s["states"]]
    heads = s["v"].shape[1]
    rep = heads // s["q"].shape[1]
    q, k, v = s["q"].float().repeat_interleave(rep, 1), s["k"].float().repeat_interleave(rep, 1), s["v"].float()
    at = slice(None) if s["slots"] is None else s["slots"].long()
    state = s["states"][at] * s["g"].exp()[..., None, None] + k[..., :, None] * v[..., None, :]
    s["states"][at] = state
    o = s["scale"] * (q[..., None, :] @ state).squeeze(-2)
    return [o.to(s["v"].dtype), s["states"]]


def _run_gdn2_step(s):
    if own:
        return [_memt().gdn2_step(s["q"], s["k"], s["v"], s["g"], s["states"], beta=s["beta"], write=s["write"],
                                  scale=s["scale"], slots=s["slots"], read_incoming=s["incoming"]), s["states"]]
    heads = s["v"].shape[1]
    rep = heads // s["q"].shape[1]
    q, v = s["q"].float().repeat_interleave(rep, 1), s["v"].float()
    k = (s["k"].float() * s["beta"].float().sqrt()[..., None]).repeat_interleave(rep, 1)
    at = slice(None) if s["slots"] is None else s["slots"].long()
    first = s["states"][at]
    g = s["g"] if s["g"].dim() == 3 else s["g"][..., None]
    state = first * g.exp()[..., :, None]
    value = v if s["write"] is None else v * s["write"].float()
    delta = value - (k[..., None, :] @ state).squeeze(-2)
    state = state + k[..., :, None] * delta[..., None, :]
    o = s["scale"] * (q[..., None, :] @ (first if s["incoming"] else state)).squeeze(-2)
    s["states"][at] = state
    return [o.to(s["v"].dtype), s["states"]]


def _run_rotary(s):
    if own:
        place = {"q_out": s["q"], "k_out": s["k"]} if s["in_place"] else {}
        return list(_memt().rotary(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=s["interleaved"],
                                   inverse=s["inverse"], attention_scale=s["attention_scale"], **place))
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos = (angle.cos() * s["attention_scale"]).float()[:, None]
    sin = (angle.sin() * (-s["attention_scale"] if s["inverse"] else s["attention_scale"])).float()[:, None]
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


_RUN = {"linear_attention": _run_linear_attention, "linear_attention_step": _run_linear_attention_step,
        "gdn2_step": _run_gdn2_step, "rotary": _run_rotary}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op, dim, heads, kh = case["op"], case["dim"], case["heads"], case["key_heads"]
    if op == "rotary":
        size = 2 if case["dtype"] == "bf16" else 4
        part = case["rotary_dim"] if case["in_place"] else dim
        rows = case["tokens"] * (heads + kh)
        return {"bytes": rows * part * 2 * size + case["tokens"] * 8, "flops": rows * case["rotary_dim"] * 3}
    n = case["sessions"]
    state = n * heads * dim * dim
    if op == "linear_attention":
        rows = sum(_lengths(case))
        gates = heads * 4 if case["decay"] == "head" else rows * heads * 4
        # the recurrence itself: decay, rank-one update and read of the state for each token and head
        # cost 5 dim^2; in chunks of C tokens the products are 4 dim^2 + 2 C dim (causal half), C = 64
        return {"bytes": rows * dim * (2 * kh + 2 * heads) * 2 + gates + 8 * state,
                "flops": rows * heads * (4 * dim * dim + 2 * 64 * dim)}
    size = 2 if case["dtype"] == "bf16" else 4
    tokens = n * dim * (2 * kh + 2 * heads) * size
    gates = {"head": heads, "token": n * heads, "channel": n * heads * dim}[case["decay"]] * 4
    if op == "gdn2_step":
        tokens += n * kh * size + (n * heads * dim * size if case["decay"] == "channel" else 0)
    return {"bytes": tokens + gates + 8 * state, "flops": state * (5 if op == "linear_attention_step" else 7)}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return [_exact_rotary(s, s["q"]), _exact_rotary(s, s["k"])]
    rep = case["heads"] // case["key_heads"]
    q, k, v = s["q"].double().repeat_interleave(rep, 1), s["k"].double().repeat_interleave(rep, 1), s["v"].double()
    states = s["states"].double()
    first = states if s["slots"] is None else states[s["slots"].long()]
    if case["op"] == "linear_attention":
        o, final = _exact_recurrence(q, k, v, s["g"].double(), first, _lengths(case))
        o = o * s["scale"]
    else:
        g = s["g"].double()
        a = torch.exp(g)[..., None] if g.dim() == 3 else torch.exp(g)[..., None, None]
        final = first * a
        if case["op"] == "gdn2_step":
            k = k * torch.sqrt(s["beta"].double()).repeat_interleave(rep, 1)[..., None]
            v = v if s["write"] is None else v * s["write"].double()
            v = v - torch.einsum("nhk,nhkv->nhv", k, final)
        final = final + torch.einsum("nhk,nhv->nhkv", k, v)
        o = s["scale"] * torch.einsum("nhk,nhkv->nhv", q, first if case.get("incoming") else final)
    if s["slots"] is not None:
        states[s["slots"].long()] = final
        final = states
    return [o, final]


def _exact_recurrence(q, k, v, g, first, lengths):
    """Token by token; the samples that still have tokens are the first ones when sorted by length."""
    rows, heads, dim = v.shape
    if g.dim() == 1:
        g = g[None, :].expand(rows, heads)
    a = torch.exp(g)
    order = sorted(range(len(lengths)), key=lambda i: -lengths[i])
    start = [sum(lengths[:i]) for i in order]
    begin = torch.tensor(start, device=q.device)
    state = first[torch.tensor(order, device=q.device)].clone()
    o = torch.zeros_like(v)
    live = len(order)
    for t in range(max(lengths)):
        while live and lengths[order[live - 1]] <= t:
            live -= 1
        at = begin[:live] + t
        S = state[:live]
        S.mul_(a[at][..., None, None])
        S.addcmul_(k[at][..., :, None], v[at][..., None, :])
        o[at] = torch.matmul(q[at][..., None, :], S)[..., 0, :]
    final = torch.empty_like(state)
    final[torch.tensor(order, device=q.device)] = state
    return o, final


def _exact_rotary(s, x):
    """Each pair as a complex number, turned by the position's angle."""
    r = s["rotary_dim"]
    x = x.double()
    turn = torch.outer(s["positions"].double(), s["inv_freq"]) * (-1.0 if s["inverse"] else 1.0)
    turn = torch.polar(torch.full_like(turn, s["attention_scale"]), turn)[:, None, :]
    y = x.clone()
    if s["interleaved"]:
        z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * turn
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * turn
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y
