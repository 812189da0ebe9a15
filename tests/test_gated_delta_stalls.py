"""What the chunked gated-delta kernel does when a wait runs out, on the host: no GPU is made to stall.

The roles are those of test_gated_delta_order, with waits that give up: a role whose wait has run out waits for no
mbarrier any more and goes through its code to the end, the MMA and load warps without issuing anything. Named barriers
count arrivals, as the hardware does. The chain's warps, which otherwise only arrive at them, join them once they have
given up (``hand_over`` in the kernel).
"""

import random
import re
import subprocess
from pathlib import Path

import pytest

from test_gated_delta_order import roles as _roles

CSRC = Path(__file__).resolve().parents[1] / "memt-1.0_b200" / "csrc"
NAMED = ("barS", "barR", "barW", "barU", "barEnd")


class _Stuck(Exception):
    pass


def _run(ns, n, seed, alias, out, lose=None, gives_up=None, joins=True):
    """Runs until every role has ended, or raises _Stuck. lose: ("tile" or "batch", k), the k-th never
    lands or completes, nor do the batches behind it; gives_up: (role, i), that role's i-th wait runs out at once.
    joins: whether the chain's warps join named barriers once they have given up. Returns the roles that gave up."""
    rng = random.Random(seed)
    bars, roles = _roles(ns, n, alias, out)
    at = {name: next(role, None) for name, role in roles.items()}
    dead, last, waits = set(), {}, dict.fromkeys(at, 0)
    batches, tiles, issued = [], [], {"tile": 0, "batch": 0}
    weight = {name: rng.choice([1, 1, 5, 30]) for name in [*at, "tensor pipe", "tma"]}

    def reach(name, bar):  # an arrival at a named barrier: at most one of a warp in a phase
        if last.get((name, bar)) == bars[bar].done:
            raise _Stuck(f"{name} arrives twice in phase {bars[bar].done} of {bar}")
        last[name, bar] = bars[bar].done
        bars[bar].arrive()

    while True:
        ready, waiting = [], []
        for name, op in at.items():
            if op is None or op[0] == "joined" and bars[op[1]].done == op[2]:
                continue
            if op[0] == "wait" and name not in dead and bars[op[1]].done % 2 == op[2] % 2:
                waiting.append(name)
                if (name, waits[name]) == gives_up:
                    dead.add(name)
                else:
                    continue
            ready.append(name)
        ready += ["tensor pipe"] * bool(batches) + ["tma"] * bool(tiles)
        if not ready:
            if not waiting:
                left = {name: op for name, op in at.items() if op is not None}
                if left:
                    raise _Stuck(str(left))
                return dead
            dead.add(rng.choice(waiting))  # half a second later
            continue
        name = rng.choices(ready, [weight[r] for r in ready])[0]
        if name == "tensor pipe":
            for b in batches.pop(0):
                bars[b].arrive()
            continue
        if name == "tma":
            bars[tiles.pop(rng.randrange(len(tiles)))].arrive()
            continue
        kind, what, more = at[name]
        if kind == "wait":
            waits[name] += 1
        elif kind == "sync" or kind == "arrive" and what[0] in NAMED and name in dead and joins:
            at[name] = "joined", what, bars[what].done
            reach(name, what)
            continue
        elif kind == "arrive":
            if what[0] in NAMED:
                reach(name, what)
            else:
                bars[what].arrive()
        elif kind in ("issue", "load") and name not in dead:
            queue, sort = (batches, "batch") if kind == "issue" else (tiles, "tile")
            if lose is None or lose[0] != sort or issued[sort] < lose[1] or sort == "tile" and issued[sort] > lose[1]:
                queue.append(what)
            issued[sort] += 1
        at[name] = next(roles[name], None)


SHAPES = [(3, False), (2, True)]


@pytest.mark.parametrize("stages,alias", SHAPES)
@pytest.mark.parametrize("out", [True, False])
def test_every_role_ends_when_nothing_is_lost(stages, alias, out):
    for seed in range(20):
        assert _run(stages, 9, seed, alias, out) == set()


@pytest.mark.parametrize("stages,alias", SHAPES)
@pytest.mark.parametrize("out", [True, False])
@pytest.mark.parametrize("lose", [("tile", 0), ("tile", 3), ("tile", 8), ("batch", 0), ("batch", 10), ("batch", 33)])
def test_every_role_ends_when_something_is_lost(stages, alias, out, lose):
    for seed in range(15):
        assert _run(stages, 9, seed, alias, out, lose=lose)


@pytest.mark.parametrize("stages,alias", SHAPES)
@pytest.mark.parametrize("out", [True, False])
@pytest.mark.parametrize("role", ["mma", "loads", "table 0", "table 1", "outputs 2", "chain 0", "chain 7", "chain 12"])
def test_every_role_ends_when_one_gives_up(stages, alias, out, role):
    """Alone, with nothing lost: the others are still waiting for it."""
    for seed in range(4):
        for i in (0, 1, 2, 5, 8, 20):
            _run(stages, 9, seed, alias, out, gives_up=(role, i))


def test_passing_a_barrier_after_giving_up_gets_stuck():
    """What hand_over is for."""
    stuck = 0
    for seed in range(40):
        try:
            _run(3, 9, seed, False, True, lose=("tile", 3), joins=False)
        except _Stuck:
            stuck += 1
    assert stuck == 40


def _code(name):
    return re.sub(r"//.*", "", (CSRC / name).read_text())


def test_the_chain_joins_named_barriers_once_it_has_given_up():
    code = _code("delta_tc.cuh")
    body = re.search(r"auto hand_over = \[&\]\(int id\) \{(.*?)\};", code, re.S).group(1)
    assert re.sub(r"\s+", " ", body).strip() == "if (alive) bar_arrive<288>(id); else bar_sync<288>(id);"
    assert code.count("bar_arrive<288>") == 1  # nowhere else
    for bar in ("kBarS", "kBarR", "kBarW", "kBarU"):
        assert f"hand_over({bar} + half)" in code and f"bar_sync<288>({bar})" in code
    # a warp of the chain has given up as a whole: behind both places where it waits
    assert code.count("alive = __all_sync(~0u, alive);") == 2


# ---------------------------------------------------------------------------
# what a CTA has stored, once one of its waits ran out
# ---------------------------------------------------------------------------

def test_a_wait_that_ran_out_is_seen_behind_the_last_barrier():
    """Whichever role's it was: all join the barrier behind which the flag is read, and set it before."""
    code = re.sub(r"\s+", " ", _code("delta_tc.cuh"))
    tail = code[code.rindex("__syncthreads();"):]
    before = code[:code.rindex("__syncthreads();")]
    assert "if (*stalled != 0) delta_lost<D, OUT>(" in tail
    assert before.rindex("*stalled = 1;") > before.rindex("hand_over(") > before.index("*stalled = 0;")
    assert "if (!alive) { atomicOr(&g_delta_status, 1); *stalled = 1; }" in before


_HOST = r"""
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>
#include <cmath>
#define __device__
#define __forceinline__ inline
struct { unsigned x; } threadIdx;
static int g_cta;
struct bf16 { uint16_t x; };
typedef bf16 __nv_bfloat16;
static float __int_as_float(int i) { float f; memcpy(&f, &i, 4); return f; }
static bool __any_sync(unsigned, bool x) { return x; }
static void store_f32(bf16* p, int64_t i, float f) { uint32_t u; memcpy(&u, &f, 4); p[i].x = u >> 16; }
struct DeltaParams { int H; float *ht, *seg_moves, *seg_states; const int32_t* slots_out; int num_out; void* out; int64_t so; };
static int64_t pool_slot(const int32_t* s, int num, int n) {
  if (s == nullptr) return n;
  return s[n] < 0 || s[n] >= num ? -1 : s[n];
}
static bool slot_taken(const int32_t* s, int n, int64_t slot, int, int) {
  bool t = false;
  if (s != nullptr && slot >= 0) for (int m = 0; m < n; ++m) t |= s[m] == slot;
  return t;
}
template <int D> struct DeltaTcCfg { static constexpr int kVB = D < 128 ? D : 128, kBlocks = D / kVB, kThreads = 768; };
FUNCTION

template <typename T> static bool nan_at(const T& x);
template <> bool nan_at(const float& x) { return std::isnan(x); }
template <> bool nan_at(const bf16& x) { return (x.x & 0x7f80) == 0x7f80 && (x.x & 0x7f); }

template <int D, bool OUT> static int check() {
  const int H = 3, N = 3, L = 23, VB = DeltaTcCfg<D>::kVB, B = D / VB;
  const int32_t slots[N] = {1, 1, -1};
  const int64_t so = H * D + 8, bos[N] = {2, 9, 9}, eos[N] = {9, 9, 20};
  int bad = 0;
  for (int pool = 0; pool < 2; ++pool)
    for (int last = 0; last < 2; ++last)
      for (g_cta = 0; g_cta < N * H * B * (OUT ? 1 : 2); ++g_cta) {
        std::vector<float> ht(N * H * D * D), mv(ht), st(ht);
        std::vector<bf16> out(L * so);
        DeltaParams p{H, ht.data(), mv.data(), st.data(), pool ? slots : nullptr, N, out.data(), so};
        const int vblk = g_cta % B, rest = g_cta / B / (OUT ? 1 : 2), unit = rest / H, h = rest % H;
        const bool moves = !OUT && g_cta / B % 2;
        for (threadIdx.x = 0; threadIdx.x < 768; ++threadIdx.x)
          delta_lost<D, OUT>(p, unit, bos[unit], eos[unit], last);
        const int slot = !pool ? unit : unit == 0 ? 1 : -1;  // (slot 1 is the first sample's)
        for (int n = 0; n < N; ++n)
          for (int g = 0; g < H; ++g)
            for (int k = 0; k < D; ++k)
              for (int v = 0; v < D; ++v) {
                const size_t at = ((size_t)n * H + g) * D * D;
                const bool cols = v / VB == vblk && g == h, own = cols && n == unit;
                bad += nan_at(ht[at + k * D + v]) != (OUT && last && cols && n == slot);
                bad += nan_at(st[at + k * D + v]) != (!OUT && !moves && own);
                bad += nan_at(mv[at + v * D + k]) != (!OUT && moves && own);  // [value column][key]
              }
        for (int t = 0; t < L; ++t)
          for (int c = 0; c < so; ++c)
            bad += nan_at(out[t * so + c]) != (OUT && t >= bos[unit] && t < eos[unit] && c / D == h && c < H * D &&
                                               c % D / VB == vblk);
      }
  return bad;
}

int main() {
  const int bad[6] = {check<64, true>(), check<64, false>(), check<128, true>(), check<128, false>(),
                      check<256, true>(), check<256, false>()};
  int all = 0;
  for (int b : bad) all += b;
  printf("%d\n", all);
  return all != 0;
}
"""


def test_what_a_cta_has_stored_becomes_nan(tmp_path):
    """The kernel's own function, compiled for the host: every element of the CTA's part and no other."""
    code = (CSRC / "delta_tc.cuh").read_text()
    begin = code.index("template <int D, bool OUT>\n__device__ __forceinline__ void delta_lost(")
    function = code[begin:code.index("\n}\n", begin) + 3]
    function, n = re.subn(r"asm volatile\([^;]*;\"[^;]*;", "cta = g_cta;", function)
    assert n == 1
    src = tmp_path / "lost.cpp"
    src.write_text(_HOST.replace("FUNCTION", function))
    exe = tmp_path / "lost"
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_a_chunk_whose_tiles_were_late_is_nan_for_the_chain():
    """The operands' kernel: all of its threads learn of it behind a barrier, T becomes NaN in both terms, and the tiles are
    waited for once more before the block ends."""
    code = re.sub(r"\s+", " ", _code("delta_chunks.cuh"))
    kernel = code[code.index("delta_chunks_kernel("):]
    wait = kernel.index("if (!mbar_wait_clock(smem_u32(bar), 0)) *late = 1;")
    branch = kernel.index("if (*late != 0) {")
    assert kernel.index("*late = 0;") < kernel.index("__syncthreads();") < wait
    between = kernel[wait:branch]
    assert "return;" not in between and "__syncthreads();" in between
    assert kernel.index("split2(f32x2_pack(lo4.x") > branch  # T is stored behind it
    body = kernel[branch:kernel.index("return; }", branch)]
    assert "0x7fff7fff" in body and "i < 2 * DeltaChunks::kTerm / 16; i += Cfg::kThreads" in body
    assert "atomicOr(&g_delta_status, 1); mbar_wait_clock(smem_u32(bar), 0);" in body


def test_a_nan_in_t_reaches_every_column_and_both_passes():
    """In 64 bits, the zeros of T included: one chunk's T as NaN leaves no finite value in the state, whatever its tokens,
    their gates and the states before are."""
    import torch

    gen = torch.Generator().manual_seed(1)
    for beta, decay, before in ((0.5, 0.9, 1.0), (0.0, 0.0, 0.0), (1.0, 1.0, 0.0)):
        k, v = torch.randn(64, 16, generator=gen).double(), torch.randn(64, 16, generator=gen).double()
        S = before * torch.randn(16, 16, generator=gen).double()
        T = torch.tril(torch.full((64, 64), float("nan"), dtype=torch.float64))  # stored up to the diagonal's blocks
        r = beta * (v - decay * (k @ S))
        u = T @ r
        assert not bool(torch.isfinite(decay * S + k.T @ (0.5 * u)).any())


@pytest.mark.parametrize("pieces", [1, 4, 5, 64, 992])
@pytest.mark.parametrize("lost", [0, 3, 63])
def test_the_join_waits_a_few_times_at_most(pieces, lost):
    """Between the passes over segments: a piece that never lands ends the waiting for later ones and their loads; what
    has been loaded is waited for once more. Waits of half a second each, in the order of the kernel's code."""
    code = re.sub(r"\s+", " ", _code("delta_join.cuh"))
    assert "if (alive) alive = mbar_wait_clock(bars + 8 * stage, (i / Cfg::kStages) & 1);" in code
    assert "if (tid == 0 && alive && i + Cfg::kStages < pieces) {" in code
    assert code.count("mbar_wait_clock(") == 2 and "j = issued > Cfg::kStages ? issued - Cfg::kStages : 0; j < issued" in code
    stages = int(re.search(r"kStages = (\d+)", code).group(1))
    alive, issued, ran_out = True, min(stages, pieces), 0
    landed = lambda i: i < lost  # noqa: E731  (in order, one after another, up to the lost one)
    for i in range(pieces):
        if alive and not landed(i):
            alive, ran_out = False, ran_out + 1
        if alive and i + stages < pieces:
            issued = i + stages + 1
    if not alive:
        waited = list(range(max(issued - stages, 0), issued))
        assert set(waited) >= {i for i in range(issued) if not landed(i)}  # nothing in flight is left out
        ran_out += sum(not landed(j) for j in waited)
    assert alive == (lost >= pieces) and ran_out <= 1 + stages
