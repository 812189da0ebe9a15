// The chain of chunks of the gated delta rule on tcgen05 tensor cores: one CTA per (sample, head, block of up to 128
// values), the chunks of 64 tokens of a sample in order. With T and B as delta_chunks.cuh makes them, G_i the sum of
// the log decays of a chunk's tokens up to and including i, w_i = e^{G_63 - G_i} and S the state before the chunk:
//     r_i  = beta_i (v_i - e^{G_i} S^T k_i),    u = T r       (the corrections of the chunk's tokens)
//     o_i  = scale e^{G_i} S^T q_i + sum_{j <= i} B_ij u_j
//     S'   = e^{G_63} S + sum_j w_j k_j u_j^T
// Everything is computed transposed, the value index as the tensor-memory lane, so that the A operands of all products
// are written into tensor memory by the threads that own a value:
//     X^T = S^T K^T, S^T Q^T   M = 128 values, N = 64 tokens each, K = D
//     U^T = R^T T^T            M = 128 values, K = 64 tokens; T is lower triangular: N = 64, 48, 32, 16
//     P^T = (w U)^T K          M = 128 values, N = D keys, K = 64 tokens
//     O^T = U^T B^T            as U
//
// Precision. The state is fp32 in registers. K and V are bf16 as given; every fp32 factor of a product that the state
// depends on (S in S^T K^T, T, R, w U) is split into two bf16 terms, which leaves 2^-16 of each value at most and a few
// 1e-6 of the state in all (one term would leave 1e-3; a third of R and w U 0.3 to 1.7e-6, for 8 to 10 % of the time). S, U and
// B are two terms for the outputs, too, which are then rounded once: 1.7e-3 from the definition, as the definition's own
// are (with one term of S and U 2.4e-3, of B also 2.9e-3). Sums of log decays are formed in 64 bits; the decay of a
// whole chunk is a pair of fp32 numbers where it is the same for every chunk.
//
// Roles (24 warps): warp 0 issues MMAs, warp 1 loads tiles, warps 2 and 3 make the decay tables of alternate chunks;
// warps 4-7 make the outputs; warps 8-23 hold the state, a quarter of the keys each warpgroup, and walk the chain
// X -> R -> U -> w U -> P -> S. What bounds a chunk is that chain: each of its three batches of MMAs has some 350
// cycles from the first arrival to the threads that read the result, beside its own time and that of the threads
// (8 x 8192 tokens, 16 heads, D = 128: 418 us in a run of its own, 3.3 us a chunk with 128 SMs at work; tensor pipe 34 %).
// So it goes in two halves, of the keys
// for S and P and of the tokens for R and U (warps 8-15 and 16-23), one half's threads working while the other
// half's products are made: X's sum over the first keys needs the first half of S only, U's first tokens only the first
// half of R (T is lower triangular), P's sum over the first tokens only the first half of w U. V is fetched while P is
// computed, and U's terms for O^T are written then, over X; S^T Q^T is issued behind X and O^T behind P. The MMA warp
// waits for the others at named barriers, which take no issue slots. (Outputs made by the chain's warps beside X cost it a quarter more.)
// At D = 256 a state thread has 64 keys in 96 registers and spills (1,310 bytes of stores, 1,416 of loads in the kernel, more
// than half of them where columns are made again; D = 128: 100 and 248): 6.3 us a chunk, warps wait for tensor memory and for
// what is spilled (4 x 2048 tokens, 16 heads: 202 us; tensor pipe 34 %).
// At D = 64 the 64 values fill half of the 128 lanes; lanes 64-127 repeat them and store half of the output rows.
//
// Values that are not finite: the zeros of T and B meet them in tokens they must not reach. Whatever spoils a token
// never leaves the state, so a CTA looks at its final state; a warp's columns of which one is not finite are made
// again token by token (DeltaAgain) from the initial state, outputs too (2 us a token). A query never enters the state: of
// columns whose state is finite and some output is not, those outputs alone are made again (an infinite query's scores
// differ in sign, and their second terms are differences of infinities), unless a NaN in the query settles them.
// Every wait for an mbarrier is bounded as in linear_tc.cuh: a thread whose wait runs out flags it and stops waiting, the
// control warps drain what they have in flight, and all that the CTA has stored becomes NaN (delta_lost). Named barriers
// have no bound of their own: the MMA warp comes to all of them, whatever it has given up, and so does each warp of the
// chain, once a phase: its waits keep it from arriving twice, and where one of them has run out it joins the barrier
// instead of passing it (hand_over).
#pragma once

#include "delta_chunks.cuh"
#include "tc.cuh"
#include "tma.h"

namespace memt {

// one chunk's decays and gates; tokens behind the sample: all but f are 0
struct DeltaTable {
  float f[kTile];              // scale e^{G_i}
  float b[kTile];              // beta_i
  float bf[kTile];             // beta_i e^{G_i}
  float w[kTile];              // e^{G_63 - G_i}
  float a_hi, a_lo;            // decay of the whole chunk
  float pad[2];
};

template <int D_>
struct DeltaTcCfg {
  static constexpr int D = D_;
  static constexpr int kVB = D < 128 ? D : 128;  // values per CTA
  static constexpr int kBlocks = D / kVB;        // CTAs per (sample, head)
  static constexpr int kThreads = 768;
  static constexpr int kKeys = D / 4;            // keys per state thread
  static constexpr int kStages = D == 256 ? 2 : 3;
  static constexpr int kTables = 4;
  static constexpr uint32_t kPanel = kTile * 128;             // 64 x 64 bf16: 8 KB
  static constexpr uint32_t kPair = 2 * kPanel;               // a panel of K and the same of Q behind it
  static constexpr uint32_t kBytesKQ = D / 64 * kPair;
  static constexpr uint32_t kBytesV = kTile * kVB * 2;
  static constexpr uint32_t kBytesTB = DeltaChunks::kBytes;
  static constexpr uint32_t kOffKQ = 0;
  static constexpr uint32_t kOffV = kOffKQ + kStages * kBytesKQ;
  static constexpr uint32_t kOffTB = kOffV + kStages * kBytesV;
  static constexpr uint32_t kOffOut = kOffTB + kStages * kBytesTB;  // two pieces of 2 KB per output warp
  static constexpr uint32_t kOffTab = kOffOut + 4 * 2 * 2048;
  static constexpr uint32_t kOffBar = kOffTab + kTables * sizeof(DeltaTable);
  static constexpr size_t kSmem = kOffBar + 512 + 1024;
  // Tensor memory columns. S: for each quarter of the keys its two terms, over which P^T is written once X has read
  // them. X: S^T K^T, then for each 16 tokens the two terms of U^T. R: for each 16 tokens the two terms of R^T. U: U^T, then
  // for each 16 tokens the two terms of (w U)^T. XQ: S^T Q^T of even and odd chunks. O has columns of its own. At D = 256 there is
  // one XQ, and O lies on U, once P has read it.
  static constexpr bool kAlias = D == 256;
  static constexpr uint32_t kColS = 0, kColX = D, kColR = kColX + 64, kColU = kColR + 64, kColXQ = kColU + 64,
                            kColO = kAlias ? kColU : kColXQ + 128, kColEnd = kAlias ? kColXQ + 64 : kColO + 64;
  // Whether the chain fetches the next chunk's V before it hands over U for the outputs. V first / U first, us: D = 256,
  // 4 x 4096 tokens 512 / 535; 8 x 8192 tokens at D = 128 702 / 646, at D = 64 593 / 543.
  static constexpr bool kFetchFirst = D == 256;
  // registers per thread after the split of the launch's 6 x 80 over the warpgroups (40, 56, 96 at D = 128: the chain a sixth
  // slower; more for the outputs, fewer for the state: the same)
  static constexpr int kRegsControl = D == 256 ? 40 : 56, kRegsOut = D == 256 ? 56 : 72,
                       kRegsState = D == 256 ? 96 : 88;
  static_assert(kRegsControl + kRegsOut + 4 * kRegsState <= 6 * 80, "no more than the launch's registers");
  static_assert(kColEnd <= 512 && kSmem <= 227 * 1024, "one CTA's resources");
};

// Named barriers of the roles (0 is __syncthreads): arrivals of one role, a wait of another, without polls. Those in
// pairs are of the chain's first and second half.
enum DeltaBarrier {
  kBarEnd = 1,  // the chain's and the outputs' warps, once
  kBarAgain = 8,  // the chain's, around columns that are made again
  kBarS = 2,    // the state's terms written: chain -> MMA
  kBarR = 4,    // R^T written: chain -> MMA
  kBarW = 6,    // (w U)^T written: chain -> MMA
  kBarU = 9     // U^T written: chain -> MMA
};
template <int THREADS>
__device__ __forceinline__ void bar_arrive(int id) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ void bar_sync(int id) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}

// 2^(h + l) for |l| far below 1
__device__ __forceinline__ float exp2_pair(float h, float l) {
  const float x = fast_exp2(h);
  return fmaf(x, l * 0.69314718f, x);
}

// NaN in `seen` (zeros before) once a pair of bf16 numbers is not finite
__device__ __forceinline__ uint32_t not_finite(uint32_t pair, uint32_t seen) {
  uint32_t x;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(x) : "r"(pair), "r"(0u), "r"(seen));
  return x;
}

// The warp's columns from `col` of one state, again, token by token from `start` (null: zeros) and with the outputs, or
// with `odd` those of them that are not finite. Once every value of the state is NaN, so is everything behind.
// (At D = 64 and 128 with what the next token needs in registers, too, the chain itself comes out slower.)
template <int D>
using DeltaAgain = DeltaColumns<D, D == 64 ? 4 : 2>;
template <int D>
__device__ __forceinline__ void delta_columns_again(const DeltaParams& p, int h, int col, int64_t bos, int64_t eos,
                                                    const float* start, float* end, bool odd) {
  using Cols = DeltaAgain<D>;
  using T = __nv_bfloat16;
  constexpr bool kAhead = D == 256;
  constexpr int M = kAhead ? Cols::kRows / 4 : 1;
  Cols cols;
  cols.load(start != nullptr ? start + col : nullptr);
  const int hk = h / (p.H / p.Hk);
  float fixed_hi, fixed_lo;
  split_decay(p.g_layout == 3 ? exp(static_cast<double>(p.g[h])) : 1.0, fixed_hi, fixed_lo);
  auto kt = [&](int64_t t) { return static_cast<const T*>(p.k) + t * p.sk + (int64_t)hk * D + Cols::row0(); };
  auto qt = [&](int64_t t) { return static_cast<const T*>(p.q) + t * p.sq + (int64_t)hk * D + Cols::row0(); };
  auto vt = [&](int64_t t) { return static_cast<const T*>(p.v) + t * p.sv + (int64_t)h * D + col; };
  auto raw = [](const T* x, int m) { return *reinterpret_cast<const uint2*>(x + 4 * Cols::kRowGroups * m); };
  auto four = [](uint2 u) {
    const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
  };
  uint2 k2[M], q2[M];  // the next token's, as loaded
  float v2 = 0.f, g2 = 0.f, b2 = 0.f;
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int m = 0; m < M; ++m) {
      k2[m] = raw(kt(t), m);
      q2[m] = raw(qt(t), m);
    }
    v2 = as_f32(vt(t)[Cols::col0() + Cols::own_col()]);
    b2 = load_beta<T>(p, t, h);
    if (p.g_layout == 1) g2 = p.g[t * p.H + h];
  };
  if (kAhead && bos < eos) fetch(bos);
  bool lost = false;
#pragma unroll 1
  for (int64_t t = bos; t < eos; ++t) {
    float out = __int_as_float(0x7fffffff);
    if (!lost) {
      uint2 k1[M], q1[M];
      float v1 = v2, beta = b2, g1 = g2;
      if constexpr (kAhead) {
#pragma unroll
        for (int m = 0; m < M; ++m) {
          k1[m] = k2[m];
          q1[m] = q2[m];
        }
        if (t + 1 < eos) fetch(t + 1);
      } else {
        beta = load_beta<T>(p, t, h);
        if (p.g_layout == 1) g1 = p.g[t * p.H + h];
      }
      const float a = p.g_layout == 1 ? expf(g1) : fixed_hi;
      auto k = [&](int m) { return four(kAhead ? k1[kAhead ? m : 0] : raw(kt(t), m)); };
      auto q = [&](int m) { return four(kAhead ? q1[kAhead ? m : 0] : raw(qt(t), m)); };
      auto v = [&](int c) { return kAhead ? v1 : as_f32(vt(t)[c]); };  // (c is this lane's own column)
      // (a low half of zero would make NaN of an infinite state)
      out = cols.template step<true>(k, q, v, a, p.g_layout == 1 ? low_half(a, 0.f) : fixed_lo, beta);
      bool nan = true;
#pragma unroll
      for (int i = 0; i < Cols::kRows / 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) nan = nan && isnan(f32x2_lo(cols.S[i][c])) && isnan(f32x2_hi(cols.S[i][c]));
      lost = __all_sync(~0u, nan);
    }
    if (Cols::writes()) {
      T* at = static_cast<T*>(p.out) + t * p.so + (int64_t)h * D + col + Cols::col0() + Cols::own_col();
      if (!odd || !isfinite(as_f32(*at))) store_f32(at, 0, p.scale * out);
    }
  }
  if (end != nullptr) cols.store(end + col);
}

// The end of the last token of the chunks odd[0] .. odd[1] whose output, in the CTA's columns from `col`, is not finite
// although no NaN in its query makes it so, to odd[2]. By the chain's 16 warps.
template <int D>
__device__ __forceinline__ void odd_tokens(const DeltaParams& p, int h, int col, int64_t bos, int64_t eos, int32_t* odd,
                                           int warp) {
  constexpr int VB = DeltaTcCfg<D>::kVB, W = VB / 64, AT = 4;  // words of a lane, tokens at once
  const int lane = threadIdx.x & 31;
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q) + (int64_t)(h / (p.H / p.Hk)) * D;
  const __nv_bfloat16* o = static_cast<const __nv_bfloat16*>(p.out) + (int64_t)h * D + col;
  int64_t end = bos + (int64_t)(odd[1] + 1) * kTile;
  if (end > eos) end = eos;
  for (int64_t t0 = bos + (int64_t)odd[0] * kTile + AT * warp; t0 < end; t0 += 16 * AT) {
    uint32_t x[AT][W] = {};
#pragma unroll
    for (int j = 0; j < AT; ++j)
      if (t0 + j < end) {
#pragma unroll
        for (int i = 0; i < W; ++i) x[j][i] = reinterpret_cast<const uint32_t*>(o + (t0 + j) * p.so)[lane + 32 * i];
      }
#pragma unroll
    for (int j = 0; j < AT; ++j) {
      uint32_t seen = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) seen = not_finite(x[j][i], seen);
      if (!__any_sync(~0u, seen != 0)) continue;
      bool nan = false;
      for (int i = lane; i < D; i += 32) nan = nan || isnan(as_f32(q[(t0 + j) * p.sq + i]));
      if (!__any_sync(~0u, nan) && lane == 0) atomicMax(odd + 2, static_cast<int>(t0) + j + 1);
    }
  }
}

// All that a CTA has stored becomes NaN: a wait of it ran out, in whichever role, and nothing of it can be relied on.
template <int D, bool OUT>
__device__ __forceinline__ void delta_lost(const DeltaParams& p, int n, int64_t bos, int64_t eos, bool last) {
  constexpr int VB = DeltaTcCfg<D>::kVB, NT = DeltaTcCfg<D>::kThreads;
  int cta;  // as in the kernel, which must not hold registers for this
  asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(cta));
  const int vblk = cta % (D / VB), rest = cta / (D / VB), h = rest / (OUT ? 1 : 2) % p.H;
  const bool moves = !OUT && rest % 2;
  const int64_t seg_state = (int64_t)(rest / (OUT ? 1 : 2)) * D * D;
  const float nan = __int_as_float(0x7fffffff);
  const int64_t out_slot = pool_slot(p.slots_out, p.num_out, n);
  const bool taken = __any_sync(~0u, slot_taken(p.slots_out, n, out_slot, threadIdx.x & 31, 32));
  float* end = OUT ? (last && out_slot >= 0 && !taken ? p.ht + (out_slot * p.H + h) * D * D : nullptr)
                   : (moves ? p.seg_moves : p.seg_states) + seg_state;
  if (end != nullptr)
    for (int i = threadIdx.x; i < D * VB; i += NT)
      end[!OUT && moves ? vblk * VB * D + i : i / VB * D + vblk * VB + i % VB] = nan;
  if constexpr (OUT) {
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + (int64_t)h * D + vblk * VB;
    for (int64_t i = threadIdx.x; i < (eos - bos) * VB; i += NT) store_f32(o, (bos + i / VB) * p.so + i % VB, nan);
  }
}

// OUT: outputs and final states. Otherwise the first pass over segments: what a segment adds to a zero state
// (seg_states) and makes of an identity without values (seg_moves, transposed), in a CTA each.
template <int D, bool OUT>
__global__ void __launch_bounds__(DeltaTcCfg<D>::kThreads, 1) delta_tc_kernel(const __grid_constant__ DeltaTcParams P) {
  using Cfg = DeltaTcCfg<D>;
  constexpr int NS = Cfg::kStages, NT = Cfg::kTables, KT = Cfg::kKeys;
  const DeltaParams& p = P.p;
  extern __shared__ __align__(1024) unsigned char smem_delta_tc[];
  // (by an offset: a pointer made from an integer would be a generic one, and every access through it)
  unsigned char* sm = smem_delta_tc + ((1024u - (smem_u32(smem_delta_tc) & 1023u)) & 1023u);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(~0u, tid >> 5, 0), quad = warp & 3;  // uniform: so are the roles' branches
  const int vblk = blockIdx.x % Cfg::kBlocks;
  const int rest = blockIdx.x / Cfg::kBlocks / (OUT ? 1 : 2), unit = rest / p.H, h = rest % p.H, hk = h / (p.H / p.Hk);
  const bool moves = !OUT && blockIdx.x / Cfg::kBlocks % 2;
  // a unit is a sample, or with segments one of a sample's `segs`
  int n = unit, seg = 0, segs = 1;
  if (p.seg_chunks > 0) {
    if (!find_segment(p, unit, n, seg, segs)) return;
    if (!OUT && seg + 1 == segs) return;  // the first pass is for what later segments start from
  } else if (p.only_long) {
    n = p.longs != nullptr ? p.longs[unit] : find_long(p, unit);
    if (n < 0) return;
  } else if (p.by_length) {
    n = sample_by_length(p, unit);
  }
  int64_t bos, eos;
  sample_range(p, n, bos, eos);
  if (eos - bos <= p.few) return;  // the token-by-token kernel's
  int first, units;
  sample_units(p, n, first, units);
  // Offsets that overlap can leave a sample without units for all of its chunks: it goes token by token, whole.
  const bool tokenwise = units < (eos - bos + kTile - 1) / kTile;
  if (tokenwise) {
    if (!OUT || seg > 0) return;
    segs = 1;
  }
  if (segs > 1) {
    first += seg * p.seg_chunks;
    bos += (int64_t)seg * p.seg_chunks * kTile;
    if (seg + 1 < segs) eos = bos + (int64_t)p.seg_chunks * kTile;
  }
  const int nchunks = tokenwise ? 0 : static_cast<int>((eos - bos + kTile - 1) / kTile);

  // mbarriers: a chunk's tiles landed (LF) and free again (LE); table written / read (TF, TE); both halves of X (XD), U
  // (UD) and P (PD) and O (OD) ready; outputs read (OE); drained (DR)
  constexpr int LF = 0, LE = LF + NS, TF = LE + NS, TE = TF + NT, XD = TE + NT, UD = XD + 2, PD = UD + 2, OD = PD + 2,
                OE = OD + 1, DR = OE + 1, NBAR = DR + 1;
  static_assert(NBAR * 8 + 48 <= 512, "barrier area");
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + Cfg::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + Cfg::kOffBar + NBAR * 8);
  // bit c: some value of the CTA's c-th group of columns (DeltaAgain) is not finite; kGivenUp: so have some of the chain's
  // or the outputs' warps
  uint32_t* spoiled = tmem_slot + 1;
  constexpr uint32_t kGivenUp = 1u << 31;
  uint32_t* stalled = tmem_slot + 2;  // a wait ran out
  int32_t* whose = reinterpret_cast<int32_t*>(tmem_slot + 3);  // sample, first and last token, whether the sample ends here
  // groups with outputs that are not finite, the first and the last chunk of them, and the end of the last token that is
  // made again for them
  uint32_t* odd_groups = tmem_slot + 7;
  int32_t* odd = reinterpret_cast<int32_t*>(tmem_slot + 8);
  const uint32_t base = smem_u32(sm), bars = smem_u32(bar);
  auto B = [&](int i) { return bars + 8 * i; };
  if (tid == 0) {
    for (int i = 0; i < NBAR; ++i) {
      uint32_t count = 1;  // TMA, tcgen05.commit or one thread
      if (i >= TE && i < XD) count = OUT ? 20 : 16;  // the chain's and the outputs' warps
      if (i == OE) count = 4;
      mbar_init(B(i), count);
    }
    mbar_fence_init();
    *spoiled = 0;
    *stalled = 0;
    whose[0] = n;
    whose[1] = static_cast<int>(bos);
    whose[2] = static_cast<int>(eos);
    whose[3] = seg + 1 == segs;
    *odd_groups = 0;
    odd[0] = INT32_MAX;
    odd[1] = odd[2] = -1;
  }
  if (warp == 0) tc::alloc(smem_u32(tmem_slot), 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem + Cfg::kColS, tX = tmem + Cfg::kColX, tR = tmem + Cfg::kColR,
                 tU = tmem + Cfg::kColU, tO = tmem + Cfg::kColO;
  auto tXQ = [&](int c) { return tmem + Cfg::kColXQ + (Cfg::kAlias ? 0 : 64 * (c & 1)); };
  DeltaTable* tab = reinterpret_cast<DeltaTable*>(sm + Cfg::kOffTab);
  auto chunk_len = [&](int c) {
    const int64_t left = eos - bos - (int64_t)c * kTile;
    return static_cast<int>(left < kTile ? left : kTile);
  };

  bool alive = true;
  auto wait = [&](int b, uint32_t phase) {
    if (alive) alive = mbar_wait_polls(B(b), phase & 1);
  };
  auto wait_long = [&](int b, uint32_t phase) {  // by a warp that is ahead of the others and need not hurry
    for (int i = 0; i < 64 && alive && !mbar_try(B(b), phase & 1); ++i) __nanosleep(100);
    wait(b, phase);
  };
  auto arrive = [&](int b) {  // one arrival per warp
    __syncwarp();
    if (lane == 0) mbar_arrive(B(b));
  };
  auto hand_over = [&](int id) {  // chain -> MMA, by a warp of which all or none have given up
    if (alive) bar_arrive<288>(id);
    else bar_sync<288>(id);
  };

  if (warp < 4) {
    regs_dec<Cfg::kRegsControl>();
    if (warp == 0) {
      // ---------------- MMA issue ----------------
      auto go = [&]() {  // nothing more is issued after a wait ran out
        tc::fence_after();
        return __all_sync(~0u, alive) && tc::elect_one();
      };
      // A operand of S's term for K step i: quarters of the keys, each with its two terms
      auto state = [&](int term, int i) {
        constexpr int per = KT / 16;  // K steps of a quarter
        return tS + KT * (i / per) + 8 * (i % per) + term * (KT / 2);
      };
      // B operand: rows t0 on of a lower triangular operand's block of columns j, as a descriptor's offset
      auto rows = [](int j, int t0) { return (DeltaChunks::block(j) + (t0 - 16 * j) * 32) >> 4; };
      // K step i of the tile's rows
      auto kq = [](int i) { return (i >> 2) * static_cast<int>(Cfg::kPair >> 4) + (i & 3) * 2; };
      for (int c = 0; c < nchunks; ++c) {
        const int s = c % NS, len = chunk_len(c);
        constexpr int kHalf = D / 32;  // K steps of half the keys
        // descriptors of the stage's tiles: an MMA's own is a sum away (made whole, it costs more than the MMA)
        const uint64_t dk = tc::desc_kmajor(base + Cfg::kOffKQ + s * Cfg::kBytesKQ, 0);
        const uint64_t dm = tc::desc_mnmajor(base + Cfg::kOffKQ + s * Cfg::kBytesKQ, Cfg::kPair, 0);
        const uint64_t dt = tc::desc_plain(base + Cfg::kOffTB + s * Cfg::kBytesTB, 128, 256);
        constexpr int kTerm = DeltaChunks::kTerm >> 4;
        wait(LF + s, c / NS);
        if (len < kTile) {  // rows of K behind the sample: zero
          const int pieces = (kTile - len) * 8;
          for (int i = lane; i < D / 64 * pieces; i += 32)
            *reinterpret_cast<uint4*>(sm + Cfg::kOffKQ + s * Cfg::kBytesKQ + i / pieces * Cfg::kPair + len * 128 +
                                      i % pieces * 16) = make_uint4(0, 0, 0, 0);
          tc::fence_smem_async();
          __syncwarp();
        }
        bar_sync<288>(kBarS);
        if (go()) {  // the first half of the keys for all tokens
#pragma unroll
          for (int i = 0; i < 2 * kHalf; ++i)
            tc::mma_bf16_ts(tX, state(i < kHalf, i % kHalf), dk + kq(i % kHalf),
                            tc::idesc(tc::kBF16, 128, 64, false, false), i > 0);
        }
        __syncwarp();
        bar_sync<288>(kBarS + 1);
        if (go()) {  // the second half for one half of the tokens after the other
#pragma unroll
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int i = 0; i < 2 * kHalf; ++i)
              tc::mma_bf16_ts(tX + 32 * half, state(i < kHalf, kHalf + i % kHalf),
                              dk + (kq(kHalf + i % kHalf) + 256 * half), tc::idesc(tc::kBF16, 128, 32, false, false), true);
            tc::commit(B(XD + half));
          }
        }
        __syncwarp();
        if (OUT && Cfg::kAlias && c > 0) wait(OE, c - 1);
        if (OUT && go()) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            tc::mma_bf16_ts(tXQ(c), state(i < D / 16, i % (D / 16)), dk + (kq(i % (D / 16)) + (Cfg::kPanel >> 4)),
                            tc::idesc(tc::kBF16, 128, 64, false, false), i > 0);
        }
        __syncwarp();
        bar_sync<288>(kBarR);
        if (go()) {  // tokens 0 .. 31 of U
#pragma unroll
          for (int i = 0; i < 3; ++i)  // first and second terms of R and T: 0 1, 1 0, 0 0
#pragma unroll
            for (int j = 0; j < 2; ++j)
              tc::mma_bf16_ts(tU + 16 * j, tR + 16 * j + 8 * (i == 1), dt + ((i == 0 ? kTerm : 0) + rows(j, 16 * j)),
                              tc::idesc(tc::kBF16, 128, 32 - 16 * j, false, false), i > 0 || j > 0);
          tc::commit(B(UD));
        }
        __syncwarp();
        bar_sync<288>(kBarR + 1);
        if (go()) {
#pragma unroll
          for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int t0 = j == 3 ? 48 : 32;
              tc::mma_bf16_ts(tU + t0, tR + 16 * j + 8 * (i == 1), dt + ((i == 0 ? kTerm : 0) + rows(j, t0)),
                              tc::idesc(tc::kBF16, 128, 64 - t0, false, false), i > 0 || j > 0);
            }
          tc::commit(B(UD + 1));
        }
        __syncwarp();
        bar_sync<288>(kBarW);
        if (go()) {  // tokens 0 .. 31 for all keys
#pragma unroll
          for (int i = 0; i < 4; ++i)
            tc::mma_bf16_ts(tS, tU + 16 * (i & 1) + 8 * (i < 2), dm + 128 * (i & 1),
                            tc::idesc(tc::kBF16, 128, D, false, true), i > 0);
        }
        __syncwarp();
        bar_sync<288>(kBarW + 1);
        if (go()) {  // the others for one half of the keys after the other (D = 64: half a panel is no operand)
          constexpr int kParts = D == 64 ? 1 : 2;
#pragma unroll
          for (int half = 0; half < kParts; ++half) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              tc::mma_bf16_ts(tS + D / 2 * half, tU + 32 + 16 * (i & 1) + 8 * (i < 2),
                              dm + (256 + 128 * (i & 1) + half * (D / 128) * (Cfg::kPair >> 4)),
                              tc::idesc(tc::kBF16, 128, D / kParts, false, true), true);
            tc::commit(B(PD + half));
          }
          if constexpr (kParts == 1) tc::commit(B(PD + 1));
        }
        __syncwarp();
        if constexpr (OUT) {
          bar_sync<288>(kBarU);
          bar_sync<288>(kBarU + 1);
          if (!Cfg::kAlias && c > 0) wait(OE, c - 1);
        }
        if (go()) {
#pragma unroll
          for (int i = 0; OUT && i < 12; ++i) {  // terms of U and B: first second, second first, first first
            const int j = i & 3;
            tc::mma_bf16_ts(tO + 16 * j, tX + 16 * j + 8 * (i >> 2 == 1), dt + ((i < 4 ? 3 : 2) * kTerm + rows(j, 16 * j)),
                            tc::idesc(tc::kBF16, 128, 64 - 16 * j, false, false), i > 0);
          }
          tc::commit(B(OD));
          tc::commit(B(LE + s));
        }
        __syncwarp();
      }
      if (nchunks > 0) {  // the last arrivals land before the barriers go
        wait(OD, nchunks - 1);
        wait(LE + (nchunks - 1) % NS, (nchunks - 1) / NS);
      }
      // a wait that ran out: nothing of this warp may still run when tensor memory is freed
      if (!__all_sync(~0u, alive)) {
        if (tc::elect_one()) tc::commit(B(DR));
        __syncwarp();
        mbar_wait_clock(B(DR), 0);
      }
    } else if (warp == 1) {
      // ---------------- tile loads ----------------
      int issued = 0;
      for (int c = 0; c < nchunks; ++c) {
        const int y = static_cast<int>(bos) + c * kTile, s = c % NS;
        if (c >= NS) wait_long(LE + s, c / NS - 1);
        if (__all_sync(~0u, alive) && tc::elect_one()) {
          mbar_expect_tx(B(LF + s), Cfg::kBytesKQ / (OUT ? 1 : 2) + Cfg::kBytesV + Cfg::kBytesTB);
          for (int i = 0; i < D / 64; ++i) {
            const uint32_t at = base + Cfg::kOffKQ + s * Cfg::kBytesKQ + i * Cfg::kPair;
            tma_load_2d(at, &P.k_map, hk * D + 64 * i, y, B(LF + s));
            if (OUT) tma_load_2d(at + Cfg::kPanel, &P.q_map, hk * D + 64 * i, y, B(LF + s));
          }
          for (int i = 0; i < Cfg::kVB / 64; ++i)
            tma_load_2d(base + Cfg::kOffV + s * Cfg::kBytesV + i * Cfg::kPanel, &P.v_map,
                        h * D + vblk * Cfg::kVB + 64 * i, y, B(LF + s));
          bulk_g2s(base + Cfg::kOffTB + s * Cfg::kBytesTB,
                   static_cast<const unsigned char*>(p.chunks) + ((int64_t)(first + c) * p.H + h) * DeltaChunks::kBytes,
                   Cfg::kBytesTB, B(LF + s));
        }
        __syncwarp();
        issued = c + 1;
      }
      // Every load lands before shared memory is released, also when a wait ran out: tiles that were never
      // issued only use up their (bounded) wait.
      if (!__all_sync(~0u, alive)) {
        for (int c = issued > NS ? issued - NS : 0; c < issued; ++c) mbar_wait_clock(B(LF + c % NS), (c / NS) & 1);
      }
    } else {
      // ---------------- decay tables: lane l has tokens 2 l and 2 l + 1 ----------------
      float xg[2], xb[2];
      auto fetch = [&](int c) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int64_t t = bos + (int64_t)c * kTile + 2 * lane + e;
          xg[e] = t < eos ? log_decay(p, t, h) : 0.f;
          xb[e] = t < eos ? load_beta<__nv_bfloat16>(p, t, h) : 0.f;
        }
      };
      fetch(warp - 2);
      for (int c = warp - 2; c < nchunks; c += 2) {
        const int len = chunk_len(c), t0 = 2 * lane;
        double g[2];
        const float beta[2] = {xb[0], xb[1]};
#pragma unroll
        for (int e = 0; e < 2; ++e)  // below e^-111 = 2^-160 a decay is a reset in fp32 whatever it multiplies; NaN stays NaN
          g[e] = 1.4426950408889634 * (xg[e] < -111.f ? -111.0 : static_cast<double>(xg[e]));
        if (c + 2 < nchunks) fetch(c + 2);
        double sum = g[0] + g[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double x = __shfl_up_sync(~0u, sum, o);
          if (lane >= o) sum += x;
        }
        const double total = __shfl_sync(~0u, sum, 31);
        const int ts = c % NT;
        if (c >= NT) wait_long(TE + ts, c / NT - 1);
        DeltaTable& t = tab[ts];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const double G = e == 0 ? sum - g[1] : sum;
          const float gh = static_cast<float>(G), gl = static_cast<float>(G - static_cast<double>(gh));
          const float a = exp2_pair(gh, gl);
          const double R = total - G;
          const float rh = static_cast<float>(R), rl = static_cast<float>(R - static_cast<double>(rh));
          t.f[t0 + e] = p.scale * a;
          t.b[t0 + e] = beta[e];
          t.bf[t0 + e] = beta[e] * a;
          t.w[t0 + e] = t0 + e < len ? exp2_pair(rh, rl) : 0.f;
        }
        if (lane == 0) chunk_decay(total, t.a_hi, t.a_lo);
        arrive(TF + ts);
      }
    }
  } else if (warp < 8) {
    // ---------------- outputs from X and O ----------------
    // Fragments of 16 values by 32 tokens, a register pair is two tokens of one value. stmatrix turns them into token
    // rows of this warp's 32 values (64 bytes, the 64-byte swizzle), which leave as one TMA box; a chunk that ends
    // inside leaves row by row instead. At D = 64 the lanes that repeat values have the other half of the tokens.
    regs_dec<Cfg::kRegsOut>();
    const int pair = 2 * (lane & 3);                                        // first column of a fragment
    const int prow = 8 * (lane >> 4) + (lane & 7), pval = (lane >> 3) & 1;  // row of an stmatrix piece
    const int col = h * D + vblk * Cfg::kVB + 32 * quad % Cfg::kVB;
    constexpr int kPieces = D >= 128 ? 2 : 1;  // of 32 tokens
    auto is_odd = [&](int value, int c) {  // of the warp's 32
      atomicOr(odd_groups, 1u << ((32 * quad + value) % Cfg::kVB / DeltaAgain<D>::kCols));
      atomicMin(odd, c);
      atomicMax(odd + 1, c);
    };
    for (int c = 0; OUT && c < nchunks; ++c) {
      const DeltaTable& t = tab[c % NT];
      const int len = chunk_len(c);
      wait(TF + c % NT, c / NT);
      wait_long(OD, c);
      __syncwarp();
      tc::fence_after();
#pragma unroll 1
      for (int piece = 0; piece < kPieces; ++piece) {
        const int t0 = 32 * (D >= 128 ? piece : quad >> 1);
        const uint32_t turn = base + Cfg::kOffOut + (2 * quad + piece) * 2048;
        if (lane == 0) {  // the box before the last (at D = 64 the last one) has left its rows
          if constexpr (kPieces == 2) bulk_wait_read_but1();
          else bulk_wait_read();
        }
        __syncwarp();
#pragma unroll 1
        for (int e = 0; e < 2; ++e) {
          uint32_t x[16], y[16];
          tc::ld_frag2<4>(tc::lane_addr(tXQ(c), 32 * quad + 16 * e, t0), tc::lane_addr(tO, 32 * quad + 16 * e, t0), x, y);
          if (piece + 1 == kPieces && e == 1) {
            tc::fence_before();
            arrive(OE);
          }
          uint32_t seen[2] = {0, 0};
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            uint32_t z[4];  // tokens 8 (i + j) + pair, + 1: of value lane / 4, of value lane / 4 + 8
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2 f = *reinterpret_cast<const float2*>(&t.f[t0 + 8 * (i + j) + pair]);
              const uint64_t ff = f32x2_pack(f.x, f.y);
#pragma unroll
              for (int v8 = 0; v8 < 2; ++v8) {
                const int k = 4 * (i + j) + 2 * v8;
                z[2 * j + v8] = f32x2_to_bf16x2(fma_f32x2(ff, (static_cast<uint64_t>(x[k + 1]) << 32) | x[k],
                                                          (static_cast<uint64_t>(y[k + 1]) << 32) | y[k]));
                seen[v8] = not_finite(z[2 * j + v8], seen[v8]);
              }
            }
            const int tok = 8 * i + prow;
            stsm_x4_t(turn + tok * 64 + (((2 * e + pval) ^ ((tok >> 1) & 3)) << 4), z[0], z[1], z[2], z[3]);
          }
          if (len == kTile) {
#pragma unroll
            for (int v8 = 0; v8 < 2; ++v8)
              if (seen[v8] != 0) is_odd(16 * e + 8 * v8, c);
          }
        }
        const int64_t tok0 = bos + (int64_t)c * kTile + t0;
        if (len == kTile) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&P.o_map, col, static_cast<int>(tok0), turn);
            bulk_commit();
          }
        } else {
          __syncwarp();
          __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + tok0 * p.so + col + 8 * (lane & 3);
          for (int tok = lane >> 2; tok < 32 && t0 + tok < len; tok += 8) {
            uint4 z;
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(z.x), "=r"(z.y), "=r"(z.z), "=r"(z.w)
                         : "r"(turn + tok * 64 + (((lane & 3) ^ ((tok >> 1) & 3)) << 4)) : "memory");
            *reinterpret_cast<uint4*>(o + tok * p.so) = z;
            if (not_finite(z.x, not_finite(z.y, not_finite(z.z, not_finite(z.w, 0)))) != 0) is_odd(8 * (lane & 3), c);
          }
        }
      }
      arrive(TE + c % NT);
    }
    if (lane == 0) bulk_wait_all();
    if (!alive) atomicOr(spoiled, kGivenUp);
    __syncwarp();
    bar_sync<640>(kBarEnd);
  } else {
    // ---------------- the state and its chain: value row of this lane, keys KT part .., tokens 16 part .. ----------------
    regs_inc<Cfg::kRegsState>();
    const int part = (warp - 8) >> 2;
    const int vr = (32 * quad + lane) % Cfg::kVB;
    const bool writes = D >= 128 || quad < 2;  // at D = 64 quadrants 2 and 3 repeat 0 and 1
    const int pair = 2 * (lane & 3);
    const int prow = 8 * (lane >> 4) + (lane & 7), pval = (lane >> 3) & 1;  // row of an ldmatrix piece
    const int64_t head = (int64_t)D * D, col_off = (int64_t)(KT * part) * D + vblk * Cfg::kVB + vr;
    const int64_t seg_state = ((int64_t)unit * p.H + h) * head;
    auto first_state = [&](int n) -> const float* {
      if (!OUT || segs > 1) return OUT ? p.seg_states + seg_state : nullptr;
      const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n);
      return p.h0 != nullptr && in_slot >= 0 ? p.h0 + (in_slot * p.H + h) * head : nullptr;
    };
    const float* start = first_state(n);
    uint64_t S[KT / 2];  // pairs of fp32: keys KT part + 2 i, + 2 i + 1 of value vr
    if (start != nullptr) {
      const float* src = start + col_off;
#pragma unroll
      for (int i = 0; i < KT; i += 2) S[i / 2] = f32x2_pack(src[i * D], src[(i + 1) * D]);
    } else {
      const int one = moves ? vblk * Cfg::kVB + vr - KT * part : -1;
#pragma unroll
      for (int i = 0; i < KT; i += 2) S[i / 2] = f32x2_pack(one == i ? 1.f : 0.f, one == i + 1 ? 1.f : 0.f);
    }
    const uint32_t own = tc::lane_addr(tS, 32 * quad, KT * part);  // of S's terms and of P
    const bool fixed = p.g_layout == 3;
    const int half = part >> 1;  // of the chain
    auto ready = [&](int b, uint32_t phase) {
      wait(b + half, phase);
      alive = __all_sync(~0u, alive);
      tc::fence_after();
    };
    // V of a chunk as fragments of 16 values by 16 tokens: a register holds two tokens of one value; and its gates
    uint32_t v[2][4];
    uint64_t minus[2];
    auto fetch = [&](int c) {
      const int s = c % NS;
      wait(LF + s, c / NS);
      wait(TF + c % NT, c / NT);
      alive = __all_sync(~0u, alive);
      const DeltaTable& t = tab[c % NT];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int val = (32 * quad + 16 * e) % Cfg::kVB + 8 * pval, tok = 16 * part + prow;
        ldsm_x4_t(v[e], base + Cfg::kOffV + s * Cfg::kBytesV + (val >> 6) * Cfg::kPanel + tok * 128 +
                            ((((val & 63) >> 3) ^ (tok & 7)) << 4));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 bf = *reinterpret_cast<const float2*>(&t.bf[16 * part + 8 * i + pair]);
        minus[i] = f32x2_pack(-bf.x, -bf.y);
      }
      if (!OUT && moves) {
#pragma unroll
        for (int e = 0; e < 2; ++e) v[e][0] = v[e][1] = v[e][2] = v[e][3] = 0;
      } else if (chunk_len(c) < kTile) {  // tokens behind the sample, whatever stands in their rows
        const int len = chunk_len(c) - 16 * part - pair;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[e][j] = 8 * (j >> 1) >= len ? 0 : 8 * (j >> 1) + 1 >= len ? v[e][j] & 0xffffu : v[e][j];
      }
    };
    if (nchunks > 0) fetch(0);
    for (int c = 0; c < nchunks; ++c) {
#pragma unroll
      for (int q = 0; q < KT / 16; ++q) {
        uint32_t first[8], second[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split2(S[8 * q + i], first[i], second[i]);
        tc::st8(own + 8 * q, first);
        tc::st8(own + KT / 2 + 8 * q, second);
      }
      tc::wait_st();
      tc::fence_before();
      hand_over(kBarS + half);
      const DeltaTable& t = tab[c % NT];
      {  // R = beta v - beta e^G X
        uint64_t y[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 b = *reinterpret_cast<const float2*>(&t.b[16 * part + 8 * (j >> 1) + pair]);
#pragma unroll
          for (int e = 0; e < 2; ++e) y[e][j] = mul_f32x2(f32x2_pack(b.x, b.y), bf16x2_to_f32x2(v[e][j]));
        }
        ready(XD, c);
        uint32_t x[2][8];
        tc::ld_frag2<2>(tc::lane_addr(tX, 32 * quad, 16 * part), tc::lane_addr(tX, 32 * quad + 16, 16 * part), x[0], x[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t first[4], second[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            split2(fma_f32x2(minus[j >> 1], (static_cast<uint64_t>(x[e][2 * j + 1]) << 32) | x[e][2 * j], y[e][j]),
                   first[j], second[j]);
          tc::st_frag8(tc::lane_addr(tR, 32 * quad + 16 * e, 16 * part), first);
          tc::st_frag8(tc::lane_addr(tR, 32 * quad + 16 * e, 16 * part + 8), second);
        }
      }
      tc::wait_st();
      tc::fence_before();
      hand_over(kBarR + half);
      uint64_t ww[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 w = *reinterpret_cast<const float2*>(&t.w[16 * part + 8 * i + pair]);
        ww[i] = f32x2_pack(w.x, w.y);
      }
      const float a_hi = t.a_hi, a_lo = t.a_lo;
      ready(UD, c);
      uint32_t x[2][8];
      tc::ld_frag2<2>(tc::lane_addr(tU, 32 * quad, 16 * part), tc::lane_addr(tU, 32 * quad + 16, 16 * part), x[0], x[1]);
      auto u = [&](int e, int j) { return (static_cast<uint64_t>(x[e][2 * j + 1]) << 32) | x[e][2 * j]; };
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t first[4], second[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split2(mul_f32x2(ww[j >> 1], u(e, j)), first[j], second[j]);
        tc::st_frag8(tc::lane_addr(tU, 32 * quad + 16 * e, 16 * part), first);
        tc::st_frag8(tc::lane_addr(tU, 32 * quad + 16 * e, 16 * part + 8), second);
      }
      tc::wait_st();
      tc::fence_before();
      hand_over(kBarW + half);
      auto hand_over_u = [&]() {  // in X's columns of the warp's own tokens, while P is made
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t first[4], second[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) split2(u(e, j), first[j], second[j]);
          tc::st_frag8(tc::lane_addr(tX, 32 * quad + 16 * e, 16 * part), first);
          tc::st_frag8(tc::lane_addr(tX, 32 * quad + 16 * e, 16 * part + 8), second);
        }
        tc::wait_st();
        tc::fence_before();
        hand_over(kBarU + half);
      };
      if (OUT && !Cfg::kFetchFirst) hand_over_u();
      arrive(TE + c % NT);
      if (c + 1 < nchunks) fetch(c + 1);
      if (OUT && Cfg::kFetchFirst) hand_over_u();
      ready(PD, c);
      // A constant decay's rounding would be the same one every chunk and is left out by a pair of numbers.
      const uint64_t ah = f32x2_splat(fixed ? a_hi : a_hi + a_lo), al = f32x2_splat(a_lo);
      constexpr int CW = KT < 32 ? KT : 32;  // columns at a time
#pragma unroll
      for (int q = 0; q < KT / CW; ++q) {
        float x[CW];
        tc::ldn<CW>(own + CW * q, x);
#pragma unroll
        for (int i = 0; i < CW; i += 2) {
          uint64_t& S2 = S[(CW * q + i) / 2];
          uint64_t y = f32x2_pack(x[i], x[i + 1]);
          if (fixed) y = fma_f32x2(al, S2, y);
          S2 = fma_f32x2(ah, S2, y);
        }
      }
    }
    const int sample = whose[0];  // (read back: registers held over the chain are few)
    const int64_t out_slot = pool_slot(p.slots_out, p.num_out, sample);
    const bool taken = OUT && __any_sync(~0u, slot_taken(p.slots_out, sample, out_slot, lane, 32));
    // No state is stored before every thread has loaded its share of the first one and, where one is not finite,
    // before columns have been made from them again, their outputs over those stored above.
    constexpr int kGroup = DeltaAgain<D>::kCols;
    uint64_t seen = 0;  // two zeros; NaN once a state is not finite
#pragma unroll
    for (int i = 0; i < KT / 2; ++i) seen = fma_f32x2(S[i], 0, seen);
    if (f32x2_lo(seen) != 0.f || f32x2_hi(seen) != 0.f) atomicOr(spoiled, 1u << (vr / kGroup));
    if (!alive) atomicOr(spoiled, kGivenUp);
    bar_sync<640>(kBarEnd);  // with the outputs' warps, once theirs have left
    float* end = out_slot >= 0 && !taken ? p.ht + (out_slot * p.H + h) * head : nullptr;
    if (OUT && seg + 1 < segs) end = nullptr;
    if (!OUT) end = (moves ? p.seg_moves : p.seg_states) + seg_state;
    // (what a segment that is not finite hands on is not made again: a column of it is spoiled as it is)
    const uint32_t again = !OUT ? 0 : tokenwise ? ~kGivenUp : *spoiled & ~kGivenUp;
    if constexpr (OUT) {
      const uint32_t rows = *odd_groups & ~again;
      if ((again | rows) != 0 && !(*spoiled & kGivenUp)) {
        // the states wait in shared memory, which no tile needs any more
        uint64_t* keep = reinterpret_cast<uint64_t*>(sm) + tid - 256;
        static_assert(512 * KT * 4 <= NS * Cfg::kBytesKQ, "room for the states");
#pragma unroll
        for (int i = 0; i < KT / 2; ++i) keep[512 * i] = S[i];
        if (rows != 0) odd_tokens<D>(p, h, vblk * Cfg::kVB, whose[1], whose[2], odd, warp - 8);
        bar_sync<512>(kBarAgain);
        for (int g = warp - 8; g < Cfg::kVB / kGroup; g += 16) {
          const bool whole = again >> g & 1;
          if (whole || (rows >> g & 1))
            delta_columns_again<D>(p, h, vblk * Cfg::kVB + g * kGroup, whose[1], whole ? whose[2] : odd[2],
                                   first_state(sample), whole ? end : nullptr, !whole);
        }
        bar_sync<512>(kBarAgain);
#pragma unroll
        for (int i = 0; i < KT / 2; ++i) S[i] = keep[512 * i];
      }
    }
    if (writes && end != nullptr && !(again >> (vr / kGroup) & 1)) {
      if (moves) {  // [value column][key], as the join reads it
        ulonglong2* dst = reinterpret_cast<ulonglong2*>(end + (int64_t)(vblk * Cfg::kVB + vr) * D + KT * part);
#pragma unroll
        for (int i = 0; i < KT / 4; ++i) dst[i] = make_ulonglong2(S[2 * i], S[2 * i + 1]);
      } else {
        float* dst = end + col_off;
#pragma unroll
        for (int i = 0; i < KT; i += 2) {
          dst[i * D] = f32x2_lo(S[i / 2]);
          dst[(i + 1) * D] = f32x2_hi(S[i / 2]);
        }
      }
    }
  }
  if (!alive) {
    atomicOr(&g_delta_status, 1);
    *stalled = 1;
  }
  tc::fence_before();
  __syncthreads();  // every wait of every role lies before
  if (warp == 0) tc::dealloc(tmem, 512);
  if (*stalled != 0) delta_lost<D, OUT>(p, whose[0], whose[1], whose[2], whose[3] != 0);
}

}  // namespace memt
