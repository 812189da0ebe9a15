// The gated delta rule over packed samples: parameters of its kernels and the token-by-token form.
//
//     S_t = a_t S_{t-1} + beta_t k_t (v_t - a_t S_{t-1}^T k_t)^T,  a_t = e^{g_t},   o_t = scale S_t^T q_t
//
// The token-by-token kernel is the definition in fp32 on CUDA cores: fp32 inputs and bf16 samples of few
// tokens. A token's correction needs a sum over all rows of the state before any of it can be written, so
// a warp owns whole columns: its lanes are row groups of four columns each, the sums over the rows are three
// (D = 256: four) exchanges between lanes, and no token waits for another warp. Both sums of a token,
// S^T k and S^T q, are taken of the state before it, where they need not wait for one another:
//     d = beta (v - a S^T k),   S <- a S + k d^T,   o = scale (a S^T q + (q.k) d)
// k and q are staged in shared memory a batch of tokens ahead as 16-byte vectors, rows of a lane in groups of
// four such that a warp reads them without bank conflicts and the packed arithmetic pairs rows.
// Bound by the states' traffic for one token, by the latency of a token's chain of exchanges for many: 0.31 us a token at
// D = 64 (2 samples of up to 1000, 8 states), 0.40 at D = 128; 256 samples of up to 16 tokens, 16 heads, D = 128: 211 us
// where the states' traffic alone takes 82.
#pragma once

#include <type_traits>

#include "linear.cuh"

namespace memt {

struct DeltaParams : LinearParams {
  const void* beta;
  int32_t beta_layout;  // MEMT_GATE_NONE / PER_HEAD (key heads) / PER_VALUE_HEAD
  // Chunked form (delta_chunks.cuh, delta_tc.cuh): what each chunk needs of its keys, queries and gates, [unit][H] of
  // DeltaChunks::kBytes. Units are the chunks of the samples of more than `few` tokens, in order; max_units of them fit,
  // as many as there can be unless offsets overlap.
  int32_t max_units;
  void* chunks;
  // Calls of many samples: where a unit's chunk is (sample, chunk; -1 behind the last), a sample's first unit [N + 1], and
  // the samples of more than `few` tokens (-1 behind the last; only_long of them). Otherwise null: searched for.
  int2* unit_table;
  int32_t* first_unit;
  int32_t* longs;
  // Segments of few long samples (linear.cuh): seg_states and, as large, what each makes of an identity.
  float* seg_moves;
};

__device__ __forceinline__ int units_of(const DeltaParams& p, int n) {
  int64_t bos, eos;
  sample_range(p, n, bos, eos);
  return eos - bos > p.few ? static_cast<int>((eos - bos + kTile - 1) / kTile) : 0;
}

// The units of sample n, by a converged warp: the first one's number and how many.
__device__ __forceinline__ void sample_units(const DeltaParams& p, int n, int& first, int& count) {
  if (p.first_unit != nullptr) {
    first = p.first_unit[n];
    count = p.first_unit[n + 1] - first;
    return;
  }
  int64_t before = 0;
  for (int m = threadIdx.x & 31; m < n; m += 32) before += units_of(p, m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(~0u, before, o);
  const int64_t end = before + units_of(p, n);
  first = static_cast<int>(before < p.max_units ? before : p.max_units);
  count = static_cast<int>(end < p.max_units ? end : p.max_units) - first;
}

// Chunk c of sample n, unit number `unit`, found by a converged warp; false when there are fewer.
__device__ __forceinline__ bool find_unit(const DeltaParams& p, int unit, int& n, int& c) {
  if (p.unit_table != nullptr) {
    const int2 x = p.unit_table[unit];
    n = x.x;
    c = x.y;
    return n >= 0;
  }
  const int lane = threadIdx.x & 31;
  int64_t base = 0;
  for (int n0 = 0; n0 < p.N; n0 += 32) {
    const int64_t own = n0 + lane < p.N ? units_of(p, n0 + lane) : 0;
    int64_t incl = base + own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(~0u, incl - base, o);
      if (lane >= o) incl += x;
    }
    const uint32_t past = __ballot_sync(~0u, incl > unit);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      n = n0 + l;
      c = static_cast<int>(unit - __shfl_sync(~0u, incl - own, l));
      return true;
    }
    base = __shfl_sync(~0u, incl, 31);
  }
  return false;
}

// The tables of a call of many samples, by one CTA: a search in every CTA of the others would take their number times
// that of the samples (4096 samples of 8 tokens, 16 heads: half of the call). num_longs: entries of `longs`.
constexpr int kPlanThreads = 1024;
__global__ void __launch_bounds__(kPlanThreads) delta_plan_kernel(const DeltaParams p, int num_longs) {
  __shared__ int64_t s_units[kPlanThreads / 32];
  __shared__ int s_longs[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto clamp = [&](int64_t u) { return static_cast<int>(u < p.max_units ? u : p.max_units); };
  int64_t base = 0;
  int long_base = 0;
  for (int n0 = 0; n0 < p.N; n0 += kPlanThreads) {
    const int n = n0 + tid;
    const int own = n < p.N ? units_of(p, n) : 0;
    int64_t incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += x;
    }
    const uint32_t longer = __ballot_sync(~0u, own > 0);
    if (lane == 31) {
      s_units[warp] = incl;
      s_longs[warp] = __popc(longer);
    }
    __syncthreads();
    int64_t first = base + incl - own;
    int rank = long_base + __popc(longer & ((1u << lane) - 1));
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w < warp) {
        first += s_units[w];
        rank += s_longs[w];
      }
      base += s_units[w];
      long_base += s_longs[w];
    }
    if (n < p.N) p.first_unit[n] = clamp(first);
    if (own > 0 && rank < num_longs) p.longs[rank] = n;
    for (uint32_t rest = longer; rest != 0; rest &= rest - 1) {  // a sample's units, by the warp
      const int l = __ffs(rest) - 1;
      const int64_t from = __shfl_sync(~0u, first, l);
      const int to = clamp(from + __shfl_sync(~0u, own, l));
      for (int64_t u = from + lane; u < to; u += 32)
        p.unit_table[u] = make_int2(n0 + 32 * warp + l, static_cast<int>(u - from));
    }
    __syncthreads();
  }
  if (tid == 0) p.first_unit[p.N] = clamp(base);
  for (int u = clamp(base) + tid; u < p.max_units; u += kPlanThreads) p.unit_table[u] = make_int2(-1, 0);
  for (int i = long_base + tid; i < num_longs; i += kPlanThreads) p.longs[i] = -1;
}

// A warp's columns of one state, four to a lane, and a token's step on them; CG: lanes across the columns.
template <int D, int CG = D == 256 ? 2 : 4>
struct DeltaColumns {
  static constexpr int kColGroups = CG;
  static constexpr int kRowGroups = 32 / kColGroups;
  static constexpr int kCols = 4 * kColGroups;         // columns of a warp
  static constexpr int kRows = D / kRowGroups;         // rows of a lane: 4 group + 4 kRowGroups m + 0 .. 3
  uint64_t S[kRows / 2][4];                            // rows 2 i, 2 i + 1 of those, column by column

  static __device__ __forceinline__ int row0() { return 4 * ((threadIdx.x & 31) / kColGroups); }
  static __device__ __forceinline__ int col0() { return 4 * ((threadIdx.x & 31) % kColGroups); }

  // states of D x D, from the warp's first column; null: zeros
  __device__ __forceinline__ void load(const float* state) {
#pragma unroll
    for (int i = 0; i < kRows / 2; ++i) {
      const int r = row0() + 4 * kRowGroups * (i >> 1) + 2 * (i & 1);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
      if (state != nullptr) {
        x = __ldcs(reinterpret_cast<const float4*>(state + r * D + col0()));
        y = __ldcs(reinterpret_cast<const float4*>(state + (r + 1) * D + col0()));
      }
      S[i][0] = f32x2_pack(x.x, y.x);
      S[i][1] = f32x2_pack(x.y, y.y);
      S[i][2] = f32x2_pack(x.z, y.z);
      S[i][3] = f32x2_pack(x.w, y.w);
    }
  }
  __device__ __forceinline__ void store(float* state) const {
#pragma unroll
    for (int i = 0; i < kRows / 2; ++i) {
      const int r = row0() + 4 * kRowGroups * (i >> 1) + 2 * (i & 1);
      __stcs(reinterpret_cast<float4*>(state + r * D + col0()),
             make_float4(f32x2_lo(S[i][0]), f32x2_lo(S[i][1]), f32x2_lo(S[i][2]), f32x2_lo(S[i][3])));
      __stcs(reinterpret_cast<float4*>(state + (r + 1) * D + col0()),
             make_float4(f32x2_hi(S[i][0]), f32x2_hi(S[i][1]), f32x2_hi(S[i][2]), f32x2_hi(S[i][3])));
    }
  }

  // Sums over the rows of eight values: afterwards lanes with bit 4 clear hold one of the first four, those
  // with it set one of the others, number own_col().
  static __device__ __forceinline__ int own_col() { return (threadIdx.x >> 2 & 1) + (threadIdx.x >> 2 & 2); }
  static __device__ __forceinline__ float sum_rows(const float (&z)[8]) {
    const bool b4 = threadIdx.x & 16, b3 = threadIdx.x & 8, b2 = threadIdx.x & 4;
    float x[4], y[2], w;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (b4 ? z[4 + i] : z[i]) + __shfl_xor_sync(~0u, b4 ? z[i] : z[4 + i], 16);
#pragma unroll
    for (int i = 0; i < 2; ++i) y[i] = (b3 ? x[2 + i] : x[i]) + __shfl_xor_sync(~0u, b3 ? x[i] : x[2 + i], 8);
    w = (b2 ? y[1] : y[0]) + __shfl_xor_sync(~0u, b2 ? y[0] : y[1], 4);
    if constexpr (kColGroups == 2) w += __shfl_xor_sync(~0u, w, 2);
    return w;
  }

  // One token: k(i), q(i) give rows 4 (kRowGroups m) + row0() .. + 3 as float4 for i = m; v(c) the value of the
  // warp's column c. Lanes for which writes() return their column's output, without the scale. PAIR: the decay
  // is a_hi + a_lo.
  static __device__ __forceinline__ bool writes() {
    return (threadIdx.x & 16) && (kColGroups == 4 || !(threadIdx.x & 2));
  }
  template <bool PAIR, typename K, typename Q, typename V>
  __device__ __forceinline__ float step(K k, Q q, V v, float a_hi, float a_lo, float beta) {
    uint64_t r2[4] = {0, 0, 0, 0}, y2[4] = {0, 0, 0, 0}, kq2 = 0;
#pragma unroll
    for (int m = 0; m < kRows / 4; ++m) {
      const float4 k4 = k(m), q4 = q(m);
      const uint64_t kk[2] = {f32x2_pack(k4.x, k4.y), f32x2_pack(k4.z, k4.w)};
      const uint64_t qq[2] = {f32x2_pack(q4.x, q4.y), f32x2_pack(q4.z, q4.w)};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        kq2 = fma_f32x2(kk[j], qq[j], kq2);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          r2[c] = fma_f32x2(S[2 * m + j][c], kk[j], r2[c]);
          y2[c] = fma_f32x2(S[2 * m + j][c], qq[j], y2[c]);
        }
      }
    }
    float z[8];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      z[c] = f32x2_lo(r2[c]) + f32x2_hi(r2[c]);
      z[4 + c] = f32x2_lo(y2[c]) + f32x2_hi(y2[c]);
    }
    float kq = f32x2_lo(kq2) + f32x2_hi(kq2);
#pragma unroll
    for (int o = kColGroups; o < 32; o <<= 1) kq += __shfl_xor_sync(~0u, kq, o);
    const float w = sum_rows(z);
    const float aw = PAIR ? fmaf(a_hi, w, a_lo * w) : a_hi * w;
    const float mine = beta * (v(col0() + own_col()) - aw);  // meant on the lanes without bit 4
    float d[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) d[c] = __shfl_sync(~0u, mine, (threadIdx.x & (kColGroups - 1)) + 4 * c);
    const float d_own = __shfl_sync(~0u, mine, threadIdx.x & 15);
    const uint64_t ah = f32x2_splat(a_hi), al = f32x2_splat(a_lo);
#pragma unroll
    for (int m = 0; m < kRows / 4; ++m) {
      const float4 k4 = k(m);
      const uint64_t kk[2] = {f32x2_pack(k4.x, k4.y), f32x2_pack(k4.z, k4.w)};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint64_t x = mul_f32x2(kk[j], f32x2_splat(d[c]));
          if constexpr (PAIR) x = fma_f32x2(al, S[2 * m + j][c], x);
          S[2 * m + j][c] = fma_f32x2(ah, S[2 * m + j][c], x);
        }
    }
    float out = fmaf(kq, d_own, aw);
    // What is not finite in the correction or the query makes terms of either sign, which k.q and S^T q would not show: the
    // new state's sum.
    if (__any_sync(~0u, !isfinite(out))) {
      uint64_t n2[4] = {0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < kRows / 4; ++m) {
        const float4 q4 = q(m);
        const uint64_t qq[2] = {f32x2_pack(q4.x, q4.y), f32x2_pack(q4.z, q4.w)};
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) n2[c] = fma_f32x2(S[2 * m + j][c], qq[j], n2[c]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) z[c] = z[4 + c] = f32x2_lo(n2[c]) + f32x2_hi(n2[c]);
      out = sum_rows(z);
    }
    return out;
  }
};

template <int D, int CG>
struct DeltaTokensCfg {
  static constexpr int kWarps = 4, kThreads = 32 * kWarps;
  static constexpr int kCols = kWarps * DeltaColumns<D, CG>::kCols, kBlocks = D / kCols;  // of a CTA; CTAs per state
  static constexpr int kBatch = 4;  // tokens between two barriers
};

template <int D, typename T, int CG>
__global__ void __launch_bounds__(DeltaTokensCfg<D, CG>::kThreads, 4) delta_tokens_kernel(const DeltaParams p) {
  using Cfg = DeltaTokensCfg<D, CG>;
  using Cols = DeltaColumns<D, CG>;
  constexpr int TB = Cfg::kBatch, NT = Cfg::kThreads, C = Cfg::kCols;
  constexpr int VE = 16 / sizeof(T), DV = D / VE, CV = C / VE;  // elements of a vector, vectors of a row
  constexpr int kVecs = TB * (2 * DV + CV), NV = (kVecs + NT - 1) / NT;
  __shared__ __align__(16) float s_x[2][TB * (2 * D + C)];  // k of the batch's tokens, then q, then v
  __shared__ float s_a[2][TB], s_b[2][TB];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int blk = blockIdx.x % Cfg::kBlocks, nh = blockIdx.x / Cfg::kBlocks;
  const int h = nh % p.H, n = nh / p.H, hk = h / (p.H / p.Hk);
  int64_t bos, eos;
  sample_range(p, n, bos, eos);
  if (eos - bos > p.few && (p.only_long == 0 || long_before(p, n) < p.only_long)) return;  // goes in chunks
  const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n), out_slot = pool_slot(p.slots_out, p.num_out, n);
  const int wcol = warp * Cols::kCols, col = blk * C + wcol;
  Cols cols;
  cols.load(p.h0 != nullptr && in_slot >= 0 ? p.h0 + (in_slot * p.H + h) * D * D + col : nullptr);
  // A decay that is the same for every token is a pair of fp32 numbers: the rounding of one would be repeated.
  float fixed_hi, fixed_lo;
  split_decay(p.g_layout == 3 ? exp(static_cast<double>(p.g[h])) : 1.0, fixed_hi, fixed_lo);

  // the next batch's vectors, as loaded: nothing waits for them before keep()
  uint4 x[NV];
  float xg = 0.f, xb = 1.f;
  auto fetch = [&](int64_t t0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = tid + i * NT;
      x[i] = make_uint4(0, 0, 0, 0);
      if (idx < 2 * TB * DV) {
        const int row = idx / DV, t = row % TB;
        const int64_t at = (int64_t)hk * D + (idx % DV) * VE;
        if (t0 + t < eos)
          x[i] = *reinterpret_cast<const uint4*>(row < TB ? static_cast<const T*>(p.k) + (t0 + t) * p.sk + at
                                                          : static_cast<const T*>(p.q) + (t0 + t) * p.sq + at);
      } else if (idx < kVecs) {
        const int t = (idx - 2 * TB * DV) / CV, e = (idx - 2 * TB * DV) % CV;
        if (t0 + t < eos)
          x[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.v) + (t0 + t) * p.sv + (int64_t)h * D +
                                                 blk * C + e * VE);
      }
    }
    if (tid < TB && t0 + tid < eos) {
      if (p.g_layout == 1) xg = p.g[(t0 + tid) * p.H + h];
      xb = load_beta<T>(p, t0 + tid, h);
    }
  };
  auto keep = [&](int buf) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = tid + i * NT;
      if (idx >= kVecs) continue;
      float4* dst = reinterpret_cast<float4*>(&s_x[buf][idx * VE]);
      if constexpr (sizeof(T) == 4) {
        *dst = make_float4(__uint_as_float(x[i].x), __uint_as_float(x[i].y), __uint_as_float(x[i].z),
                           __uint_as_float(x[i].w));
      } else {
        const float2 a = unpack_bf16x2(x[i].x), b = unpack_bf16x2(x[i].y), c = unpack_bf16x2(x[i].z),
                     d = unpack_bf16x2(x[i].w);
        dst[0] = make_float4(a.x, a.y, b.x, b.y);
        dst[1] = make_float4(c.x, c.y, d.x, d.y);
      }
    }
    if (tid < TB) {
      s_a[buf][tid] = p.g_layout == 1 ? expf(xg) : fixed_hi;
      s_b[buf][tid] = xb;
    }
  };
  fetch(bos);
  keep(0);
  __syncthreads();
  int b = 0;
  for (int64_t t0 = bos; t0 < eos; t0 += TB, b ^= 1) {
    fetch(t0 + TB);
#pragma unroll 1
    for (int t = 0; t < TB; ++t) {
      if (t0 + t >= eos) break;
      const float* kt = &s_x[b][t * D + Cols::row0()];
      const float* vt = &s_x[b][TB * 2 * D + t * C + wcol];
      auto k = [&](int m) { return *reinterpret_cast<const float4*>(kt + 4 * Cols::kRowGroups * m); };
      auto q = [&](int m) { return *reinterpret_cast<const float4*>(kt + TB * D + 4 * Cols::kRowGroups * m); };
      auto v = [&](int c) { return vt[c]; };
      const float out = p.g_layout == 3 ? cols.template step<true>(k, q, v, fixed_hi, fixed_lo, s_b[b][t])
                                        : cols.template step<false>(k, q, v, s_a[b][t], 0.f, s_b[b][t]);
      if (Cols::writes())
        store_f32(static_cast<T*>(p.out), (t0 + t) * p.so + (int64_t)h * D + col + Cols::col0() + Cols::own_col(),
                  p.scale * out);
    }
    keep(b ^ 1);
    __syncthreads();
  }
  const bool taken = __any_sync(~0u, slot_taken(p.slots_out, n, out_slot, lane, 32));
  if (out_slot < 0 || taken) return;
  cols.store(p.ht + (out_slot * p.H + h) * D * D + col);
}

}  // namespace memt
