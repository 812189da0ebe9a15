// Causal linear attention with a decay for each head, packed samples: parameters of its kernels
// and the token-by-token form.
//
//     S_t = e^{g_t} S_{t-1} + k_t v_t^T,    o_t = scale S_t^T q_t
//
// The token-by-token kernel is the definition in fp32 on CUDA cores. It serves fp32 inputs (as the
// fp32 mode of the update does) and bf16 samples of few tokens, where the states are most of the
// traffic and a 64-token chunk is mostly padding. The state is in registers as in the single-token
// step (16-byte vectors of whole rows, 64 value columns a CTA); tokens come in batches of four, whose
// vectors are fetched a batch ahead and whose outputs share one barrier. One token costs the states'
// traffic (256 samples, 16 heads, D = 128: 83 us, the floor 83); each one more from 5 us to 11, the work
// of folding it in. fp32 prompts (8 x 8192 tokens, 16 heads, D = 128): 4.4 ms, with four columns a warp and all
// lanes on the rows 8.4.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "step.cuh"

namespace memt {

struct LinearParams {
  int32_t N, H, Hk;
  int64_t L;
  const int32_t* cu;
  const void* q;
  const void* k;
  const void* v;
  int64_t sq, sk, sv, so;  // elements per token row
  const float* g;
  int32_t g_layout;  // MEMT_GATE_NONE / PER_HEAD / CONSTANT
  float scale;
  void* out;
  const float* h0;  // null: zero states
  float* ht;
  const int32_t* slots_in;
  const int32_t* slots_out;
  int32_t num_in, num_out;
  // Samples of up to `few` tokens go token by token, longer ones in chunks (fp32: all and none).
  int32_t few;
  // Chunked form of few long samples: 0, or 64-token chunks per segment, and the segments' states
  // [segment][H][D][D] (first their own sums, then the state before each) and decays [segment][H].
  int32_t seg_chunks;
  int32_t max_segments;
  int32_t by_length;   // whole samples, the longest first
  int32_t only_long;   // 0, or the CTAs a head where each finds one of the samples of more than `few` tokens
  float* seg_states;
  float2* seg_decays;
};

// tokens [bos, eos) of sample n, clamped to the packed rows
__device__ __forceinline__ void sample_range(const LinearParams& p, int n, int64_t& bos, int64_t& eos) {
  bos = p.cu[n];
  eos = p.cu[n + 1];
  bos = bos < 0 ? 0 : (bos > p.L ? p.L : bos);
  eos = eos < bos ? bos : (eos > p.L ? p.L : eos);
}

// Segments of a sample: runs of seg_chunks chunks of 64 tokens, at least one.
__device__ __forceinline__ int segments_of(const LinearParams& p, int64_t tokens) {
  const int64_t run = (int64_t)p.seg_chunks * kTile;
  return tokens > run ? static_cast<int>((tokens + run - 1) / run) : 1;
}

// Segments of samples 0 .. n, of the `sum` that their lengths make: bounded such that the call's fit into
// max_segments with at least one for each sample. Only offsets that overlap reach the bound; the last
// segment of a sample then runs to its end.
__device__ __forceinline__ int segments_up_to(const LinearParams& p, int n, int sum) {
  const int room = p.max_segments - (p.N - 1 - n);
  return sum < room ? sum : room;
}

// Sample n, segment s of its `count`, of the call's segment number `unit` (samples in order), found by
// a converged warp; false when there are fewer segments.
__device__ __forceinline__ bool find_segment(const LinearParams& p, int unit, int& n, int& s, int& count) {
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int n0 = 0; n0 < p.N; n0 += 32) {
    int own = 0;
    if (n0 + lane < p.N) {
      int64_t bos, eos;
      sample_range(p, n0 + lane, bos, eos);
      own = segments_of(p, eos - bos);
    }
    int incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += x;
    }
    const int last = segments_up_to(p, n0 + lane, base + incl);
    const int first = n0 + lane == 0 ? 0 : segments_up_to(p, n0 + lane - 1, base + incl - own);
    const uint32_t past = __ballot_sync(~0u, n0 + lane < p.N && last > unit);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      n = n0 + l;
      const int at = __shfl_sync(~0u, first, l);
      count = __shfl_sync(~0u, last, l) - at;
      s = unit - at;
      return true;
    }
    base += __shfl_sync(~0u, incl, 31);
  }
  return false;
}

// The sample with the rank-th longest token range (ties: the lower index first), found by a converged
// warp. N is small: every lane ranks its samples against all.
__device__ __forceinline__ int sample_by_length(const LinearParams& p, int rank) {
  const int lane = threadIdx.x & 31;
  int found = 0;
  for (int n0 = 0; n0 < p.N; n0 += 32) {
    const int n = n0 + lane;
    int64_t bos, eos, len = -1;
    if (n < p.N) {
      sample_range(p, n, bos, eos);
      len = eos - bos;
    }
    int ahead = 0;
    for (int m = 0; m < p.N; ++m) {
      sample_range(p, m, bos, eos);
      ahead += eos - bos > len || (eos - bos == len && m < n);
    }
    const uint32_t hit = __ballot_sync(~0u, n < p.N && ahead == rank);
    if (hit != 0) found = n0 + __ffs(hit) - 1;
  }
  return found;
}

// The unit-th sample of more than p.few tokens, found by a converged warp; -1 when there are fewer.
__device__ __forceinline__ int find_long(const LinearParams& p, int unit) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int n0 = 0; n0 < p.N; n0 += 32) {
    int64_t bos = 0, eos = 0;
    const bool own = n0 + lane < p.N;
    if (own) sample_range(p, n0 + lane, bos, eos);
    const uint32_t longer = __ballot_sync(~0u, own && eos - bos > p.few);
    const int rank = before + __popc(longer & ((1u << lane) - 1));
    const uint32_t hit = __ballot_sync(~0u, rank == unit && (longer >> lane & 1));
    if (hit != 0) return n0 + __ffs(hit) - 1;
    before += __popc(longer);
  }
  return -1;
}

// Samples before n of more than p.few tokens, counted by a converged warp: offsets that overlap can make
// more of them than there are CTAs to find them, and the token-by-token kernel takes the rest.
__device__ __forceinline__ int long_before(const LinearParams& p, int n) {
  int count = 0;
  for (int n0 = 0; n0 < n; n0 += 32) {
    const int m = n0 + (threadIdx.x & 31);
    int64_t bos = 0, eos = 0;
    if (m < n) sample_range(p, m, bos, eos);
    count += __popc(__ballot_sync(~0u, m < n && eos - bos > p.few));
  }
  return count;
}

// A decay as a pair of fp32 numbers, hi + lo. Neither is negative, and lo is above zero where hi is, so that
// an infinite state stays infinite with its sign: hi inf + (lo inf + u). (2^-149 of a state changes no sum.)
__device__ __forceinline__ float low_half(float hi, float lo) { return hi > 0.f ? fmaxf(lo, 1.4e-45f) : lo; }
__device__ __forceinline__ void split_decay(double a, float& hi, float& lo) {
  hi = __double2float_rd(a);
  lo = low_half(hi, static_cast<float>(a - static_cast<double>(hi)));
}

__device__ __forceinline__ float log_decay(const LinearParams& p, int64_t t, int h) {
  return p.g_layout == 1 ? p.g[t * p.H + h] : (p.g_layout == 3 ? p.g[h] : 0.f);
}

// an earlier sample of this call writes the same slot
__device__ __forceinline__ bool slot_taken(const int32_t* slots, int n, int64_t slot, int tid, int threads) {
  bool taken = false;
  if (slots != nullptr)
    for (int i = tid; i < n; i += threads) taken |= slots[i] == static_cast<int32_t>(slot);
  return taken;
}

// Between the two passes over segments: the state before each one. A thread owns four values of one
// (sample, head) state and walks over its segments; the segments' own sums are replaced in place.
__global__ void __launch_bounds__(256) linear_segments_kernel(const LinearParams p, int D) {
  const int per_state = D * D / 4, blocks = (per_state + 255) / 256;
  const int at = (blockIdx.x % blocks) * 256 + threadIdx.x;
  const int nh = blockIdx.x / blocks, h = nh % p.H, n = nh / p.H;
  int64_t bos, eos;
  int first = 0, count = 1;
  {  // this sample's first segment: every warp sums the samples before it
    const int lane = threadIdx.x & 31;
    for (int m = lane; m < n; m += 32) {
      sample_range(p, m, bos, eos);
      first += segments_of(p, eos - bos);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) first += __shfl_xor_sync(~0u, first, o);
    sample_range(p, n, bos, eos);
    count = segments_up_to(p, n, first + segments_of(p, eos - bos));
    first = n == 0 ? 0 : segments_up_to(p, n - 1, first);
    count -= first;
  }
  if (count == 1 || at >= per_state) return;  // one segment starts from the sample's own state
  const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n);
  float4 S = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p.h0 != nullptr && in_slot >= 0)
    S = reinterpret_cast<const float4*>(p.h0 + (in_slot * p.H + h) * D * D)[at];
  for (int s = 0; s < count; ++s) {
    const int64_t seg = (int64_t)(first + s) * p.H + h;
    float4* state = reinterpret_cast<float4*>(p.seg_states + seg * D * D) + at;
    float4 own = make_float4(0.f, 0.f, 0.f, 0.f);
    float2 a = make_float2(0.f, 0.f);
    if (s + 1 < count) {  // the last one's sum is not made: the second pass ends with it
      own = *state;
      a = p.seg_decays[seg];
    }
    *state = S;
    S.x = fmaf(a.x, S.x, fmaf(a.y, S.x, own.x));
    S.y = fmaf(a.x, S.y, fmaf(a.y, S.y, own.y));
    S.z = fmaf(a.x, S.z, fmaf(a.y, S.z, own.z));
    S.w = fmaf(a.x, S.w, fmaf(a.y, S.w, own.w));
  }
}

// Token-by-token form: fp32 inputs, and bf16 samples of few tokens.
template <int D>
struct LinearTokensCfg {
  static constexpr int kCols = 64, kBlocks = D / kCols;  // value columns per CTA, CTAs per (sample, head)
  static constexpr int kRows = D == 64 ? 4 : 8;          // state rows per thread, 8 columns of each
  static constexpr int kWarps = D / (4 * kRows);         // four row groups of eight lanes a warp
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kBatch = 4;                       // tokens between two barriers
  static constexpr int kPer = (D + kThreads - 1) / kThreads;
  static constexpr int kMinCtas = D == 256 ? 2 : (D == 128 ? 4 : 6);
};

template <int D, typename T>
__global__ void __launch_bounds__(LinearTokensCfg<D>::kThreads, LinearTokensCfg<D>::kMinCtas)
    linear_tokens_kernel(const LinearParams p) {
  using Cfg = LinearTokensCfg<D>;
  constexpr int R = Cfg::kRows, W = Cfg::kWarps, TB = Cfg::kBatch, NT = Cfg::kThreads, C = Cfg::kCols, NP = Cfg::kPer;
  __shared__ __align__(16) float s_k[2][TB][D], s_q[2][TB][D], s_v[2][TB][C];
  __shared__ float s_a[2][TB];
  __shared__ __align__(16) float s_o[2][W][TB][C];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int blk = blockIdx.x % Cfg::kBlocks, nh = blockIdx.x / Cfg::kBlocks;
  const int h = nh % p.H, n = nh / p.H, hk = h / (p.H / p.Hk);
  // rows row0 + i, columns col .. col + 3 and col + 32 .. col + 35: a warp's load covers four rows' 128-byte
  // lines, and a token costs two reads of shared memory for each of k, q and v
  const int row0 = (4 * warp + (lane >> 3)) * R, col = 4 * (lane & 7);
  int64_t bos, eos;
  sample_range(p, n, bos, eos);
  if (eos - bos > p.few && (p.only_long == 0 || long_before(p, n) < p.only_long)) return;  // goes in chunks
  const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n), out_slot = pool_slot(p.slots_out, p.num_out, n);
  const int64_t at = (int64_t)row0 * D + blk * C + col;
  uint64_t S[R][4];  // fp32 pairs
  if (p.h0 != nullptr && in_slot >= 0) {
    const float* src = p.h0 + (in_slot * p.H + h) * D * D + at;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float4 x = __ldcs(reinterpret_cast<const float4*>(src + i * D + 32 * e));
        S[i][2 * e] = f32x2_pack(x.x, x.y);
        S[i][2 * e + 1] = f32x2_pack(x.z, x.w);
      }
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) S[i][0] = S[i][1] = S[i][2] = S[i][3] = 0;
  }
  // A decay that is the same for every token is a pair of fp32 numbers: the rounding of one, repeated
  // for every token, would drift (7e-6 over 16384 tokens).
  float fixed_hi, fixed_lo;
  split_decay(p.g_layout == 3 ? exp(static_cast<double>(p.g[h])) : 1.0, fixed_hi, fixed_lo);
  const uint64_t a_lo = f32x2_splat(fixed_lo);

  // the next batch's vectors, as loaded: nothing waits for them before keep()
  T xk[TB][NP], xq[TB][NP], xv[TB];
  float xg = 0.f;
  auto fetch = [&](int64_t t0) {
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      const bool live = t0 + t < eos;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int c = tid + i * NT;
        xk[t][i] = xq[t][i] = T(0.f);
        if (live && c < D) {
          xk[t][i] = static_cast<const T*>(p.k)[(t0 + t) * p.sk + (int64_t)hk * D + c];
          xq[t][i] = static_cast<const T*>(p.q)[(t0 + t) * p.sq + (int64_t)hk * D + c];
        }
      }
      xv[t] = T(0.f);
      if (live && tid < C) xv[t] = static_cast<const T*>(p.v)[(t0 + t) * p.sv + (int64_t)h * D + blk * C + tid];
    }
    xg = 0.f;
    if (p.g_layout == 1 && tid < TB && t0 + tid < eos) xg = p.g[(t0 + tid) * p.H + h];
  };
  auto keep = [&](int buf) {
#pragma unroll
    for (int t = 0; t < TB; ++t) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int c = tid + i * NT;
        if (c < D) {
          s_k[buf][t][c] = as_f32(xk[t][i]);
          s_q[buf][t][c] = as_f32(xq[t][i]);
        }
      }
      if (tid < C) s_v[buf][t][tid] = as_f32(xv[t]);
    }
    if (tid < TB) s_a[buf][tid] = p.g_layout == 1 ? expf(xg) : fixed_hi;
  };
  auto fold = [&](int buf, int t, uint64_t (&o)[4], auto pair) {  // one token into the state, its partial output
    uint64_t v[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float4 x = *reinterpret_cast<const float4*>(&s_v[buf][t][col + 32 * e]);
      v[2 * e] = f32x2_pack(x.x, x.y);
      v[2 * e + 1] = f32x2_pack(x.z, x.w);
    }
    const uint64_t a = f32x2_splat(s_a[buf][t]);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = 0;
#pragma unroll
    for (int i0 = 0; i0 < R; i0 += 4) {
      const float4 k4 = *reinterpret_cast<const float4*>(&s_k[buf][t][row0 + i0]);
      const float4 q4 = *reinterpret_cast<const float4*>(&s_q[buf][t][row0 + i0]);
      const float ks[4] = {k4.x, k4.y, k4.z, k4.w}, qs[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t k = f32x2_splat(ks[j]), q = f32x2_splat(qs[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint64_t x = mul_f32x2(k, v[e]);
          if constexpr (decltype(pair)::value) x = fma_f32x2(a_lo, S[i0 + j][e], x);
          S[i0 + j][e] = fma_f32x2(a, S[i0 + j][e], x);
          o[e] = fma_f32x2(S[i0 + j][e], q, o[e]);
        }
      }
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
      uint64_t o[4];
      if (p.g_layout == 3) fold(b, t, o, std::true_type{});
      else fold(b, t, o, std::false_type{});
      // sums over the warp's four row groups: each exchange halves the columns a lane is left with
      const bool hi = lane & 8, hi2 = lane & 16;
      float z[4];  // columns of half `hi`
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint64_t mine = hi ? o[2 + e] : o[e], give = hi ? o[e] : o[2 + e];
        z[2 * e] = f32x2_lo(mine) + __shfl_xor_sync(0xffffffffu, f32x2_lo(give), 8);
        z[2 * e + 1] = f32x2_hi(mine) + __shfl_xor_sync(0xffffffffu, f32x2_hi(give), 8);
      }
      float2 y;  // columns 2 hi2, 2 hi2 + 1 of those
      y.x = (hi2 ? z[2] : z[0]) + __shfl_xor_sync(0xffffffffu, hi2 ? z[0] : z[2], 16);
      y.y = (hi2 ? z[3] : z[1]) + __shfl_xor_sync(0xffffffffu, hi2 ? z[1] : z[3], 16);
      *reinterpret_cast<float2*>(&s_o[b][warp][t][col + (hi ? 32 : 0) + (hi2 ? 2 : 0)]) = y;
    }
    keep(b ^ 1);
    __syncthreads();
    for (int i = tid; i < TB * C; i += NT) {
      const int t = i / C, c = i % C;
      if (t0 + t >= eos) break;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += s_o[b][w][t][c];
      store_f32(static_cast<T*>(p.out), (t0 + t) * p.so + (int64_t)h * D + blk * C + c, p.scale * sum);
    }
  }
  const bool taken = __any_sync(0xffffffffu, slot_taken(p.slots_out, n, out_slot, lane, 32));
  if (out_slot < 0 || taken) return;
  float* dst = p.ht + (out_slot * p.H + h) * D * D + at;
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      __stcs(reinterpret_cast<float4*>(dst + i * D + 32 * e),
             make_float4(f32x2_lo(S[i][2 * e]), f32x2_hi(S[i][2 * e]), f32x2_lo(S[i][2 * e + 1]),
                         f32x2_hi(S[i][2 * e + 1])));
}

}  // namespace memt
