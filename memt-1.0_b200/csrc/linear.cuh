// Causal linear attention with a decay for each head, packed samples: parameters of its kernels
// and the token-by-token form.
//
//     S_t = e^{g_t} S_{t-1} + k_t v_t^T,    o_t = scale S_t^T q_t
//
// The token-by-token kernel is the definition in fp32 on CUDA cores. It serves fp32 inputs (as
// the fp32 mode of the update does) and is bound by the latency of the token chain.
// One warp owns kCols value columns of one (sample, head): the state's D rows are spread over the
// lanes (D / 32 rows each), so a token costs D / 32 * kCols * 2 multiply-adds a lane and one
// butterfly sum over the lanes, without any barrier between warps. The next token's vectors are
// fetched while this one is folded in.
#pragma once

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
  // Chunked form of few long samples: 0, or 64-token chunks per segment, and the segments' states
  // [segment][H][D][D] (first their own sums, then the state before each) and decays [segment][H].
  int32_t seg_chunks;
  int32_t max_segments;
  int32_t by_length;  // whole samples, the longest first
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
    const uint32_t past = __ballot_sync(~0u, base + incl > unit);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      n = n0 + l;
      count = __shfl_sync(~0u, own, l);
      s = unit - (base + __shfl_sync(~0u, incl, l) - count);
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
    count = segments_of(p, eos - bos);
  }
  if (count == 1 || at >= per_state) return;  // one segment starts from the sample's own state
  const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n);
  float4 S = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p.h0 != nullptr && in_slot >= 0)
    S = reinterpret_cast<const float4*>(p.h0 + (in_slot * p.H + h) * D * D)[at];
  // (offsets that overlap, which no packed batch has, could make more segments than there is room for)
  for (int s = 0; s < count && first + s < p.max_segments; ++s) {
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

struct LinearRecurrentCfg {
  static constexpr int kCols = 4;   // value columns per warp
  static constexpr int kWarps = 4;  // warps per CTA, consecutive column groups
};

template <int D>
__global__ void __launch_bounds__(LinearRecurrentCfg::kWarps * 32) linear_recurrent_kernel(const LinearParams p) {
  constexpr int C = LinearRecurrentCfg::kCols, W = LinearRecurrentCfg::kWarps, R = D / 32;
  constexpr int kBlocks = D / (C * W);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blk = blockIdx.x % kBlocks, nh = blockIdx.x / kBlocks;
  const int h = nh % p.H, n = nh / p.H, hk = h / (p.H / p.Hk);
  const int col = (blk * W + warp) * C, row = lane * R;
  int64_t bos, eos;
  sample_range(p, n, bos, eos);
  const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n), out_slot = pool_slot(p.slots_out, p.num_out, n);
  float S[R][C];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int e = 0; e < C; ++e)
      S[i][e] = p.h0 != nullptr && in_slot >= 0 ? p.h0[((in_slot * p.H + h) * D + row + i) * D + col + e] : 0.f;
  float q[R], k[R], v[C], g = 0.f;
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      q[i] = load_f32<float>(p.q, t * p.sq + (int64_t)hk * D + row + i);
      k[i] = load_f32<float>(p.k, t * p.sk + (int64_t)hk * D + row + i);
    }
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = load_f32<float>(p.v, t * p.sv + (int64_t)h * D + col + e);
    g = log_decay(p, t, h);
  };
  if (bos < eos) fetch(bos);
  // A decay that is the same for every token is a pair of fp32 numbers: the rounding of one, repeated
  // for every token, would drift (7e-6 over 16384 tokens).
  const double fixed = p.g_layout == 3 ? exp(static_cast<double>(p.g[h])) : 1.0;
  const float fixed_hi = static_cast<float>(fixed), fixed_lo = static_cast<float>(fixed - fixed_hi);
  for (int64_t t = bos; t < eos; ++t) {
    float o[C] = {0.f, 0.f, 0.f, 0.f};
    const float a = p.g_layout == 1 ? expf(g) : fixed_hi, a_lo = p.g_layout == 1 ? 0.f : fixed_lo;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int e = 0; e < C; ++e) {
        S[i][e] = fmaf(a, S[i][e], fmaf(a_lo, S[i][e], k[i] * v[e]));
        o[e] = fmaf(S[i][e], q[i], o[e]);
      }
    if (t + 1 < eos) fetch(t + 1);
#pragma unroll
    for (int e = 0; e < C; ++e)
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) o[e] += __shfl_xor_sync(0xffffffffu, o[e], m);
    if (lane < C) {
      const float x = lane == 0 ? o[0] : lane == 1 ? o[1] : lane == 2 ? o[2] : o[3];
      store_f32(static_cast<float*>(p.out), t * p.so + (int64_t)h * D + col + lane, p.scale * x);
    }
  }
  const bool taken = __any_sync(0xffffffffu, slot_taken(p.slots_out, n, out_slot, lane, 32));
  if (out_slot < 0 || taken) return;
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int e = 0; e < C; ++e) p.ht[((out_slot * p.H + h) * D + row + i) * D + col + e] = S[i][e];
}

}  // namespace memt
