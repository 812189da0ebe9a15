// One token of a matrix-state recurrence for each session, the states updated in place.
//
//   linear attention   S <- e^g S + k v^T,                               o = scale S^T q
//   stable GDN-2       S~ = diag(e^g) S,  d = w v - S~^T (b k'),  S <- S~ + k' d^T,
//                      o = scale S^T q, with the new state or the incoming one
//   gated delta rule   S~ = e^g S,  d = beta (v - S~^T k),  S <- S~ + k d^T,     o = scale S^T q
// with k' = sqrt(beta) k. All arithmetic is fp32 on the fp32 state; the output is rounded once.
//
// Bound by HBM: the state is read and written once, 8 D^2 bytes for each (session, head), every
// byte of it in registers in between. A warp holds whole rows (one 16-byte vector a lane), so
// that its loads and stores are full lines and a column's sum over the rows is a sum over
// registers, then over warps through shared memory. All state loads are issued before the
// token's vectors are fetched. A CTA takes 64 value columns, so that several on an SM are in different
// phases, and marks its loads and stores as read and written once. 256 sessions x 16 heads x 128 x 128
// (537 MB): 83.4 us linear, 87.1 us stable GDN-2, 0.99 and 0.95 of the measured copy rate (per call 85.7, 93.3, and 90.0
// with the gated delta rule's one decay and beta a head). Measured for GDN-2: 128 columns 95 us (93 without the
// marks), 64 without the marks on loads 96, on stores 97; states streamed through shared memory by bulk copies in a
// persistent CTA 104.
#pragma once

#include "common.cuh"

namespace memt {

struct StepParams {
  int32_t N, H, Hk;
  const void* q;
  const void* k;
  const void* v;
  int64_t sq, sk, sv, so;  // elements per token row
  const float* g;
  int32_t g_layout;  // MEMT_GATE_NONE / PER_HEAD / PER_CHANNEL / CONSTANT
  const void* beta;
  int32_t beta_layout;
  const void* erase;
  const void* write;
  float scale;
  float* states;
  const int32_t* slots;
  int32_t num_slots;
  int32_t incoming;
  int32_t gated;  // DELTA: the gated delta rule, beta on the correction instead of the key
  void* out;
};

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ float load_f32(const void* base, int64_t i) {
  return as_f32(static_cast<const T*>(base)[i]);
}
__device__ __forceinline__ void store_f32(float* base, int64_t i, float x) { base[i] = x; }
__device__ __forceinline__ void store_f32(__nv_bfloat16* base, int64_t i, float x) { base[i] = __float2bfloat16_rn(x); }

// beta of a token and value head, given for each value head or its key head; none: 1
template <typename T, typename P>
__device__ __forceinline__ float load_beta(const P& p, int64_t t, int h) {
  if (p.beta_layout == 0) return 1.f;
  return p.beta_layout == 4 ? load_f32<T>(p.beta, t * p.H + h) : load_f32<T>(p.beta, t * p.Hk + h / (p.H / p.Hk));
}

template <int D>
struct StepCfg {
  static constexpr int kCols = 64;  // value columns per CTA
  static constexpr int kBlocks = D / kCols;           // CTAs per (session, head)
  static constexpr int kLanes = kCols / 4;            // lanes across one row
  static constexpr int kRowsPerWarp = 32 / kLanes;    // rows a warp loads at once
  static constexpr int kVecs = D == 64 ? 8 : 16;      // 16-byte vectors of state per thread
  static constexpr int kWarps = D / (kVecs * kRowsPerWarp);
  static constexpr int kThreads = 32 * kWarps;
};

// DELTA: the rules with a correction. T: type of q, k, v, the gates and the output.
template <int D, bool DELTA, typename T>
__global__ void __launch_bounds__(StepCfg<D>::kThreads) step_kernel(const StepParams p) {
  using Cfg = StepCfg<D>;
  constexpr int NV = Cfg::kVecs, C = Cfg::kCols, NT = Cfg::kThreads;
  constexpr int G = Cfg::kWarps * Cfg::kRowsPerWarp;  // row groups: row = r * G + group
  __shared__ float s_q[D], s_k[D], s_kb[DELTA ? D : 1], s_a[D];
  __shared__ __align__(16) float s_o[G][C];
  __shared__ __align__(16) float s_r[DELTA ? G : 1][C];
  __shared__ float s_kq[Cfg::kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int blk = blockIdx.x % Cfg::kBlocks;
  const int nh = blockIdx.x / Cfg::kBlocks;
  const int h = nh % p.H, n = nh / p.H;
  const int hk = h / (p.H / p.Hk);
  const int64_t slot = pool_slot(p.slots, p.num_slots, n);
  if (slot < 0) return;
  const int group = warp * Cfg::kRowsPerWarp + lane / Cfg::kLanes;
  const int col = 4 * (lane % Cfg::kLanes);
  float4* st = reinterpret_cast<float4*>(p.states + (slot * p.H + h) * D * D + (int64_t)group * D + blk * C + col);
  constexpr int kStep = G * D / 4;  // float4s from one of this thread's rows to the next
  float4 S[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) S[i] = __ldcs(st + i * kStep);
  // a slot named by an earlier sample of this call belongs to that sample
  int taken = 0;
  if (p.slots != nullptr)
    for (int i = tid; i < n; i += NT) taken |= p.slots[i] == static_cast<int32_t>(slot);
  const int64_t qrow = (int64_t)n * p.sq + (int64_t)hk * D, krow = (int64_t)n * p.sk + (int64_t)hk * D;
  const float beta = DELTA && p.gated ? load_beta<T>(p, n, h) : 1.f;
  for (int i = tid; i < D; i += NT) {
    s_q[i] = load_f32<T>(p.q, qrow + i);
    float k = load_f32<T>(p.k, krow + i);
    float a = 1.f;
    if (p.g_layout == 1) a = expf(p.g[(int64_t)n * p.H + h]);
    if (p.g_layout == 2) a = expf(p.g[((int64_t)n * p.H + h) * D + i]);
    if (p.g_layout == 3) a = expf(p.g[h]);
    s_a[i] = a;
    if constexpr (DELTA) {
      if (!p.gated && p.beta_layout == 1) k *= sqrtf(load_f32<T>(p.beta, (int64_t)n * p.Hk + hk));
      if (p.beta_layout == 2) k *= sqrtf(load_f32<T>(p.beta, ((int64_t)n * p.Hk + hk) * D + i));
      s_kb[i] = p.erase != nullptr ? k * load_f32<T>(p.erase, ((int64_t)n * p.Hk + hk) * D + i) : k;
    }
    s_k[i] = k;
  }
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = blk * C + col + e;
    v[e] = load_f32<T>(p.v, (int64_t)n * p.sv + (int64_t)h * D + c);
    if (DELTA && p.write != nullptr) v[e] *= load_f32<T>(p.write, ((int64_t)n * p.H + h) * D + c);
  }
  if (__syncthreads_or(taken)) return;
  float o[4] = {0.f, 0.f, 0.f, 0.f}, r[4] = {0.f, 0.f, 0.f, 0.f};
  float kq = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int row = i * G + group;
    const float a = s_a[row], q = s_q[row], k = s_k[row];
    float x[4] = {S[i].x, S[i].y, S[i].z, S[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DELTA) {
        if (p.incoming) o[e] = fmaf(x[e], q, o[e]);
        x[e] *= a;
        r[e] = fmaf(x[e], s_kb[row], r[e]);
      } else {
        x[e] = fmaf(a, x[e], k * v[e]);
      }
      if (!DELTA || !p.incoming) o[e] = fmaf(x[e], q, o[e]);
    }
    if constexpr (DELTA) kq = fmaf(k, q, kq);
    S[i] = make_float4(x[0], x[1], x[2], x[3]);
    if constexpr (!DELTA) __stcs(st + i * kStep, S[i]);
  }
  *reinterpret_cast<float4*>(&s_o[group][col]) = make_float4(o[0], o[1], o[2], o[3]);
  if constexpr (DELTA) {
    *reinterpret_cast<float4*>(&s_r[group][col]) = make_float4(r[0], r[1], r[2], r[3]);
    // rows of this warp's lane groups (each lane of a group holds the group's sum)
    if constexpr (Cfg::kRowsPerWarp == 2) kq += __shfl_xor_sync(0xffffffffu, kq, 16);
    if (lane == 0) s_kq[warp] = kq;
  }
  bool any_odd = false;  // some value of this CTA's is not finite, where its output would show it
  if (DELTA && p.gated) {
    float seen = kq + beta;
#pragma unroll
    for (int e = 0; e < 4; ++e) seen = fmaf(0.f, o[e] + r[e], fmaf(0.f, v[e], seen));
    any_odd = __syncthreads_or(!isfinite(seen));
  } else {
    __syncthreads();
  }
  if constexpr (DELTA) {
    float d[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const float4 x = *reinterpret_cast<const float4*>(&s_r[j][col]);
      d[0] -= x.x;
      d[1] -= x.y;
      d[2] -= x.z;
      d[3] -= x.w;
    }
    if (p.gated) {
#pragma unroll
      for (int e = 0; e < 4; ++e) d[e] *= beta;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float k = s_k[i * G + group];
      __stcs(st + i * kStep, make_float4(fmaf(k, d[0], S[i].x), fmaf(k, d[1], S[i].y), fmaf(k, d[2], S[i].z),
                                  fmaf(k, d[3], S[i].w)));
    }
    bool odd[4] = {};  // outputs that are not finite
    if (group == 0) {
      // o = S~^T q + (k'.q) d for the new state; the incoming one does not know d, which may not be finite
      float all = 0.f;
      if (p.incoming) {
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = 0.f;
      } else {
#pragma unroll
        for (int j = 0; j < Cfg::kWarps; ++j) all += s_kq[j];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < G; ++j) sum += s_o[j][col + e];
        const float out = fmaf(all, d[e], sum);
        odd[e] = !isfinite(out);
        store_f32(static_cast<T*>(p.out), (int64_t)n * p.so + (int64_t)h * D + blk * C + col + e, p.scale * out);
      }
    }
    // A correction or a query that is not finite makes terms of either sign, which k.q and S~^T q do not show: the
    // new state's sum.
    if (any_odd) {
      __syncthreads();
      float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const float k = s_k[i * G + group], q = s_q[i * G + group];
        const float x[4] = {S[i].x, S[i].y, S[i].z, S[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaf(q, fmaf(k, d[e], x[e]), y[e]);
      }
      *reinterpret_cast<float4*>(&s_o[group][col]) = make_float4(y[0], y[1], y[2], y[3]);
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!odd[e]) continue;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < G; ++j) sum += s_o[j][col + e];
        store_f32(static_cast<T*>(p.out), (int64_t)n * p.so + (int64_t)h * D + blk * C + col + e, p.scale * sum);
      }
    }
  } else {
    for (int c = tid; c < C; c += NT) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < G; ++j) sum += s_o[j][c];
      store_f32(static_cast<T*>(p.out), (int64_t)n * p.so + (int64_t)h * D + blk * C + c, p.scale * sum);
    }
  }
}

}  // namespace memt
