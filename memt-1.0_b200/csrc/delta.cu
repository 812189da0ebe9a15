// memt_gated_delta: argument checks and launch of the gated delta rule over prompts.
#include <algorithm>

#include "delta.cuh"
#include "delta_join.cuh"
#include "launch.h"
#include "prompts.h"

namespace {

using namespace memt;

// Columns (samples x heads x D) up to which a warp has 8 instead of 16 of them: half the work between the sums over rows,
// which is what a token waits for, but more warps that load its row. 500 tokens, fp32, us with 8 / 16 columns:
// D = 64: 8 heads 162 / 193, 192 218 / 242, 256 265 / 242; D = 128: 8 heads 201 / 275, 96 301 / 344, 128 377 / 347.
constexpr int64_t kFewColumns = 12288;

template <int D, typename T, int CG>
int launch_tokens(const DeltaParams& p, cudaStream_t s) {
  using Cfg = DeltaTokensCfg<D, CG>;
  const int64_t grid = int64_t(p.N) * p.H * Cfg::kBlocks;
  ProfScope prof(kProfLinear, s);
  delta_tokens_kernel<D, T, CG><<<static_cast<unsigned>(grid), Cfg::kThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError());
}

template <int D, typename T>
int launch_tokens(const DeltaParams& p, cudaStream_t s) {
  if constexpr (D < 256) {
    if (int64_t(p.N) * p.H * D <= kFewColumns) return launch_tokens<D, T, 2>(p, s);
  }
  return launch_tokens<D, T, D == 256 ? 2 : 4>(p, s);
}

template <typename T>
int launch_tokens(int D, const DeltaParams& p, cudaStream_t s) {
  switch (D) {
    case 64: return launch_tokens<64, T>(p, s);
    case 128: return launch_tokens<128, T>(p, s);
    default: return launch_tokens<256, T>(p, s);
  }
}

// Multiprocessors the calls are planned for (the workspace size is known without a device).
constexpr int kPlanSms = 148;

// 64-token chunks per segment, or 0: one CTA per (sample, head, value block) walks a whole sample. Few of them leave
// SMs idle for as long as a sample takes. With S segments a sample, a first pass goes over all but the last of them twice
// (once for what they add to a zero state, once for what they make of an identity), a kernel joins them one after the other,
// and a second pass over all makes the outputs. Measured at D = 64 / 128 / 256: a chunk of a whole sample takes
// 1.9 / 2.4 / 5.5 us, 0.85 of it in a wave of the first pass, 1.25 in a full wave of the second; a segment's join
// 2.1 / 4 / 11 (the rule counts 8 for the last); a start of a wave some 6. Samples of unequal length can make one segment more each.
// The rule counts samples, not tokens: short samples beside a long one can leave it whole.
int plan_segment_chunks(int64_t N, int64_t L, int64_t H, int D) {
  const int64_t ctas = N * H * (D == 256 ? 2 : 1), chunks = (L + kTile - 1) / kTile / N;  // of a mean sample
  if (ctas * 2 > kPlanSms) return 0;
  const double chunk_us = D == 64 ? 1.9 : (D == 128 ? 2.4 : 5.5), join_us = D == 64 ? 2.1 : (D == 128 ? 3.7 : 8);
  auto waves = [](int64_t n) { return static_cast<double>((n + kPlanSms - 1) / kPlanSms); };
  const double joins = waves(N * H * (D / 16)) * join_us;
  int64_t best = 1;
  double best_us = chunks * chunk_us + 6;
  for (int64_t S = 2; S <= 32 && S <= chunks; ++S) {
    const double run = ((chunks + S - 1) / S) * chunk_us + 6;
    const double us = (0.85 * waves(2 * ctas * (S - 1)) + 1.25 * waves(ctas * S)) * run + S * joins + 15;
    if (us < 0.95 * best_us) {
      best_us = us;
      best = S;
    }
  }
  return best == 1 ? 0 : static_cast<int>((chunks + best - 1) / best);
}
int64_t max_segments(int64_t N, int64_t L, int seg_chunks) { return L / (int64_t(seg_chunks) * kTile) + N; }

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Tokens up to which a bf16 sample runs token by token. Measured, the token kernel alone against chunks alone, 16 heads,
// us: 256 samples at D = 64: 8 tokens 95 / 342, 32 264 / 356, 48 349 / 363; D = 128: 8 tokens 211 / 455, 20 427 / 459, 24
// 498 / 459; 64 samples at D = 256: 6 tokens 209 / 351, 12 298 / 355, 16 361 / 356. (The token kernel's times include
// launches for chunks that find no sample.)
int few_tokens(int D) { return D == 64 ? 40 : (D == 128 ? 20 : 14); }

// Whether both forms run, each for its samples by their own lengths: up to 64 tokens a sample in the mean.
bool mixed(int64_t N, int64_t L) { return N > 1 && L <= 64 * N; }

// chunks of 64 tokens that the samples that go in chunks can have between them
int64_t max_units(int64_t N, int64_t L, int D) {
  const int64_t samples = mixed(N, L) ? std::min(N, L / (few_tokens(D) + 1)) : N;
  return L / kTile + samples;
}

size_t units_bytes(int64_t N, int64_t L, int64_t H, int D) {
  return align256(size_t(max_units(N, L, D)) * H * DeltaChunks::kBytes);
}

// Tables of a call of many samples (delta_plan_kernel), behind the units: the bytes of all and of each.
struct Tables {
  size_t units, first, longs;
  Tables(int64_t N, int64_t L, int D) : units(0), first(0), longs(0) {
    if (N <= 32) return;  // a warp finds its sample at once
    units = align256(size_t(max_units(N, L, D)) * sizeof(int2));
    first = align256(size_t(N + 1) * sizeof(int32_t));
    longs = align256(size_t(L / (few_tokens(D) + 1)) * sizeof(int32_t));
  }
  size_t bytes() const { return units + first + longs; }
};

// Whether a launch of the call could have more CTAs than a grid holds (at most eight a unit or sample and head: some 10^10
// tokens and heads, more than memory does).
bool too_large(int64_t N, int64_t L, int64_t H, int D) {
  return double(std::max(max_units(N, L, D), N)) * double(H) * 8 > INT32_MAX;
}

template <int D, bool OUT>
int launch_pass(const DeltaTcParams& P, int64_t units, cudaStream_t s) {
  using Cfg = DeltaTcCfg<D>;
  const cudaError_t e = ensure_smem(delta_tc_kernel<D, OUT>, Cfg::kSmem);
  if (e != cudaSuccess) return cuda_status(e);
  const int64_t grid = units * P.p.H * Cfg::kBlocks * (OUT ? 1 : 2);
  ProfScope prof(kProfLinear, s);
  delta_tc_kernel<D, OUT><<<static_cast<unsigned>(grid), Cfg::kThreads, Cfg::kSmem, s>>>(P);
  return cuda_status(cudaGetLastError());
}

template <int D>
int launch_chunked(const DeltaParams& p, cudaStream_t s) {
  using Pre = DeltaChunksCfg<D>;
  DeltaTcParams P;
  P.p = p;
  const uint64_t rows = static_cast<uint64_t>(p.L);
  cudaError_t e = make_tmap_bf16_2d(&P.q_map, p.q, uint64_t(p.Hk) * D, rows, uint64_t(p.sq) * 2, 64, kTile);
  if (e == cudaSuccess) e = make_tmap_bf16_2d(&P.k_map, p.k, uint64_t(p.Hk) * D, rows, uint64_t(p.sk) * 2, 64, kTile);
  if (e == cudaSuccess) e = make_tmap_bf16_2d(&P.v_map, p.v, uint64_t(p.H) * D, rows, uint64_t(p.sv) * 2, 64, kTile);
  if (e == cudaSuccess) e = make_tmap_bf16_2d_sw64(&P.o_map, p.out, uint64_t(p.H) * D, rows, uint64_t(p.so) * 2, 32);
  if (e == cudaSuccess) e = ensure_smem(delta_chunks_kernel<D>, Pre::kSmem);
  if (e != cudaSuccess) return cuda_status(e);
  const int64_t units = p.max_units * int64_t(p.H);
  {
    ProfScope prof(kProfLinear, s);
    delta_chunks_kernel<D><<<static_cast<unsigned>(units), Pre::kThreads, Pre::kSmem, s>>>(P);
    const int st = cuda_status(cudaGetLastError());
    if (st != MEMT_OK) return st;
  }
  if (p.seg_chunks == 0) {
    // More CTAs than SMs: the longest samples first, so that no SM is left with one at the end.
    P.p.by_length = p.N > 1 && p.N <= 32 && int64_t(p.N) * p.H * DeltaTcCfg<D>::kBlocks > kPlanSms && p.L / p.N >= 1024;
    return launch_pass<D, true>(P, p.only_long > 0 ? p.only_long : p.N, s);
  }
  int st = launch_pass<D, false>(P, p.max_segments, s);
  if (st != MEMT_OK) return st;
  {
    using Join = DeltaJoinCfg<D>;
    e = ensure_smem(delta_join_kernel<D>, Join::kSmem);
    if (e != cudaSuccess) return cuda_status(e);
    ProfScope prof(kProfLinear, s);
    const int grid = p.N * p.H * (D / Join::kCols);  // (N H <= kPlanSms)
    delta_join_kernel<D><<<grid, D, Join::kSmem, s>>>(P.p);
    st = cuda_status(cudaGetLastError());
    if (st != MEMT_OK) return st;
  }
  return launch_pass<D, true>(P, p.max_segments, s);
}

int launch_chunked(int D, const DeltaParams& p, cudaStream_t s) {
  switch (D) {
    case 64: return launch_chunked<64>(p, s);
    case 128: return launch_chunked<128>(p, s);
    default: return launch_chunked<256>(p, s);
  }
}

int check_delta(const memt_gated_delta_args* a) {
  const int st = check_prompts(a);
  if (st != MEMT_OK) return st;
  if (a->beta_layout != MEMT_GATE_NONE && a->beta_layout != MEMT_GATE_PER_HEAD &&
      a->beta_layout != MEMT_GATE_PER_VALUE_HEAD)
    return MEMT_ERR_INVALID_ARGUMENT;
  // (a tensor without tokens has no address)
  if (a->beta == nullptr ? a->beta_layout != MEMT_GATE_NONE && a->total_tokens > 0 : a->beta_layout == MEMT_GATE_NONE)
    return MEMT_ERR_INVALID_ARGUMENT;
  return MEMT_OK;
}

}  // namespace

extern "C" {

size_t memt_gated_delta_workspace_size(int32_t N, int64_t L, int32_t H, int32_t D, int32_t dtype) {
  if (N < 1 || L < 0 || H < 1 || (D != 64 && D != 128 && D != 256)) return 0;
  if ((dtype != MEMT_F32 && dtype != MEMT_BF16) || too_large(N, L, H, D)) return 0;
  if (dtype == MEMT_F32 || L <= few_tokens(D)) return 256;  // token by token
  const int seg_chunks = mixed(N, L) ? 0 : plan_segment_chunks(N, L, H, D);
  const size_t states =
      seg_chunks == 0 ? 0 : align256(size_t(max_segments(N, L, seg_chunks)) * H * D * D * sizeof(float));
  return units_bytes(N, L, H, D) + Tables(N, L, D).bytes() + 2 * states;
}

int memt_gated_delta(const memt_gated_delta_args* a, void* workspace, size_t workspace_bytes,
                     memt_stream_t stream) try {
  const int st = check_delta(a);
  if (st != MEMT_OK) return st;
  if (too_large(a->num_samples, a->total_tokens, a->num_heads, a->head_dim)) return MEMT_ERR_UNSUPPORTED;
  const size_t need =
      memt_gated_delta_workspace_size(a->num_samples, a->total_tokens, a->num_heads, a->head_dim, a->dtype);
  // (256 stands for none)
  if (need > 256 &&
      (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return MEMT_ERR_WORKSPACE;
  const int64_t size = a->dtype == MEMT_BF16 ? 2 : 4;
  const int64_t gates = a->beta_layout == MEMT_GATE_PER_HEAD ? a->num_key_heads : a->num_heads;
  if (prompts_overlap(a, need > 256 ? workspace : nullptr, need, Rows(a->beta, a->total_tokens * gates * size)))
    return MEMT_ERR_INVALID_ARGUMENT;
  DeltaParams p{};
  p.N = a->num_samples;
  p.H = a->num_heads;
  p.Hk = a->num_key_heads;
  p.L = a->total_tokens;
  p.cu = a->cu_seqlens;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.sq = a->q_stride;
  p.sk = a->k_stride;
  p.sv = a->v_stride;
  p.so = a->out_stride;
  p.g = a->g;
  p.g_layout = a->g_layout;
  p.beta = a->beta;
  p.beta_layout = a->beta_layout;
  p.scale = a->scale;
  p.out = a->out;
  p.h0 = a->initial_state;
  p.ht = a->final_state;
  p.slots_in = a->initial_slots;
  p.num_in = a->num_initial_slots;
  p.slots_out = a->final_slots;
  p.num_out = a->num_final_slots;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // fp32, and calls without tokens, which only copy the states: all samples token by token
  p.few = INT32_MAX;
  if (a->dtype == MEMT_F32 || a->total_tokens == 0) return launch_tokens<float>(a->head_dim, p, s);
  const int few = few_tokens(a->head_dim);
  if (a->total_tokens <= few) return launch_tokens<__nv_bfloat16>(a->head_dim, p, s);
  const int D = a->head_dim;
  const bool both = mixed(p.N, p.L);
  const int64_t most = p.L / (few + 1);  // samples of more than `few` tokens, unless offsets overlap
  p.few = both ? few : -1;
  p.only_long = both && most <= p.N / 2 ? static_cast<int32_t>(most) : 0;
  p.max_units = static_cast<int32_t>(max_units(p.N, p.L, D));
  unsigned char* at = static_cast<unsigned char*>(workspace);
  p.chunks = at;
  at += units_bytes(p.N, p.L, p.H, D);
  const Tables tables(p.N, p.L, D);
  if (tables.bytes() > 0) {
    p.unit_table = reinterpret_cast<int2*>(at);
    p.first_unit = reinterpret_cast<int32_t*>(at + tables.units);
    p.longs = reinterpret_cast<int32_t*>(at + tables.units + tables.first);
    at += tables.bytes();
    ProfScope prof(kProfLinear, s);
    delta_plan_kernel<<<1, kPlanThreads, 0, s>>>(p, p.only_long);
    const int st_plan = cuda_status(cudaGetLastError());
    if (st_plan != MEMT_OK) return st_plan;
  }
  if (both) {
    const int st_few = launch_tokens<__nv_bfloat16>(D, p, s);
    if (st_few != MEMT_OK) return st_few;
  }
  p.seg_chunks = mixed(p.N, p.L) ? 0 : plan_segment_chunks(p.N, p.L, p.H, D);
  if (p.seg_chunks > 0) {
    const int64_t segments = max_segments(p.N, p.L, p.seg_chunks);
    p.max_segments = static_cast<int32_t>(segments);
    p.seg_states = reinterpret_cast<float*>(at);
    p.seg_moves = reinterpret_cast<float*>(at + align256(size_t(segments) * p.H * D * D * sizeof(float)));
  }
  return launch_chunked(D, p, s);
} catch (...) {  // the launch bookkeeping may run out of host memory
  return MEMT_ERR_CUDA;
}

int memt_gated_delta_status(memt_stream_t stream, int32_t* status_out) {
  if (status_out == nullptr) return MEMT_ERR_INVALID_ARGUMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int zero = 0;
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_delta_status, sizeof(v), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_delta_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return cuda_status(e);
  *status_out = v;
  return MEMT_OK;
}

}  // extern "C"
