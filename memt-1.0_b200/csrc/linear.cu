// memt_linear_attention: argument checks and launch of the causal linear attention.
#include <algorithm>

#include "launch.h"
#include "linear.cuh"
#include "linear_tc.cuh"
#include "overlap.h"

namespace {

using namespace memt;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int D, typename T>
int launch_tokens(const LinearParams& p, cudaStream_t s) {
  using Cfg = LinearTokensCfg<D>;
  const int64_t grid = int64_t(p.N) * p.H * Cfg::kBlocks;
  if (grid > INT32_MAX) return MEMT_ERR_UNSUPPORTED;
  ProfScope prof(kProfLinear, s);
  linear_tokens_kernel<D, T><<<static_cast<unsigned>(grid), Cfg::kThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError());
}

template <typename T>
int launch_tokens(int D, const LinearParams& p, cudaStream_t s) {
  switch (D) {
    case 64: return launch_tokens<64, T>(p, s);
    case 128: return launch_tokens<128, T>(p, s);
    default: return launch_tokens<256, T>(p, s);
  }
}

// Multiprocessors the split is planned for (the workspace size is known without a device).
constexpr int kPlanSms = 148;

// 64-token chunks per segment, or 0: one CTA per (sample, head, value block) walks a whole sample. Few of
// them leave SMs idle for as long as a sample takes: 16 heads of one 65536-token sample 1.51 ms. Segments of a
// mean sample's chunks over the free SMs fill them once (samples of unequal length can make one more each,
// and the second pass then takes a second wave), at the price of a first pass that sums their states (k and
// v are read twice) and a pass that joins them: 0.43 ms. The rule counts samples, not tokens: short samples
// beside a long one can leave it whole. A chunk takes 1.2 / 1.55 / 2.6 us in one CTA at D = 64 / 128 / 256,
// 0.65 of that more in the first pass, and the launches about 18 us. Measured on either side, whole against
// segments in us: 16 heads of one sample, D = 128: 512 tokens 19 / 27, 1024 31 / 30, 2048 55 / 36, 8192
// 203 / 72; of two: 1024 31 / 33, 2048 55 / 45; two segments never pay (four samples: 8192 207 / 207).
int plan_segment_chunks(int64_t N, int64_t L, int64_t H, int D) {
  const int64_t ctas = N * H * (D == 256 ? 2 : 1);
  const int64_t split = kPlanSms / ctas;
  if (split < 3) return 0;
  const int64_t chunks = (L + kTile - 1) / kTile / N;  // of a mean sample
  const double chunk_us = D == 64 ? 1.2 : (D == 128 ? 1.55 : 2.6);
  if (chunks * chunk_us * (1.0 - 1.65 / split) < 18.0) return 0;
  return static_cast<int>((chunks + split - 1) / split);
}
int64_t max_segments(int64_t N, int64_t L, int seg_chunks) { return L / (int64_t(seg_chunks) * kTile) + N; }

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

template <int D, bool OUT>
int launch_pass(const LinearTcParams& P, int64_t units, cudaStream_t s) {
  using Cfg = LinearTcCfg<D>;
  const cudaError_t e = ensure_smem(linear_tc_kernel<D, OUT>, Cfg::kSmem);
  if (e != cudaSuccess) return cuda_status(e);
  const int64_t grid = units * P.p.H * Cfg::kBlocks;
  if (grid > INT32_MAX) return MEMT_ERR_UNSUPPORTED;
  ProfScope prof(kProfLinear, s);
  linear_tc_kernel<D, OUT><<<static_cast<unsigned>(grid), Cfg::kThreads, Cfg::kSmem, s>>>(P);
  return cuda_status(cudaGetLastError());
}

template <int D>
int launch_chunked(const LinearParams& p, void* workspace, cudaStream_t s) {
  using Cfg = LinearTcCfg<D>;
  LinearTcParams P;
  P.p = p;
  const uint64_t rows = static_cast<uint64_t>(p.L);
  cudaError_t e = make_tmap_bf16_2d(&P.q_map, p.q, uint64_t(p.Hk) * D, rows, uint64_t(p.sq) * 2, 64, kTile);
  if (e == cudaSuccess) e = make_tmap_bf16_2d(&P.k_map, p.k, uint64_t(p.Hk) * D, rows, uint64_t(p.sk) * 2, 64, kTile);
  if (e == cudaSuccess) e = make_tmap_bf16_2d(&P.v_map, p.v, uint64_t(p.H) * D, rows, uint64_t(p.sv) * 2, 64, kTile);
  if (e == cudaSuccess)
    e = make_tmap_bf16_2d_sw64(&P.o_map, p.out, uint64_t(p.H) * D, rows, uint64_t(p.so) * 2, Cfg::kOutTokens);
  if (e != cudaSuccess) return cuda_status(e);
  const int seg_chunks = plan_segment_chunks(p.N, p.L, p.H, D);
  if (seg_chunks == 0) {
    // More CTAs than SMs: the longest samples first, so that no SM is left with one at the end (16 samples of
    // 0 to 16384 tokens, 16 heads, d = 128: 617 us in order of the samples, 594 by length). Every CTA ranks
    // the samples for itself, which short or many samples would not repay.
    P.p.by_length = p.N > 1 && p.N <= 32 && int64_t(p.N) * p.H * Cfg::kBlocks > kPlanSms && p.L / p.N >= 1024;
    return launch_pass<D, true>(P, p.only_long > 0 ? p.only_long : p.N, s);
  }
  const int64_t units = max_segments(p.N, p.L, seg_chunks);
  P.p.seg_chunks = seg_chunks;
  P.p.max_segments = static_cast<int32_t>(units);
  P.p.seg_states = static_cast<float*>(workspace);
  P.p.seg_decays = reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) +
                                             align256(size_t(units) * p.H * D * D * sizeof(float)));
  int st = launch_pass<D, false>(P, units, s);
  if (st != MEMT_OK) return st;
  {
    ProfScope prof(kProfLinear, s);
    const unsigned grid = static_cast<unsigned>(p.N * p.H * ((D * D / 4 + 255) / 256));  // N * H < kPlanSms: small
    linear_segments_kernel<<<grid, 256, 0, s>>>(P.p, D);
    st = cuda_status(cudaGetLastError());
    if (st != MEMT_OK) return st;
  }
  return launch_pass<D, true>(P, units, s);
}

int launch_chunked(int D, const LinearParams& p, void* workspace, cudaStream_t s) {
  switch (D) {
    case 64: return launch_chunked<64>(p, workspace, s);
    case 128: return launch_chunked<128>(p, workspace, s);
    default: return launch_chunked<256>(p, workspace, s);
  }
}

// Tokens up to which a bf16 sample runs token by token. Measured, the token kernel alone against chunks alone,
// 16 heads, us: 256 samples at D = 64: 1 token 24 / 149, 16 74 / 154, 24 104 / 152, 32 134 / 152; D = 128: 1 token
// 83 / 201, 8 138 / 201, 12 182 / 203; 64 samples at D = 256: 1 token 96 / 168, 6 137 / 169, 8 156 / 170. The
// chunks' launch that finds no sample costs up to 36 us more (D = 256, 64 samples: 19).
int few_tokens(int D) { return D == 64 ? 24 : (D == 128 ? 8 : 6); }

int check_linear(const memt_linear_attention_args* a) {
  if (a == nullptr || a->struct_size != sizeof(memt_linear_attention_args)) return MEMT_ERR_INVALID_ARGUMENT;
  if (a->num_samples < 1 || a->num_heads < 1 || a->num_key_heads < 1 || a->num_heads % a->num_key_heads != 0 ||
      a->total_tokens < 0 || a->total_tokens > INT32_MAX - 1 || (a->dtype != MEMT_BF16 && a->dtype != MEMT_F32))
    return MEMT_ERR_INVALID_ARGUMENT;
  const int D = a->head_dim;
  if (D != 64 && D != 128 && D != 256) return MEMT_ERR_UNSUPPORTED;
  if (a->cu_seqlens == nullptr || a->final_state == nullptr) return MEMT_ERR_INVALID_ARGUMENT;
  if (a->total_tokens > 0 && (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->out == nullptr))
    return MEMT_ERR_INVALID_ARGUMENT;
  if (a->g_layout != MEMT_GATE_NONE && a->g_layout != MEMT_GATE_PER_HEAD && a->g_layout != MEMT_GATE_CONSTANT)
    return MEMT_ERR_INVALID_ARGUMENT;
  // (an [L, H] tensor without tokens has no address; a constant decay is read whatever the tokens are)
  const bool no_g = a->g_layout == MEMT_GATE_NONE || (a->g_layout == MEMT_GATE_PER_HEAD && a->total_tokens == 0);
  if (a->g == nullptr ? !no_g : a->g_layout == MEMT_GATE_NONE) return MEMT_ERR_INVALID_ARGUMENT;
  const int64_t row = int64_t(a->num_heads) * D, krow = int64_t(a->num_key_heads) * D;
  if (a->q_stride < krow || a->k_stride < krow || a->v_stride < row || a->out_stride < row)
    return MEMT_ERR_INVALID_ARGUMENT;
  if ((a->initial_slots != nullptr && (a->num_initial_slots < 1 || a->initial_state == nullptr)) ||
      (a->final_slots != nullptr && a->num_final_slots < 1))
    return MEMT_ERR_INVALID_ARGUMENT;
  // A sample must not end where another one starts from. Without slots, states are one tensor or apart; pools may
  // share whole states, which the slots then tell apart.
  if (a->initial_state != nullptr) {
    const uintptr_t in = reinterpret_cast<uintptr_t>(a->initial_state);
    const uintptr_t fin = reinterpret_cast<uintptr_t>(a->final_state);
    const uint64_t state = uint64_t(a->num_heads) * D * D * sizeof(float), off = in < fin ? fin - in : in - fin;
    const uint64_t n_in = a->initial_slots != nullptr ? a->num_initial_slots : a->num_samples;
    const uint64_t n_fin = a->final_slots != nullptr ? a->num_final_slots : a->num_samples;
    const bool shared = off < state * (in < fin ? n_in : n_fin);
    const bool pools = a->initial_slots != nullptr || a->final_slots != nullptr;
    if (shared && (pools ? off % state != 0 : off != 0)) return MEMT_ERR_INVALID_ARGUMENT;
  }
  const int64_t vec = a->dtype == MEMT_BF16 ? 8 : 4;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out) ||
      !aligned16(a->initial_state) || !aligned16(a->final_state) || a->q_stride % vec != 0 ||
      a->k_stride % vec != 0 || a->v_stride % vec != 0 || a->out_stride % vec != 0)
    return MEMT_ERR_MISALIGNED;
  return MEMT_OK;
}

// What the call writes, against all that it reads and the rest of what it writes (states may be one tensor).
bool writes_overlap(const memt_linear_attention_args* a, const void* workspace, size_t workspace_bytes) {
  const int64_t size = a->dtype == MEMT_BF16 ? 2 : 4, L = a->total_tokens, N = a->num_samples;
  const int64_t row = int64_t(a->num_heads) * a->head_dim * size, krow = int64_t(a->num_key_heads) * a->head_dim * size;
  const int64_t state = int64_t(a->num_heads) * a->head_dim * a->head_dim * 4;
  const Rows out(a->out, row, a->out_stride * size, L);
  const Rows fin(a->final_state, state * (a->final_slots != nullptr ? a->num_final_slots : N));
  const Rows ws(workspace, static_cast<int64_t>(workspace_bytes));
  const Rows q(a->q, krow, a->q_stride * size, L), k(a->k, krow, a->k_stride * size, L);
  const Rows v(a->v, row, a->v_stride * size, L);
  const Rows g(a->g, int64_t(a->num_heads) * 4 * (a->g_layout == MEMT_GATE_PER_HEAD ? L : 1));
  const Rows cu(a->cu_seqlens, (N + 1) * 4);
  const Rows in(a->initial_state, state * (a->initial_slots != nullptr ? a->num_initial_slots : N));
  const Rows from(a->initial_slots, N * 4), to(a->final_slots, N * 4);
  return overlaps_any(out, {q, k, v, g, cu, in, from, to, fin, ws}) ||
         overlaps_any(fin, {q, k, v, g, cu, from, to, ws}) || overlaps_any(ws, {q, k, v, g, cu, in, from, to});
}

}  // namespace

extern "C" {

size_t memt_linear_attention_workspace_size(int32_t N, int64_t L, int32_t H, int32_t D, int32_t dtype) {
  if (N < 1 || L < 0 || H < 1 || (D != 64 && D != 128 && D != 256)) return 0;
  if (dtype != MEMT_F32 && dtype != MEMT_BF16) return 0;
  const int seg_chunks = dtype == MEMT_BF16 ? plan_segment_chunks(N, L, H, D) : 0;
  if (seg_chunks == 0) return 256;
  const size_t units = static_cast<size_t>(max_segments(N, L, seg_chunks));
  return align256(units * H * D * D * sizeof(float)) + align256(units * H * sizeof(float2));
}

int memt_linear_attention(const memt_linear_attention_args* a, void* workspace, size_t workspace_bytes,
                          memt_stream_t stream) try {
  const int st = check_linear(a);
  if (st != MEMT_OK) return st;
  const size_t need =
      memt_linear_attention_workspace_size(a->num_samples, a->total_tokens, a->num_heads, a->head_dim, a->dtype);
  // (256 stands for none)
  if (need > 256 &&
      (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return MEMT_ERR_WORKSPACE;
  if (writes_overlap(a, need > 256 ? workspace : nullptr, need)) return MEMT_ERR_INVALID_ARGUMENT;
  LinearParams p{};
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
  // Up to 64 tokens a sample in the mean, both kernels run, each for its samples by their own lengths; where no
  // sample is short, the idle launch costs 4 to 11 us of 136 to 206. Above, all samples run in chunks: a short
  // sample's result may then differ in its last bits.
  const int few = few_tokens(a->head_dim);
  if (a->total_tokens <= few) return launch_tokens<__nv_bfloat16>(a->head_dim, p, s);
  p.few = -1;
  if (a->num_samples > 1 && a->total_tokens <= int64_t(64) * a->num_samples) {
    p.few = few;
    // No more than L / (few + 1) samples are longer. Where that is up to half of them, so many CTAs a head look for
    // one each; otherwise every sample has its CTAs, and those of short ones end at once. 256 samples, 16 heads,
    // D = 64: empty CTAs for all 31 us; CTAs that look and find none 7 us for 10 samples, 36 us for 122, 70 us
    // for 248.
    const int64_t most = p.L / (few + 1);
    p.only_long = most <= p.N / 2 ? static_cast<int32_t>(most) : 0;
    const int st_few = launch_tokens<__nv_bfloat16>(a->head_dim, p, s);
    if (st_few != MEMT_OK) return st_few;
  }
  return launch_chunked(a->head_dim, p, workspace, s);
} catch (...) {  // the launch bookkeeping may run out of host memory
  return MEMT_ERR_CUDA;
}

int memt_linear_attention_status(memt_stream_t stream, int32_t* status_out) {
  if (status_out == nullptr) return MEMT_ERR_INVALID_ARGUMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int zero = 0;
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_linear_status, sizeof(v), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_linear_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return cuda_status(e);
  *status_out = v;
  return MEMT_OK;
}

}  // extern "C"
