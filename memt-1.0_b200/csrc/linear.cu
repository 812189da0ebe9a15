// memt_linear_attention: argument checks and launch of the causal linear attention.
#include "launch.h"
#include "linear.cuh"

namespace {

using namespace memt;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int D, typename T>
int launch_recurrent_form(const LinearParams& p, cudaStream_t s) {
  constexpr int kBlocks = D / (LinearRecurrentCfg::kCols * LinearRecurrentCfg::kWarps);
  const int64_t grid = int64_t(p.N) * p.H * kBlocks;
  if (grid > INT32_MAX) return MEMT_ERR_UNSUPPORTED;
  ProfScope prof(kProfLinear, s);
  linear_recurrent_kernel<D, T><<<static_cast<unsigned>(grid), LinearRecurrentCfg::kWarps * 32, 0, s>>>(p);
  return cuda_status(cudaGetLastError());
}

template <typename T>
int launch_recurrent_form(int D, const LinearParams& p, cudaStream_t s) {
  switch (D) {
    case 64: return launch_recurrent_form<64, T>(p, s);
    case 128: return launch_recurrent_form<128, T>(p, s);
    default: return launch_recurrent_form<256, T>(p, s);
  }
}

int check_linear(const memt_linear_attention_args* a) {
  if (a == nullptr || a->struct_size != sizeof(memt_linear_attention_args)) return MEMT_ERR_INVALID_ARGUMENT;
  if (a->num_samples < 1 || a->num_heads < 1 || a->num_key_heads < 1 || a->num_heads % a->num_key_heads != 0 ||
      a->total_tokens < 0 || a->total_tokens > INT32_MAX - 1 || (a->dtype != MEMT_BF16 && a->dtype != MEMT_F32))
    return MEMT_ERR_INVALID_ARGUMENT;
  const int D = a->head_dim;
  if (D != 64 && D != 128 && D != 256) return MEMT_ERR_UNSUPPORTED;
  if (a->cu_seqlens == nullptr || a->q == nullptr || a->k == nullptr || a->v == nullptr || a->out == nullptr ||
      a->final_state == nullptr)
    return MEMT_ERR_INVALID_ARGUMENT;
  if (a->g_layout != MEMT_GATE_NONE && a->g_layout != MEMT_GATE_PER_HEAD && a->g_layout != MEMT_GATE_CONSTANT)
    return MEMT_ERR_INVALID_ARGUMENT;
  if ((a->g_layout == MEMT_GATE_NONE) != (a->g == nullptr)) return MEMT_ERR_INVALID_ARGUMENT;
  const int64_t row = int64_t(a->num_heads) * D, krow = int64_t(a->num_key_heads) * D;
  if (a->q_stride < krow || a->k_stride < krow || a->v_stride < row || a->out_stride < row)
    return MEMT_ERR_INVALID_ARGUMENT;
  if ((a->initial_slots != nullptr && (a->num_initial_slots < 1 || a->initial_state == nullptr)) ||
      (a->final_slots != nullptr && a->num_final_slots < 1))
    return MEMT_ERR_INVALID_ARGUMENT;
  const int64_t vec = a->dtype == MEMT_BF16 ? 8 : 4;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out) ||
      !aligned16(a->initial_state) || !aligned16(a->final_state) || a->q_stride % vec != 0 ||
      a->k_stride % vec != 0 || a->v_stride % vec != 0 || a->out_stride % vec != 0)
    return MEMT_ERR_MISALIGNED;
  return MEMT_OK;
}

}  // namespace

extern "C" {

size_t memt_linear_attention_workspace_size(int32_t N, int64_t L, int32_t H, int32_t D, int32_t dtype) {
  if (N < 1 || L < 0 || H < 1 || (D != 64 && D != 128 && D != 256)) return 0;
  if (dtype != MEMT_F32 && dtype != MEMT_BF16) return 0;
  return 256;
}

int memt_linear_attention(const memt_linear_attention_args* a, void* workspace, size_t workspace_bytes,
                          memt_stream_t stream) {
  const int st = check_linear(a);
  if (st != MEMT_OK) return st;
  const size_t need =
      memt_linear_attention_workspace_size(a->num_samples, a->total_tokens, a->num_heads, a->head_dim, a->dtype);
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return MEMT_ERR_WORKSPACE;
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
  return a->dtype == MEMT_F32 ? launch_recurrent_form<float>(a->head_dim, p, s)
                              : launch_recurrent_form<__nv_bfloat16>(a->head_dim, p, s);
}

}  // extern "C"
