// memt_recurrent_step: argument checks and launch of the single-token recurrences (step.cuh).
#include "launch.h"
#include "overlap.h"
#include "step.cuh"

namespace {

using namespace memt;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int D, bool DELTA, typename T>
int launch(const StepParams& p, cudaStream_t s) {
  using Cfg = StepCfg<D>;
  const int64_t grid = int64_t(p.N) * p.H * Cfg::kBlocks;
  if (grid > INT32_MAX) return MEMT_ERR_UNSUPPORTED;
  ProfScope prof(kProfStep, s);
  step_kernel<D, DELTA, T><<<static_cast<unsigned>(grid), Cfg::kThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError());
}

template <int D>
int launch_step(const StepParams& p, bool delta, bool bf16, cudaStream_t s) {
  if (delta) return bf16 ? launch<D, true, __nv_bfloat16>(p, s) : launch<D, true, float>(p, s);
  return bf16 ? launch<D, false, __nv_bfloat16>(p, s) : launch<D, false, float>(p, s);
}

// What the call writes (output rows, states), against all that it reads and each other: several CTAs share
// a head, each reads whole rows of the gates and writes its columns of the output.
bool writes_overlap(const memt_recurrent_step_args* a) {
  const int64_t size = a->dtype == MEMT_BF16 ? 2 : 4, N = a->num_samples, H = a->num_heads, Hk = a->num_key_heads;
  const int64_t D = a->head_dim, row = H * D * size, krow = Hk * D * size;
  const Rows out(a->out, row, a->out_stride * size, N);
  const Rows states(a->states, H * D * D * 4 * (a->slots != nullptr ? a->num_slots : N));
  const Rows q(a->q, krow, a->q_stride * size, N), k(a->k, krow, a->k_stride * size, N);
  const Rows v(a->v, row, a->v_stride * size, N);
  const Rows g(a->g, H * 4 * (a->g_layout == MEMT_GATE_CONSTANT ? 1 : N) * (a->g_layout == MEMT_GATE_PER_CHANNEL ? D : 1));
  const Rows beta(a->beta, N * (a->beta_layout == MEMT_GATE_PER_CHANNEL ? krow
                                : a->beta_layout == MEMT_GATE_PER_VALUE_HEAD ? H * size : Hk * size));
  const Rows erase(a->erase, N * krow), write(a->write, N * row), slots(a->slots, N * 4);
  return overlaps_any(out, {q, k, v, g, beta, erase, write, slots, states}) ||
         overlaps_any(states, {q, k, v, g, beta, erase, write, slots});
}

}  // namespace

extern "C" int memt_recurrent_step(const memt_recurrent_step_args* a, memt_stream_t stream) try {
  if (a == nullptr || a->struct_size != sizeof(memt_recurrent_step_args)) return MEMT_ERR_INVALID_ARGUMENT;
  if (a->rule != MEMT_RULE_LINEAR && a->rule != MEMT_RULE_GDN2 && a->rule != MEMT_RULE_GATED_DELTA) return MEMT_ERR_INVALID_ARGUMENT;
  const bool delta = a->rule != MEMT_RULE_LINEAR, gated = a->rule == MEMT_RULE_GATED_DELTA;
  if (a->num_samples < 0 || a->num_heads < 1 || a->num_key_heads < 1 || a->num_heads % a->num_key_heads != 0 ||
      (a->dtype != MEMT_BF16 && a->dtype != MEMT_F32))
    return MEMT_ERR_INVALID_ARGUMENT;
  const int D = a->head_dim;
  if (D != 64 && D != 128 && D != 256) return MEMT_ERR_UNSUPPORTED;
  if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->states == nullptr || a->out == nullptr)
    return MEMT_ERR_INVALID_ARGUMENT;
  if (a->g_layout < MEMT_GATE_NONE || a->g_layout > MEMT_GATE_CONSTANT ||
      (a->g_layout == MEMT_GATE_NONE) != (a->g == nullptr))
    return MEMT_ERR_INVALID_ARGUMENT;
  if (!delta && (a->g_layout == MEMT_GATE_PER_CHANNEL || a->beta != nullptr || a->erase != nullptr ||
                 a->write != nullptr || a->read_incoming != 0))
    return MEMT_ERR_UNSUPPORTED;
  if (a->beta_layout < MEMT_GATE_NONE || a->beta_layout > MEMT_GATE_PER_VALUE_HEAD ||
      a->beta_layout == MEMT_GATE_CONSTANT ||
      (a->beta_layout == MEMT_GATE_NONE) != (a->beta == nullptr))
    return MEMT_ERR_INVALID_ARGUMENT;
  if (gated ? a->g_layout == MEMT_GATE_PER_CHANNEL || a->beta_layout == MEMT_GATE_PER_CHANNEL ||
                  a->erase != nullptr || a->write != nullptr || a->read_incoming != 0
            : a->beta_layout == MEMT_GATE_PER_VALUE_HEAD)
    return MEMT_ERR_UNSUPPORTED;
  const int64_t row = int64_t(a->num_heads) * D, krow = int64_t(a->num_key_heads) * D;
  if (a->q_stride < krow || a->k_stride < krow || a->v_stride < row || a->out_stride < row)
    return MEMT_ERR_INVALID_ARGUMENT;
  if (a->slots != nullptr && a->num_slots < 1) return MEMT_ERR_INVALID_ARGUMENT;
  if (!aligned16(a->states)) return MEMT_ERR_MISALIGNED;
  if (a->num_samples == 0) return MEMT_OK;
  if (writes_overlap(a)) return MEMT_ERR_INVALID_ARGUMENT;
  StepParams p{};
  p.N = a->num_samples;
  p.H = a->num_heads;
  p.Hk = a->num_key_heads;
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
  p.erase = a->erase;
  p.write = a->write;
  p.scale = a->scale;
  p.states = a->states;
  p.slots = a->slots;
  p.num_slots = a->num_slots;
  p.incoming = a->read_incoming != 0;
  p.gated = gated;
  p.out = a->out;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf16 = a->dtype == MEMT_BF16;
  switch (D) {
    case 64: return launch_step<64>(p, delta, bf16, s);
    case 128: return launch_step<128>(p, delta, bf16, s);
    default: return launch_step<256>(p, delta, bf16, s);
  }
} catch (...) {  // the launch bookkeeping may run out of host memory
  return MEMT_ERR_CUDA;
}
