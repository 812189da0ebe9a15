// Argument checks that the operators over packed prompts share (linear attention, the gated delta rule): their
// argument structs name the same fields.
#pragma once

#include <cstdint>

#include "memt_gdn2.h"
#include "overlap.h"

namespace memt {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename Args>
int check_prompts(const Args* a) {
  if (a == nullptr || a->struct_size != sizeof(Args)) return MEMT_ERR_INVALID_ARGUMENT;
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

// What the call writes, against all that it reads and the rest of what it writes (states may be one
// tensor). `more`: what it reads besides.
template <typename Args>
bool prompts_overlap(const Args* a, const void* workspace, size_t workspace_bytes, const Rows& more = Rows(nullptr, 0)) {
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
  return overlaps_any(out, {q, k, v, g, cu, in, from, to, fin, ws, more}) ||
         overlaps_any(fin, {q, k, v, g, cu, from, to, ws, more}) ||
         overlaps_any(ws, {q, k, v, g, cu, in, from, to, more});
}

}  // namespace memt
