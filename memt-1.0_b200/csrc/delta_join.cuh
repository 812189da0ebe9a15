// Few long samples of the gated delta rule, between the two passes over their segments: the state before each segment.
//
// A segment takes the state before it to M S + H, with the matrix M that the rule makes of an identity without values
// and H that it makes of a zero state; the first pass has stored both. The products depend on one another, so a
// (sample, head) state is shared out by value columns: a CTA has 16 of them and walks over the segments, in fp32, S in
// shared memory, each H replaced in place by the state before its segment. All of M goes through every CTA: pieces
// of it are copied ahead of the walk (they do not wait for S) and lie transposed, so that a thread with two rows and
// eight columns of S reads pairs of rows beside its neighbours'. Measured: 2.1 / 4 / 11 us a segment at
// D = 64 / 128 / 256 (2 heads, 16 and 10 segments), bound by the products (16 D^2 in a CTA); more threads that split the sum over keys were 20 to 60
// percent faster for short segments and up to twice as slow behind long ones.
#pragma once

#include "delta_tc.cuh"

namespace memt {

template <int D>
struct DeltaJoinCfg {
  static constexpr int kCols = 16;
  static constexpr int kRows = D == 64 ? 64 : 8192 / D;  // of the transposed M in a piece
  static constexpr int kPiece = kRows * D * 4;
  static constexpr int kStages = 4;
  static constexpr int kOffS = kStages * kPiece;  // two buffers
  static constexpr int kOffBar = kOffS + 2 * D * kCols * 4;
  static constexpr int kSmem = kOffBar + kStages * 8;
};

template <int D>
__global__ void __launch_bounds__(D) delta_join_kernel(const DeltaParams p) {
  using Cfg = DeltaJoinCfg<D>;
  constexpr int C = Cfg::kCols, kPieces = D / Cfg::kRows;
  extern __shared__ __align__(128) unsigned char sm_join[];
  const int tid = threadIdx.x, blk = blockIdx.x % (D / C), nh = blockIdx.x / (D / C), h = nh % p.H, n = nh / p.H;
  int64_t bos, eos;
  int first = 0, count;
  {  // this sample's first segment: every warp sums the samples before it
    for (int m = tid & 31; m < n; m += 32) {
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
  if (count <= 1) return;  // one segment starts from the sample's own state
  const uint32_t base = smem_u32(sm_join), bars = base + Cfg::kOffBar;
  const int pieces = (count - 1) * kPieces;
  auto load = [&](int i) {  // piece i of the walk
    const float* M = p.seg_moves + ((int64_t)(first + i / kPieces) * p.H + h) * D * D;
    const int s = i % Cfg::kStages;
    mbar_expect_tx(bars + 8 * s, Cfg::kPiece);
    bulk_g2s(base + s * Cfg::kPiece, M + i % kPieces * (Cfg::kPiece / 4), Cfg::kPiece, bars + 8 * s);
  };
  if (tid == 0) {
    for (int s = 0; s < Cfg::kStages; ++s) mbar_init(bars + 8 * s, 1);
    mbar_fence_init();
    for (int i = 0; i < Cfg::kStages && i < pieces; ++i) load(i);
  }
  const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n);
  const int r = 2 * (tid % (D / 2)), col = 8 * (tid / (D / 2));
  const int64_t at = (int64_t)r * D + blk * C + col;
  auto read = [&](const float* x, uint64_t (&y)[2][4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(x + (e >> 1) * D + 4 * (e & 1));
      y[e >> 1][2 * (e & 1)] = f.x;
      y[e >> 1][2 * (e & 1) + 1] = f.y;
    }
  };
  auto write = [&](float* x, int row, const uint64_t (&y)[2][4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<ulonglong2*>(x + (e >> 1) * row + 4 * (e & 1)) =
          make_ulonglong2(y[e >> 1][2 * (e & 1)], y[e >> 1][2 * (e & 1) + 1]);
  };
  uint64_t S[2][4] = {}, H[2][4];
  if (p.h0 != nullptr && in_slot >= 0) read(p.h0 + (in_slot * p.H + h) * D * D + at, S);
  read(p.seg_states + ((int64_t)first * p.H + h) * D * D + at, H);
  bool alive = true;
  int i = 0, issued = pieces < Cfg::kStages ? pieces : Cfg::kStages;
  __syncthreads();
  for (int s = 0; s < count; ++s) {
    write(p.seg_states + ((int64_t)(first + s) * p.H + h) * D * D + at, D, S);
    if (s + 1 == count) break;  // the second pass ends with it
    float* shared = reinterpret_cast<float*>(sm_join + Cfg::kOffS) + (s & 1) * D * C;
    write(shared + r * C + col, C, S);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) S[e >> 2][e & 3] = H[e >> 2][e & 3];
    if (s + 2 < count) read(p.seg_states + ((int64_t)(first + s + 1) * p.H + h) * D * D + at, H);
    for (int piece = 0; piece < kPieces; ++piece, ++i) {
      const int stage = i % Cfg::kStages;
      if (alive) alive = mbar_wait_clock(bars + 8 * stage, (i / Cfg::kStages) & 1);
      const float* M = reinterpret_cast<const float*>(sm_join + stage * Cfg::kPiece) + r;
      const float* x = shared + piece * Cfg::kRows * C + col;
#pragma unroll 8
      for (int j = 0; j < Cfg::kRows; ++j) {
        const float2 m = *reinterpret_cast<const float2*>(M + j * D);
        const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(x + j * C);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(x + j * C + 4);
        const uint64_t y[4] = {a.x, a.y, b.x, b.y}, mx = f32x2_splat(m.x), my = f32x2_splat(m.y);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          S[0][q] = fma_f32x2(mx, y[q], S[0][q]);
          S[1][q] = fma_f32x2(my, y[q], S[1][q]);
        }
      }
      __syncthreads();
      if (tid == 0 && alive && i + Cfg::kStages < pieces) {
        load(i + Cfg::kStages);
        issued = i + Cfg::kStages + 1;
      }
    }
    if (!alive) {  // a wait that ran out: nothing more is waited for or loaded, and the caller sees it in the state
#pragma unroll
      for (int e = 0; e < 8; ++e) S[e >> 2][e & 3] = f32x2_splat(__int_as_float(0x7fffffff));
    }
  }
  if (!alive) {
    atomicOr(&g_delta_status, 1);
    if (tid == 0)  // what has been loaded lands before shared memory is released
      for (int j = issued > Cfg::kStages ? issued - Cfg::kStages : 0; j < issued; ++j)
        mbar_wait_clock(bars + 8 * (j % Cfg::kStages), (j / Cfg::kStages) & 1);
  }
}

}  // namespace memt
