// What a chunk of the gated delta rule needs of its keys, queries and gates alone, for every (chunk of 64 tokens,
// value head) at once: with G_i the sum of the log decays up to and including token i of the chunk
//     A_ij = beta_i e^{G_i - G_j} k_i.k_j  (j < i),    T = (I + A)^-1,    B_ij = scale e^{G_i - G_j} q_i.k_j  (j <= i)
// T and B leave as two bf16 terms each, in the layout of the operands that the chain of chunks (delta_tc.cuh) multiplies
// by: for each block of 16 columns j the rows from the diagonal block on, in core matrices of 8 rows by 16 bytes, the
// two of 16 columns behind one another. What lies above the diagonal's blocks is neither made nor stored.
//
// One CTA of four warps a unit, six an SM (D = 256: three). K and Q land by TMA. K K^T and Q K^T are on mma.sync (bf16 products, fp32
// sums): two warps each, one the last 16 rows, one the rows before, columns up to the diagonal. The inverse of the unit
// lower triangular I + A is fp32: 16 x 16 blocks by forward substitution, a lane a column, then two doublings
// T_21 = -T_22 (A_21 T_11) with 3xTF32 products (both factors as two terms of 11 bits, 2^-21 of each left out; on
// CUDA cores their reads of shared memory, 16 bytes for 16 additions, bound them). Sums of log decays are formed in 64
// bits and kept as pairs of fp32 numbers, so that their differences are those of the tokens in between whatever
// came before them.
// Measured at 8 x 8192 tokens, 16 heads, D = 128 (16,384 units, 870 MB): 226 us, 3.8 TB/s. Some 7,300 warp instructions
// a unit at 0.48 a cycle and scheduler; of ten resident warps four wait at a barrier between the steps, two for a fixed
// latency. With one term of B
// 219 us; five CTAs an SM (A beside K instead of over it) a twentieth more; one warp a unit, no barriers but 12 warps an
// SM, 300; weights of blocks left of the diagonal as products of a row's and a column's 2 % less at D = 128, 3 % more
// at 64.
#pragma once

#include "delta.cuh"
#include "tc.cuh"
#include "tma.h"

namespace memt {

struct DeltaChunks {
  // bytes of a unit: T's two terms and B's, each for its blocks of columns 64, 48, 32 and 16 rows of 32 bytes
  static constexpr int kTerm = (64 + 48 + 32 + 16) * 32, kBytes = 4 * kTerm;
  // first byte of column block j
  static __host__ __device__ constexpr int block(int j) { return 32 * (64 * j - 8 * j * (j - 1)); }
  // byte of row r, columns col .. col + 7 (col a multiple of 8)
  static __device__ __forceinline__ int at(int r, int col) {
    const int j = col >> 4;
    return block(j) + ((r >> 3) - 2 * j) * 256 + ((col >> 3) & 1) * 128 + (r & 7) * 16;
  }
};
static_assert(DeltaChunks::block(1) == 2048 && DeltaChunks::block(2) == 3584 && DeltaChunks::block(3) == 4608 &&
                  DeltaChunks::block(4) == DeltaChunks::kTerm,
              "column blocks lie behind one another");

// Two bf16 terms of a pair of fp32 numbers: first + second.
__device__ __forceinline__ void split2(uint64_t x, uint32_t& first, uint32_t& second) {
  first = f32x2_to_bf16x2(x);
  second = f32x2_to_bf16x2(sub_f32x2(x, bf16x2_to_f32x2(first)));
}

// bit 0: a wait of the chunked form ran out (memt_gated_delta_status)
static __device__ int g_delta_status;

struct DeltaTcParams {
  CUtensorMap q_map, k_map, v_map;  // bf16 token rows, boxes of 64 channels x 64 tokens
  CUtensorMap o_map;                // boxes of 32 channels x 32 tokens
  DeltaParams p;
};

template <int D>
struct DeltaChunksCfg {
  static constexpr int kThreads = 128;
  // floats per row of A, of the transpose of T's first 32 x 32 block and of that of its third 16 x 16 block: 8 or 24 more
  // than a multiple of 32, for 8-byte reads of fragments without conflicts
  static constexpr int kRow = 72, kRowT = 40, kRowT2 = 24;
  static constexpr uint32_t kOffK = 0, kBytesK = kTile * D * 2;
  static constexpr uint32_t kOffQ = kOffK + kBytesK;
  // A and the inverse's scratch lie over K and Q, which the scores are made of before
  static constexpr uint32_t kOffA = kOffK, kOffT = kOffA + kTile * kRow * 4;
  static constexpr uint32_t kBytesA = (kTile * kRow + 32 * kRowT + 16 * kRowT2) * 4;
  static constexpr uint32_t kOffG = kBytesA > 2 * kBytesK ? (kBytesA + 15) / 16 * 16 : 2 * kBytesK;
  static constexpr size_t kSmem = kOffG + 3 * kTile * 4 + 16 + 1024;
};

template <int D>
__global__ void __launch_bounds__(128, D == 256 ? 3 : 6) delta_chunks_kernel(const __grid_constant__ DeltaTcParams P) {
  using Cfg = DeltaChunksCfg<D>;
  using T16 = __nv_bfloat16;
  constexpr int RL = Cfg::kRow, RT = Cfg::kRowT, RT2 = Cfg::kRowT2;
  constexpr uint32_t kPanel = kTile * 128;
  const DeltaParams& p = P.p;
  extern __shared__ __align__(1024) unsigned char smem_delta_chunks[];
  unsigned char* sm = smem_delta_chunks + ((1024u - (smem_u32(smem_delta_chunks) & 1023u)) & 1023u);
  const int tid = threadIdx.x, lane = tid & 31, iw = __shfl_sync(~0u, tid >> 5, 0);
  const int unit = blockIdx.x / p.H, h = blockIdx.x % p.H, hk = h / (p.H / p.Hk);
  int n, c;
  if (!find_unit(p, unit, n, c)) return;
  int64_t bos, eos;
  sample_range(p, n, bos, eos);
  bos += (int64_t)c * kTile;
  const int len = eos - bos < kTile ? static_cast<int>(eos - bos) : kTile;

  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + Cfg::kOffG + 3 * kTile * 4);
  uint32_t* late = reinterpret_cast<uint32_t*>(bar + 1);  // some thread has waited too long for the tiles
  if (tid == 0) {
    *late = 0;
    mbar_init(smem_u32(bar), 1);
    mbar_fence_init();
    mbar_expect_tx(smem_u32(bar), 2 * Cfg::kBytesK);
    for (int i = 0; i < D / 64; ++i) {
      tma_load_2d(smem_u32(sm + Cfg::kOffK + i * kPanel), &P.k_map, hk * D + 64 * i, static_cast<int>(bos), smem_u32(bar));
      tma_load_2d(smem_u32(sm + Cfg::kOffQ + i * kPanel), &P.q_map, hk * D + 64 * i, static_cast<int>(bos), smem_u32(bar));
    }
  }
  // minus the log2 decay from the chunk's start up to i, as a pair, and beta
  float* gh = reinterpret_cast<float*>(sm + Cfg::kOffG);
  float* gl = gh + kTile;
  float* gb = gl + kTile;
  if (iw == 1) {  // lane l has tokens 2 l and 2 l + 1
    double g[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t t = bos + 2 * lane + e;
      const bool live = 2 * lane + e < len;
      const float x = live ? log_decay(p, t, h) : 0.f;
      // below e^-111 = 2^-160 a decay is a reset in fp32 whatever it multiplies; NaN stays NaN
      g[e] = -1.4426950408889634 * (x < -111.f ? -111.0 : static_cast<double>(x));
      gb[2 * lane + e] = live ? load_beta<T16>(p, t, h) : 0.f;
    }
    double sum = g[0] + g[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += x;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const double G = e == 0 ? sum - g[1] : sum;
      const float hi = static_cast<float>(G);
      gh[2 * lane + e] = hi;
      gl[2 * lane + e] = static_cast<float>(G - static_cast<double>(hi));
    }
  }
  __syncthreads();
  if (!mbar_wait_clock(smem_u32(bar), 0)) *late = 1;  // half a second: goes on with what is there, up to the stores
  if (len < kTile) {  // rows of K behind the sample: zero (those of Q make rows of B that nothing reads)
    const int pieces = (kTile - len) * 8;
    for (int i = tid; i < D / 64 * pieces; i += 128)
      *reinterpret_cast<uint4*>(sm + Cfg::kOffK + i / pieces * kPanel + len * 128 + i % pieces * 16) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }

  // Scores in blocks of 16 x 16: warps 0 and 1 the last 16 rows of K K^T and Q K^T, warps 2 and 3 the rows before
  const bool of_q = iw & 1, last = iw < 2;
  const int fg = lane >> 2, ft = 2 * (lane & 3);
  float acc[6][2][4];  // last: blocks (3, J); else (0, 0), (1, 0), (1, 1), (2, 0), (2, 1), (2, 2)
#pragma unroll
  for (int i = 0; i < 6; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][e][j] = 0.f;
  {
    // rows of 16: pieces (two of rows by two of columns) in the order of an A fragment; a B fragment takes them crosswise
    const int row = lane & 15;
    const uint32_t at = row * 128, flip = row & 7, right = lane >> 4;
    const uint32_t from = smem_u32(sm + (of_q ? Cfg::kOffQ : Cfg::kOffK)) + at, keys = smem_u32(sm + Cfg::kOffK) + at;
    auto mul = [&](float (&x)[2][4], const uint32_t (&a)[4], const uint32_t (&k)[4]) {
      const uint32_t b0[2] = {k[0], k[2]}, b1[2] = {k[1], k[3]};
      mma_bf16_16816(x[0], a, b0);
      mma_bf16_16816(x[1], a, b1);
    };
#pragma unroll 2
    for (int d = 0; d < D / 16; ++d) {
      const uint32_t off = (d >> 2) * kPanel + (((2 * (d & 3) + right) ^ flip) << 4);
      uint32_t k[4][4];
#pragma unroll
      for (int J = 0; J < 3; ++J) ldsm_x4(k[J], keys + off + J * 2048);
      if (last) {
        uint32_t a[4];
        ldsm_x4(k[3], keys + off + 3 * 2048);
        ldsm_x4(a, from + off + 3 * 2048);
#pragma unroll
        for (int J = 0; J < 4; ++J) mul(acc[J], a, k[J]);
      } else {
#pragma unroll
        for (int m = 0; m < 3; ++m) {
          uint32_t a[4];
          ldsm_x4(a, from + off + m * 2048);
#pragma unroll
          for (int J = 0; J <= m; ++J) mul(acc[m * (m + 1) / 2 + J], a, k[J]);
        }
      }
    }
  }
  __syncthreads();  // A lies over K and Q
  float* A = reinterpret_cast<float*>(sm + Cfg::kOffA);
  float* TT = reinterpret_cast<float*>(sm + Cfg::kOffT);
  float* T2 = TT + 32 * RT;
  unsigned char* out = static_cast<unsigned char*>(p.chunks) + ((int64_t)unit * p.H + h) * DeltaChunks::kBytes;
  // A_ij or B_ij of one block: decays, and beta of the row or the scale; masked by selection
  auto weigh = [&](float (&acc)[2][4], int m, int J) {
    const int r0 = 16 * m + fg;
    const float h0 = -gh[r0], l0 = -gl[r0], h1 = -gh[r0 + 8], l1 = -gl[r0 + 8];
    const float f0 = of_q ? p.scale : gb[r0], f1 = of_q ? p.scale : gb[r0 + 8];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = 16 * J + 8 * e + ft;
      const float2 hj = *reinterpret_cast<const float2*>(gh + col), lj = *reinterpret_cast<const float2*>(gl + col);
      float (&x)[4] = acc[e];
      x[0] *= f0 * fast_exp2((h0 + hj.x) + (l0 + lj.x));
      x[1] *= f0 * fast_exp2((h0 + hj.y) + (l0 + lj.y));
      x[2] *= f1 * fast_exp2((h1 + hj.x) + (l1 + lj.x));
      x[3] *= f1 * fast_exp2((h1 + hj.y) + (l1 + lj.y));
      if (J == m) {
        const int most = of_q ? fg : fg - 1, cc = 8 * e + ft;
        if (cc > most) x[0] = 0.f;
        if (cc + 1 > most) x[1] = 0.f;
        if (cc > most + 8) x[2] = 0.f;
        if (cc + 1 > most + 8) x[3] = 0.f;
      }
      if (of_q) {
        uint32_t* to = reinterpret_cast<uint32_t*>(out + 2 * DeltaChunks::kTerm + DeltaChunks::at(16 * m, 16 * J + 8 * e) +
                                                   fg * 16 + ft * 2);
        constexpr int kNext = DeltaChunks::kTerm / 4;
        split2(f32x2_pack(x[0], x[1]), to[0], to[kNext]);
        split2(f32x2_pack(x[2], x[3]), to[64], to[kNext + 64]);  // eight rows on
      } else {
        *reinterpret_cast<float2*>(A + r0 * RL + col) = make_float2(x[0], x[1]);
        *reinterpret_cast<float2*>(A + (r0 + 8) * RL + col) = make_float2(x[2], x[3]);
      }
    }
  };
  if (last) {
#pragma unroll
    for (int J = 0; J < 4; ++J) weigh(acc[J], 3, J);
  } else {
#pragma unroll
    for (int m = 0; m < 3; ++m)
#pragma unroll
      for (int J = 0; J <= m; ++J) weigh(acc[m * (m + 1) / 2 + J], m, J);
  }
  __syncthreads();

  // The inverse in place of A. A product takes its left factor by rows and its right one by columns, as its transpose: TT
  // is that of T's first 32 x 32 block, T2 of its third 16 x 16 block; a product's, YT, lies in the unused quarter of A
  // right of the diagonal.
  float* YT = A + 32;  // rows 0 .. 31
  auto row4 = [](const float* x) { return *reinterpret_cast<const float4*>(x); };
  auto terms = [](const float* x, uint32_t (&hi)[2], uint32_t (&lo)[2]) {  // of two values
    const float2 v = *reinterpret_cast<const float2*>(x);
    hi[0] = __float_as_uint(v.x) & 0xffffe000u;
    hi[1] = __float_as_uint(v.y) & 0xffffe000u;
    lo[0] = __float_as_uint(v.x - __uint_as_float(hi[0]));
    lo[1] = __float_as_uint(v.y - __uint_as_float(hi[1]));
  };
  // y[j] = 16 rows at a (k contiguous) times the columns 8 j .. of b (rows SB apart, k contiguous), k0 <= k < k1; the
  // sum's index is permuted within a step of 8, for both factors alike
  auto product = [&](const float* a, const float* b, int SB, int k0, int k1, auto& y) {
    constexpr int NJ = std::extent<std::remove_reference_t<decltype(y)>>::value;
#pragma unroll
    for (int j = 0; j < NJ; ++j) y[j][0] = y[j][1] = y[j][2] = y[j][3] = 0.f;
#pragma unroll 1
    for (int k = k0; k < k1; k += 8) {
      uint32_t h0[2], l0[2], h1[2], l1[2];
      terms(a + fg * RL + k + ft, h0, l0);
      terms(a + (fg + 8) * RL + k + ft, h1, l1);
      const uint32_t ah[4] = {h0[0], h1[0], h0[1], h1[1]}, al[4] = {l0[0], l1[0], l0[1], l1[1]};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        uint32_t bh[2], bl[2];
        terms(b + (8 * j + fg) * SB + k + ft, bh, bl);
        mma_tf32_1688(y[j], al, bh);
        mma_tf32_1688(y[j], ah, bl);
        mma_tf32_1688(y[j], ah, bh);
      }
    }
  };
  // the transpose of a product's 8 columns from n on
  auto put_t = [&](float* t, int stride, int n, const float (&y)[4], float sign) {
    t[(n + ft) * stride + fg] = sign * y[0];
    t[(n + ft + 1) * stride + fg] = sign * y[1];
    t[(n + ft) * stride + fg + 8] = sign * y[2];
    t[(n + ft + 1) * stride + fg + 8] = sign * y[3];
  };
  auto put = [&](float* x, const float (&y)[4], float sign) {
    *reinterpret_cast<float2*>(x + fg * RL + ft) = make_float2(sign * y[0], sign * y[1]);
    *reinterpret_cast<float2*>(x + (fg + 8) * RL + ft) = make_float2(sign * y[2], sign * y[3]);
  };
  if (iw < 2) {  // 16 x 16 blocks on the diagonal, two a warp: a lane solves for one column,
                 // x_i = [i = column] - sum_{m < i} A_im x_m
    const int b16 = 2 * iw + (lane >> 4), col = lane & 15;
    float* blk = A + 16 * b16 * (RL + 1);
    float x[16];
    x[0] = col == 0 ? 1.f : 0.f;
#pragma unroll
    for (int i = 1; i < 16; ++i) {
      float sum[2] = {i == col ? 1.f : 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < i; m += 4) {
        const float4 f = row4(blk + i * RL + m);
        const float as[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (m + e < i) sum[e & 1] = fmaf(-as[e], x[m + e], sum[e & 1]);
      }
      x[i] = sum[0] + sum[1];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) blk[i * RL + col] = x[i];
    if (b16 < 3) {  // the transpose
      float* t = b16 < 2 ? TT + (16 * b16 + col) * RT + 16 * b16 : T2 + col * RT2;
#pragma unroll
      for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(t + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
  }
  __syncthreads();
  {  // two 32 x 32 blocks: T_21 = -T_22 (A_21 T_11), each by two warps, 8 columns from n on each
    float* blk = A + 32 * (iw >> 1) * (RL + 1);
    const int n8 = 8 * (iw & 1);
    float y[1][4];
    if (iw < 2) product(blk + 16 * RL, TT + n8 * RT, RT, n8, 16, y);
    else product(blk + 16 * RL, T2 + n8 * RT2, RT2, n8, 16, y);
    put_t(YT, RL, 8 * iw, y[0], 1.f);
    __syncthreads();  // (both warps of a pair have read A_21)
    product(blk + 16 * (RL + 1), YT + 8 * iw * RL, RL, 0, 16, y);
    put(blk + 16 * RL + n8, y[0], -1.f);
    if (iw < 2) put_t(TT + 16, RT, n8, y[0], -1.f);
  }
  __syncthreads();
  {  // the 64 x 64 block: 16 rows from m on by 16 columns from n on each
    const int m = 16 * (iw >> 1), n16 = 16 * (iw & 1);
    float y[2][4];
    product(A + (32 + m) * RL, TT + n16 * RT, RT, n16, 32, y);  // T_11 is zero above its diagonal
    put_t(YT + m, RL, n16, y[0], 1.f);
    put_t(YT + m, RL, n16 + 8, y[1], 1.f);
    __syncthreads();
    product(A + (32 + m) * RL + 32, YT + n16 * RL, RL, 0, m + 16, y);  // and so is T_22
    put(A + (32 + m) * RL + n16, y[0], -1.f);
    put(A + (32 + m) * RL + n16 + 8, y[1], -1.f);
  }
  __syncthreads();
  if (*late != 0) {
    // T as NaN: every correction of the chunk and with them all columns of the state become NaN, which the chain makes again
    // token by token, without T and B (in a first pass over segments the state stays NaN). The tiles land before
    // shared memory is released.
    const uint4 nan = make_uint4(0x7fff7fff, 0x7fff7fff, 0x7fff7fff, 0x7fff7fff);
    for (int i = tid; i < 2 * DeltaChunks::kTerm / 16; i += Cfg::kThreads) reinterpret_cast<uint4*>(out)[i] = nan;
    if (tid == 0) {
      atomicOr(&g_delta_status, 1);
      mbar_wait_clock(smem_u32(bar), 0);
    }
    return;
  }
  // two bf16 terms, eight columns at a time: warp m the rows 16 m on, up to column 16 m + 15
#pragma unroll 1
  for (int i = 0; i <= iw; ++i) {
    const int r = 16 * iw + (lane >> 1), col = 16 * i + 8 * (lane & 1);
    const float4 lo4 = row4(A + r * RL + col), hi4 = row4(A + r * RL + col + 4);
    uint32_t u[4], v[4];
    split2(f32x2_pack(lo4.x, lo4.y), u[0], v[0]);
    split2(f32x2_pack(lo4.z, lo4.w), u[1], v[1]);
    split2(f32x2_pack(hi4.x, hi4.y), u[2], v[2]);
    split2(f32x2_pack(hi4.z, hi4.w), u[3], v[3]);
    const int at = DeltaChunks::at(r, col);
    *reinterpret_cast<uint4*>(out + at) = make_uint4(u[0], u[1], u[2], u[3]);
    *reinterpret_cast<uint4*>(out + DeltaChunks::kTerm + at) = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

}  // namespace memt
