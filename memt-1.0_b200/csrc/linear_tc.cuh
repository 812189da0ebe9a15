// Causal linear attention with a decay for each head, in chunks of 64 tokens on tcgen05 tensor
// cores: one CTA per (sample, head, block of up to 128 values), the chunks of a sample in order.
//
// With G_i the sum of the log decays of a chunk's tokens up to and including i, R_j the sum over
// the tokens behind j and S the state before the chunk:
//     o_i = scale [ e^{G_i} S^T q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j ]
//     S'  = e^{G_63} S + sum_j (e^{R_j} k_j) v_j^T
// Everything is computed transposed, so that the value index is the tensor-memory lane:
//     Sc   = Q K^T              M = 64 tokens i, N = 64 tokens j, K = D
//     Y^T  = V^T P^T            M = 128 values, N = 64 tokens i, K = 64 tokens j, P = masked, decayed Sc
//     X^T  = bf16(S)^T Q^T      M = 128 values, N = 64 tokens, K = D, A operand in tensor memory
//     U^T  = V^T (e^R K)        M = 128 values, N = D keys, K = 64 tokens, three times (below)
// Q, K and V tiles arrive by TMA with the 128-byte swizzle and are used in place: Q and K as
// K-major operands, V as the MN-major A operand, e^R K in K's own layout as the MN-major B operand.
//
// Precision. The state is fp32 in registers. e^R K is not rounded to bf16 but split into three bf16
// terms (8 bits each), so that the sum over a chunk is an fp32 sum and the final state is what the
// fp32 recurrence gives (measured 1e-7 relative; one bf16 term leaves 1e-3, two 2e-6). The chunk's
// decay is applied as a pair of fp32 numbers: one number, its rounding repeated for every chunk of a
// constant decay, would drift by 2^-25 a chunk. Scores P and the copy of the state that X reads are
// bf16 (2^-9 relative each), as is the output; no other value is rounded below fp32.
// Decay weights never come from differences of long sums: P's weight is the product of the decay from
// its row's 16-token block start, of whole blocks between, and to its column's block end; inside a
// block of 16 it is one difference. So every factor is <= 1 for any decay, a reset (e^g = 0) included.
//
// What bounds it: 64 tokens of Q, K, V and O are 8 x 64 D bytes, 2.5k cycles of an SM's share of
// HBM at D = 128; the MMAs take 1.4k, the 16 worker warps about 2k issue slots a scheduler.
// Roles: warps 0-15 work, warp 16 issues MMAs, warp 17 loads tiles and makes the decay tables.
// A worker's chunk: fold U of the previous chunk into its registers and write bf16(S); P from Sc;
// the split e^R K; the output from X and Y. MMAs of a chunk: X, Y, U, then Sc of the next one. The
// only wait between chunks is U -> state -> X; loads run a stage ahead.
// The last chunk of a sample is padded with whatever the TMA brings (the next sample's rows, or
// zeros past the last row): those columns of P are masked by selection, those rows of e^R K and of
// V's tile are set to zero (0 x NaN would not be), and those tokens' outputs are not stored.
// At D = 64 the 64 values fill half of the 128 lanes; V's tile is loaded twice so that lanes 64-127
// repeat lanes 0-63 and share their output stores.
// Every wait is bounded: a thread whose wait runs out flags it and stops waiting, the control warps
// drain what they have in flight, and the final state stays unwritten.
#pragma once

#include "linear.cuh"
#include "tc.cuh"
#include "tma.h"

namespace memt {

struct LinearTcParams {
  CUtensorMap q_map, k_map, v_map;  // bf16 token rows, boxes of 64 channels x 64 tokens
  LinearParams p;
};

// bit 0: a wait of linear_tc_kernel ran out (memt_linear_attention_status)
static __device__ int g_linear_status;

template <int D_>
struct LinearTcCfg {
  static constexpr int D = D_;
  static constexpr int kVB = D < 128 ? D : 128;     // values per CTA
  static constexpr int kBlocks = D / kVB;           // CTAs per (sample, head)
  static constexpr int kWorkers = 16;
  static constexpr int kThreads = (kWorkers + 2) * 32;
  static constexpr int kPanelsU = D < 128 ? 1 : D / 128;  // U and e^R K go in panels of up to 128 keys
  static constexpr int kPanelKeys = D / kPanelsU;
  static constexpr int kKeysPerThread = kPanelKeys / 4;   // state columns per thread and panel
  static constexpr int kStagesQK = D == 256 ? 1 : (D == 128 ? 3 : 4);
  static constexpr int kStagesV = D == 256 ? 2 : kStagesQK;
  static constexpr uint32_t kPanel = kTile * 128;         // 64 x 64 bf16: 8 KB
  static constexpr uint32_t kBytesQK = kTile * D * 2;
  static constexpr uint32_t kBytesV = kTile * 128 * 2;    // 128 lanes of values, also at D = 64
  static constexpr uint32_t kOffQ = 0;
  static constexpr uint32_t kOffK = kOffQ + kStagesQK * kBytesQK;
  static constexpr uint32_t kOffV = kOffK + kStagesQK * kBytesQK;
  static constexpr uint32_t kOffKt = kOffV + kStagesV * kBytesV;  // three terms, [term][D / 64] panels
  static constexpr uint32_t kOffP = kOffKt + 3 * kBytesQK;
  static constexpr uint32_t kOffTab = kOffP + kPanel;
  static constexpr uint32_t kTabFloats = 5 * kTile + 16 + 4 + 12;  // 352 floats
  static constexpr uint32_t kOffBar = kOffTab + 2 * kTabFloats * 4;
  static constexpr size_t kSmem = kOffBar + 512 + 1024;
  // tensor memory columns
  static constexpr uint32_t kColU = 0, kColSb = D, kColX = D + D / 2, kColY = kColX + 64;
  static constexpr uint32_t kColSc = D == 256 ? kColY : kColY + 64;  // D = 256: no room of its own
  static constexpr bool kAlias = kColSc == kColY;
  static_assert(kColSc + 64 <= 512 && kSmem <= 227 * 1024, "one CTA's resources");
};

// one chunk's decay tables
struct DecayTable {
  float f[kTile];      // e^{G_i}
  float w[kTile];      // e^{R_j}, 0 behind the sample
  float row[kTile];    // decay from the start of i's 16-token block up to i
  float col[kTile];    // decay behind j up to the end of j's block
  float local[kTile];  // log2 decay from the start of i's block up to i
  float between[16];   // [I][J]: decay of the blocks strictly between J and I
  float a_hi, a_lo;    // decay of the whole chunk
  float pad[14];
};

template <int D, bool OUT>
__global__ void __launch_bounds__(LinearTcCfg<D>::kThreads, 1) linear_tc_kernel(const __grid_constant__ LinearTcParams P) {
  using Cfg = LinearTcCfg<D>;
  constexpr int NQK = Cfg::kStagesQK, NV = Cfg::kStagesV, NP = Cfg::kPanelsU, KT = Cfg::kKeysPerThread;
  static_assert(sizeof(DecayTable) == Cfg::kTabFloats * 4, "table size");
  const LinearParams& p = P.p;
  extern __shared__ __align__(1024) unsigned char smem_linear_tc[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_linear_tc) + 1023) &
                                                       ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int vblk = blockIdx.x % Cfg::kBlocks, nh = blockIdx.x / Cfg::kBlocks;
  const int h = nh % p.H, n = nh / p.H, hk = h / (p.H / p.Hk);

  // barriers: Q, K, V tiles landed (QF, KF, VF) and free again (QE, KE, VE); decay table written /
  // read (TF, TE); Sc ready (SC); P written (BP); bf16(S)^T written (SB); X and Y ready (XY); e^R K
  // panel written (BK); U panel ready (BU); outputs read from tensor memory (BE)
  constexpr int QF = 0, KF = QF + NQK, VF = KF + NQK, QE = VF + NV, KE = QE + NQK, VE = KE + NQK, TF = VE + NV,
                TE = TF + 2, SC = TE + 2, BP = SC + 1, SB = BP + 1, XY = SB + 1, BK = XY + 1, BU = BK + NP,
                BE = BU + NP, DR = BE + 1, NBAR = DR + 1;
  static_assert(NBAR * 8 + 8 <= 512, "barrier area");
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + Cfg::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + Cfg::kOffBar + NBAR * 8);
  auto B = [&](int i) { return smem_u32(&bar[i]); };
  if (tid == 0) {
    for (int i = 0; i < NBAR; ++i) {
      const bool by_warps = (i >= KE && i < VE) || i == TE || i == TE + 1 || i == BP || i == SB || i == BE ||
                            (i >= BK && i < BU);
      mbar_init(B(i), by_warps ? Cfg::kWorkers : 1);
    }
    mbar_fence_init();
  }
  if (warp == Cfg::kWorkers) tc::alloc(smem_u32(tmem_slot), 512);
  // blocks of P above the diagonal are zero in every chunk
  for (int i = tid; i < int(Cfg::kPanel / 16); i += Cfg::kThreads)
    reinterpret_cast<uint4*>(sm + Cfg::kOffP)[i] = make_uint4(0, 0, 0, 0);
  tc::fence_smem_async();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tU = tmem + Cfg::kColU, tSb = tmem + Cfg::kColSb, tX = tmem + Cfg::kColX, tY = tmem + Cfg::kColY,
                 tSc = tmem + Cfg::kColSc;
  DecayTable* tab = reinterpret_cast<DecayTable*>(sm + Cfg::kOffTab);

  int64_t bos, eos;
  sample_range(p, n, bos, eos);
  const int nchunks = static_cast<int>((eos - bos + kTile - 1) / kTile);

  bool alive = true;
  auto wait = [&](int b, uint32_t parity) {
    if (alive && !mbar_wait(B(b), parity)) {
      alive = false;
      atomicOr(&g_linear_status, 1);
    }
  };

  if (warp == Cfg::kWorkers) {
    // ---------------- MMA issue ----------------
    constexpr uint32_t kIdSc = tc::idesc(tc::kBF16, 64, 64, false, false);
    constexpr uint32_t kIdX = tc::idesc(tc::kBF16, 128, 64, false, false);   // Sb^T in TMEM, Q K-major
    constexpr uint32_t kIdY = tc::idesc(tc::kBF16, 128, 64, true, false);    // V^T MN-major, P K-major
    constexpr uint32_t kIdU = tc::idesc(tc::kBF16, 128, Cfg::kPanelKeys, true, true);
    const uint32_t base = smem_u32(sm);
    auto scores = [&](int c) {
      const int s = c % NQK;
      const uint32_t ph = (c / NQK) & 1;
      wait(QF + s, ph);
      wait(KF + s, ph);
      tc::fence_after();
      if (__all_sync(~0u, alive) && tc::elect_one()) {
        const uint32_t q = base + Cfg::kOffQ + s * Cfg::kBytesQK, k = base + Cfg::kOffK + s * Cfg::kBytesQK;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          tc::mma_bf16(tSc, tc::desc_kmajor(q + (ks >> 2) * Cfg::kPanel, (ks & 3) * 32),
                       tc::desc_kmajor(k + (ks >> 2) * Cfg::kPanel, (ks & 3) * 32), kIdSc, ks > 0);
        tc::commit(B(SC));
      }
      __syncwarp();
    };
    if (OUT && nchunks > 0) scores(0);
    for (int c = 0; c < nchunks; ++c) {
      const uint32_t ph = c & 1;
      const int sv = c % NV;
      const uint32_t v = base + Cfg::kOffV + sv * Cfg::kBytesV;
      if constexpr (OUT) {
        const int sq = c % NQK;
        wait(SB, ph);  // and the outputs of chunk c - 1 have been read: X and Y may be overwritten
        tc::fence_after();
        if (__all_sync(~0u, alive) && tc::elect_one()) {
          const uint32_t q = base + Cfg::kOffQ + sq * Cfg::kBytesQK;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            tc::mma_bf16_ts(tX, tSb + 8 * ks, tc::desc_kmajor(q + (ks >> 2) * Cfg::kPanel, (ks & 3) * 32), kIdX, ks > 0);
          tc::commit(B(QE + sq));
        }
        __syncwarp();
      }
      wait(VF + sv, (c / NV) & 1);
      if constexpr (OUT) {
        wait(BP, ph);
        tc::fence_after();
        if (__all_sync(~0u, alive) && tc::elect_one()) {
          const uint32_t pt = base + Cfg::kOffP;
#pragma unroll
          for (int ks = 0; ks < kTile / 16; ++ks)
            tc::mma_bf16(tY, tc::desc_mnmajor(v, Cfg::kPanel, ks), tc::desc_kmajor(pt, ks * 32), kIdY, ks > 0);
          tc::commit(B(XY));
        }
        __syncwarp();
      }
#pragma unroll
      for (int u = 0; u < NP; ++u) {
        wait(BK + u, ph);
        tc::fence_after();
        if (__all_sync(~0u, alive) && tc::elect_one()) {
          // smallest term first, so that the accumulator's truncations are those of small sums
#pragma unroll
          for (int term = 2; term >= 0; --term) {
            const uint32_t kt = base + Cfg::kOffKt + term * Cfg::kBytesQK + u * (Cfg::kPanelKeys / 64) * Cfg::kPanel;
#pragma unroll
            for (int ks = 0; ks < kTile / 16; ++ks)
              tc::mma_bf16(tU + u * Cfg::kPanelKeys, tc::desc_mnmajor(v, Cfg::kPanel, ks),
                           tc::desc_mnmajor(kt, Cfg::kPanel, ks), kIdU, term < 2 || ks > 0);
          }
          tc::commit(B(BU + u));
          if (u == NP - 1) tc::commit(B(VE + sv));
        }
        __syncwarp();
      }
      if (OUT && c + 1 < nchunks) {
        if constexpr (Cfg::kAlias) {
          wait(BE, ph);
          tc::fence_after();
        }
        scores(c + 1);
      }
    }
    // a wait that ran out: nothing of this warp may still run when tensor memory is freed
    if (!__all_sync(~0u, alive)) {
      if (tc::elect_one()) tc::commit(B(DR));
      __syncwarp();
      mbar_wait(B(DR), 0);
    }
  } else if (warp == Cfg::kWorkers + 1) {
    // ---------------- tiles and decay tables ----------------
    const uint32_t base = smem_u32(sm);
    int issued = 0;
    for (int c = 0; c < nchunks; ++c) {
      const int y = static_cast<int>(bos) + c * kTile;
      const int s = c % NQK, sv = c % NV;
      if (c >= NQK) {
        if constexpr (OUT) wait(QE + s, ((c / NQK) - 1) & 1);
        wait(KE + s, ((c / NQK) - 1) & 1);
      }
      if (c >= NV) wait(VE + sv, ((c / NV) - 1) & 1);
      if (__all_sync(~0u, alive)) {
        if (tc::elect_one()) {
          if constexpr (OUT) {
            mbar_expect_tx(B(QF + s), Cfg::kBytesQK);
#pragma unroll
            for (int b = 0; b < D / 64; ++b)
              tma_load_2d(base + Cfg::kOffQ + s * Cfg::kBytesQK + b * Cfg::kPanel, &P.q_map, hk * D + 64 * b, y, B(QF + s));
          }
          mbar_expect_tx(B(KF + s), Cfg::kBytesQK);
#pragma unroll
          for (int b = 0; b < D / 64; ++b)
            tma_load_2d(base + Cfg::kOffK + s * Cfg::kBytesQK + b * Cfg::kPanel, &P.k_map, hk * D + 64 * b, y, B(KF + s));
          mbar_expect_tx(B(VF + sv), Cfg::kBytesV);
#pragma unroll
          for (int b = 0; b < 2; ++b)
            tma_load_2d(base + Cfg::kOffV + sv * Cfg::kBytesV + b * Cfg::kPanel, &P.v_map,
                        h * D + vblk * Cfg::kVB + (D == 64 ? 0 : 64 * b), y, B(VF + sv));
        }
        issued = c + 1;
      }
      __syncwarp();
      // decay table: lane l has tokens 2 l and 2 l + 1, eight lanes a block of 16
      const int len = static_cast<int>(eos - y < kTile ? eos - y : kTile);
      constexpr float kLog2e = 1.44269504f;
      float g[2];
      double total = 0.0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = 2 * lane + e;
        const float x = t < len ? log_decay(p, y + t, h) : 0.f;
        // below 2^-160 a decay is a reset in fp32 whatever it multiplies; NaN stays NaN
        g[e] = x * kLog2e < -160.f ? -160.f : x * kLog2e;
        total += x < -111.f ? -111.0 : static_cast<double>(x);
      }
      float sum = g[0] + g[1], fwd = sum, bwd = sum;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const float a = __shfl_up_sync(~0u, fwd, o, 8), b = __shfl_down_sync(~0u, bwd, o, 8);
        if ((lane & 7) >= o) fwd += a;
        if ((lane & 7) + o < 8) bwd += b;
      }
      float before = __shfl_up_sync(~0u, fwd, 1, 8), behind = __shfl_down_sync(~0u, bwd, 1, 8);
      if ((lane & 7) == 0) before = 0.f;
      if ((lane & 7) == 7) behind = 0.f;
      float blk[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) blk[b] = __shfl_sync(~0u, fwd, 8 * b + 7);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
      const int I = lane >> 3;
      float pre = 0.f, post = 0.f;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (b < I) pre += blk[b];
        if (b > I) post += blk[b];
      }
      const float L0 = before + g[0], L1 = L0 + g[1], R1 = behind, R0 = behind + g[1];
      const int ts = c & 1;
      if (c >= 2) wait(TE + ts, ((c >> 1) - 1) & 1);
      DecayTable& t = tab[ts];
      const int t0 = 2 * lane;
      t.local[t0] = L0;
      t.local[t0 + 1] = L1;
      t.row[t0] = exp2f(L0);
      t.row[t0 + 1] = exp2f(L1);
      t.col[t0] = exp2f(R0);
      t.col[t0 + 1] = exp2f(R1);
      t.f[t0] = exp2f(pre + L0);
      t.f[t0 + 1] = exp2f(pre + L1);
      t.w[t0] = t0 < len ? exp2f(R0 + post) : 0.f;
      t.w[t0 + 1] = t0 + 1 < len ? exp2f(R1 + post) : 0.f;
      if (lane < 16) {
        const int bi = lane >> 2, bj = lane & 3;
        float x = 0.f;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (b > bj && b < bi) x += blk[b];
        t.between[lane] = exp2f(x);
      }
      if (lane == 0) {
        const double a = exp(total);
        t.a_hi = static_cast<float>(a);
        t.a_lo = static_cast<float>(a - static_cast<double>(t.a_hi));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(B(TF + ts));
    }
    // a wait that ran out: the loads in flight must land before shared memory is released
    if (!__all_sync(~0u, alive)) {
      for (int c = issued > NQK ? issued - NQK : 0; c < issued; ++c) {
        if constexpr (OUT) mbar_wait(B(QF + c % NQK), (c / NQK) & 1);
        mbar_wait(B(KF + c % NQK), (c / NQK) & 1);
      }
      for (int c = issued > NV ? issued - NV : 0; c < issued; ++c) mbar_wait(B(VF + c % NV), (c / NV) & 1);
    }
  } else {
    // ---------------- workers ----------------
    const int quad = warp & 3, kq = warp >> 2;  // tensor-memory lane quadrant; key and token column group
    const int vr = (32 * quad + lane) % Cfg::kVB;
    const bool writes = D >= 128 || quad < 2;  // at D = 64 quadrants 2 and 3 repeat 0 and 1
    const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n), out_slot = pool_slot(p.slots_out, p.num_out, n);
    const int64_t col_off = (int64_t)(KT * kq) * D + vblk * Cfg::kVB + vr;  // key KT kq of panel 0
    float S[NP][KT];  // S[panel u][key KT kq + i][value vr]
#pragma unroll
    for (int u = 0; u < NP; ++u)
#pragma unroll
      for (int i = 0; i < KT; ++i)
        S[u][i] = p.h0 != nullptr && in_slot >= 0
                      ? p.h0[(in_slot * p.H + h) * D * D + col_off + (int64_t)(u * Cfg::kPanelKeys + i) * D]
                      : 0.f;
    auto fold = [&](int u, float a_hi, float a_lo) {  // S = a S + U^T
      const uint64_t ah = f32x2_splat(a_hi), al = f32x2_splat(a_lo);
#pragma unroll
      for (int q = 0; q < KT / 16; ++q) {
        float x[16];
        tc::ld16(tc::lane_addr(tU, 32 * quad, u * Cfg::kPanelKeys + KT * kq + 16 * q), x);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float& s0 = S[u][16 * q + i];
          float& s1 = S[u][16 * q + i + 1];
          const uint64_t s = f32x2_pack(s0, s1);
          const uint64_t y = fma_f32x2(ah, s, fma_f32x2(al, s, f32x2_pack(x[i], x[i + 1])));
          s0 = f32x2_lo(y);
          s1 = f32x2_hi(y);
        }
      }
    };
    auto write_sb = [&](int u) {  // bf16(S)^T: keys 2 c, 2 c + 1 in column c
#pragma unroll
      for (int q = 0; q < KT / 16; ++q) {
        uint32_t r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = pack_bf16x2(S[u][16 * q + 2 * i], S[u][16 * q + 2 * i + 1]);
        tc::st8(tc::lane_addr(tSb, 32 * quad, (u * Cfg::kPanelKeys + KT * kq + 16 * q) / 2), r);
      }
    };
    auto arrive = [&](int b) {
      __syncwarp();
      if (lane == 0) mbar_arrive(B(b));
    };
    const int prow = 16 * quad + (lane & 15);  // row of P; its columns are 16 kq ..
    for (int c = 0; c < nchunks; ++c) {
      const uint32_t ph = c & 1;
      const int ts = c & 1;
      const int64_t tok0 = bos + (int64_t)c * kTile;
      const int len = static_cast<int>(eos - tok0 < kTile ? eos - tok0 : kTile);
      // ---- the previous chunk's U into the state ----
      if (c > 0) {
        const DecayTable& t = tab[ts ^ 1];
        const float a_hi = t.a_hi, a_lo = t.a_lo;
#pragma unroll
        for (int u = 0; u < NP; ++u) {
          wait(BU + u, ph ^ 1);
          __syncwarp();
          tc::fence_after();
          fold(u, a_hi, a_lo);
          if constexpr (OUT) write_sb(u);
        }
        arrive(TE + (ts ^ 1));
      } else if constexpr (OUT) {
#pragma unroll
        for (int u = 0; u < NP; ++u) write_sb(u);
      }
      if constexpr (OUT) {
        tc::wait_st();
        tc::fence_before();
        arrive(SB);
      }
      wait(TF + ts, (c >> 1) & 1);
      const DecayTable& t = tab[ts];
      if (len < kTile) {  // rows of V behind the sample
        wait(VF + c % NV, (c / NV) & 1);
        unsigned char* v = sm + Cfg::kOffV + (c % NV) * Cfg::kBytesV;
        for (int i = tid; i < 2 * (kTile - len) * 8; i += Cfg::kWorkers * 32) {
          const int panel = i & 1, piece = i >> 1;
          *reinterpret_cast<uint4*>(v + panel * Cfg::kPanel + len * 128 + piece * 16) = make_uint4(0, 0, 0, 0);
        }
        tc::fence_smem_async();
      }
      if constexpr (OUT) {
        // ---- P: scores masked and decayed ----
        wait(SC, ph);
        __syncwarp();
        tc::fence_after();
        if (kq <= quad) {
          float x[16];
          tc::ld16(tc::lane_addr(tSc, 32 * quad, 16 * kq), x);
          if (kq < quad) {
            const float r = t.row[prow] * t.between[quad * 4 + kq];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= r * t.col[16 * kq + i];
          } else {
            const float l = t.local[prow];
#pragma unroll
            for (int i = 0; i < 16; ++i)
              x[i] = 16 * kq + i <= prow ? x[i] * fast_exp2(l - t.local[16 * kq + i]) : 0.f;
          }
          if (len < kTile) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 16 * kq + i < len ? x[i] : 0.f;
          }
          if (lane < 16) {
            unsigned char* row = sm + Cfg::kOffP + prow * 128;
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<uint4*>(row + (((2 * kq + e) ^ (prow & 7)) << 4)) =
                  make_uint4(pack_bf16x2(x[8 * e], x[8 * e + 1]), pack_bf16x2(x[8 * e + 2], x[8 * e + 3]),
                             pack_bf16x2(x[8 * e + 4], x[8 * e + 5]), pack_bf16x2(x[8 * e + 6], x[8 * e + 7]));
          }
          tc::fence_smem_async();
        }
        tc::fence_before();
        arrive(BP);
      }
      // ---- e^R K in three bf16 terms, in K's layout ----
      wait(KF + c % NQK, (c / NQK) & 1);
      const unsigned char* kt = sm + Cfg::kOffK + (c % NQK) * Cfg::kBytesQK;
#pragma unroll
      for (int u = 0; u < NP; ++u) {
        constexpr int kPieces = Cfg::kPanelKeys / 64 * kTile * 8;  // 16-byte pieces of a panel
#pragma unroll
        for (int i0 = 0; i0 < kPieces; i0 += Cfg::kWorkers * 32) {
          const int off = (u * kPieces + i0 + tid) * 16;
          const int row = (off >> 7) & 63;
          const float w = t.w[row];
          const uint4 x = *reinterpret_cast<const uint4*>(kt + off);
          const uint32_t in[4] = {x.x, x.y, x.z, x.w};
          uint32_t r[3][4];
          const uint64_t ww = f32x2_splat(w);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint64_t y = mul_f32x2(bf16x2_to_f32x2(in[e]), ww);
            if (row >= len) y = 0;
            r[0][e] = f32x2_to_bf16x2(y);
            y = sub_f32x2(y, bf16x2_to_f32x2(r[0][e]));
            r[1][e] = f32x2_to_bf16x2(y);
            y = sub_f32x2(y, bf16x2_to_f32x2(r[1][e]));
            r[2][e] = f32x2_to_bf16x2(y);
          }
#pragma unroll
          for (int term = 0; term < 3; ++term)
            *reinterpret_cast<uint4*>(sm + Cfg::kOffKt + term * Cfg::kBytesQK + off) =
                make_uint4(r[term][0], r[term][1], r[term][2], r[term][3]);
        }
        tc::fence_smem_async();
        tc::fence_before();  // this panel's U has been read above
        arrive(BK + u);
      }
      arrive(KE + c % NQK);
      if constexpr (OUT) {
        // ---- outputs of this thread's value for 16 tokens ----
        wait(XY, ph);
        __syncwarp();
        tc::fence_after();
        float x[16], y[16];
        tc::ld16(tc::lane_addr(tX, 32 * quad, 16 * kq), x);
        tc::ld16(tc::lane_addr(tY, 32 * quad, 16 * kq), y);
        tc::fence_before();
        if constexpr (Cfg::kAlias) arrive(BE);
        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + (tok0 + 16 * kq) * p.so + (int64_t)h * D +
                           vblk * Cfg::kVB + vr;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool mine = D >= 128 || (quad < 2) == (i < 8);
          const float z = p.scale * fmaf(t.f[16 * kq + i], x[i], y[i]);
          if (mine && 16 * kq + i < len) o[i * p.so] = __float2bfloat16_rn(z);
        }
      }
    }
    if (nchunks > 0) {
      const DecayTable& t = tab[(nchunks - 1) & 1];
#pragma unroll
      for (int u = 0; u < NP; ++u) {
        wait(BU + u, (nchunks - 1) & 1);
        __syncwarp();
        tc::fence_after();
        fold(u, t.a_hi, t.a_lo);
      }
    }
    const bool taken = __any_sync(~0u, slot_taken(p.slots_out, n, out_slot, lane, 32));
    if (__all_sync(~0u, alive) && writes && out_slot >= 0 && !taken) {
#pragma unroll
      for (int u = 0; u < NP; ++u)
#pragma unroll
        for (int i = 0; i < KT; ++i)
          p.ht[(out_slot * p.H + h) * D * D + col_off + (int64_t)(u * Cfg::kPanelKeys + i) * D] = S[u][i];
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == Cfg::kWorkers) tc::dealloc(tmem, 512);
}

}  // namespace memt
