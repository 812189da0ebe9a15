// The gated delta rule in chunks of 64 tokens on tcgen05 tensor cores: one CTA per (sample, head, block of up
// to 128 values), the chunks of a sample in order.
//
// With G_i the sum of the log decays of a chunk's tokens up to and including i and S the state before the chunk:
//     A_ij = beta_i e^{G_i - G_j} k_i.k_j  (j < i),    T = (I + A)^-1
//     r_i  = beta_i (v_i - e^{G_i} S^T k_i),           u = T r       (the corrections of the chunk's tokens)
//     o_i  = scale [ e^{G_i} S^T q_i + sum_{j <= i} e^{G_i - G_j} (q_i.k_j) u_j ]
//     S'   = e^{G_63} S + sum_j e^{G_63 - G_j} k_j u_j^T
// Everything that the state enters is computed transposed, the value index as the tensor-memory lane, so that its A
// operand is written into tensor memory by the threads that own a value:
//     Sc  = [K; Q] K^T         M = 128 rows, N = 64, K = D
//     X^T = S^T K^T, S^T Q^T   M = 128 values, N = 64 tokens each, K = D
//     U^T = R^T T^T            M = 128 values, N = 64 tokens, K = 64; T is lower triangular: smaller N
//     P^T = (w U)^T K          M = 128 values, N = D keys, K = 64 tokens
//     O^T = U^T B^T            M = 128 values, N = 64 tokens, K = 64; B = masked, decayed Q K^T: smaller N
//
// Precision. The state is fp32 in registers. K and V are bf16 as given; every fp32 factor of a product that the state
// depends on (S in S^T K^T, T, R, w U) is split into two bf16 terms, which leaves 2^-16 of each value at most and a few
// 1e-6 of the state in all (one term would leave 1e-3). A and its inverse are fp32 on CUDA cores: a unit lower
// triangular inverse by forward substitution of 16 x 16 blocks and two doublings. S^T Q^T reads the first term only, B
// and the U of O^T are bf16: what only the output sees is rounded like the output. Sums of log decays are formed in
// 64 bits and kept as pairs of fp32 numbers, so that their differences are those of the tokens in between whatever
// came before them; the decay of a whole chunk is a pair too.
//
// Roles (20 warps): warp 0 issues MMAs, warp 1 loads tiles, warps 2 and 3 make the decay tables of alternate chunks
// (and set rows behind the sample to zero); warps 4-7 invert I + A; warps 8-11 make A and B of the next chunk from Sc
// and then the outputs of the previous one; warps 12-19 hold the state, half of the keys each warpgroup, and walk the
// chain X -> R -> U -> w U -> P -> S. What bounds a chunk is that chain: three batches of MMAs of 540, 290 and 530
// cycles at D = 128, each with some 350 cycles from the first arrival to the threads that read the result, and
// the threads' work between them. Products off the chain are issued where it leaves the tensor pipe idle: the next chunk's
// Sc behind S^T K^T, S^T Q^T behind U, O^T behind P.
// At D = 64 the 64 values fill half of the 128 lanes; lanes 64-127 repeat them and take half of the output rows.
//
// Values that are not finite: the zeros of T and B meet them in tokens they must not reach. Whatever spoils a token
// never leaves the state, so a CTA looks at its final state; a warp's columns of which one is not finite are made
// again token by token (DeltaColumns) from the initial state.
// Every wait is bounded as in linear_tc.cuh: a thread whose wait runs out flags it and stops waiting, the control
// warps drain what they have in flight, and the final state is NaN.
#pragma once

#include "delta.cuh"
#include "tc.cuh"
#include "tma.h"

namespace memt {

struct DeltaTcParams {
  CUtensorMap q_map, k_map, v_map;  // bf16 token rows, boxes of 64 channels x 64 tokens
  CUtensorMap o_map;                // boxes of 32 channels x 32 tokens
  DeltaParams p;
};

// bit 0: a wait of delta_tc_kernel ran out (memt_gated_delta_status)
static __device__ int g_delta_status;

// one chunk's decays and gates; tokens behind the sample: no decay, everything but f and gh 0
struct DeltaTable {
  float gh[kTile], gl[kTile];  // log2 decay from the chunk's start up to i, as a pair
  float f[kTile];              // scale e^{G_i}
  float b[kTile];              // beta_i
  float bf[kTile];             // beta_i e^{G_i}
  float w[kTile];              // e^{G_63 - G_i}
  float a_hi, a_lo;            // decay of the whole chunk
  float pad[14];
};

template <int D_>
struct DeltaTcCfg {
  static constexpr int D = D_;
  static constexpr int kVB = D < 128 ? D : 128;  // values per CTA
  static constexpr int kBlocks = D / kVB;        // CTAs per (sample, head)
  static constexpr int kThreads = 640;
  static constexpr int kKeys = D / 2;            // keys per state thread
  static constexpr int kStages = D == 128 ? 3 : 4;
  static constexpr int kTables = 4;
  static constexpr int kRow = 68;                // floats per row of A: 16-byte reads of 8 rows without conflicts
  static constexpr uint32_t kPanel = kTile * 128;             // 64 x 64 bf16: 8 KB
  static constexpr uint32_t kPair = 2 * kPanel;               // a panel of K and the same of Q behind it
  static constexpr uint32_t kBytesKQ = D / 64 * kPair;
  static constexpr uint32_t kBytesV = kTile * kVB * 2;
  static constexpr uint32_t kOffKQ = 0;
  static constexpr uint32_t kOffV = kOffKQ + kStages * kBytesKQ;
  static constexpr uint32_t kOffT = kOffV + kStages * kBytesV;  // two terms
  static constexpr uint32_t kOffB = kOffT + 2 * kPanel;
  static constexpr uint32_t kOffOut = kOffB + kPanel;           // two pieces of 2 KB per output warp
  static constexpr uint32_t kOffA = kOffOut + 4 * 2 * 2048;     // fp32 [64][kRow]
  static constexpr uint32_t kOffY = kOffA + kTile * kRow * 4;   // fp32 [32][36]
  static constexpr uint32_t kOffTab = kOffY + 32 * 36 * 4;
  static constexpr uint32_t kOffBar = kOffTab + kTables * sizeof(DeltaTable);
  static constexpr size_t kSmem = kOffBar + 512 + 1024;
  // Tensor memory columns. S: for each half of the keys its two terms, over which P^T is written once X has read
  // them. R: two terms of R^T, then of (w U)^T. X: S^T K^T, then in its first half bf16(U)^T.
  static constexpr uint32_t kColS = 0, kColX = D, kColXQ = kColX + 64, kColR = kColXQ + 64, kColU = kColR + 64,
                            kColO = kColU + 64, kColSc = kColO + 64;
  // registers per thread after the split of the launch's 5 x 96 over the warpgroups
  static constexpr int kRegsControl = 56, kRegsInvert = 72, kRegsPrepare = 80, kRegsState = 136;
  static_assert(kRegsControl + kRegsInvert + kRegsPrepare + 2 * kRegsState <= 5 * 96, "the launch's registers");
  static_assert(kColSc + 64 <= 512 && kSmem <= 227 * 1024, "one CTA's resources");
};

// Two bf16 terms of a pair of fp32 numbers: first + second.
__device__ __forceinline__ void split2(uint64_t x, uint32_t& first, uint32_t& second) {
  first = f32x2_to_bf16x2(x);
  second = f32x2_to_bf16x2(sub_f32x2(x, bf16x2_to_f32x2(first)));
}

// 2^(h + l) for |l| far below 1
__device__ __forceinline__ float exp2_pair(float h, float l) {
  const float x = fast_exp2(h);
  return fmaf(x, l * 0.69314718f, x);
}

// The warp's columns from `col` of one state, again, token by token from `start` (null: zeros) and with the outputs.
// Once every value of the state is NaN, so is everything behind.
template <int D>
__device__ __forceinline__ void delta_columns_again(const DeltaParams& p, int h, int col, int64_t bos, int64_t eos,
                                                 const float* start, float* end) {
  using Cols = DeltaColumns<D>;
  using T = __nv_bfloat16;
  Cols cols;
  cols.load(start != nullptr ? start + col : nullptr);
  const int hk = h / (p.H / p.Hk);
  float fixed_hi, fixed_lo;
  split_decay(p.g_layout == 3 ? exp(static_cast<double>(p.g[h])) : 1.0, fixed_hi, fixed_lo);
  bool lost = false;
#pragma unroll 1
  for (int64_t t = bos; t < eos; ++t) {
    float out = __int_as_float(0x7fffffff);
    if (!lost) {
      const T* kt = static_cast<const T*>(p.k) + t * p.sk + (int64_t)hk * D + Cols::row0();
      const T* qt = static_cast<const T*>(p.q) + t * p.sq + (int64_t)hk * D + Cols::row0();
      const T* vt = static_cast<const T*>(p.v) + t * p.sv + (int64_t)h * D + col;
      auto four = [](const T* x) {
        const uint2 u = *reinterpret_cast<const uint2*>(x);
        const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
        return make_float4(a.x, a.y, b.x, b.y);
      };
      auto k = [&](int m) { return four(kt + 4 * Cols::kRowGroups * m); };
      auto q = [&](int m) { return four(qt + 4 * Cols::kRowGroups * m); };
      auto v = [&](int c) { return as_f32(vt[c]); };
      const float beta = load_beta<T>(p, t, h);
      const float a = p.g_layout == 1 ? expf(p.g[t * p.H + h]) : fixed_hi;
      out = cols.template step<true>(k, q, v, a, p.g_layout == 1 ? 0.f : fixed_lo, beta);
      bool nan = true;
#pragma unroll
      for (int i = 0; i < Cols::kRows / 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) nan = nan && isnan(f32x2_lo(cols.S[i][c])) && isnan(f32x2_hi(cols.S[i][c]));
      lost = __all_sync(~0u, nan);
    }
    if (Cols::writes())
      store_f32(static_cast<T*>(p.out), t * p.so + (int64_t)h * D + col + Cols::col0() + Cols::own_col(), p.scale * out);
  }
  if (end != nullptr) cols.store(end + col);
}

template <int D>
__global__ void __launch_bounds__(DeltaTcCfg<D>::kThreads, 1) delta_tc_kernel(const __grid_constant__ DeltaTcParams P) {
  using Cfg = DeltaTcCfg<D>;
  constexpr int NS = Cfg::kStages, NT = Cfg::kTables, KT = Cfg::kKeys, RL = Cfg::kRow;
  const DeltaParams& p = P.p;
  extern __shared__ __align__(1024) unsigned char smem_delta_tc[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_delta_tc) + 1023) &
                                                       ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(~0u, tid >> 5, 0), quad = warp & 3;  // uniform: so are the roles' branches
  const int vblk = blockIdx.x % Cfg::kBlocks, unit = blockIdx.x / Cfg::kBlocks / p.H;
  const int h = blockIdx.x / Cfg::kBlocks % p.H, hk = h / (p.H / p.Hk);
  int n = unit;
  if (p.only_long) {
    n = find_long(p, unit);
    if (n < 0) return;
  } else if (p.by_length) {
    n = sample_by_length(p, unit);
  }
  int64_t bos, eos;
  sample_range(p, n, bos, eos);
  if (eos - bos <= p.few) return;  // the token-by-token kernel's

  // barriers: K with Q and V tiles landed (KF, VF) and free again (KE, VE); table written / read (TF, TE); scores ready
  // (SC) and read (SR); A written (AW) and used (AE); T's operand written (TW); B's (BW); the state's terms written
  // (SB); X (XD), U (UD), P (PD) and O (OD) ready; R^T written (RW), (w U)^T and U^T written (WW); outputs read (OE);
  // drained (DR)
  constexpr int KF = 0, VF = KF + NS, KE = VF + NS, VE = KE + NS, TF = VE + NS, TE = TF + NT, SC = TE + NT, SR = SC + 1,
                AW = SR + 1, AE = AW + 1, TW = AE + 1, BW = TW + 1, SB = BW + 1, XD = SB + 1, RW = XD + 1, UD = RW + 1,
                WW = UD + 1, PD = WW + 1, OD = PD + 1, OE = OD + 1, DR = OE + 1, NBAR = DR + 1;
  static_assert(NBAR * 8 + 24 <= 512, "barrier area");
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + Cfg::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + Cfg::kOffBar + NBAR * 8);
  uint32_t* spoiled = tmem_slot + 1;  // bit c: some value of the CTA's columns 4 c .. 4 c + 3 is not finite
  uint32_t* stalled = tmem_slot + 2;  // a wait ran out
  const uint32_t base = smem_u32(sm), bars = smem_u32(bar);
  auto B = [&](int i) { return bars + 8 * i; };
  if (tid == 0) {
    for (int i = 0; i < NBAR; ++i) {
      uint32_t count = 1;  // TMA, tcgen05.commit or one thread
      if (i == SB || i == RW || i == WW || (i >= VE && i < TF)) count = 8;  // the state's warps
      if (i >= TE && i < SC) count = 12;                                    // and those of A, B and the outputs
      if (i == SR || i == OE || i == AE || i == TW) count = 4;
      if (i == AW || i == BW) count = 2;
      mbar_init(B(i), count);
    }
    mbar_fence_init();
    *spoiled = 0;
    *stalled = 0;
  }
  if (warp == 0) tc::alloc(smem_u32(tmem_slot), 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem + Cfg::kColS, tX = tmem + Cfg::kColX, tXQ = tmem + Cfg::kColXQ, tR = tmem + Cfg::kColR,
                 tU = tmem + Cfg::kColU, tO = tmem + Cfg::kColO, tSc = tmem + Cfg::kColSc;
  DeltaTable* tab = reinterpret_cast<DeltaTable*>(sm + Cfg::kOffTab);
  const int nchunks = static_cast<int>((eos - bos + kTile - 1) / kTile);
  auto chunk_len = [&](int c) {
    const int64_t left = eos - bos - (int64_t)c * kTile;
    return static_cast<int>(left < kTile ? left : kTile);
  };

  bool alive = true;
  auto wait = [&](int b, uint32_t phase) {  // a wait that ran out is known to all before anything follows it
    if (alive) {
      alive = mbar_wait_clock(B(b), phase & 1);
      }
  };
  auto arrive = [&](int b) {  // one arrival per warp
    __syncwarp();
    if (lane == 0) mbar_arrive(B(b));
  };

  if (warp < 4) {
    regs_dec<Cfg::kRegsControl>();
    if (warp == 0) {
      // ---------------- MMA issue ----------------
      auto go = [&]() {  // nothing more is issued after a wait ran out
        tc::fence_after();
        return __all_sync(~0u, alive) && tc::elect_one();
      };
      auto kq = [&](int s, int i) {  // K step i of the tile's rows, as a descriptor's offset
        return tc::desc_kmajor(base + Cfg::kOffKQ + s * Cfg::kBytesKQ, 0) + (i >> 2) * (Cfg::kPair >> 4) + (i & 3) * 2;
      };
      auto scores = [&](int c) {
        const int s = c % NS;
        wait(KF + s, c / NS);
        if (chunk_len(c) < kTile) {  // rows of K behind the sample: zero
          const int len = chunk_len(c), pieces = (kTile - len) * 8;
          for (int i = lane; i < D / 64 * pieces; i += 32)
            *reinterpret_cast<uint4*>(sm + Cfg::kOffKQ + s * Cfg::kBytesKQ + i / pieces * Cfg::kPair + len * 128 +
                                      i % pieces * 16) = make_uint4(0, 0, 0, 0);
          tc::fence_smem_async();
          __syncwarp();
        }
        if (c > 0) wait(SR, c - 1);
        if (go()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            tc::mma_bf16(tSc, kq(s, i), kq(s, i), tc::idesc(tc::kBF16, 128, 64, false, false), i > 0);
          tc::commit(B(SC));
        }
        __syncwarp();
      };
      // A operand of S's term for K step i: the halves of the keys lie D / 2 columns apart, each with its two terms
      auto state = [&](int term, int i) {
        constexpr int per = D / 32;  // K steps of a half
        return tS + (D / 2) * (i / per) + 8 * (i % per) + term * (D / 4);
      };
      // M = 128 values, lower triangular 64 x 64 operand of rows 16 i on for the tokens 16 i .. 16 i + 15
      auto triangle = [&](uint32_t d, uint32_t a, uint32_t tile, bool acc) {
        const uint64_t desc = tc::desc_kmajor(tile, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tc::mma_bf16_ts(d + 16 * i, a + 8 * i, desc + 130 * i, tc::idesc(tc::kBF16, 128, 64 - 16 * i, false, false),
                          acc || i > 0);
      };
      if (nchunks > 0) scores(0);
      for (int c = 0; c < nchunks; ++c) {
        const int s = c % NS;
        constexpr uint32_t kIdX = tc::idesc(tc::kBF16, 128, 64, false, false);
        wait(SB, c);
        if (go()) {
          // the smaller term first, so that the accumulator's truncations are those of small sums
#pragma unroll
          for (int i = 0; i < 2 * (D / 16); ++i) {
            const int term = i < D / 16 ? 1 : 0, step = i % (D / 16);
            tc::mma_bf16_ts(tX, state(term, step), kq(s, step), kIdX, i > 0);
          }
          tc::commit(B(XD));
        }
        __syncwarp();
        if (c + 1 < nchunks) scores(c + 1);
        wait(RW, c);
        wait(TW, c);
        if (go()) {
          triangle(tU, tR, base + Cfg::kOffT + Cfg::kPanel, false);
          triangle(tU, tR + 32, base + Cfg::kOffT, true);
          triangle(tU, tR, base + Cfg::kOffT, true);
          tc::commit(B(UD));
        }
        __syncwarp();
        if (c > 0) wait(OE, c - 1);
        if (go()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            tc::mma_bf16_ts(tXQ, state(0, i), kq(s, i) + (Cfg::kPanel >> 4), kIdX, i > 0);
        }
        __syncwarp();
        wait(WW, c);
        if (go()) {
          const uint64_t dk = tc::desc_mnmajor(base + Cfg::kOffKQ + s * Cfg::kBytesKQ, Cfg::kPair, 0);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            tc::mma_bf16_ts(tS, tR + 8 * (i ^ 4), dk + 128 * (i & 3), tc::idesc(tc::kBF16, 128, D, false, true), i > 0);
          tc::commit(B(PD));
          tc::commit(B(KE + s));
        }
        __syncwarp();
        wait(BW, c);
        if (go()) {
          triangle(tO, tX, base + Cfg::kOffB, false);
          tc::commit(B(OD));
        }
        __syncwarp();
      }
      // a wait that ran out: nothing of this warp may still run when tensor memory is freed
      if (!__all_sync(~0u, alive)) {
        if (tc::elect_one()) tc::commit(B(DR));
        __syncwarp();
        mbar_wait_clock(B(DR), 0);
      }
    } else if (warp == 1) {
      // ---------------- tile loads ----------------
      int issued = 0;
      for (int c = 0; c < nchunks; ++c) {
        const int y = static_cast<int>(bos) + c * kTile, s = c % NS;
        if (c >= NS) wait(KE + s, c / NS - 1);
        if (__all_sync(~0u, alive) && tc::elect_one()) {
          mbar_expect_tx(B(KF + s), Cfg::kBytesKQ);
          for (int i = 0; i < D / 64; ++i) {
            const uint32_t at = base + Cfg::kOffKQ + s * Cfg::kBytesKQ + i * Cfg::kPair;
            tma_load_2d(at, &P.k_map, hk * D + 64 * i, y, B(KF + s));
            tma_load_2d(at + Cfg::kPanel, &P.q_map, hk * D + 64 * i, y, B(KF + s));
          }
        }
        __syncwarp();
        if (c >= NS) wait(VE + s, c / NS - 1);
        if (__all_sync(~0u, alive)) {
          if (tc::elect_one()) {
            mbar_expect_tx(B(VF + s), Cfg::kBytesV);
            for (int i = 0; i < Cfg::kVB / 64; ++i)
              tma_load_2d(base + Cfg::kOffV + s * Cfg::kBytesV + i * Cfg::kPanel, &P.v_map,
                          h * D + vblk * Cfg::kVB + 64 * i, y, B(VF + s));
          }
        }
        __syncwarp();
        issued = c + 1;
      }
      // Every load lands before shared memory is released, also when a wait ran out: tiles that were never
      // issued only use up their (bounded) wait.
      if (!__all_sync(~0u, alive)) {
        for (int c = issued > NS ? issued - NS : 0; c < issued; ++c) {
          mbar_wait_clock(B(KF + c % NS), (c / NS) & 1);
          mbar_wait_clock(B(VF + c % NS), (c / NS) & 1);
        }
      }
    } else {
      // ---------------- decay tables: lane l has tokens 2 l and 2 l + 1 ----------------
      float xg[2], xb[2];
      auto fetch = [&](int c) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int64_t t = bos + (int64_t)c * kTile + 2 * lane + e;
          xg[e] = t < eos ? log_decay(p, t, h) : 0.f;
          xb[e] = t < eos ? load_beta<__nv_bfloat16>(p, t, h) : 0.f;
        }
      };
      fetch(warp - 2);
      for (int c = warp - 2; c < nchunks; c += 2) {
        const int len = chunk_len(c), t0 = 2 * lane;
        double g[2];
        const float beta[2] = {xb[0], xb[1]};
#pragma unroll
        for (int e = 0; e < 2; ++e)  // below e^-111 = 2^-160 a decay is a reset in fp32 whatever it multiplies; NaN stays NaN
          g[e] = 1.4426950408889634 * (xg[e] < -111.f ? -111.0 : static_cast<double>(xg[e]));
        if (c + 2 < nchunks) fetch(c + 2);
        double sum = g[0] + g[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double x = __shfl_up_sync(~0u, sum, o);
          if (lane >= o) sum += x;
        }
        const double total = __shfl_sync(~0u, sum, 31);
        const int ts = c % NT;
        if (c >= NT) wait(TE + ts, c / NT - 1);
        DeltaTable& t = tab[ts];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const double G = e == 0 ? sum - g[1] : sum;
          const float gh = static_cast<float>(G), gl = static_cast<float>(G - static_cast<double>(gh));
          const float a = exp2_pair(gh, gl);
          const double R = total - G;
          const float rh = static_cast<float>(R), rl = static_cast<float>(R - static_cast<double>(rh));
          t.gh[t0 + e] = gh;
          t.gl[t0 + e] = gl;
          t.f[t0 + e] = p.scale * a;
          t.b[t0 + e] = beta[e];
          t.bf[t0 + e] = beta[e] * a;
          t.w[t0 + e] = t0 + e < len ? exp2_pair(rh, rl) : 0.f;
        }
        if (lane == 0) chunk_decay(total, t.a_hi, t.a_lo);
        arrive(TF + ts);
      }
    }
  } else if (warp < 8) {
    // ---------------- T = (I + A)^-1 in place of A, then as the U products' operand ----------------
    if constexpr (Cfg::kRegsInvert > 96) regs_inc<Cfg::kRegsInvert>(); else regs_dec<Cfg::kRegsInvert>();
    float* A = reinterpret_cast<float*>(sm + Cfg::kOffA);
    float* Y = reinterpret_cast<float*>(sm + Cfg::kOffY);
    const int iw = warp - 4;
    auto meet = [&]() { asm volatile("bar.sync 3, 128;" ::: "memory"); };
    auto row4 = [](const float* x) { return *reinterpret_cast<const float4*>(x); };
    // R rows from a on, 4 RL apart and N long (16-byte aligned), times four columns at b, rows LB apart. Eight terms a
    // turn: with more loads in flight the registers would not do.
    auto product = [&](const float* a, const float* b, int LB, int N, auto& y) {
      constexpr int R = std::extent<std::remove_reference_t<decltype(y)>>::value;
#pragma unroll
      for (int r = 0; r < R; ++r) y[r][0] = y[r][1] = 0;
#pragma unroll 1
      for (int k = 0; k < N; k += 8) {
        float4 b4[8], a4[R][2];
#pragma unroll
        for (int e = 0; e < 8; ++e) b4[e] = row4(b + (k + e) * LB);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          a4[r][0] = row4(a + 4 * r * RL + k);
          a4[r][1] = row4(a + 4 * r * RL + k + 4);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float4 f = a4[r][e >> 2];
            const uint64_t aa = f32x2_splat((e & 3) == 0 ? f.x : (e & 3) == 1 ? f.y : (e & 3) == 2 ? f.z : f.w);
            y[r][0] = fma_f32x2(aa, f32x2_pack(b4[e].x, b4[e].y), y[r][0]);
            y[r][1] = fma_f32x2(aa, f32x2_pack(b4[e].z, b4[e].w), y[r][1]);
          }
        }
      }
    };
    auto put = [](float* x, const uint64_t (&y)[2], float sign) {
      *reinterpret_cast<float4*>(x) = make_float4(sign * f32x2_lo(y[0]), sign * f32x2_hi(y[0]), sign * f32x2_lo(y[1]),
                                                  sign * f32x2_hi(y[1]));
    };
    for (int c = 0; c < nchunks; ++c) {
      wait(AW, c);
      __syncwarp();
      {  // 16 x 16 blocks on the diagonal: a lane solves for one column, x_i = [i = column] - sum_{m < i} A_im x_m
        float* blk = A + (16 * iw) * RL + 16 * iw;
        const int col = lane & 15;
        float x[16];
        float4 next[4];
        x[0] = col == 0 ? 1.f : 0.f;
        next[0] = row4(blk + RL);
#pragma unroll
        for (int i = 1; i < 16; ++i) {
          float4 a4[4];
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            a4[m] = next[m];
            if (i < 15 && 4 * m < i + 1) next[m] = row4(blk + (i + 1) * RL + 4 * m);
          }
          float sum[2] = {i == col ? 1.f : 0.f, 0.f};
#pragma unroll
          for (int m = 0; m < i; ++m) {
            const float4 f = a4[m >> 2];
            const float am = (m & 3) == 0 ? f.x : (m & 3) == 1 ? f.y : (m & 3) == 2 ? f.z : f.w;
            sum[m & 1] = fmaf(-am, x[m], sum[m & 1]);
          }
          x[i] = sum[0] + sum[1];
          __syncwarp();  // one row is fetched ahead: more would not fit into registers
        }
        __syncwarp();
        if (lane < 16) {
#pragma unroll
          for (int i = 0; i < 16; ++i) blk[i * RL + col] = x[i];
        }
      }
      meet();
      {  // two 32 x 32 blocks: T_21 = -T_22 (A_21 T_11), each by two warps
        float* blk = A + 32 * (iw >> 1) * (RL + 1);
        float* y = Y + 16 * (iw >> 1) * 36;
        const int r = 8 * (iw & 1) + (lane >> 2), col = 4 * (lane & 3);
        uint64_t z[1][2];
        product(blk + (16 + r) * RL, blk + col, RL, 16, z);
        put(y + r * 36 + col, z[0], 1.f);
        meet();
        product(blk + (16 + r) * RL + 16, y + col, 36, 16, z);
        put(blk + (16 + r) * RL + col, z[0], -1.f);
      }
      meet();
      {  // the 64 x 64 block, rows r and r + 4 of this warp's eight
        const int r = 8 * iw + (lane >> 3), col = 4 * (lane & 7);
        uint64_t z[2][2];
        product(A + (32 + r) * RL, A + col, RL, 32, z);
        put(Y + r * 36 + col, z[0], 1.f);
        put(Y + (r + 4) * 36 + col, z[1], 1.f);
        meet();
        product(A + (32 + r) * RL + 32, Y + col, 36, 32, z);
        put(A + (32 + r) * RL + col, z[0], -1.f);
        put(A + (36 + r) * RL + col, z[1], -1.f);
      }
      meet();
      if (c > 0) wait(UD, c - 1);  // U has read the previous chunk's operand
      __syncwarp();
      {  // two bf16 terms, half a row a thread; what lies right of the diagonal's blocks is never read
        const int t = tid - 128, r = t >> 1, half = t & 1;
        if (half == 0 || r >= 32) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 lo4 = row4(A + r * RL + 32 * half + 8 * j), hi4 = row4(A + r * RL + 32 * half + 8 * j + 4);
            uint32_t u[4], v[4];
            split2(f32x2_pack(lo4.x, lo4.y), u[0], v[0]);
            split2(f32x2_pack(lo4.z, lo4.w), u[1], v[1]);
            split2(f32x2_pack(hi4.x, hi4.y), u[2], v[2]);
            split2(f32x2_pack(hi4.z, hi4.w), u[3], v[3]);
            unsigned char* at = sm + Cfg::kOffT + r * 128 + (((4 * half + j) ^ (r & 7)) << 4);
            *reinterpret_cast<uint4*>(at) = make_uint4(u[0], u[1], u[2], u[3]);
            *reinterpret_cast<uint4*>(at + Cfg::kPanel) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      }
      tc::fence_smem_async();
      arrive(TW);
      if (lane == 0) mbar_arrive(B(AE));
    }
  } else if (warp < 12) {
    // ---------------- A and B from the scores; outputs from X and O ----------------
    regs_dec<Cfg::kRegsPrepare>();
    const int pair = 2 * (lane & 3);                                        // first column of a fragment
    const int prow = 8 * (lane >> 4) + (lane & 7), pval = (lane >> 3) & 1;  // row of an stmatrix piece
    const int r = 32 * (quad & 1) + lane;  // row of K K^T (quads 0, 1) or Q K^T
    const bool isB = quad >= 2;
    auto prepare = [&](int c) {
      const DeltaTable& t = tab[c % NT];
      wait(TF + c % NT, c / NT);
      wait(SC, c);
      if (c > 0) wait(isB ? OD : AE, c - 1);  // the previous one has been used
      __syncwarp();
      tc::fence_after();
      const float gh = t.gh[r], gl = t.gl[r], factor = isB ? p.scale : t.b[r];
      const int most = isB ? r : r - 1;  // last column that counts
#pragma unroll 1
      for (int J = 0; J <= (quad & 1); ++J) {
        float x[32];
        tc::ld32(tc::lane_addr(tSc, 32 * quad, 32 * J), x);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 h4 = *reinterpret_cast<const float4*>(&t.gh[32 * J + i]);
          const float4 l4 = *reinterpret_cast<const float4*>(&t.gl[32 * J + i]);
          const float hs[4] = {h4.x, h4.y, h4.z, h4.w}, ls[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // masked by selection
            const float y = x[i + e] * (factor * fast_exp2((gh - hs[e]) + (gl - ls[e])));
            x[i + e] = 32 * J + i + e <= most ? y : 0.f;
          }
        }
        if (isB) {
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            *reinterpret_cast<uint4*>(sm + Cfg::kOffB + r * 128 + (((4 * J + i / 8) ^ (r & 7)) << 4)) =
                make_uint4(pack_bf16x2(x[i], x[i + 1]), pack_bf16x2(x[i + 2], x[i + 3]),
                           pack_bf16x2(x[i + 4], x[i + 5]), pack_bf16x2(x[i + 6], x[i + 7]));
        } else {
          float* row = reinterpret_cast<float*>(sm + Cfg::kOffA) + r * RL + 32 * J;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(row + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        }
      }
      tc::fence_before();
      if (isB) tc::fence_smem_async();
      arrive(SR);
      if (lane == 0) mbar_arrive(B(isB ? BW : AW));
    };
    // Outputs: fragments of 16 values by 32 tokens, a register pair is two tokens of one value. stmatrix turns them
    // into token rows of this warp's 32 values (64 bytes, the 64-byte swizzle), which leave as one TMA box; a
    // chunk that ends inside leaves row by row instead.
    const int col = h * D + vblk * Cfg::kVB + (D >= 128 ? 32 * quad : 32 * (quad & 1));
    auto write_out = [&](int c) {
      const DeltaTable& t = tab[c % NT];
      const int len = chunk_len(c);
      wait(OD, c);
      __syncwarp();
      tc::fence_after();
      constexpr int kPieces = D >= 128 ? 2 : 1;  // of 32 tokens
#pragma unroll 1
      for (int piece = 0; piece < kPieces; ++piece) {
        const int t0 = 32 * (D >= 128 ? piece : quad >> 1);
        const uint32_t turn = base + Cfg::kOffOut + (2 * (warp - 8) + piece) * 2048;
        if (lane == 0) {  // the box before the last (at D = 64 the last one) has left its rows
          if constexpr (kPieces == 2) bulk_wait_read_but1();
          else bulk_wait_read();
        }
        __syncwarp();
#pragma unroll 1
        for (int e = 0; e < 2; ++e) {
          uint32_t x[16], y[16];
          tc::ld_frag2<4>(tc::lane_addr(tXQ, 32 * quad + 16 * e, t0), tc::lane_addr(tO, 32 * quad + 16 * e, t0), x, y);
          if (piece + 1 == kPieces && e == 1) {
            tc::fence_before();
            arrive(OE);
          }
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            uint32_t z[4];  // tokens 8 (i + j) + pair, + 1: of value lane / 4, of value lane / 4 + 8
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2 f = *reinterpret_cast<const float2*>(&t.f[t0 + 8 * (i + j) + pair]);
              const uint64_t ff = f32x2_pack(f.x, f.y);
#pragma unroll
              for (int v8 = 0; v8 < 2; ++v8) {
                const int k = 4 * (i + j) + 2 * v8;
                z[2 * j + v8] = f32x2_to_bf16x2(fma_f32x2(ff, (static_cast<uint64_t>(x[k + 1]) << 32) | x[k],
                                                          (static_cast<uint64_t>(y[k + 1]) << 32) | y[k]));
              }
            }
            const int tok = 8 * i + prow;
            stsm_x4_t(turn + tok * 64 + (((2 * e + pval) ^ ((tok >> 1) & 3)) << 4), z[0], z[1], z[2], z[3]);
          }
        }
        const int64_t tok0 = bos + (int64_t)c * kTile + t0;
        if (len == kTile) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&P.o_map, col, static_cast<int>(tok0), turn);
            bulk_commit();
          }
        } else {
          __syncwarp();
          __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + tok0 * p.so + col + 8 * (lane & 3);
          for (int tok = lane >> 2; tok < 32 && t0 + tok < len; tok += 8) {
            uint4 z;
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(z.x), "=r"(z.y), "=r"(z.z), "=r"(z.w)
                         : "r"(turn + tok * 64 + (((lane & 3) ^ ((tok >> 1) & 3)) << 4)) : "memory");
            *reinterpret_cast<uint4*>(o + tok * p.so) = z;
          }
        }
      }
      arrive(TE + c % NT);
    };
    for (int c = 0; c < nchunks; ++c) {
      prepare(c);
      if (c > 0) write_out(c - 1);
    }
    if (nchunks > 0) write_out(nchunks - 1);
    if (lane == 0) bulk_wait_all();
    __syncwarp();
    asm volatile("bar.sync 2, 384;" ::: "memory");
  } else {
    // ---------------- the state and its chain: value row of this lane, keys KT half .. ----------------
    regs_inc<Cfg::kRegsState>();
    const int half = (warp - 12) >> 2;
    const int vr = (32 * quad + lane) % Cfg::kVB;
    const bool writes = D >= 128 || quad < 2;  // at D = 64 quadrants 2 and 3 repeat 0 and 1
    const int pair = 2 * (lane & 3);
    const int prow = 8 * (lane >> 4) + (lane & 7), pval = (lane >> 3) & 1;  // row of an ldmatrix piece
    const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n), out_slot = pool_slot(p.slots_out, p.num_out, n);
    const int64_t head = (int64_t)D * D, col_off = (int64_t)(KT * half) * D + vblk * Cfg::kVB + vr;
    const float* start = p.h0 != nullptr && in_slot >= 0 ? p.h0 + (in_slot * p.H + h) * head : nullptr;
    uint64_t S[KT / 2];  // pairs of fp32: keys KT half + 2 i, + 2 i + 1 of value vr
    if (start != nullptr) {
      const float* src = start + col_off;
#pragma unroll
      for (int i = 0; i < KT; i += 2) S[i / 2] = f32x2_pack(src[i * D], src[(i + 1) * D]);
    } else {
#pragma unroll
      for (int i = 0; i < KT / 2; ++i) S[i] = 0;
    }
    const uint32_t own = tc::lane_addr(tS, 32 * quad, KT * half);  // of S's terms and of P
    for (int c = 0; c < nchunks; ++c) {
#pragma unroll
      for (int q = 0; q < KT / 16; ++q) {
        uint32_t first[8], second[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split2(S[8 * q + i], first[i], second[i]);
        tc::st8(own + 8 * q, first);
        tc::st8(own + KT / 2 + 8 * q, second);
      }
      tc::wait_st();
      tc::fence_before();
      arrive(SB);
      // V as fragments of 16 values by 32 tokens: a register holds two tokens of one value
      const int s = c % NS;
      wait(VF + s, c / NS);
      wait(TF + c % NT, c / NT);
      const DeltaTable& t = tab[c % NT];
      __syncwarp();
      uint32_t v[2][8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int val = (32 * quad + 16 * e) % Cfg::kVB + 8 * pval;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t x[4];
          const int tok = 32 * half + 16 * q + prow;
          ldsm_x4_t(x, base + Cfg::kOffV + s * Cfg::kBytesV + (val >> 6) * Cfg::kPanel + tok * 128 +
                           ((((val & 63) >> 3) ^ (tok & 7)) << 4));
#pragma unroll
          for (int i = 0; i < 4; ++i) v[e][4 * q + i] = x[i];
        }
      }
      arrive(VE + s);
      if (chunk_len(c) < kTile) {  // tokens behind the sample, whatever stands in their rows
        const int len = chunk_len(c) - 32 * half - pair;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            v[e][j] = 8 * (j >> 1) >= len ? 0 : 8 * (j >> 1) + 1 >= len ? v[e][j] & 0xffffu : v[e][j];
      }
      wait(XD, c);
      __syncwarp();
      tc::fence_after();
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // R = beta v - beta e^G X
        uint32_t x[16], first[8], second[8];
        tc::ld_frag<4>(tc::lane_addr(tX, 32 * quad + 16 * e, 32 * half), x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 b = *reinterpret_cast<const float2*>(&t.b[32 * half + 8 * i + pair]);
          const float2 bf = *reinterpret_cast<const float2*>(&t.bf[32 * half + 8 * i + pair]);
          const uint64_t bb = f32x2_pack(b.x, b.y), minus = f32x2_pack(-bf.x, -bf.y);
#pragma unroll
          for (int v8 = 0; v8 < 2; ++v8) {
            const int k = 4 * i + 2 * v8, j = 2 * i + v8;
            const uint64_t y = mul_f32x2(bb, bf16x2_to_f32x2(v[e][j]));
            split2(fma_f32x2(minus, (static_cast<uint64_t>(x[k + 1]) << 32) | x[k], y), first[j], second[j]);
          }
        }
        tc::st_frag16(tc::lane_addr(tR, 32 * quad + 16 * e, 16 * half), first);
        tc::st_frag16(tc::lane_addr(tR, 32 * quad + 16 * e, 32 + 16 * half), second);
      }
      tc::wait_st();
      tc::fence_before();
      arrive(RW);
      wait(UD, c);
      __syncwarp();
      tc::fence_after();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t x[16], first[8], second[8], whole[8];
        tc::ld_frag<4>(tc::lane_addr(tU, 32 * quad + 16 * e, 32 * half), x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 w = *reinterpret_cast<const float2*>(&t.w[32 * half + 8 * i + pair]);
          const uint64_t ww = f32x2_pack(w.x, w.y);
#pragma unroll
          for (int v8 = 0; v8 < 2; ++v8) {
            const int k = 4 * i + 2 * v8, j = 2 * i + v8;
            const uint64_t u = (static_cast<uint64_t>(x[k + 1]) << 32) | x[k];
            whole[j] = f32x2_to_bf16x2(u);
            split2(mul_f32x2(ww, u), first[j], second[j]);
          }
        }
        tc::st_frag16(tc::lane_addr(tR, 32 * quad + 16 * e, 16 * half), first);
        tc::st_frag16(tc::lane_addr(tR, 32 * quad + 16 * e, 32 + 16 * half), second);
        tc::st_frag16(tc::lane_addr(tX, 32 * quad + 16 * e, 16 * half), whole);
      }
      tc::wait_st();
      tc::fence_before();
      const uint64_t ah = f32x2_splat(t.a_hi), al = f32x2_splat(t.a_lo);
      arrive(WW);
      if (lane == 0) mbar_arrive(B(TE + c % NT));
      wait(PD, c);
      __syncwarp();
      tc::fence_after();
#pragma unroll
      for (int q = 0; q < KT / 32; ++q) {
        float x[32];
        tc::ld32(own + 32 * q, x);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          uint64_t& x2 = S[(32 * q + i) / 2];
          x2 = fma_f32x2(ah, x2, fma_f32x2(al, x2, f32x2_pack(x[i], x[i + 1])));
        }
      }
    }
    const bool taken = __any_sync(~0u, slot_taken(p.slots_out, n, out_slot, lane, 32));
    // No state is stored before every thread has loaded its share of the first one and, where one is not finite,
    // before columns have been made from them again.
    constexpr int kGroup = DeltaColumns<D>::kCols;
    uint64_t seen = 0;  // two zeros; NaN once a state is not finite
#pragma unroll
    for (int i = 0; i < KT / 2; ++i) seen = fma_f32x2(S[i], 0, seen);
    if (f32x2_lo(seen) != 0.f || f32x2_hi(seen) != 0.f) atomicOr(spoiled, 1u << (vr / kGroup));
    asm volatile("bar.sync 2, 384;" ::: "memory");  // with the outputs' warps, once theirs have left
    float* end = out_slot >= 0 && !taken ? p.ht + (out_slot * p.H + h) * head : nullptr;
    const uint32_t again = *spoiled;
    const bool lost = *stalled != 0;
    if (lost) {  // the caller sees it in the state
#pragma unroll
      for (int i = 0; i < KT / 2; ++i) S[i] = f32x2_splat(__int_as_float(0x7fffffff));
    }
    if (writes && end != nullptr && (lost || !(again >> (vr / kGroup) & 1))) {
      float* dst = end + col_off;
#pragma unroll
      for (int i = 0; i < KT; i += 2) {
        dst[i * D] = f32x2_lo(S[i / 2]);
        dst[(i + 1) * D] = f32x2_hi(S[i / 2]);
      }
    }
    if (again != 0 && !lost) {
      for (int g = warp - 12; g < Cfg::kVB / kGroup; g += 8)
        if (again >> g & 1) delta_columns_again<D>(p, h, vblk * Cfg::kVB + g * kGroup, bos, eos, start, end);
    }
  }
  if (!alive) atomicOr(&g_delta_status, 1);
  tc::fence_before();
  __syncthreads();
  if (warp == 0) tc::dealloc(tmem, 512);
}

}  // namespace memt
