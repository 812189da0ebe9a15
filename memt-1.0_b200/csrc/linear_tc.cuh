// Causal linear attention with a decay for each head, in chunks of 64 tokens on tcgen05 tensor
// cores: one CTA per (sample, head, block of up to 128 values), the chunks of a sample in order.
//
// With G_i the sum of the log decays of a chunk's tokens up to and including i, R_j the sum over
// the tokens behind j and S the state before the chunk:
//     o_i = scale [ e^{G_i} S^T q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j ]
//     S'  = e^{G_63} S + sum_j (e^{R_j} k_j) v_j^T
// Everything is computed transposed, so that the value index is the tensor-memory lane:
//     Sc   = Q K^T              M = 64 tokens i, N = 64 tokens j, K = D
//     U^T  = (e^R V)^T K        M = 128 values, N = up to 128 keys, K = 64 tokens, three times (below)
//     X^T  = bf16(S)^T Q^T      M = 128 values, N = 64 tokens, K = D
//     Y^T  = V^T P^T            M = 128 values, N = 64 tokens i, K = 64 tokens j, P = masked, decayed Sc
// Q, K and V tiles arrive by TMA with the 128-byte swizzle and are operands in place (Q and K K-major,
// K for U and V for Y MN-major). The A operands of U and X are written into tensor memory by
// threads that own a value: what bounds a chunk of three-term U products from shared memory is
// not the tensor pipe but the 8 KB that each of them would read for 64 cycles of work, all that shared
// memory delivers (the split of e^R K in shared memory took 7700 cycles a chunk at D = 128).
//
// Precision. The state is fp32 in registers. e^R V is not rounded to bf16 but split into three bf16
// terms (8 bits each), so that the sum over a chunk is an fp32 sum and the final state is what the
// fp32 recurrence gives (measured 1e-7 relative; one bf16 term leaves 1e-3, two 2e-6). The chunk's
// decay is applied as a pair of fp32 numbers: one number, its rounding repeated for every chunk of a
// constant decay, would drift by 2^-25 a chunk. Neither of the pair is negative, so that an infinite state
// stays one. Scores P and the copy of the state that X reads are bf16 (at most 2^-8 relative each), as is
// the output; no other value is rounded below fp32.
// Decay weights never come from differences of long sums: P's weight is the product of the decay from
// its row's 16-token block start, of whole blocks between, and to its column's block end; inside a
// block of 16 it is one difference. So every factor is <= 1 for any decay, a reset (e^g = 0) included.
//
// Roles (20 warps): warp 0 issues MMAs, warp 1 loads tiles, warps 2 and 3 make the decay tables of
// alternate chunks; warps 4-11 split e^R V of a chunk and then make the outputs of the previous one,
// half of the tokens each warpgroup; warps 12-19 hold the state, half of the keys each warpgroup: they
// write bf16(S), make P from Sc (alternate column blocks) and fold U into S. U of a chunk does not depend on
// the state, so no MMA waits for another one's chunk; the loop that closes is U -> e^R V of the next
// chunk -> U. A form in which 16 warps did all of this in lockstep took 6200 cycles a chunk at D = 128, most of
// it the latency of its phases; one with a role for each product was bound by instruction fetch
// (every role's code runs once a chunk), hence few roles and rolled loops.
// The last chunk of a sample is padded with whatever the TMA brings (the next sample's rows, or
// zeros past the last row): those columns of P are masked by selection, those rows of K's and V's
// tiles are set to zero (0 x NaN would not be), and those tokens' outputs are not stored.
// A v that is not finite meets the zero weights of up to 15 earlier tokens in Y, and its three terms would be
// a difference of infinities. A sample whose final state is not finite therefore looks for such values once
// its chunks are done and makes what they spoil again, token by token (8 x 8192 tokens, 16 heads, D = 128:
// 220 us in a short run, 350 with a NaN near a sample's start, 2.2 ms near its end).
// Looking for them in every chunk, in the split or in the table warps, cost 4 to 16 % of every call.
// At D = 64 the 64 values fill half of the 128 lanes; V's tile is loaded twice so that lanes 64-127
// repeat lanes 0-63 and take half of the output rows.
// Every wait is bounded: a thread whose wait runs out flags it and stops waiting, the control warps
// drain what they have in flight, and the final state is NaN.
#pragma once

#include "linear.cuh"
#include "tc.cuh"
#include "tma.h"

namespace memt {

struct LinearTcParams {
  CUtensorMap q_map, k_map, v_map;  // bf16 token rows, boxes of 64 channels x 64 tokens
  CUtensorMap o_map;                // boxes of 32 channels x the tokens of an output warp
  LinearParams p;
};

// bit 0: a wait of linear_tc_kernel ran out (memt_linear_attention_status)
static __device__ int g_linear_status;

// one chunk's decay tables
struct DecayTable {
  float f[kTile];      // scale e^{G_i}
  float w[kTile];      // e^{R_j}, 0 behind the sample
  float row[kTile];    // scale times the decay from the start of i's 16-token block up to i
  float col[kTile];    // decay behind j up to the end of j's block
  float local[kTile];  // log2 decay from the start of i's block up to i
  float between[16];   // [I][J]: decay of the blocks strictly between J and I
  float a_hi, a_lo;    // decay of the whole chunk
  float pad[14];
};

template <int D_>
struct LinearTcCfg {
  static constexpr int D = D_;
  static constexpr int kVB = D < 128 ? D : 128;  // values per CTA
  static constexpr int kBlocks = D / kVB;        // CTAs per (sample, head)
  static constexpr int kThreads = 640;
  static constexpr int kPanels = D < 128 ? 1 : D / 128;  // U and e^R K go in units of up to 128 keys
  static constexpr int kPanelKeys = D / kPanels;
  static constexpr int kKeys = D / 2;            // keys per state thread
  static constexpr int kStages = D == 256 ? 2 : (D == 128 ? 3 : 4);
  static constexpr int kTables = 4;
  static constexpr uint32_t kPanel = kTile * 128;  // 64 x 64 bf16: 8 KB
  static constexpr uint32_t kBytesQK = kTile * D * 2;
  static constexpr uint32_t kBytesV = kTile * 128 * 2;          // 128 lanes of values, also at D = 64
  static constexpr uint32_t kOffQ = 0;
  static constexpr uint32_t kOffK = kOffQ + kStages * kBytesQK;
  static constexpr uint32_t kOffV = kOffK + kStages * kBytesQK;
  static constexpr uint32_t kOffP = kOffV + kStages * kBytesV;
  static constexpr uint32_t kOffOut = kOffP + kPanel;           // 2 KB per output warp
  static constexpr uint32_t kOffTab = kOffOut + 8 * 2048;
  static constexpr uint32_t kOffSpoiled = kOffTab + kTables * sizeof(DecayTable);  // kVB tokens, two flags
  static constexpr uint32_t kOffBar = kOffSpoiled + 1024;
  static constexpr size_t kSmem = kOffBar + 512 + 1024;
  // tensor memory columns: U^T of one unit, the three terms of (e^R V)^T, bf16(S)^T, X^T, Y^T, Sc
  static constexpr uint32_t kColU = 0, kColW = kPanelKeys, kColSb = kColW + 96, kColX = kColSb + D / 2,
                            kColY = kColX + 64;
  static constexpr bool kAlias = kColY + 128 > 512;  // D = 256: no columns for Sc, it lies on Y^T
  static constexpr uint32_t kColSc = kAlias ? kColY : kColY + 64;
  // registers per thread after the split of the launch's 5 x 96 over the warpgroups
  static constexpr int kRegsControl = D == 256 ? 32 : 64, kRegsState = D == 256 ? 152 : 104,
                       kRegsWork = D == 256 ? 72 : 104;
  static constexpr int kOutTokens = D >= 128 ? kTile / 2 : kTile / 4;  // tokens of an output warp
  static constexpr int kCols = D == 256 ? 8 : 32;  // columns of U that a state thread holds at a time
  static_assert(kRegsControl + 2 * kRegsState + 2 * kRegsWork <= 5 * 96, "no more than the launch's registers");
  static_assert(kColSc + 64 <= 512 && kSmem <= 227 * 1024, "one CTA's resources");
};

// Between the two passes over segments: the state before each one. A thread owns four values of one
// (sample, head) state and walks over its segments; the segments' own sums are replaced in place.
__global__ void __launch_bounds__(256) linear_segments_kernel(const LinearParams p, int D) {
  const int per_state = D * D / 4, blocks = (per_state + 255) / 256;
  const int at = (blockIdx.x % blocks) * 256 + threadIdx.x;
  const int nh = blockIdx.x / blocks, h = nh % p.H, n = nh / p.H;
  int64_t bos, eos;
  int first = 0, count = 1;
  {  // this sample's first segment: every warp sums the samples before it
    const int lane = threadIdx.x & 31;
    for (int m = lane; m < n; m += 32) {
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
  if (count == 1 || at >= per_state) return;  // one segment starts from the sample's own state
  const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n);
  float4 S = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p.h0 != nullptr && in_slot >= 0)
    S = reinterpret_cast<const float4*>(p.h0 + (in_slot * p.H + h) * D * D)[at];
  for (int s = 0; s < count; ++s) {
    const int64_t seg = (int64_t)(first + s) * p.H + h;
    float4* state = reinterpret_cast<float4*>(p.seg_states + seg * D * D) + at;
    float4 own = make_float4(0.f, 0.f, 0.f, 0.f);
    float2 a = make_float2(0.f, 0.f);
    if (s + 1 < count) {  // the last one's sum is not made: the second pass ends with it
      own = *state;
      a = p.seg_decays[seg];
    }
    *state = S;
    S.x = fmaf(a.x, S.x, fmaf(a.y, S.x, own.x));
    S.y = fmaf(a.x, S.y, fmaf(a.y, S.y, own.y));
    S.z = fmaf(a.x, S.z, fmaf(a.y, S.z, own.z));
    S.w = fmaf(a.x, S.w, fmaf(a.y, S.w, own.w));
  }
}

// Value column `col` again, by a warp in fp32, token by token from the state `start` (null: zeros) up to its
// token t1 (from bos), the first whose v is not finite: the outputs of t1's block of 16 before it. Behind a NaN the
// state and the outputs are NaN already. An infinity makes the whole column infinite (or NaN), which only other
// such tokens and full resets change; the last state goes to `end` (null: nowhere). The outputs behind stay NaN.
template <int D, bool OUT>
__device__ __forceinline__ void column_again(const LinearParams& p, int h, int col, int64_t bos, int tokens, int t1,
                                             const float* start, float* end) {
  constexpr int R = D / 32;
  const int lane = threadIdx.x & 31, hk = h / (p.H / p.Hk);
  const int64_t vcol = (int64_t)h * D + col, krow = (int64_t)hk * D + R * lane;
  if (isnan(load_f32<__nv_bfloat16>(p.v, (bos + t1) * p.sv + vcol))) end = nullptr;
  const bool outputs = OUT && (t1 & 15) != 0;
  if (!outputs && end == nullptr) return;
  const int upto = t1 + (end != nullptr);
  float S[R];
#pragma unroll
  for (int i = 0; i < R; ++i) S[i] = start != nullptr ? start[(R * lane + i) * D + col] : 0.f;
  // tokens whose loads are in flight together: a long column 2.1 ms where one by one 4.7; more than one at D = 256
  // spills in the chunks' loops as well (4 % of every call)
  constexpr int B = D == 256 ? 1 : 4;
  for (int tb = 0; tb < upto; tb += B) {
    float a[B], v[B], k[B][R];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const bool live = tb + j < upto;  // behind the last one: e^0 S + 0
      const int64_t row = bos + tb + (live ? j : 0);
      a[j] = live ? log_decay(p, row, h) : 0.f;
      v[j] = live ? load_f32<__nv_bfloat16>(p.v, row * p.sv + vcol) : 0.f;
#pragma unroll
      for (int i = 0; i < R; ++i) k[j][i] = live ? load_f32<__nv_bfloat16>(p.k, row * p.sk + krow + i) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int64_t row = bos + tb + j;
#pragma unroll
      for (int i = 0; i < R; ++i) S[i] = fmaf(expf(a[j]), S[i], k[j][i] * v[j]);
      if (outputs && tb + j >= (t1 & ~15) && tb + j < t1) {
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) o = fmaf(load_f32<__nv_bfloat16>(p.q, row * p.sq + krow + i), S[i], o);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) o += __shfl_xor_sync(~0u, o, x);
        if (lane == 0) store_f32(static_cast<__nv_bfloat16*>(p.out), row * p.so + vcol, p.scale * o);
      }
    }
  }
  if (end != nullptr) {
    for (int tb = upto; tb < tokens; tb += 32) {
      const int64_t at = bos + tb + lane;
      const bool mine = tb + lane < tokens && (!isfinite(load_f32<__nv_bfloat16>(p.v, at * p.sv + vcol)) ||
                                               expf(log_decay(p, at, h)) == 0.f);
      uint32_t hits = __ballot_sync(~0u, mine);
      if (hits != 0) {
        bool all_nan = true;
#pragma unroll
        for (int i = 0; i < R; ++i) all_nan &= isnan(S[i]);
        if (__all_sync(~0u, all_nan)) break;
      }
      for (; hits != 0; hits &= hits - 1) {
        const int64_t row = bos + tb + __ffs(hits) - 1;
        const float a = expf(log_decay(p, row, h)), v = load_f32<__nv_bfloat16>(p.v, row * p.sv + vcol);
#pragma unroll
        for (int i = 0; i < R; ++i) S[i] = fmaf(a, S[i], load_f32<__nv_bfloat16>(p.k, row * p.sk + krow + i) * v);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) end[(R * lane + i) * D + col] = S[i];
  }
}

template <int D, bool OUT>
__global__ void __launch_bounds__(LinearTcCfg<D>::kThreads, 1)
    linear_tc_kernel(const __grid_constant__ LinearTcParams P) {
  using Cfg = LinearTcCfg<D>;
  constexpr int NS = Cfg::kStages, NP = Cfg::kPanels, NT = Cfg::kTables, KT = Cfg::kKeys, CW = Cfg::kCols;
  const LinearParams& p = P.p;
  extern __shared__ __align__(1024) unsigned char smem_linear_tc[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_linear_tc) + 1023) &
                                                       ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(~0u, tid >> 5, 0), quad = warp & 3;  // uniform: so are the roles' branches
  const int vblk = blockIdx.x % Cfg::kBlocks, unit = blockIdx.x / Cfg::kBlocks / p.H;
  const int h = blockIdx.x / Cfg::kBlocks % p.H, hk = h / (p.H / p.Hk);
  // a unit is a sample, or with segments one of a sample's `segs`
  int n = unit, seg = 0, segs = 1;
  if (p.seg_chunks > 0) {
    if (!find_segment(p, unit, n, seg, segs)) return;
    if (!OUT && seg + 1 == segs) return;  // the first pass sums what later segments start from
  } else if (p.only_long) {
    n = find_long(p, unit);
    if (n < 0) return;
  } else if (p.by_length) {
    n = sample_by_length(p, unit);
  }
  int64_t bos, eos;
  sample_range(p, n, bos, eos);
  if (eos - bos <= p.few) return;  // the token-by-token kernel's
  if (segs > 1) {
    bos += (int64_t)seg * p.seg_chunks * kTile;
    if (seg + 1 < segs) eos = bos + (int64_t)p.seg_chunks * kTile;
  }

  // barriers: Q, K, V tiles landed (QF, KF, VF) and free again (QE, KE, VE); decay table written /
  // read (TF, TE); V's operand written (VW); U of a unit ready (BU) and read (UE); scores ready (SC),
  // P written and scores read (BP); bf16(S)^T written (SB) and read (XD); X and Y ready (XY)
  // and read (OE); drained (DR)
  constexpr int QF = 0, KF = QF + NS, VF = KF + NS, QE = VF + NS, KE = QE + NS, VE = KE + NS, TF = VE + NS,
                TE = TF + NT, VW = TE + NT, BU = VW + 1, UE = BU + NP, SC = UE + NP, BP = SC + 1, SB = BP + 1,
                XD = SB + 1, XY = XD + 1, OE = XY + 1, DR = OE + 1, NBAR = DR + 1;
  static_assert(NBAR * 8 + 8 <= 512, "barrier area");
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + Cfg::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + Cfg::kOffBar + NBAR * 8);
  const uint32_t base = smem_u32(sm), bars = smem_u32(bar);
  auto B = [&](int i) { return bars + 8 * i; };
  if (tid == 0) {
    for (int i = 0; i < NBAR; ++i) {
      uint32_t count = 1;                                      // TMA, tcgen05.commit or one thread
      if (i == VW || i == BP || i == OE || i == SB) count = 8;
      if (i >= TE && i < VW) count = 16;                // every warp that reads the table
      if (i >= UE && i < SC) count = NP == 1 ? 8 : 4;   // the state warps that read the unit
      mbar_init(B(i), count);
    }
    mbar_fence_init();
  }
  // of each value the first token whose v is not finite, whether some value's state is not, whether a wait
  // ran out
  int32_t* spoiled_at = reinterpret_cast<int32_t*>(sm + Cfg::kOffSpoiled);
  int32_t* any_spoiled = spoiled_at + Cfg::kVB;
  int32_t* stalled = any_spoiled + 1;
  if (tid < Cfg::kVB + 2) spoiled_at[tid] = tid < Cfg::kVB ? INT32_MAX : 0;
  if (warp == 0) tc::alloc(smem_u32(tmem_slot), 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tU = tmem + Cfg::kColU, tW = tmem + Cfg::kColW, tSb = tmem + Cfg::kColSb,
                 tX = tmem + Cfg::kColX, tY = tmem + Cfg::kColY, tSc = tmem + Cfg::kColSc;
  DecayTable* tab = reinterpret_cast<DecayTable*>(sm + Cfg::kOffTab);

  const int64_t seg_state = ((int64_t)unit * p.H + h) * D * D;  // of seg_states
  const int nchunks = static_cast<int>((eos - bos + kTile - 1) / kTile);
  auto chunk_len = [&](int c) {
    const int64_t left = eos - bos - (int64_t)c * kTile;
    return static_cast<int>(left < kTile ? left : kTile);
  };

  bool alive = true;
  auto wait = [&](int b, uint32_t phase) {
    if (alive) alive = mbar_wait_clock(B(b), phase & 1);
  };
  auto arrive = [&](int b) {  // one arrival per warp
    __syncwarp();
    if (lane == 0) mbar_arrive(B(b));
  };

  if (warp < 4) {
    regs_dec<Cfg::kRegsControl>();
    if (warp == 0) {
      // ---------------- MMA issue ----------------
      constexpr uint32_t kIdSc = tc::idesc(tc::kBF16, 64, 64, false, false);
      constexpr uint32_t kIdX = tc::idesc(tc::kBF16, 128, 64, false, false);  // A in tensor memory, Q K-major
      constexpr uint32_t kIdU = tc::idesc(tc::kBF16, 128, Cfg::kPanelKeys, false, true);  // K MN-major
      auto go = [&]() {  // nothing more is issued after a wait ran out
        tc::fence_after();
        return __all_sync(~0u, alive) && tc::elect_one();
      };
      auto scores = [&](int c) {
        const int s = c % NS;
        wait(QF + s, c / NS);
        wait(KF + s, c / NS);
        if (go()) {
          const uint64_t dq = tc::desc_kmajor(base + Cfg::kOffQ + s * Cfg::kBytesQK, 0);
          const uint64_t dk = tc::desc_kmajor(base + Cfg::kOffK + s * Cfg::kBytesQK, 0);
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            tc::mma_bf16(tSc, dq + (i >> 2) * (Cfg::kPanel >> 4) + (i & 3) * 2,
                         dk + (i >> 2) * (Cfg::kPanel >> 4) + (i & 3) * 2, kIdSc, i > 0);
          tc::commit(B(SC));
        }
        __syncwarp();
      };
      auto state_sums = [&](int c, int u) {
        const int s = c % NS;
        if (u == 0) {
          if (!OUT) wait(KF + s, c / NS);
          wait(VW, c);
        }
        if (u > 0) wait(UE, c);
        else if (c > 0) wait(UE + NP - 1, c - 1);
        if (go()) {
          const uint64_t dk = tc::desc_mnmajor(
              base + Cfg::kOffK + s * Cfg::kBytesQK + u * (Cfg::kPanelKeys / 64) * Cfg::kPanel, Cfg::kPanel, 0);
          // smallest term first, so that the accumulator's truncations are those of small sums
#pragma unroll
          for (int i = 0; i < 12; ++i)
            tc::mma_bf16_ts(tU, tW + 8 * i, dk + 128 * (i & 3), kIdU, i > 0);
          tc::commit(B(BU + u));
          if (u == NP - 1) tc::commit(B(KE + s));
          if (!OUT && u == NP - 1) tc::commit(B(VE + s));
        }
        __syncwarp();
      };
      auto outputs = [&](int c) {
        const int s = c % NS;
        wait(SB, c);
        if (!Cfg::kAlias && c > 0) wait(OE, c - 1);
        if (go()) {
          const uint64_t dq = tc::desc_kmajor(base + Cfg::kOffQ + s * Cfg::kBytesQK, 0);
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            tc::mma_bf16_ts(tX, tSb + 8 * i, dq + (i >> 2) * (Cfg::kPanel >> 4) + (i & 3) * 2, kIdX, i > 0);
          tc::commit(B(XD));
          tc::commit(B(QE + s));
        }
        __syncwarp();
        wait(BP, c);
        if (go()) {
          const uint64_t dv = tc::desc_mnmajor(base + Cfg::kOffV + s * Cfg::kBytesV, Cfg::kPanel, 0);
          const uint64_t dp = tc::desc_kmajor(base + Cfg::kOffP, 0);
          // tokens 16 i .. 16 i + 15 are seen by the columns from 16 i on only: smaller products, and the blocks
          // of P above the diagonal are never read
#pragma unroll
          for (int i = 0; i < kTile / 16; ++i)
            tc::mma_bf16(tY + 16 * i, dv + 128 * i, dp + 128 * i + 2 * i,
                         tc::idesc(tc::kBF16, 128, kTile - 16 * i, true, false), i > 0);
          tc::commit(B(XY));
          tc::commit(B(VE + s));
        }
        __syncwarp();
      };
      // Between the U products of two units (which share their columns and wait for the state warps
      // and, across chunks, for V's operands) the pipe has X, Y and the next scores to do.
      if (OUT && nchunks > 0) scores(0);
      for (int c = 0; c < nchunks; ++c) {
        state_sums(c, 0);
        if constexpr (OUT) outputs(c);
        if constexpr (NP == 2) state_sums(c, 1);
        if (OUT && c + 1 < nchunks) {
          if (Cfg::kAlias) wait(OE, c);
          scores(c + 1);
        }
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
        const int y = static_cast<int>(bos) + c * kTile;
        const int s = c % NS;
        auto load = [&](int full, int free, const CUtensorMap* map, uint32_t off, uint32_t bytes, int x, int step) {
          if (c >= NS) wait(free + s, c / NS - 1);
          if (__all_sync(~0u, alive) && tc::elect_one()) {
            mbar_expect_tx(B(full + s), bytes);
            for (uint32_t b = 0; b < bytes / Cfg::kPanel; ++b)
              tma_load_2d(base + off + s * bytes + b * Cfg::kPanel, map, x + step * b, y, B(full + s));
          }
          __syncwarp();
        };
        load(VF, VE, &P.v_map, Cfg::kOffV, Cfg::kBytesV, h * D + vblk * Cfg::kVB, D == 64 ? 0 : 64);
        if constexpr (OUT) load(QF, QE, &P.q_map, Cfg::kOffQ, Cfg::kBytesQK, hk * D, 64);
        load(KF, KE, &P.k_map, Cfg::kOffK, Cfg::kBytesQK, hk * D, 64);
        issued = c + 1;
      }
      // Every load lands before shared memory is released, also when a wait ran out: tiles that
      // were never issued only use up their (bounded) wait.
      if (!__all_sync(~0u, alive)) {
        for (int c = issued > NS ? issued - NS : 0; c < issued; ++c) {
          if constexpr (OUT) mbar_wait_clock(B(QF + c % NS), (c / NS) & 1);
          mbar_wait_clock(B(KF + c % NS), (c / NS) & 1);
          mbar_wait_clock(B(VF + c % NS), (c / NS) & 1);
        }
      }
    } else {
      // ---------------- decay tables: lane l has tokens 2 l and 2 l + 1, eight lanes a block of 16 ----------------
      constexpr float kLog2e = 1.44269504f;
      float next[2];
      auto fetch = [&](int c) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int64_t t = bos + (int64_t)c * kTile + 2 * lane + e;
          next[e] = t < eos ? log_decay(p, t, h) : 0.f;
        }
      };
      fetch(warp - 2);
      for (int c = warp - 2; c < nchunks; c += 2) {
        const int len = chunk_len(c);
        float g[2];
        double total = 0.0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = next[e];
          // below 2^-160 a decay is a reset in fp32 whatever it multiplies; NaN stays NaN
          g[e] = x * kLog2e < -160.f ? -160.f : x * kLog2e;
          total += x < -111.f ? -111.0 : static_cast<double>(x);
        }
        if (c + 2 < nchunks) fetch(c + 2);
        float fwd = g[0] + g[1], bwd = fwd;
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
        const int ts = c % NT;
        if (c >= NT) wait(TE + ts, c / NT - 1);
        DecayTable& t = tab[ts];
        const int t0 = 2 * lane;
        t.local[t0] = L0;
        t.local[t0 + 1] = L1;
        t.row[t0] = p.scale * fast_exp2(L0);
        t.row[t0 + 1] = p.scale * fast_exp2(L1);
        t.col[t0] = fast_exp2(R0);
        t.col[t0 + 1] = fast_exp2(R1);
        t.f[t0] = p.scale * fast_exp2(pre + L0);
        t.f[t0 + 1] = p.scale * fast_exp2(pre + L1);
        t.w[t0] = t0 < len ? fast_exp2(R0 + post) : 0.f;
        t.w[t0 + 1] = t0 + 1 < len ? fast_exp2(R1 + post) : 0.f;
        if (lane < 16) {
          const int bi = lane >> 2, bj = lane & 3;
          float x = 0.f;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (b > bj && b < bi) x += blk[b];
          t.between[lane] = fast_exp2(x);
        }
        if (lane == 0) {
          chunk_decay(total * 1.4426950408889634, t.a_hi, t.a_lo);
        }
        arrive(TF + ts);
      }
    }
  } else if (warp < 12) {
    // ---------------- (e^R V)^T in three bf16 terms into tensor memory; outputs from X and Y ----------------
    if constexpr (Cfg::kRegsWork > 96) regs_inc<Cfg::kRegsWork>(); else regs_dec<Cfg::kRegsWork>();
    const int half = (warp - 4) >> 2;        // tokens 32 half ..
    const int pair = 2 * (lane & 3);         // first column of a fragment
    // Values go through registers in the fragment layout: ldmatrix turns 8 x 8 pieces of V's tile, so that
    // a register holds two tokens of one value, and the fragment store puts them in that value's lane.
    // This lane's row of the four pieces (two of tokens by two of values) of an ldmatrix or stmatrix:
    const int prow = 8 * (lane >> 4) + (lane & 7), pval = (lane >> 3) & 1;
    auto split_v = [&](int c) {
      const int s = c % NS, len = chunk_len(c);
      const uint32_t v = base + Cfg::kOffV + s * Cfg::kBytesV;
      wait(VF + s, c / NS);
      if (len < kTile) {  // rows of K and V behind the sample
        wait(KF + s, c / NS);
        const int pieces = (kTile - len) * 8;
        for (int i = tid - 128; i < (D / 64 + 2) * pieces; i += 256) {
          const int pan = i / pieces;
          unsigned char* tile = pan < 2 ? sm + Cfg::kOffV + s * Cfg::kBytesV + pan * Cfg::kPanel
                                        : sm + Cfg::kOffK + s * Cfg::kBytesQK + (pan - 2) * Cfg::kPanel;
          *reinterpret_cast<uint4*>(tile + len * 128 + (i % pieces) * 16) = make_uint4(0, 0, 0, 0);
        }
        tc::fence_smem_async();
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the eight warps read each other's zeros
      }
      wait(TF + c % NT, c / NT);
      const DecayTable& t = tab[c % NT];
      if (c > 0) wait(BU + NP - 1, c - 1);  // U has read the previous chunk's operand
      __syncwarp();
      tc::fence_after();
#pragma unroll 1
      for (int e = 0; e < 2; ++e) {  // 16 values by 32 tokens
        const int val = (32 * quad + 16 * e) % Cfg::kVB + 8 * pval;
        uint32_t r[3][8];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t x[4];
          const int tok = 32 * half + 16 * q + prow;
          ldsm_x4_t(x, v + (val >> 6) * Cfg::kPanel + tok * 128 + ((((val & 63) >> 3) ^ (tok & 7)) << 4));
#pragma unroll
          for (int i = 0; i < 4; ++i) r[0][4 * q + i] = x[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 w = *reinterpret_cast<const float2*>(&t.w[32 * half + 8 * i + pair]);
          const uint64_t ww = f32x2_pack(w.x, w.y);
#pragma unroll
          for (int j = 2 * i; j < 2 * i + 2; ++j) {
            uint64_t y = mul_f32x2(bf16x2_to_f32x2(r[0][j]), ww);
            r[0][j] = f32x2_to_bf16x2(y);
            y = sub_f32x2(y, bf16x2_to_f32x2(r[0][j]));
            r[1][j] = f32x2_to_bf16x2(y);
            y = sub_f32x2(y, bf16x2_to_f32x2(r[1][j]));
            r[2][j] = f32x2_to_bf16x2(y);
          }
        }
#pragma unroll
        for (int term = 0; term < 3; ++term)
          tc::st_frag16(tc::lane_addr(tW, 32 * quad + 16 * e, 32 * (2 - term) + 16 * half), r[term]);
      }
      tc::wait_st();
      tc::fence_before();
      arrive(VW);
      if (!OUT && lane == 0) mbar_arrive(B(TE + c % NT));
    };
    // Outputs: fragments of 16 values by tokens, a register pair is two tokens of one value. stmatrix
    // turns them into token rows of this warp's 32 values (64 bytes, the 64-byte swizzle), which leave
    // as one TMA box; a chunk that ends inside leaves row by row instead.
    constexpr int kTok = Cfg::kOutTokens, kGroups = kTok / 8;
    const int t0 = 32 * half + (D >= 128 ? 0 : kTok * (quad >> 1));
    const int col = h * D + vblk * Cfg::kVB + (D >= 128 ? 32 * quad : 32 * (quad & 1));
    const uint32_t turn = base + Cfg::kOffOut + (warp - 4) * 2048;
    auto write_out = [&](int c) {
      const DecayTable& t = tab[c % NT];
      const int len = chunk_len(c);
      wait(XY, c);
      if (lane == 0) bulk_wait_read();  // the previous box has left the rows
      __syncwarp();
      tc::fence_after();
#pragma unroll 1
      for (int e = 0; e < 2; ++e) {
        uint32_t x[4 * kGroups], y[4 * kGroups];
        tc::ld_frag2<kGroups>(tc::lane_addr(tX, 32 * quad + 16 * e, t0), tc::lane_addr(tY, 32 * quad + 16 * e, t0), x,
                              y);
        if (e == 1) {
          tc::fence_before();
          arrive(OE);
        }
#pragma unroll
        for (int i = 0; i < kGroups; i += 2) {
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
      if (lane == 0) mbar_arrive(B(TE + c % NT));
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
        for (int tok = lane >> 2; tok < kTok && t0 + tok < len; tok += 8) {
          uint4 z;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(z.x), "=r"(z.y), "=r"(z.z), "=r"(z.w)
                       : "r"(turn + tok * 64 + (((lane & 3) ^ ((tok >> 1) & 3)) << 4)) : "memory");
          *reinterpret_cast<uint4*>(o + tok * p.so) = z;
        }
        __syncwarp();
      }
    };
    // With the scores on Y's columns the next ones wait for the outputs, which then come first.
    for (int c = 0; c < nchunks; ++c) {
      split_v(c);
      if constexpr (OUT) {
        if (Cfg::kAlias) write_out(c);
        else if (c > 0) write_out(c - 1);
      }
    }
    if (OUT && !Cfg::kAlias && nchunks > 0) write_out(nchunks - 1);
    if (lane == 0) bulk_wait_all();
    if (!alive) *stalled = 1;
    __syncwarp();
    asm volatile("bar.sync 2, 512;" ::: "memory");
    if (*any_spoiled) {
      // A v that is not finite: Y has weighed it by zero for earlier tokens of its block of 16, which leaves
      // them NaN, and its three terms are a difference of infinities. Find the first one of every value.
      constexpr int kLanes = Cfg::kVB / 8, kStep = 8 * 32 / kLanes;  // lanes a token, tokens of all warps' loads
      const int T = static_cast<int>(eos - bos), val = 8 * (lane % kLanes);
      const __nv_bfloat16* v =
          static_cast<const __nv_bfloat16*>(p.v) + bos * p.sv + (int64_t)h * D + vblk * Cfg::kVB + val;
      for (int t0 = (warp - 4) * (32 / kLanes) + lane / kLanes; t0 < T; t0 += 4 * kStep) {
        uint4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = t0 + j * kStep < T ? *reinterpret_cast<const uint4*>(v + (t0 + j * kStep) * p.sv)
                                    : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if ((w[e >> 1] >> (16 * (e & 1)) & 0x7f80) == 0x7f80 && t0 + j * kStep < spoiled_at[val + e])
              atomicMin(spoiled_at + val + e, t0 + j * kStep);
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n), out_slot = pool_slot(p.slots_out, p.num_out, n);
      const bool taken = __any_sync(~0u, slot_taken(p.slots_out, n, out_slot, lane, 32));
      const float* start = p.h0 != nullptr && in_slot >= 0 ? p.h0 + (in_slot * p.H + h) * D * D : nullptr;
      float* end = seg + 1 == segs && out_slot >= 0 && !taken ? p.ht + (out_slot * p.H + h) * D * D : nullptr;
      if (segs > 1) start = OUT ? p.seg_states + seg_state : nullptr;
      if (!OUT) end = p.seg_states + seg_state;
      for (int c = warp - 4; c < Cfg::kVB; c += 8) {
        const int t1 = spoiled_at[c];
        if (t1 == INT32_MAX) continue;
        const int64_t col = vblk * Cfg::kVB + c;
        column_again<D, OUT>(p, h, static_cast<int>(col), bos, T, t1, start, end);
        const bool stored = !isnan(load_f32<__nv_bfloat16>(p.v, (bos + t1) * p.sv + (int64_t)h * D + col));
        __syncwarp();
        if (lane == 0 && stored) spoiled_at[c] = -1;
      }
      asm volatile("bar.sync 2, 512;" ::: "memory");
    }
  } else {
    // ---------------- the state: value row of this lane, keys KT half .. ----------------
    regs_inc<Cfg::kRegsState>();
    const int half = (warp - 12) >> 2;
    const int vr = (32 * quad + lane) % Cfg::kVB;
    const bool writes = D >= 128 || quad < 2;  // at D = 64 quadrants 2 and 3 repeat 0 and 1
    const int64_t in_slot = pool_slot(p.slots_in, p.num_in, n), out_slot = pool_slot(p.slots_out, p.num_out, n);
    const int64_t col_off = (int64_t)(KT * half) * D + vblk * Cfg::kVB + vr;
    // P's fragments: first row and column of this lane's, and its row of the four pieces (two of rows by
    // two of columns) that one stmatrix writes
    const int r0 = 16 * quad + (lane >> 2), pair = 2 * (lane & 3);
    const int prow = 16 * quad + 8 * ((lane >> 3) & 1) + (lane & 7), pcol = lane >> 4;
    float2 seg_a = make_float2(1.f, 0.f);
    uint64_t S[KT / 2];  // pairs of fp32: keys KT half + 2 i, + 2 i + 1 of value vr
    const bool given = OUT && (segs > 1 || (p.h0 != nullptr && in_slot >= 0));
    if (given) {
      const float* src = (segs > 1 ? p.seg_states + seg_state : p.h0 + (in_slot * p.H + h) * D * D) + col_off;
#pragma unroll
      for (int i = 0; i < KT; i += 2) S[i / 2] = f32x2_pack(src[i * D], src[(i + 1) * D]);
    } else {
#pragma unroll
      for (int i = 0; i < KT / 2; ++i) S[i] = 0;
    }
    for (int c = 0; c < nchunks; ++c) {
      if constexpr (OUT) {  // bf16(S)^T before chunk c: keys 2 i, 2 i + 1 in column i
        if (c > 0) wait(XD, c - 1);
        __syncwarp();
        tc::fence_after();
#pragma unroll
        for (int q = 0; q < KT / 16; ++q) {
          uint32_t r[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) r[i] = f32x2_to_bf16x2(S[8 * q + i]);
          tc::st8(tc::lane_addr(tSb, 32 * quad, (KT * half + 16 * q) / 2), r);
        }
        tc::wait_st();
        tc::fence_before();
        arrive(SB);
      }
      wait(TF + c % NT, c / NT);
      const DecayTable& t = tab[c % NT];
      if constexpr (OUT) {
        const int len = chunk_len(c);
        const uint32_t row = base + Cfg::kOffP + prow * 128;
        wait(SC, c);
        __syncwarp();
        tc::fence_after();
        const float f0 = t.row[r0], f1 = t.row[r0 + 8];
#pragma unroll 1
        for (int J = half; J <= quad; J += 2) {  // 16 x 16 blocks up to the diagonal: decays, bf16 into the operand
          uint32_t x[8], z[4];  // x: columns 8 e + pair, + 1 of row r0, then of row r0 + 8, e = 0, 1
          tc::ld_frag<2>(tc::lane_addr(tSc, 32 * quad, 16 * J), x);
          if (J < quad) {
            const float bt = t.between[quad * 4 + J];
            const uint64_t g0 = f32x2_splat(f0 * bt), g1 = f32x2_splat(f1 * bt);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 cl = *reinterpret_cast<const float2*>(&t.col[16 * J + 8 * e + pair]);
              const uint64_t cc = f32x2_pack(cl.x, cl.y);
              const uint64_t x0 = (static_cast<uint64_t>(x[4 * e + 1]) << 32) | x[4 * e];
              const uint64_t x1 = (static_cast<uint64_t>(x[4 * e + 3]) << 32) | x[4 * e + 2];
              z[2 * e] = f32x2_to_bf16x2(mul_f32x2(x0, mul_f32x2(cc, g0)));
              z[2 * e + 1] = f32x2_to_bf16x2(mul_f32x2(x1, mul_f32x2(cc, g1)));
            }
          } else {
            const float l0 = t.local[r0], l1 = t.local[r0 + 8];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = 16 * J + 8 * e + pair;
              const float2 lj = *reinterpret_cast<const float2*>(&t.local[j]);
              const float d[4] = {l0 - lj.x, l0 - lj.y, l1 - lj.x, l1 - lj.y};
              float y[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {  // masked by selection, tokens behind the sample too
                const int jj = j + (i & 1);
                y[i] = jj <= r0 + 8 * (i >> 1) && jj < len
                           ? __uint_as_float(x[4 * e + i]) * (p.scale * fast_exp2(d[i])) : 0.f;
              }
              z[2 * e] = pack_bf16x2(y[0], y[1]);
              z[2 * e + 1] = pack_bf16x2(y[2], y[3]);
            }
          }
          stsm_x4(row + (((2 * J + pcol) ^ (prow & 7)) << 4), z[0], z[1], z[2], z[3]);
        }
        tc::fence_smem_async();
        tc::fence_before();
        arrive(BP);
      }
      // S = a S + U; a unit is both halves' keys, or at D = 256 this half's
      const int u = NP == 2 ? half : 0;
      const uint32_t col = tU + (NP == 2 ? 0 : KT * half);
      const float a_hi = t.a_hi, a_lo = t.a_lo;
      const uint64_t ah = f32x2_splat(a_hi), al = f32x2_splat(a_lo);
      arrive(TE + c % NT);
      if constexpr (!OUT) {  // the segment's decay, a pair of fp32 numbers too
        const float hi = __fmul_rd(seg_a.x, a_hi);
        seg_a.y = low_half(hi, fmaf(seg_a.x, a_hi, -hi) + fmaf(seg_a.x, a_lo, seg_a.y * a_hi));
        seg_a.x = hi;
      }
      wait(BU + u, c);
      __syncwarp();
      tc::fence_after();
#pragma unroll
      for (int q = 0; q < KT / CW; ++q) {
        float x[CW];
        tc::ldn<CW>(tc::lane_addr(col, 32 * quad, CW * q), x);
#pragma unroll
        for (int i = 0; i < CW; i += 2) {
          uint64_t& x2 = S[(CW * q + i) / 2];
          x2 = fma_f32x2(ah, x2, fma_f32x2(al, x2, f32x2_pack(x[i], x[i + 1])));
        }
      }
      tc::fence_before();
      arrive(UE + u);
    }
    if (!OUT && tid == 12 * 32 && vblk == 0) p.seg_decays[(int64_t)unit * p.H + h] = seg_a;
    const bool last = seg + 1 == segs;  // of its sample: its state is the final one
    const bool taken = OUT && last && __any_sync(~0u, slot_taken(p.slots_out, n, out_slot, lane, 32));
    // No state is stored before the first one's loads are done (in place at D = 64 quadrants 2 and 3 load the
    // rows that 0 and 1 store), and, where one is not finite, before columns have been made from them again
    // (those with a state of their own are marked as stored).
    uint64_t seen = 0;  // two zeros; NaN once a state is not finite
#pragma unroll
    for (int i = 0; i < KT / 2; ++i) seen = fma_f32x2(S[i], 0, seen);
    if (f32x2_lo(seen) != 0.f || f32x2_hi(seen) != 0.f) *any_spoiled = 1;
    if (!alive) *stalled = 1;
    asm volatile("bar.sync 2, 512;" ::: "memory");
    if (*any_spoiled) asm volatile("bar.sync 2, 512;" ::: "memory");
    if (*stalled) {  // the caller sees it in the state
#pragma unroll
      for (int i = 0; i < KT / 2; ++i) S[i] = f32x2_splat(__int_as_float(0x7fffffff));
    }
    if (writes && (spoiled_at[vr] >= 0 || *stalled) && (OUT ? last && out_slot >= 0 && !taken : true)) {
      float* dst = (OUT ? p.ht + (out_slot * p.H + h) * D * D : p.seg_states + seg_state) + col_off;
#pragma unroll
      for (int i = 0; i < KT; i += 2) {
        dst[i * D] = f32x2_lo(S[i / 2]);
        dst[(i + 1) * D] = f32x2_hi(S[i / 2]);
      }
    }
  }
  if (!alive) atomicOr(&g_linear_status, 1);
  tc::fence_before();
  __syncthreads();
  if (warp == 0) tc::dealloc(tmem, 512);
}

}  // namespace memt
