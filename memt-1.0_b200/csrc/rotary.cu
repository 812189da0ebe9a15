// memt_rotary, memt_rotary_axes: rotary positions of queries and keys, both in one launch.
//
// Pair i of a head (elements i and i + R/2 in the half layout, 2i and 2i + 1 in the interleaved
// one) at position p is turned by the angle p * inv_freq[i]:
//     y_a = c x_a - s x_b,   y_b = c x_b + s x_a,   (c, s) = scale * (cos, sin)(p * inv_freq[i])
// and the inverse (the operator's own backward pass) turns by the negative angle. With several axes (AXES)
// a token has a position on each and pair i takes that of its axis (65,536 tokens, 16 + 16 heads of 128, bf16, per call:
// 176 us with three axes, 169 with one, 164 at the measured copy rate).
//
// The angle is formed and reduced to a fraction of a turn in 64 bits: at position 10^6 an fp32
// product is off by 0.03 radians. Sine and cosine of the fraction, and the rotation, are fp32;
// the result is rounded once.
//
// Bound by HBM: every element is read and written once, in 16-byte vectors. A thread owns one
// vector of pairs of one token, evaluates its sines and cosines once and walks over heads with
// them, four heads in flight, so their cost is shared by the heads it walks. Few tokens leave SMs idle
// that way; the heads of a token are then spread over more threads, which each evaluate the angles
// again. The vectors behind the rotary part are copied by threads of their own, behind all others
// in the grid, so that no warp does both.
#include "launch.h"
#include "overlap.h"

namespace {

using namespace memt;

struct RotaryParams {
  int64_t L;
  int32_t Hq, Hk, D, R;
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int64_t sq, sk, sqo, sko;  // elements per token row
  const void* pos;
  int32_t pos64;
  int32_t axes;              // AXES: rows of pos, pos_stride elements apart
  int64_t pos_stride;
  const int32_t* pair_axes;  // row of each pair; a pair outside of them stays at position 0
  const double* inv_freq;
  float scale;
  int32_t inverse, interleaved;
  int32_t groups;     // threads a token's heads are spread over
  int32_t rot_units;  // vectors (pairs of vectors in the half layout) that turn, per head
  int32_t copy_units;  // vectors behind the rotary part that are copied, per head
};

// Thread `idx` of `per_token` for each token -> (token, thread of it); 32-bit division where it suffices.
__device__ __forceinline__ int64_t split(int64_t idx, int per_token, int& rest) {
  if (idx <= 0xffffffffll) {
    const uint32_t t = static_cast<uint32_t>(idx) / static_cast<uint32_t>(per_token);
    rest = static_cast<int>(static_cast<uint32_t>(idx) - t * per_token);
    return t;
  }
  const int64_t t = idx / per_token;
  rest = static_cast<int>(idx - t * per_token);
  return t;
}

__device__ __forceinline__ double position(const RotaryParams& p, int64_t t) {
  return p.pos64 ? static_cast<double>(static_cast<const int64_t*>(p.pos)[t])
                 : static_cast<double>(static_cast<const int32_t*>(p.pos)[t]);
}

__device__ __forceinline__ void angle(const RotaryParams& p, double pos, int pair, float& c, float& s) {
  constexpr double kInvTwoPi = 0.15915494309189533577;
  double turns = pos * p.inv_freq[pair] * kInvTwoPi;
  turns -= rint(turns);
  sincospif(2.0f * static_cast<float>(turns), &s, &c);
  c *= p.scale;
  s *= p.inverse ? -p.scale : p.scale;
}

// the position that turns `pair` of token t (`pos`: the token's only one, without axes)
template <bool AXES>
__device__ __forceinline__ double pair_position(const RotaryParams& p, double pos, int64_t t, int pair) {
  if constexpr (!AXES) return pos;
  const int axis = p.pair_axes[pair];
  return axis >= 0 && axis < p.axes ? position(p, axis * p.pos_stride + t) : 0.0;
}

// one 16-byte vector as fp32 values, and back
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = unpack_bf16x2(w[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

template <typename T>
__device__ __forceinline__ void head_ptrs(const RotaryParams& p, int64_t t, int h, const T*& x, T*& y) {
  if (h < p.Hq) {
    x = static_cast<const T*>(p.q) + t * p.sq + (int64_t)h * p.D;
    y = static_cast<T*>(p.q_out) + t * p.sqo + (int64_t)h * p.D;
  } else {
    x = static_cast<const T*>(p.k) + t * p.sk + (int64_t)(h - p.Hq) * p.D;
    y = static_cast<T*>(p.k_out) + t * p.sko + (int64_t)(h - p.Hq) * p.D;
  }
}

// 16-byte vectors. kHeads heads are in flight per thread at a time.
template <typename T, bool INTERLEAVED, bool AXES>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  constexpr int V = Vec<T>::N;
  constexpr int kPairs = INTERLEAVED ? V / 2 : V;
  constexpr int kHeads = 4;
  int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int H = p.Hq + p.Hk;
  const int64_t turning = p.L * p.rot_units * p.groups;
  int rest;
  if (idx >= turning) {  // behind the rotary part: copied
    if (p.copy_units == 0) return;
    const int64_t t = split(idx - turning, p.copy_units * p.groups, rest);
    if (t >= p.L) return;
    const int group = rest / p.copy_units, col = p.R + (rest - group * p.copy_units) * V;
    for (int h0 = group; h0 < H; h0 += kHeads * p.groups) {
      uint4 a[kHeads];
#pragma unroll
      for (int j = 0; j < kHeads; ++j) {
        const int h = h0 + j * p.groups;
        const T* x;
        T* y;
        if (h < H) {
          head_ptrs(p, t, h, x, y);
          a[j] = *reinterpret_cast<const uint4*>(x + col);
        }
      }
#pragma unroll
      for (int j = 0; j < kHeads; ++j) {
        const int h = h0 + j * p.groups;
        const T* x;
        T* y;
        if (h < H) {
          head_ptrs(p, t, h, x, y);
          *reinterpret_cast<uint4*>(y + col) = a[j];
        }
      }
    }
    return;
  }
  const int64_t t = split(idx, p.rot_units * p.groups, rest);
  const int group = rest / p.rot_units, unit = rest - group * p.rot_units;
  float c[kPairs], s[kPairs];
  const double pos = AXES ? 0.0 : position(p, t);
#pragma unroll
  for (int i = 0; i < kPairs; ++i)
    angle(p, pair_position<AXES>(p, pos, t, unit * kPairs + i), unit * kPairs + i, c[i], s[i]);
  const int col = unit * V, half = p.R >> 1;
  for (int h0 = group; h0 < H; h0 += kHeads * p.groups) {
    uint4 a[kHeads], b[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = h0 + j * p.groups;
      if (h < H) {
        const T* x;
        T* y;
        head_ptrs(p, t, h, x, y);
        a[j] = *reinterpret_cast<const uint4*>(x + col);
        if constexpr (!INTERLEAVED) b[j] = *reinterpret_cast<const uint4*>(x + half + col);
      }
    }
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = h0 + j * p.groups;
      if (h < H) {
        const T* x;
        T* y;
        head_ptrs(p, t, h, x, y);
        float fa[V], fb[V], ya[V], yb[V];
        Vec<T>::unpack(a[j], fa);
        if constexpr (INTERLEAVED) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            ya[2 * i] = c[i] * fa[2 * i] - s[i] * fa[2 * i + 1];
            ya[2 * i + 1] = c[i] * fa[2 * i + 1] + s[i] * fa[2 * i];
          }
        } else {
          Vec<T>::unpack(b[j], fb);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            ya[i] = c[i] * fa[i] - s[i] * fb[i];
            yb[i] = c[i] * fb[i] + s[i] * fa[i];
          }
          *reinterpret_cast<uint4*>(y + half + col) = Vec<T>::pack(yb);
        }
        *reinterpret_cast<uint4*>(y + col) = Vec<T>::pack(ya);
      }
    }
  }
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void store(float* y, float x) { *y = x; }
__device__ __forceinline__ void store(__nv_bfloat16* y, float x) { *y = __float2bfloat16_rn(x); }

// Rows or rotary parts that are not whole 16-byte vectors: one pair (or copied element) a thread.
template <typename T, bool AXES>
__global__ void __launch_bounds__(256) rotary_scalar_kernel(const RotaryParams p) {
  constexpr int kHeads = 4;
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int units = p.rot_units + p.copy_units;
  int rest;
  const int64_t t = split(idx, units * p.groups, rest);
  if (t >= p.L) return;
  const int group = rest / units, unit = rest - group * units;
  const int H = p.Hq + p.Hk, half = p.R >> 1;
  const bool turns = unit < p.rot_units;
  const int ia = turns ? (p.interleaved ? 2 * unit : unit) : p.R + unit - p.rot_units;
  const int ib = turns ? (p.interleaved ? ia + 1 : ia + half) : ia;
  float c = 1.f, s = 0.f;
  if (turns) angle(p, pair_position<AXES>(p, AXES ? 0.0 : position(p, t), t, unit), unit, c, s);
  for (int h0 = group; h0 < H; h0 += kHeads * p.groups) {
    T a[kHeads], b[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = h0 + j * p.groups;
      const T* x;
      T* y;
      if (h < H) {
        head_ptrs(p, t, h, x, y);
        a[j] = x[ia];
        b[j] = x[ib];
      }
    }
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = h0 + j * p.groups;
      const T* x;
      T* y;
      if (h < H) {
        head_ptrs(p, t, h, x, y);
        if (turns) {
          const float fa = to_float(a[j]), fb = to_float(b[j]);
          store(y + ia, c * fa - s * fb);
          store(y + ib, c * fb + s * fa);
        } else {
          y[ia] = a[j];
        }
      }
    }
  }
}

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

template <typename T, bool AXES>
int launch_rotary(RotaryParams& p, bool copy_rest, int sms, cudaStream_t s) {
  constexpr int V = Vec<T>::N;
  bool vec = p.D % V == 0 && (p.interleaved ? p.R % V == 0 : p.R % (2 * V) == 0);
  const int64_t strides[] = {p.sq, p.sqo, p.Hk > 0 ? p.sk : 0, p.Hk > 0 ? p.sko : 0};
  for (int64_t st : strides) vec = vec && st % V == 0;
  vec = vec && aligned16(p.q) && aligned16(p.q_out) && aligned16(p.k) && aligned16(p.k_out);
  const int per_unit = vec ? (p.interleaved ? V : 2 * V) : 2;  // rotary elements per unit
  p.rot_units = p.R / per_unit;
  p.copy_units = copy_rest ? (p.D - p.R) / (vec ? V : 1) : 0;
  // threads for two full waves at 1024 threads an SM, as far as there are heads to spread
  const int64_t want = int64_t(sms) * 2048, have = p.L * (p.rot_units + p.copy_units);
  const int H = p.Hq + p.Hk;
  int64_t groups = have > 0 ? (want + have - 1) / have : 1;
  if (groups > H) groups = H;
  if (groups < 1) groups = 1;
  p.groups = static_cast<int32_t>(groups);
  const int64_t blocks = (have * groups + 255) / 256;
  if (blocks > INT32_MAX) return MEMT_ERR_UNSUPPORTED;
  ProfScope prof(kProfRotary, s);
  const unsigned grid = static_cast<unsigned>(blocks);
  if (!vec)
    rotary_scalar_kernel<T, AXES><<<grid, 256, 0, s>>>(p);
  else if (p.interleaved)
    rotary_kernel<T, true, AXES><<<grid, 256, 0, s>>>(p);
  else
    rotary_kernel<T, false, AXES><<<grid, 256, 0, s>>>(p);
  return cuda_status(cudaGetLastError());
}

// Both entry points: `a` without its struct_size; axes 0: one position a token, else as in memt_rotary_axes_args.
int rotary(const memt_rotary_args* a, int axes, const int32_t* pair_axes, int64_t pos_stride, cudaStream_t s) {
  if (a->total_tokens < 0 || a->num_heads < 1 || a->num_key_heads < 0 || a->head_dim < 2 || a->rotary_dim < 2 ||
      a->rotary_dim % 2 != 0 || a->rotary_dim > a->head_dim || (a->dtype != MEMT_BF16 && a->dtype != MEMT_F32) ||
      a->inv_freq == nullptr || a->positions == nullptr || a->q == nullptr || a->q_out == nullptr)
    return MEMT_ERR_INVALID_ARGUMENT;
  const int64_t qrow = int64_t(a->num_heads) * a->head_dim, krow = int64_t(a->num_key_heads) * a->head_dim;
  if (a->q_stride < qrow || a->q_out_stride < qrow) return MEMT_ERR_INVALID_ARGUMENT;
  if (a->num_key_heads > 0 &&
      (a->k == nullptr || a->k_out == nullptr || a->k_stride < krow || a->k_out_stride < krow))
    return MEMT_ERR_INVALID_ARGUMENT;
  if (a->total_tokens == 0) return MEMT_OK;
  {  // every thread reads positions and angles, other threads' outputs must not lie there
    const int64_t size = a->dtype == MEMT_BF16 ? 2 : 4, L = a->total_tokens, each = a->positions_int64 != 0 ? 8 : 4;
    const Rows pos(a->positions, L * each, axes > 1 ? pos_stride * each : L * each, axes > 1 ? axes : 1);
    const Rows inv(a->inv_freq, int64_t(a->rotary_dim) * 4), pairs(pair_axes, int64_t(a->rotary_dim) * 2);
    const Rows qo(a->q_out, qrow * size, a->q_out_stride * size, L);
    const Rows ko(a->num_key_heads > 0 ? a->k_out : nullptr, krow * size, a->k_out_stride * size, L);
    if (overlaps_any(qo, {pos, inv, pairs}) || overlaps_any(ko, {pos, inv, pairs})) return MEMT_ERR_INVALID_ARGUMENT;
  }
  RotaryParams p{};
  p.L = a->total_tokens;
  p.Hq = a->num_heads;
  p.Hk = a->num_key_heads;
  p.D = a->head_dim;
  p.R = a->rotary_dim;
  p.q = a->q;
  p.q_out = a->q_out;
  p.sq = a->q_stride;
  p.sqo = a->q_out_stride;
  if (p.Hk > 0) {
    p.k = a->k;
    p.k_out = a->k_out;
    p.sk = a->k_stride;
    p.sko = a->k_out_stride;
  }
  p.pos = a->positions;
  p.pos64 = a->positions_int64 != 0;
  p.axes = axes;
  p.pos_stride = pos_stride;
  p.pair_axes = pair_axes;
  p.inv_freq = a->inv_freq;
  p.scale = a->attention_scale;
  p.inverse = a->inverse != 0;
  p.interleaved = a->interleaved != 0;
  int sms = 0;
  const int st = device_sms(&sms);
  if (st != MEMT_OK) return st;
  // in place, the elements behind the rotary part stay where they are
  const bool in_place = p.q == p.q_out && (p.Hk == 0 || p.k == p.k_out);
  if (axes > 0)
    return a->dtype == MEMT_BF16 ? launch_rotary<__nv_bfloat16, true>(p, !in_place, sms, s)
                                 : launch_rotary<float, true>(p, !in_place, sms, s);
  return a->dtype == MEMT_BF16 ? launch_rotary<__nv_bfloat16, false>(p, !in_place, sms, s)
                               : launch_rotary<float, false>(p, !in_place, sms, s);
}

}  // namespace

extern "C" {

int memt_rotary(const memt_rotary_args* a, memt_stream_t stream) try {
  if (a == nullptr || a->struct_size != sizeof(memt_rotary_args)) return MEMT_ERR_INVALID_ARGUMENT;
  return rotary(a, 0, nullptr, 0, reinterpret_cast<cudaStream_t>(stream));
} catch (...) {  // the launch bookkeeping may run out of host memory
  return MEMT_ERR_CUDA;
}

int memt_rotary_axes(const memt_rotary_axes_args* a, memt_stream_t stream) try {
  if (a == nullptr || a->struct_size != sizeof(memt_rotary_axes_args)) return MEMT_ERR_INVALID_ARGUMENT;
  if (a->num_axes < 1 || a->pair_axes == nullptr || (a->num_axes > 1 && a->position_stride < a->total_tokens))
    return MEMT_ERR_INVALID_ARGUMENT;
  const memt_rotary_args one = {sizeof(memt_rotary_args), a->num_heads, a->num_key_heads, a->head_dim, a->rotary_dim,
                                a->dtype, a->total_tokens, a->q, a->q_stride, a->k, a->k_stride, a->q_out,
                                a->q_out_stride, a->k_out, a->k_out_stride, a->positions, a->positions_int64,
                                a->interleaved, a->inv_freq, a->attention_scale, a->inverse};
  return rotary(&one, a->num_axes, a->pair_axes, a->position_stride, reinterpret_cast<cudaStream_t>(stream));
} catch (...) {
  return MEMT_ERR_CUDA;
}

}  // extern "C"
