// Pieces of the gated linear recurrence: types, strided inputs, the gate, the shape of a tile.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace frnnt {

// Steps between two states that the forward keeps for the backward, and of one tile: one float
// per channel every 128 steps is 1.6 % of 16-bit values and gates, and the backward recomputes
// a tile from its state instead of reading h.
constexpr int kRecChunk = 128;
constexpr int kRecThreads = 128;
constexpr int kRecWarps = kRecThreads / 32;

// states, and everything computed, are 32 bits wide (64 for doubles)
template <typename T> struct RecStateOf { using type = float; };
template <> struct RecStateOf<double> { using type = double; };
template <typename T> using RecState = typename RecStateOf<T>::type;

// [B][T][D] with channels side by side and any strides (in elements) between batches and steps
struct RecTensor {
  const void *data;
  long long batch, step;
};

// steps of utterance b, within [0, T] whatever the tensor holds
__device__ __forceinline__ int steps_of(const int64_t *lengths, int b, int T) {
  if (lengths == nullptr) return T;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : n > T ? T : (int)n;
}

// ---- bytes <-> values -----------------------------------------------------------
template <int BYTES> struct RecPackOf;
template <> struct RecPackOf<2> { using type = uint16_t; };
template <> struct RecPackOf<4> { using type = uint32_t; };
template <> struct RecPackOf<8> { using type = uint2; };
template <> struct RecPackOf<16> { using type = uint4; };
template <typename T, int VEC> using RecPack = typename RecPackOf<(int)sizeof(T) * VEC>::type;

template <typename T> __device__ __forceinline__ RecState<T> rec_value(T v) { return in_f32(v); }
template <> __device__ __forceinline__ double rec_value<double>(double v) { return v; }
// the one rounding of an output to its 16-bit type
template <typename T> __device__ __forceinline__ T rec_round(RecState<T> v) { return v; }
template <> __device__ __forceinline__ __half rec_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rec_round<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <typename T, int VEC>
__device__ __forceinline__ void rec_unpack(const RecPack<T, VEC> &p, RecState<T> (&v)[VEC]) {
  T e[VEC];
  memcpy(e, &p, sizeof(p));
#pragma unroll
  for (int k = 0; k < VEC; ++k) v[k] = rec_value<T>(e[k]);
}
// a vector of one value
template <typename T, int VEC> __device__ __forceinline__ RecPack<T, VEC> rec_fill(float value) {
  T e[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) e[k] = T(value);
  RecPack<T, VEC> p;
  memcpy(&p, e, sizeof(p));
  return p;
}
template <typename T, int VEC> __device__ __forceinline__ RecPack<T, VEC> rec_pack(const RecState<T> (&v)[VEC]) {
  T e[VEC];
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {   // two at a time
#pragma unroll
    for (int k = 0; k < VEC; k += 2) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 q = __floats2half2_rn(v[k], v[k + 1]);
        e[k] = q.x, e[k + 1] = q.y;
      } else {
        const __nv_bfloat162 q = __floats2bfloat162_rn(v[k], v[k + 1]);
        e[k] = q.x, e[k + 1] = q.y;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) e[k] = rec_round<T>(v[k]);
  }
  RecPack<T, VEC> p;
  memcpy(&p, e, sizeof(p));
  return p;
}

// ---- arithmetic on the channels of a thread: floats two at a time (half the instructions) -------
#define FRNNT_REC_EACH(PAIR, ONE)                                              \
  if constexpr (sizeof(real) == 4 && VEC % 2 == 0) {                           \
    _Pragma("unroll") for (int k = 0; k < VEC; k += 2) {                       \
      const float2 r = PAIR;                                                   \
      out[k] = r.x, out[k + 1] = r.y;                                          \
    }                                                                          \
  } else {                                                                     \
    _Pragma("unroll") for (int k = 0; k < VEC; ++k) out[k] = ONE;              \
  }
#define FRNNT_REC_PAIR(v) make_float2((float)v[k], (float)v[k + 1])
template <typename real, int VEC>
__device__ __forceinline__ void vmul(real (&out)[VEC], const real (&a)[VEC], const real (&b)[VEC]) {
  FRNNT_REC_EACH(__fmul2_rn(FRNNT_REC_PAIR(a), FRNNT_REC_PAIR(b)), a[k] * b[k])
}
template <typename real, int VEC>
__device__ __forceinline__ void vadd(real (&out)[VEC], const real (&a)[VEC], const real (&b)[VEC]) {
  FRNNT_REC_EACH(__fadd2_rn(FRNNT_REC_PAIR(a), FRNNT_REC_PAIR(b)), a[k] + b[k])
}
template <typename real, int VEC>
__device__ __forceinline__ void vfma(real (&out)[VEC], const real (&a)[VEC], const real (&b)[VEC], const real (&c)[VEC]) {
  FRNNT_REC_EACH(__ffma2_rn(FRNNT_REC_PAIR(a), FRNNT_REC_PAIR(b), FRNNT_REC_PAIR(c)), a[k] * b[k] + c[k])
}
template <typename real, int VEC>   // a - b
__device__ __forceinline__ void vsub(real (&out)[VEC], const real (&a)[VEC], const real (&b)[VEC]) {
  FRNNT_REC_EACH(__ffma2_rn(FRNNT_REC_PAIR(b), make_float2(-1.0f, -1.0f), FRNNT_REC_PAIR(a)), a[k] - b[k])
}
template <typename real, int VEC> __device__ __forceinline__ void vset(real (&out)[VEC], real value) {
#pragma unroll
  for (int k = 0; k < VEC; ++k) out[k] = value;
}
#undef FRNNT_REC_EACH
#undef FRNNT_REC_PAIR

// keep = sigmoid(g) and take = 1 - keep from one exponential of -|g|, which cannot overflow.  The
// smaller of the two is a product, never the difference of two numbers near one, and the larger is
// one less that product, rounded once: off by 2^-25 where the other is small.  (As the reciprocal of
// the rounded 1 + e it was off by up to 2^-23: the state after 30000 steps at a gate of 12 by 1.7e-3,
// now 1.2e-4; the one instruction more costs a hundredth of the time.)  The reciprocal of 1 .. 2 is
// the hardware's (within one unit in the last place); for 16-bit inputs the exponential is, too: a
// relative error of (4 + 1.3 |g|) 2^-24, 2^-17 at most where it is not zero, below the 2^-9 / 2^-12
// of their outputs.
template <typename T> __device__ __forceinline__ RecState<T> rec_exp(RecState<T> x) { return exp_r(x); }
__device__ __forceinline__ float rec_exp_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}
template <> __device__ __forceinline__ float rec_exp<__half>(float x) { return rec_exp_fast(x); }
template <> __device__ __forceinline__ float rec_exp<__nv_bfloat16>(float x) { return rec_exp_fast(x); }
__device__ __forceinline__ float rec_reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ double rec_reciprocal(double x) { return 1.0 / x; }
template <typename T> __device__ __forceinline__ void gate_pair(RecState<T> g, RecState<T> &keep, RecState<T> &take) {
  const RecState<T> e = rec_exp<T>(-fabs(g)), r = rec_reciprocal(1 + e), small = e * r, large = fma(-e, r, RecState<T>(1));
  keep = g >= 0 ? large : small;
  take = g >= 0 ? small : large;
}

// ---- the tile of a CTA ------------------------------------------------------------
// kRecChunk steps of LC * VEC channels: LC lanes of a warp side by side along the channels, each
// with VEC of them, the 32 / LC groups of lanes and then the warps one after the other along
// time, kSteps consecutive steps each ("piece").
template <typename T_, int VEC_, int LC_> struct RecShape {
  using T = T_;
  using real = RecState<T>;
  static constexpr int VEC = VEC_, LC = LC_;
  static constexpr int kGroups = 32 / LC;                       // of lanes along time
  static constexpr int kPieces = kRecWarps * kGroups;           // of a tile along time
  static constexpr int kSteps = kRecChunk / kPieces;            // of a piece
  static constexpr int kWidth = LC * VEC;                       // channels
  // joining the pieces: kJoin threads per channel with kRun consecutive pieces each
  static constexpr int kRun = kPieces < 8 ? kPieces : 8;
  static constexpr int kJoin = kPieces / kRun;
  static constexpr int kSegment = 8 * kJoin;                    // lanes with all runs of eight channels
  static_assert(kSteps * kPieces == kRecChunk && kJoin * kWidth <= kRecThreads && kJoin <= 4 && kWidth % 8 == 0, "shape");
  // offset of (piece, channel) in the exchange: runs are skewed by 8 so that the kJoin threads
  // of eight channels, which share a warp, hit different banks
  static __device__ __forceinline__ int at(int piece, int c) { return piece * kWidth + (piece / kRun) * 8 + c; }
  static constexpr int kExchange = kPieces * kWidth + kJoin * 8;   // values of one array
  static constexpr int kStage = kRecThreads * kSteps * VEC * (int)sizeof(T);   // bytes of one input's tile
};

}  // namespace frnnt
