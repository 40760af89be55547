// Pieces of the gated linear recurrence: types, strided inputs, the gate, the shape of a tile.
#pragma once
#include "common.cuh"

namespace frnnt {

// Steps between two states that the forward keeps for the backward, and of one tile: one float
// per channel every 128 steps is 1.6 % of 16-bit values and gates, and the backward recomputes
// a tile from its state instead of reading h.
constexpr int kRecChunk = 128;
constexpr int kRecThreads = 256;
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
template <typename T, int VEC> __device__ __forceinline__ RecPack<T, VEC> rec_pack(const RecState<T> (&v)[VEC]) {
  T e[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) e[k] = rec_round<T>(v[k]);
  RecPack<T, VEC> p;
  memcpy(&p, e, sizeof(p));
  return p;
}

// keep = sigmoid(g) and take = 1 - keep from one exponential of -|g|, which cannot overflow;
// take is never the difference of two numbers near one.  16-bit inputs take the hardware's
// exponential and division (relative error 2^-20, far below the 2^-9 / 2^-12 of their outputs).
template <typename T> __device__ __forceinline__ void gate_pair(RecState<T> g, RecState<T> &keep, RecState<T> &take) {
  using real = RecState<T>;
  real e, r;
  if constexpr (sizeof(T) == 2) {
    e = __expf(-fabsf(g));
    r = __fdividef(1.0f, 1.0f + e);
  } else {
    e = exp_r(-fabs(g));
    r = real(1) / (real(1) + e);
  }
  keep = g >= 0 ? r : e * r;
  take = g >= 0 ? e * r : r;
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
  static constexpr int kJoiners = kJoin * kWidth;
  static_assert(kSteps * kPieces == kRecChunk && kJoiners <= kRecThreads && kJoin <= 4, "shape");
  // offset of (piece, channel) in the exchange: runs are skewed by 8 so that the kJoin threads
  // of eight channels, which share a warp, hit different banks
  static __device__ __forceinline__ int at(int piece, int c) { return piece * kWidth + (piece / kRun) * 8 + c; }
  static constexpr int kExchange = kPieces * kWidth + kJoin * 8;   // values of one array
  static constexpr int kStage = kRecThreads * kSteps * VEC * (int)sizeof(T);   // bytes of one input's tile
};

}  // namespace frnnt
