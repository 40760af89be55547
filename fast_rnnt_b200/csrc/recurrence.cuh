// Pieces of the gated linear recurrence: types, strided inputs, the gate.
#pragma once
#include "common.cuh"

namespace frnnt {

// Steps between two states that the forward keeps for the backward: one float per channel every
// 128 steps is 1.6 % of 16-bit values and gate, and the backward recomputes a chunk from its state.
constexpr int kRecChunk = 128;

// states, and everything computed, are 32 bits wide (64 for doubles)
template <typename T> struct RecStateOf { using type = float; };
template <> struct RecStateOf<double> { using type = double; };
template <typename T> using RecState = typename RecStateOf<T>::type;

// [B][T][D] with channels side by side and any strides (in elements) between batches and steps
struct RecTensor {
  const void *data;
  long long batch, step;
  template <typename T> __device__ __forceinline__ const T *row(int b, int t) const {
    return (const T *)data + b * batch + t * step;
  }
};

template <typename T> __device__ __forceinline__ RecState<T> rec_load(const T *p) { return in_f32(*p); }
template <> __device__ __forceinline__ double rec_load<double>(const double *p) { return *p; }

// the one rounding of an output to its 16-bit type
template <typename T> __device__ __forceinline__ T rec_store(RecState<T> v) { return v; }
template <> __device__ __forceinline__ __half rec_store<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rec_store<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// keep = sigmoid(g) and take = 1 - keep from one exponential of -|g|, which cannot overflow;
// take is never the difference of two numbers near one.
template <typename real> __device__ __forceinline__ void gate_pair(real g, real &keep, real &take) {
  const real e = exp_r(-fabs(g)), r = real(1) / (real(1) + e);
  keep = g >= 0 ? r : e * r;
  take = g >= 0 ? e * r : r;
}

}  // namespace frnnt
