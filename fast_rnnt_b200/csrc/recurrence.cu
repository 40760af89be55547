// Gated linear recurrence: h_t = f_t h_{t-1} + (1 - f_t) x_t with f = sigmoid(gate).
//
// Forward and backward over whole sequences, and one token for decoding.
#include "common.cuh"
#include "recurrence.cuh"

namespace frnnt {

constexpr int kRecThreads = 128;

// steps of utterance b, within [0, T] whatever the tensor holds
__device__ __forceinline__ int steps_of(const int64_t *lengths, int b, int T) {
  if (lengths == nullptr) return T;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : n > T ? T : (int)n;
}

template <typename T>
__global__ void __launch_bounds__(kRecThreads)
recurrence_forward_kernel(RecTensor x, RecTensor gate, const RecState<T> *__restrict__ initial,
                          const int64_t *__restrict__ lengths, T *__restrict__ h,
                          RecState<T> *__restrict__ last, RecState<T> *__restrict__ saved, int steps, int D) {
  using real = RecState<T>;
  const int b = blockIdx.y, d = blockIdx.x * kRecThreads + threadIdx.x;
  if (d >= D) return;
  const int n = steps_of(lengths, b, steps);
  const T *X = x.row<T>(b, 0) + d, *G = gate.row<T>(b, 0) + d;
  T *H = h + (size_t)b * steps * D + d;
  const int chunks = (steps + kRecChunk - 1) / kRecChunk;
  real state = initial != nullptr ? initial[(size_t)b * D + d] : real(0);
  for (int t = 0; t < n; ++t) {
    if (saved != nullptr && t % kRecChunk == 0) saved[((size_t)b * chunks + t / kRecChunk) * D + d] = state;
    real keep, take;
    gate_pair(rec_load(G + t * gate.step), keep, take);
    state = keep * state + take * rec_load(X + t * x.step);
    H[(size_t)t * D] = rec_store<T>(state);
  }
  for (int t = n; t < steps; ++t) H[(size_t)t * D] = rec_store<T>(real(0));
  last[(size_t)b * D + d] = state;
}

template <typename T>
__global__ void __launch_bounds__(kRecThreads)
recurrence_backward_kernel(RecTensor x, RecTensor gate, const int64_t *__restrict__ lengths,
                           const RecState<T> *__restrict__ saved, RecTensor dh,
                           const RecState<T> *__restrict__ dlast, T *__restrict__ dx, T *__restrict__ dgate,
                           RecState<T> *__restrict__ dinitial, int steps, int D) {
  using real = RecState<T>;
  const int b = blockIdx.y, d = blockIdx.x * kRecThreads + threadIdx.x;
  if (d >= D) return;
  const int n = steps_of(lengths, b, steps);
  const T *X = x.row<T>(b, 0) + d, *G = gate.row<T>(b, 0) + d;
  const T *DH = dh.data != nullptr ? dh.row<T>(b, 0) + d : nullptr;
  T *DX = dx + (size_t)b * steps * D + d, *DG = dgate + (size_t)b * steps * D + d;
  const int chunks = (steps + kRecChunk - 1) / kRecChunk;
  real flow = dlast != nullptr ? dlast[(size_t)b * D + d] : real(0);
  for (int t = n; t < steps; ++t) DX[(size_t)t * D] = DG[(size_t)t * D] = rec_store<T>(real(0));
  real before[kRecChunk];
  for (int c = (n + kRecChunk - 1) / kRecChunk - 1; c >= 0; --c) {
    const int t0 = c * kRecChunk, t1 = min(n, t0 + kRecChunk);
    real state = saved[((size_t)b * chunks + c) * D + d], keep, take;
    for (int t = t0; t < t1; ++t) {
      before[t - t0] = state;
      gate_pair(rec_load(G + t * gate.step), keep, take);
      state = keep * state + take * rec_load(X + t * x.step);
    }
    for (int t = t1 - 1; t >= t0; --t) {
      gate_pair(rec_load(G + t * gate.step), keep, take);
      const real lam = flow + (DH != nullptr ? rec_load(DH + t * dh.step) : real(0));
      DX[(size_t)t * D] = rec_store<T>(take * lam);
      DG[(size_t)t * D] = rec_store<T>(lam * (before[t - t0] - rec_load(X + t * x.step)) * keep * take);
      flow = keep * lam;
    }
  }
  if (dinitial != nullptr) dinitial[(size_t)b * D + d] = flow;
}

// One token: every row reads the state of its parent (its own without parents; zero where the
// parent is not one of the K rows) and writes the new state and its rounding to x's type.
template <typename T>
__global__ void __launch_bounds__(kRecThreads)
recurrence_step_kernel(const T *__restrict__ x, long long x_row, const T *__restrict__ gate, long long gate_row,
                       const RecState<T> *__restrict__ state, const int64_t *__restrict__ parents,
                       T *__restrict__ h, RecState<T> *__restrict__ next, long long rows, int beams, int K, int D) {
  using real = RecState<T>;
  const int d = blockIdx.x * kRecThreads + threadIdx.x;
  if (d >= D) return;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    long long from = row;
    if (parents != nullptr) {
      const int64_t p = parents[row];
      from = p < 0 || p >= K ? -1 : div_rows(row, beams) * K + p;
    }
    real keep, take;
    gate_pair(rec_load(gate + row * gate_row + d), keep, take);
    const real old = from < 0 ? real(0) : state[from * D + d];
    const real now = keep * old + take * rec_load(x + row * x_row + d);
    next[row * D + d] = now;
    if (h != nullptr) h[row * D + d] = rec_store<T>(now);
  }
}

}  // namespace frnnt

using namespace frnnt;

#define FRNNT_REC_TYPES(CALL) \
  switch (dtype) {            \
    case FRNNT_F32: CALL(float); break;           \
    case FRNNT_F64: CALL(double); break;          \
    case FRNNT_F16: CALL(__half); break;          \
    default: CALL(__nv_bfloat16); break;          \
  }

static bool rec_dtype(int dtype) {
  return dtype == FRNNT_F32 || dtype == FRNNT_F64 || dtype == FRNNT_F16 || dtype == FRNNT_BF16;
}
static bool rec_sizes(int B, int T, int D) { return B >= 0 && T >= 0 && D >= 0; }

extern "C" size_t frnnt_recurrence_saved_bytes(int dtype, int B, int T, int D) {
  if (!rec_dtype(dtype) || B <= 0 || T <= 0 || D <= 0) return 0;
  return (size_t)B * ((T + kRecChunk - 1) / kRecChunk) * D * (dtype == FRNNT_F64 ? 8 : 4);
}

extern "C" int frnnt_recurrence_forward(int dtype, const void *x, long long x_batch, long long x_step,
                                        const void *gate, long long gate_batch, long long gate_step,
                                        const void *initial, const int64_t *lengths, void *h, void *last,
                                        void *saved, int B, int T, int D, void *stream) {
  FRNNT_REQUIRE(rec_dtype(dtype), FRNNT_EINVAL, "dtype must be FRNNT_F32, _F64, _F16 or _BF16");
  FRNNT_REQUIRE(rec_sizes(B, T, D), FRNNT_EINVAL, "bad sizes");
  FRNNT_REQUIRE(B <= 65535, FRNNT_EUNSUPPORTED, "B too large for the grid");
  if (B == 0 || D == 0) return FRNNT_OK;
  FRNNT_REQUIRE(last && (T == 0 || (x && gate && h)), FRNNT_EINVAL, "NULL argument");
  cudaStream_t st = (cudaStream_t)stream;
  const RecTensor X{x, x_batch, x_step}, G{gate, gate_batch, gate_step};
  const dim3 grid((unsigned)((D + kRecThreads - 1) / kRecThreads), (unsigned)B);
#define FRNNT_REC_FORWARD(TYPE)                                                             \
  FRNNT_KERNEL(recurrence_forward_kernel<TYPE><<<grid, kRecThreads, 0, st>>>(               \
      X, G, (const RecState<TYPE> *)initial, lengths, (TYPE *)h, (RecState<TYPE> *)last,    \
      (RecState<TYPE> *)saved, T, D))
  FRNNT_REC_TYPES(FRNNT_REC_FORWARD)
#undef FRNNT_REC_FORWARD
  FRNNT_CUDA(cudaGetLastError());
  return FRNNT_OK;
}

extern "C" int frnnt_recurrence_backward(int dtype, const void *x, long long x_batch, long long x_step,
                                         const void *gate, long long gate_batch, long long gate_step,
                                         const int64_t *lengths, const void *saved, const void *dh,
                                         long long dh_batch, long long dh_step, const void *dlast, void *dx,
                                         void *dgate, void *dinitial, int B, int T, int D, void *stream) {
  FRNNT_REQUIRE(rec_dtype(dtype), FRNNT_EINVAL, "dtype must be FRNNT_F32, _F64, _F16 or _BF16");
  FRNNT_REQUIRE(rec_sizes(B, T, D), FRNNT_EINVAL, "bad sizes");
  FRNNT_REQUIRE(B <= 65535, FRNNT_EUNSUPPORTED, "B too large for the grid");
  if (B == 0 || D == 0) return FRNNT_OK;
  FRNNT_REQUIRE(T == 0 || (x && gate && saved && dx && dgate), FRNNT_EINVAL, "NULL argument");
  cudaStream_t st = (cudaStream_t)stream;
  const RecTensor X{x, x_batch, x_step}, G{gate, gate_batch, gate_step}, DH{dh, dh_batch, dh_step};
  const dim3 grid((unsigned)((D + kRecThreads - 1) / kRecThreads), (unsigned)B);
#define FRNNT_REC_BACKWARD(TYPE)                                                            \
  FRNNT_KERNEL(recurrence_backward_kernel<TYPE><<<grid, kRecThreads, 0, st>>>(              \
      X, G, lengths, (const RecState<TYPE> *)saved, DH, (const RecState<TYPE> *)dlast,      \
      (TYPE *)dx, (TYPE *)dgate, (RecState<TYPE> *)dinitial, T, D))
  FRNNT_REC_TYPES(FRNNT_REC_BACKWARD)
#undef FRNNT_REC_BACKWARD
  FRNNT_CUDA(cudaGetLastError());
  return FRNNT_OK;
}

extern "C" int frnnt_recurrence_step(int dtype, const void *x, long long x_row, const void *gate,
                                     long long gate_row, const void *state, const int64_t *parents, void *h,
                                     void *next, long long rows, int beams, int K, int D, void *stream) {
  FRNNT_REQUIRE(rec_dtype(dtype), FRNNT_EINVAL, "dtype must be FRNNT_F32, _F64, _F16 or _BF16");
  FRNNT_REQUIRE(rows >= 0 && beams >= 1 && K >= 1 && D >= 0, FRNNT_EINVAL, "bad sizes");
  if (rows == 0 || D == 0) return FRNNT_OK;
  FRNNT_REQUIRE(x && gate && state && next, FRNNT_EINVAL, "NULL argument");
  FRNNT_REQUIRE(state != next, FRNNT_EINVAL, "the new states may not overwrite the old ones");
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid((unsigned)((D + kRecThreads - 1) / kRecThreads), (unsigned)(rows < 65535 ? rows : 65535));
#define FRNNT_REC_STEP(TYPE)                                                                \
  FRNNT_KERNEL(recurrence_step_kernel<TYPE><<<grid, kRecThreads, 0, st>>>(                  \
      (const TYPE *)x, x_row, (const TYPE *)gate, gate_row, (const RecState<TYPE> *)state,  \
      parents, (TYPE *)h, (RecState<TYPE> *)next, rows, beams, K, D))
  FRNNT_REC_TYPES(FRNNT_REC_STEP)
#undef FRNNT_REC_STEP
  FRNNT_CUDA(cudaGetLastError());
  return FRNNT_OK;
}
