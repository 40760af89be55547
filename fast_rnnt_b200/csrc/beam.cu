// Beam search: the best continuations over beams and vocabulary, and the reordering of states.
#include <climits>

#include "common.cuh"

namespace frnnt {

constexpr int kSelThreads = 256;
constexpr int kSelBeams = 1024;   // most rows of logits of one utterance
constexpr int kSelMost = 32;      // most continuations

template <typename T>
__global__ void __launch_bounds__(kSelThreads)
beam_select_kernel(const T *__restrict__ logits, long long batch, long long row, const float *__restrict__ scores,
                   const uint8_t *__restrict__ finished, int blank, float *__restrict__ out_scores,
                   int64_t *__restrict__ out_parents, int64_t *__restrict__ out_tokens, int K, int V, int beam) {
  __shared__ float tops[kSelBeams];
  __shared__ double logs[kSelBeams];
  __shared__ double part[kSelThreads / 32];
  __shared__ long long part_at[kSelThreads / 32];
  __shared__ double s_key;
  __shared__ long long s_at;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = warp; i < K; i += kSelThreads / 32) {
    const T *X = logits + b * batch + i * row;
    float top = neg_inf<float>();
    for (int v = lane; v < V; v += 32) top = fmaxf(top, in_f32(X[v]));
    top = warp_max(top);
    double sum = 0;
    for (int v = lane; v < V; v += 32) sum += (double)expf(in_f32(X[v]) - top);
    sum = warp_sum(sum);
    if (lane == 0) tops[i] = top, logs[i] = log(sum);
  }
  __syncthreads();
  double bound = INFINITY;
  long long bound_at = -1;   // what was chosen last: the next one comes after it
  for (int j = 0; j < beam; ++j) {
    double best = -INFINITY;
    long long at = LLONG_MAX;
    for (long long n = tid; n < (long long)K * V; n += kSelThreads) {
      const int i = (int)(n / V), v = (int)(n - (long long)i * V);
      const double score = scores[(size_t)b * K + i];
      const bool done = finished != nullptr && finished[(size_t)b * K + i];
      const double key = done ? (v == blank ? score : -INFINITY)
                              : score + (((double)in_f32(logits[b * batch + i * row + v]) - tops[i]) - logs[i]);
      if (!(key > -INFINITY)) continue;
      if (key > bound || (key == bound && n <= bound_at)) continue;
      if (key > best || (key == best && n < at)) best = key, at = n;
    }
    for (int o = 16; o > 0; o >>= 1) {
      const double k2 = __shfl_xor_sync(0xffffffffu, best, o);
      const long long a2 = __shfl_xor_sync(0xffffffffu, at, o);
      if (k2 > best || (k2 == best && a2 < at)) best = k2, at = a2;
    }
    if (lane == 0) part[warp] = best, part_at[warp] = at;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kSelThreads / 32; ++w)
        if (part[w] > best || (part[w] == best && part_at[w] < at)) best = part[w], at = part_at[w];
      const bool none = at == LLONG_MAX;
      const size_t o = (size_t)b * beam + j;
      out_scores[o] = (float)best;
      out_parents[o] = none ? -1 : at / V;
      out_tokens[o] = none ? -1 : at % V;
      s_key = best;
      s_at = at;
    }
    __syncthreads();
    bound = s_key;
    bound_at = s_at;
  }
}

// ------------------------------------------------------------------------------
constexpr int kReorderMost = 32;   // tensors of one launch
struct ReorderList {
  const char *from[kReorderMost];
  char *to[kReorderMost];
  long long batch[kReorderMost], beam[kReorderMost];   // strides of `from` in bytes
  long long bytes[kReorderMost];                       // of one row
};

template <typename W>
__device__ __forceinline__ void copy_row(const char *from, char *to, long long bytes) {
  for (long long n = threadIdx.x; n < bytes / (long long)sizeof(W); n += blockDim.x)
    reinterpret_cast<W *>(to)[n] = from == nullptr ? W{} : reinterpret_cast<const W *>(from)[n];
}

__global__ void __launch_bounds__(128)
beam_reorder_kernel(const __grid_constant__ ReorderList list, const int64_t *__restrict__ parents, long long rows,
                    int beams, int K) {
  const int n = blockIdx.y;
  const long long bytes = list.bytes[n];
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t p = parents[row];
    const char *from = p < 0 || p >= K ? nullptr
                                       : list.from[n] + div_rows(row, beams) * list.batch[n] + p * list.beam[n];
    char *to = list.to[n] + row * bytes;
    const uintptr_t low = (uintptr_t)from | (uintptr_t)to | (uintptr_t)bytes;
    if (low % 16 == 0) copy_row<uint4>(from, to, bytes);
    else if (low % 4 == 0) copy_row<uint32_t>(from, to, bytes);
    else if (low % 2 == 0) copy_row<uint16_t>(from, to, bytes);
    else copy_row<uint8_t>(from, to, bytes);
  }
}

}  // namespace frnnt

using namespace frnnt;

extern "C" int frnnt_beam_select(int dtype, const void *logits, long long batch, long long row, const float *scores,
                                 const uint8_t *finished, int blank, float *out_scores, int64_t *out_parents,
                                 int64_t *out_tokens, int B, int K, int V, int beam, void *stream) {
  FRNNT_REQUIRE(dtype == FRNNT_F32 || is_half_input(dtype), FRNNT_EINVAL, "dtype must be FRNNT_F32, _F16 or _BF16");
  FRNNT_REQUIRE(B >= 0 && K >= 1 && V >= 1, FRNNT_EINVAL, "bad sizes");
  FRNNT_REQUIRE(beam >= 1 && beam <= kSelMost, FRNNT_EUNSUPPORTED, "beam must be 1 to %d", kSelMost);
  FRNNT_REQUIRE(K <= kSelBeams, FRNNT_EUNSUPPORTED, "at most %d beams", kSelBeams);
  FRNNT_REQUIRE((long long)K * V < INT_MAX, FRNNT_EUNSUPPORTED, "beams times vocabulary must be below 2^31");
  FRNNT_REQUIRE(finished == nullptr || (blank >= 0 && blank < V), FRNNT_EINVAL, "termination symbol out of range");
  if (B == 0) return FRNNT_OK;
  FRNNT_REQUIRE(logits && scores && out_scores && out_parents && out_tokens, FRNNT_EINVAL, "NULL argument");
  cudaStream_t st = (cudaStream_t)stream;
#define FRNNT_SELECT(TYPE)                                                                               \
  FRNNT_KERNEL(beam_select_kernel<TYPE><<<B, kSelThreads, 0, st>>>((const TYPE *)logits, batch, row,     \
      scores, finished, blank, out_scores, out_parents, out_tokens, K, V, beam))
  if (dtype == FRNNT_F32) FRNNT_SELECT(float);
  else if (dtype == FRNNT_F16) FRNNT_SELECT(__half);
  else FRNNT_SELECT(__nv_bfloat16);
#undef FRNNT_SELECT
  FRNNT_CUDA(cudaGetLastError());
  return FRNNT_OK;
}

extern "C" int frnnt_beam_reorder(int count, const void *const *from, const long long *batch, const long long *beam,
                                  void *const *to, const long long *bytes, const int64_t *parents, int B, int beams,
                                  int K, void *stream) {
  FRNNT_REQUIRE(count >= 0 && B >= 0 && beams >= 0 && K >= 1, FRNNT_EINVAL, "bad sizes");
  const long long rows = (long long)B * beams;
  if (count == 0 || rows == 0) return FRNNT_OK;
  FRNNT_REQUIRE(from && batch && beam && to && bytes && parents, FRNNT_EINVAL, "NULL argument");
  for (int n = 0; n < count; ++n) {
    FRNNT_REQUIRE(bytes[n] >= 0 && (bytes[n] == 0 || (from[n] && to[n])), FRNNT_EINVAL, "NULL argument");
    FRNNT_REQUIRE(bytes[n] == 0 || from[n] != to[n], FRNNT_EINVAL, "a tensor cannot be reordered in place");
  }
  cudaStream_t st = (cudaStream_t)stream;
  for (int first = 0; first < count; first += kReorderMost) {
    ReorderList list{};
    const int m = count - first < kReorderMost ? count - first : kReorderMost;
    for (int n = 0; n < m; ++n) {
      list.from[n] = (const char *)from[first + n];
      list.to[n] = (char *)to[first + n];
      list.batch[n] = batch[first + n];
      list.beam[n] = beam[first + n];
      list.bytes[n] = bytes[first + n];
    }
    const long long most = (long long)sm_count() * 64;
    FRNNT_KERNEL(beam_reorder_kernel<<<dim3((unsigned)(rows < most ? rows : most), (unsigned)m), 128, 0, st>>>(
        list, parents, rows, beams, K));
    FRNNT_CUDA(cudaGetLastError());
  }
  return FRNNT_OK;
}
