// Beam search: the best continuations over beams and vocabulary, and the reordering of states.
//
// beam_select, bound by one read of the logits.  A cluster of CTAs has an utterance; a CTA takes
// whole rows (hypotheses) in turn, or one part of a row where there are fewer rows than CTAs.
//
//   stream   every thread reads 16 bytes at a time, keeping the running maximum and the sum of
//            exponentials, and in which of its vectors the maximum lies: one pass gives the
//            log-sum and, for every thread's share ("column"), its best symbol.
//   columns  the `beam` threads with the largest maxima.  Whatever is among the best `beam` of the
//            row lies in one of their columns: anything else is less than `beam` maxima.
//   collect  those columns again (from L1 / L2, beam / 256 of the row), for all that is no less
//            than the least of the chosen maxima: rarely more than `beam` and a few.
//   order    by counting, for each, the greater ones.
//
// Lists of different rows are joined by the rank of each entry, which a binary search in the
// other lists gives: no entry moves more than once, and there is no order in which atomics
// could change the outcome.  Rows are read as vectors of the same elements wherever they begin
// in memory (two aligned loads shifted into one off a 16-byte boundary), so that equal rows
// have equal sums to the last bit and their ties are ties.
//
// Exponentials are the hardware's, in 32 bits relative to the maximum; the sums of the threads
// are added, and scores kept and compared, in 64 bits.
#include <cooperative_groups.h>

#include <climits>
#include <type_traits>

#include "common.cuh"

namespace frnnt {

constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelBeams = 1024;   // most rows of logits of one utterance
constexpr int kSelMost = 32;      // most continuations
constexpr int kSelCluster = 8;    // most CTAs of an utterance
constexpr int kSelLists = 8;      // of rows, before they are joined; one per CTA of a cluster at the end
constexpr int kSelBuffer = 1024;  // candidates of a row
static_assert(kSelLists >= kSelCluster && kSelMost <= 32, "a list per CTA, a lane per entry");

// order of floats as order of unsigned integers; the two zeros are one number
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u ^ ((uint32_t)((int32_t)~u >> 31) | 0x80000000u));
}
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered(uint64_t u) {
  return __longlong_as_double((long long)(u ^ ((uint64_t)((int64_t)~u >> 63) | 0x8000000000000000ull)));
}
// (value, place): larger values first, then lower places; 0 is less than any
__device__ __forceinline__ uint64_t placed(float x, uint32_t place) {
  return (uint64_t)ordered(x) << 32 | (0xffffffffu - place);
}
__device__ __forceinline__ uint32_t place_of(uint64_t p) { return 0xffffffffu - (uint32_t)p; }
__device__ __forceinline__ float value_of(uint64_t p) { return unordered((uint32_t)(p >> 32)); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// exp(x - top) for x <= top; 0 where both are -inf
__device__ __forceinline__ float exp_below(float x, float top) {
  return exp2_fast((x - (top == neg_inf<float>() ? 0.0f : top)) * 1.4426950408889634f);
}

// ---- a row of logits as vectors of 16 bytes --------------------------------------------
template <typename T> struct SelRow {
  static constexpr int EV = 16 / (int)sizeof(T);
  const T *row;
  int V, off, safe_lo, safe_hi;   // elements behind a 16-byte boundary; vectors that need no care
  __device__ SelRow(const T *row_, int V_) : row(row_), V(V_) {
    off = (int)((uintptr_t)row % 16) / (int)sizeof(T);
    safe_lo = off ? 1 : 0;
    safe_hi = off ? (int)(((long long)V + off) / EV) - 1 : V / EV;
  }
  // vector j: elements EV j .. EV j + EV - 1, -inf behind the end
  __device__ __forceinline__ uint4 load(int j) const {
    if (j >= safe_lo && j < safe_hi) {
      const uint4 *p = reinterpret_cast<const uint4 *>(row - off) + j;
      const uint4 q = __ldg(p);
      if (off == 0) return q;
      const uint4 r = __ldg(p + 1);
      uint32_t w[8] = {q.x, q.y, q.z, q.w, r.x, r.y, r.z, r.w};
      const int words = off * (int)sizeof(T) / 4;
#pragma unroll
      for (int n = 0; n < 7; ++n) w[n] = words & 1 ? w[n + 1] : w[n];
#pragma unroll
      for (int n = 0; n < 5; ++n) w[n] = words & 2 ? w[n + 2] : w[n];
      if constexpr (sizeof(T) == 2) {
        const int half = off & 1 ? 16 : 0;
#pragma unroll
        for (int n = 0; n < 4; ++n) w[n] = __funnelshift_r(w[n], w[n + 1], half);
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
    T e[EV];
#pragma unroll
    for (int n = 0; n < EV; ++n) {
      const long long v = (long long)j * EV + n;
      e[n] = v < V ? row[v] : minus_inf();
    }
    uint4 q;
    memcpy(&q, e, 16);
    return q;
  }
  __device__ static __forceinline__ T minus_inf() {
    if constexpr (sizeof(T) == 4) return -INFINITY;
    else if constexpr (std::is_same<T, __half>::value) return __ushort_as_half(0xfc00);
    else return __ushort_as_bfloat16(0xff80);
  }
  __device__ static __forceinline__ void unpack(const uint4 &q, float (&x)[EV]) {
    T e[EV];
    memcpy(e, &q, 16);
#pragma unroll
    for (int n = 0; n < EV; ++n) x[n] = in_f32(e[n]);
  }
};

// ---- lists of continuations, best first --------------------------------------------------
struct SelEntry {
  uint64_t key;     // ordered score
  uint64_t symbol;  // (logit, symbol)
  int row;
};
struct SelList {
  uint64_t key[kSelMost], symbol[kSelMost];
  int row[kSelMost], size;
  __device__ __forceinline__ SelEntry get(int n) const { return {key[n], symbol[n], row[n]}; }
  __device__ __forceinline__ void set(int n, const SelEntry &e) { key[n] = e.key, symbol[n] = e.symbol, row[n] = e.row; }
};
// Equal scores: the lower hypothesis; of one hypothesis the larger logit, then the lower symbol
// (logits whose difference 64 bits of score do not show are in the order of the row's list too).
__device__ __forceinline__ bool before(const SelEntry &a, const SelEntry &b) {
  if (a.key != b.key) return a.key > b.key;
  if (a.row != b.row) return a.row < b.row;
  return a.symbol > b.symbol;
}
// how many entries of a list come before `e`
__device__ __forceinline__ int rank_in(const SelList &list, const SelEntry &e) {
  int lo = 0, hi = list.size;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (before(list.get(mid), e)) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

struct SelShared {
  alignas(16) uint64_t buffer[kSelBuffer];
  alignas(16) uint64_t lanes[kSelWarps][32];
  uint64_t sorted[kSelWarps][32];
  uint64_t top[kSelMost];
  SelList lists[kSelLists], joined;
  float part_top[kSelWarps];
  double part_sum[kSelWarps];
  float parts_top[kSelCluster];   // of a row in parts, from the CTAs of its parts
  double parts_sum[kSelCluster];
  float row_top;
  double row_sum;
  int found;
};

// lists[0 .. n-1] -> lists[0]
__device__ void join_lists(SelShared &sm, int n, int beam) {
  __syncthreads();
  int total = 0;
  for (int l = 0; l < n; ++l) total += sm.lists[l].size;
  for (int e = threadIdx.x; e < n * beam; e += kSelThreads) {
    const int l = e / beam, pos = e - l * beam;
    if (pos >= sm.lists[l].size) continue;
    const SelEntry own = sm.lists[l].get(pos);
    int rank = pos;
    for (int o = 0; o < n; ++o)
      if (o != l) rank += rank_in(sm.lists[o], own);
    if (rank < beam) sm.joined.set(rank, own);
  }
  __syncthreads();
  const int size = total < beam ? total : beam;
  if (threadIdx.x < size) sm.lists[0].set(threadIdx.x, sm.joined.get(threadIdx.x));
  if (threadIdx.x == 0) sm.lists[0].size = size;
  __syncthreads();
}

// The best `beam` symbols of vectors [first, end) of a row in sm.top, best first (0: none), and the
// maximum and sum of exponentials in sm.row_top, sm.row_sum.
template <typename T>
__device__ void select_row(SelShared &sm, const SelRow<T> &row, int first, int end, int beam) {
  constexpr int EV = SelRow<T>::EV, U = 4;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // stream
  float top = neg_inf<float>(), sum = 0;
  int top_at = 0;
  for (int j0 = first + tid; j0 < end; j0 += U * kSelThreads) {
    uint4 q[U];
#pragma unroll
    for (int n = 0; n < U; ++n)
      if (j0 + n * kSelThreads < end) q[n] = row.load(j0 + n * kSelThreads);
#pragma unroll
    for (int n = 0; n < U; ++n) {
      const int j = j0 + n * kSelThreads;
      if (j >= end) break;
      float x[EV], most;
      SelRow<T>::unpack(q[n], x);
      most = x[0];
#pragma unroll
      for (int e = 1; e < EV; ++e) most = fmaxf(most, x[e]);
      if (most > top) {
        sum *= exp_below(top, most);
        top = most;
        top_at = j;
      }
#pragma unroll
      for (int e = 0; e < EV; ++e) sum += exp_below(x[e], top);
    }
  }
  // columns: in order within the warp, then among the warps
  const uint64_t mine = top > neg_inf<float>() ? placed(top, (uint32_t)top_at) : 0;
  sm.lanes[warp][lane] = mine;
  sm.sorted[warp][lane] = 0;
  if (tid < kSelMost) sm.top[tid] = 0;
  if (tid == 0) sm.found = 0;
  const float warp_top = warp_max(top);
  const double warp_total = warp_sum((double)(sum * exp_below(top, warp_top)));
  if (lane == 0) sm.part_top[warp] = warp_top, sm.part_sum[warp] = warp_total;
  __syncwarp();
  int rank = 0;
#pragma unroll
  for (int o = 0; o < 32; o += 2) {
    const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(&sm.lanes[warp][o]);
    rank += (two.x > mine) + (two.y > mine);
  }
  if (mine != 0) sm.sorted[warp][rank] = mine;
  __syncthreads();
  if (lane < beam && sm.sorted[warp][lane] != 0) {
    const uint64_t key = sm.sorted[warp][lane];
    int at[kSelWarps] = {};
#pragma unroll
    for (int step = 16; step > 0; step >>= 1)
#pragma unroll
      for (int w = 0; w < kSelWarps; ++w)
        if (sm.sorted[w][at[w] + step - 1] > key) at[w] += step;
    int total = 0;
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) total += w == warp ? lane : at[w] + (at[w] == 31 && sm.sorted[w][31] > key);
    if (total < beam) sm.top[total] = key;
  }
  if (warp == kSelWarps - 1 && lane < kSelWarps) {   // the row's maximum and sum
    const unsigned mask = (1u << kSelWarps) - 1;
    float m = sm.part_top[lane];
    double s = sm.part_sum[lane];
#pragma unroll
    for (int o = kSelWarps / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(mask, m, o));
    s *= (double)exp_below(sm.part_top[lane], m);
#pragma unroll
    for (int o = kSelWarps / 2; o > 0; o >>= 1) s += __shfl_xor_sync(mask, s, o);
    if (lane == 0) sm.row_top = m, sm.row_sum = s;
  }
  __syncthreads();
  // collect
  int columns = 0;
  while (columns < beam && sm.top[columns] != 0) ++columns;
  if (columns == 0) return;   // the whole CTA
  // with fewer columns than `beam` there are no better ones elsewhere: all above -inf
  const bool few = columns < beam;
  const uint64_t least = sm.top[columns - 1];
  const float least_value = few ? neg_inf<float>() : value_of(least);
  const int least_at = few ? -1 : (int)place_of(least), deep = (end - first + kSelThreads - 1) / kSelThreads;
  const auto each = [&](auto &&take) {
    for (int p = tid; p < columns * deep; p += kSelThreads) {
      const int c = p % columns;
      const int j = first + ((int)place_of(sm.top[c]) - first) % kSelThreads + p / columns * kSelThreads;
      if (j >= end) continue;
      float x[EV];
      SelRow<T>::unpack(row.load(j), x);
#pragma unroll
      for (int e = 0; e < EV; ++e)
        if (x[e] > least_value || (x[e] == least_value && j <= least_at)) take(placed(x[e], (uint32_t)(j * EV + e)));
    }
  };
  each([&](uint64_t p) {
    const int n = atomicAdd(&sm.found, 1);
    if (n < kSelBuffer) sm.buffer[n] = p;
  });
  __syncthreads();
  const int found = sm.found;
  if (found <= kSelBuffer) {
    // order
    for (int c = tid; c < found; c += kSelThreads) {
      const uint64_t own = sm.buffer[c];
      int greater = 0;
      for (int o = 0; o < found; ++o) greater += sm.buffer[o] > own;
      if (greater < beam) sm.top[greater] = own;
    }
  } else {
    // more than the buffer holds, where the best ones lie in few columns: one at a time
    uint64_t bound = ~0ull;
    for (int n = 0; n < beam; ++n) {
      uint64_t best = 0;
      each([&](uint64_t p) { best = p < bound && p > best ? p : best; });
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
      }
      if (lane == 0) sm.lanes[0][warp] = best;
      __syncthreads();
      for (int w = 0; w < kSelWarps; ++w) best = sm.lanes[0][w] > best ? sm.lanes[0][w] : best;
      if (tid == 0) sm.buffer[n] = best;
      bound = best;
      __syncthreads();
    }
    if (tid < beam) sm.top[tid] = sm.buffer[tid];
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kSelThreads, 4)
beam_select_kernel(const T *__restrict__ logits, long long batch, long long row_stride,
                   const float *__restrict__ scores, const uint8_t *__restrict__ finished, int blank,
                   float *__restrict__ out_scores, int64_t *__restrict__ out_parents,
                   int64_t *__restrict__ out_tokens, int K, int V, int parts, int beam) {
  __shared__ SelShared sm;
  namespace cg = cooperative_groups;
  const int rank = blockIdx.x, ranks = gridDim.x, b = blockIdx.y, tid = threadIdx.x;
  const int vectors = (int)(((long long)V + SelRow<T>::EV - 1) / SelRow<T>::EV);
  const int share = (vectors + parts - 1) / parts;
  if (parts > 1) {
    if (tid < kSelCluster) sm.parts_top[tid] = neg_inf<float>(), sm.parts_sum[tid] = 0;
    cg::this_cluster().sync();   // all have started, and have cleared theirs
  }
  int lists = 0;
  for (int unit = rank; unit < K * parts; unit += ranks) {
    const int i = unit / parts, part = unit - i * parts;
    const float score = scores[(size_t)b * K + i];
    const bool none = !(fabsf(score) < INFINITY);
    const bool done = !none && finished != nullptr && finished[(size_t)b * K + i] != 0;
    const bool stream = !none && !done;
    if (stream) {
      const int first = part * share, end = min(vectors, first + share);
      select_row<T>(sm, SelRow<T>(logits + b * batch + i * row_stride, V), first, end, beam);
    }
    if (parts > 1) {   // one unit per CTA: the parts of a row tell each other their sums
      if (stream && tid < parts) {
        SelShared *peer = cg::this_cluster().map_shared_rank(&sm, i * parts + tid);
        peer->parts_top[part] = sm.row_top;
        peer->parts_sum[part] = sm.row_sum;
      }
      cg::this_cluster().sync();
      if (stream && tid == 0) {
        float m = neg_inf<float>();
        double s = 0;
        for (int p = 0; p < parts; ++p) m = fmaxf(m, sm.parts_top[p]);
        for (int p = 0; p < parts; ++p) s += sm.parts_sum[p] * (double)exp_below(sm.parts_top[p], m);
        sm.row_top = m;
        sm.row_sum = s;
      }
      __syncthreads();
    }
    SelList &list = sm.lists[lists];
    if (stream) {
      const float m = sm.row_top;
      const bool fine = fabsf(m) < INFINITY && sm.row_sum < (double)INFINITY;   // no NaN either
      if (tid < 32) {
        const double log_sum = log(sm.row_sum);
        const uint64_t symbol = tid < beam ? sm.top[tid] : 0;
        const unsigned have = __ballot_sync(0xffffffffu, fine && symbol != 0);
        if (symbol != 0)
          list.set(tid, {ordered((double)score + (((double)value_of(symbol) - (double)m) - log_sum)), symbol, i});
        if (tid == 0) list.size = __popc(have);
      }
      ++lists;
    } else if (done && part == 0) {
      if (tid == 0) {
        list.set(0, {ordered((double)score), placed(0.0f, (uint32_t)blank), i});
        list.size = 1;
      }
      ++lists;
    }
    if (lists == kSelLists) {
      join_lists(sm, lists, beam);
      lists = 1;
    }
    __syncthreads();
  }
  if (lists == 0) {
    if (tid == 0) sm.lists[0].size = 0;
    lists = 1;
  }
  if (lists > 1) join_lists(sm, lists, beam);
  if (ranks > 1) {
    cg::this_cluster().sync();
    if (rank == 0) {
      for (int e = tid; e < (ranks - 1) * beam; e += kSelThreads) {
        const int l = 1 + e / beam, pos = e % beam;
        const SelList &from = cg::this_cluster().map_shared_rank(&sm, l)->lists[0];
        if (pos < from.size) sm.lists[l].set(pos, from.get(pos));
        if (pos == 0) sm.lists[l].size = from.size;
      }
    }
    cg::this_cluster().sync();   // nobody reads another's lists any more
    if (rank != 0) return;
    join_lists(sm, ranks, beam);
  }
  if (tid < beam) {
    const bool have = tid < sm.lists[0].size;
    const SelEntry e = have ? sm.lists[0].get(tid) : SelEntry{};
    const size_t o = (size_t)b * beam + tid;
    out_scores[o] = have ? (float)unordered(e.key) : neg_inf<float>();
    out_parents[o] = have ? e.row : -1;
    out_tokens[o] = have ? (int64_t)place_of(e.symbol) : -1;
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

// Rows over the CTAs of a cluster: as many rows each as it takes for up to eight; with fewer
// rows than that, rows in parts, each of two rounds of vectors or more.
template <typename T>
static int select_launch(const T *logits, long long batch, long long row, const float *scores,
                         const uint8_t *finished, int blank, float *out_scores, int64_t *out_parents,
                         int64_t *out_tokens, int B, int K, int V, int beam, cudaStream_t st) {
  const int each = (K + kSelCluster - 1) / kSelCluster, vectors = (V + SelRow<T>::EV - 1) / SelRow<T>::EV;
  int parts = 1, ranks = (K + each - 1) / each;
  while (ranks + K <= kSelCluster && (parts + 1) * 2 * kSelThreads <= vectors) ++parts, ranks += K;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)ranks, (unsigned)B);
  config.blockDim = dim3(kSelThreads);
  config.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = ranks > 1 ? 1 : 0;
  FRNNT_CUDA(FRNNT_KERNEL(cudaLaunchKernelEx(&config, beam_select_kernel<T>, logits, batch, row, scores, finished,
                                             blank, out_scores, out_parents, out_tokens, K, V, parts, beam)));
  return FRNNT_OK;
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
  FRNNT_REQUIRE(B <= 65535, FRNNT_EUNSUPPORTED, "B too large for the grid");
#define FRNNT_SELECT(TYPE)                                                                                \
  return select_launch<TYPE>((const TYPE *)logits, batch, row, scores, finished, blank, out_scores,       \
                             out_parents, out_tokens, B, K, V, beam, (cudaStream_t)stream)
  if (dtype == FRNNT_F32) FRNNT_SELECT(float);
  if (dtype == FRNNT_F16) FRNNT_SELECT(__half);
  FRNNT_SELECT(__nv_bfloat16);
#undef FRNNT_SELECT
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
