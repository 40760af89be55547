// Beam search: the best continuations over beams and vocabulary, and the reordering of states.
//
// beam_select, bound by one read of the logits, in two launches.  The first has a CTA for every
// row (hypothesis), or for parts of rows where they are few, and leaves the `beam` best symbols
// and the sum of exponentials of each; the second joins an utterance's rows.
//
//   stream   every thread reads 16 bytes at a time and keeps the sum of exponentials of its
//            share ("column"), the maximum, which vector holds it, and the next vector's maximum.
//   bound    a logit that at least `beam` of the threads' maxima reach: the least, over the
//            warps, of their m-th largest, with the warps' m making up `beam`.  Nothing below it
//            is among the best `beam` of the row.
//   collect  the vectors whose maximum reaches the bound, again (from L1 / L2), for all that
//            does: two to three times `beam` where logits are in no special order.  Of a column
//            whose next maximum reaches it too, all vectors are looked at.
//   order    by counting, for each, those before it.
//
// The second launch does the same with the entries of the rows' lists in place of logits.  Equal
// logits of a row are in the order of their symbols and equal scores in that of i V + v, so that
// no order of atomics could change the outcome.  Rows are read as vectors of the same elements
// wherever they begin in memory (two aligned loads shifted into one off a 16-byte boundary), so
// that equal rows have equal sums to the last bit and their ties are ties.
//
// Exponentials are the hardware's, in 32 bits; the sums of a row's warps are added, and scores
// computed and compared, in 64 bits.
#include <cfloat>
#include <climits>
#include <type_traits>

#include "common.cuh"

namespace frnnt {

// Small CTAs, many of them: a row's short phases after the stream run beside other rows' streams
// (96 x 16 x 31999 fp16: 35 us; 12 CTAs a multiprocessor, with too few registers for that, 40, 256
// threads and 5 CTAs 39, 64 threads and 24 CTAs 48; the same loads for their maxima alone take 21
// to 24).  Chosen on that size only.
constexpr int kSelThreads = 128, kSelResident = 10;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelBeams = 1024;   // most rows of logits of one utterance
constexpr int kSelMost = 32;      // most continuations
constexpr int kSelParts = 16;     // most parts of a row
constexpr int kSelBuffer = 512;   // candidates, of a row or of an utterance's lists

// order of floating values as order of unsigned integers; the two zeros are one number
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

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// exp(x - top) for x <= top; 0 where both are -inf
__device__ __forceinline__ float exp_below(float x, float top) {
  return exp2_fast((x - (top == neg_inf<float>() ? 0.0f : top)) * 1.4426950408889634f);
}
// log(x), x >= 1, off by 2^-26: the exponent's share in 64 bits, the rest below 0.35 in 32
__device__ __forceinline__ double log_of(double x) {
  const int e = (int)(((uint64_t)__double_as_longlong(x * 1.4142135623730951) >> 52) & 0x7ff) - 1023;
  const double m = x * __longlong_as_double((long long)((uint64_t)(1023 - e) << 52));
  const float f = (float)m;
  return e * 0.6931471805599453 + (double)(logf(f) + (float)(m - (double)f) / f);
}

// ---- a row of logits as vectors of 16 bytes --------------------------------------------
// Vector j holds elements EV j .. EV j + EV - 1 wherever the row begins; in memory it is the end
// of one 16-byte granule and the beginning of the next (`off` elements on), or just a granule.
// The granules of vectors 1 .. count - 3 lie within the row; the elements of the first and the
// last two ("edges") are read one by one, a lane for each.
template <typename T> struct SelRow {
  static constexpr int EV = 16 / (int)sizeof(T);
  const T *row;
  int V, off, half;   // off in elements; half: the bits of an odd 16-bit value's offset
  __device__ SelRow(const T *row_, int V_) : row(row_), V(V_) {
    off = (int)((uintptr_t)row % 16) / (int)sizeof(T);
    half = sizeof(T) == 2 && off % 2 ? 16 : 0;
  }
  __device__ __forceinline__ static int vectors(int V) { return (int)(((long long)V + EV - 1) / EV); }
  // the symbol of a lane's edge element, -1: none
  __device__ __forceinline__ int edge_symbol(int lane) const {
    const long long v = lane < EV ? lane : (long long)max(1, vectors(V) - 2) * EV + lane - EV;
    return lane < 3 * EV && v < V ? (int)v : -1;
  }
  // whole 32-bit words that the row begins behind a boundary; -1: on one
  __device__ __forceinline__ int words() const { return off == 0 ? -1 : off * (int)sizeof(T) / 4; }
  struct Raw {
    uint4 q, r;   // a vector's granule and, off a boundary, the next one
  };
  template <int W> __device__ __forceinline__ Raw load(int j) const {
    const uint4 *p = reinterpret_cast<const uint4 *>(row - off) + j;
    if constexpr (W < 0) return {__ldg(p), {}};
    else return {__ldg(p), __ldg(p + 1)};
  }
  template <int W> __device__ __forceinline__ uint4 vector_of(const Raw &raw) const {
    if constexpr (W < 0) {
      return raw.q;
    } else {
      const uint32_t w[8] = {raw.q.x, raw.q.y, raw.q.z, raw.q.w, raw.r.x, raw.r.y, raw.r.z, raw.r.w};
      if constexpr (sizeof(T) == 4) return make_uint4(w[W], w[W + 1], w[W + 2], w[W + 3]);
      else
        return make_uint4(__funnelshift_r(w[W], w[W + 1], half), __funnelshift_r(w[W + 1], w[W + 2], half),
                          __funnelshift_r(w[W + 2], w[W + 3], half), __funnelshift_r(w[W + 3], w[(W + 4) % 8], half));
    }
  }
  __device__ static __forceinline__ void unpack(const uint4 &q, float (&x)[EV]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if constexpr (sizeof(T) == 4) {
        x[n] = __uint_as_float(w[n]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[n]));
        x[2 * n] = f.x, x[2 * n + 1] = f.y;
      } else {
        x[2 * n] = __uint_as_float(w[n] << 16), x[2 * n + 1] = __uint_as_float(w[n] & 0xffff0000u);
      }
    }
  }
  // the largest value that is a number
  __device__ static __forceinline__ float most_of(const uint4 &q, const float (&x)[EV]) {
    if constexpr (sizeof(T) == 4) {
      return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2 *h = reinterpret_cast<const T2 *>(&q);
      const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(in_f32(m.x), in_f32(m.y));
    }
  }
};

// vector j, the shift at run time (the collection's few vectors: one copy of that code)
template <typename T> __device__ __forceinline__ uint4 load_any(const SelRow<T> &row, int j) {
  const uint4 *p = reinterpret_cast<const uint4 *>(row.row - row.off) + j;
  const uint4 q = __ldg(p);
  if (row.off == 0) return q;
  const uint4 r = __ldg(p + 1);
  uint32_t w[8] = {q.x, q.y, q.z, q.w, r.x, r.y, r.z, r.w};
  const int words = row.words();
#pragma unroll
  for (int n = 0; n < 7; ++n) w[n] = words & 1 ? w[n + 1] : w[n];
#pragma unroll
  for (int n = 0; n < 5; ++n) w[n] = words & 2 ? w[n + 2] : w[n];
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int n = 0; n < 4; ++n) w[n] = __funnelshift_r(w[n], w[n + 1], row.half);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// What a thread keeps of its share of a row.  The sum of exponentials is relative to `ref`, which
// follows the maximum only when that is far above it: nearly every vector raises some lane's
// maximum, hardly one needs the sum rescaled.  All of it is arithmetic on differences of logits, and
// so is what it is decided by: rows that differ by a constant (which the subtraction leaves exact)
// have equal sums.
struct SelShare {
  float top = neg_inf<float>(), next = neg_inf<float>(), ref = -FLT_MAX;
  float2 sum = {0, 0};
  int at = 0;   // the vector of `top`; `next` is the maximum of the others
  static constexpr float kLog2e = 1.4426950408889634f, kSlack = 10.0f;
  template <int EV> __device__ __forceinline__ void add(const float (&x)[EV], float most, int j) {
    next = fmaxf(next, fminf(top, most));
    if (most > top) top = most, at = j;
    if (top - ref > kSlack) {
      const float by = exp2_fast((ref - top) * kLog2e);
      sum.x *= by;
      sum.y *= by;
      ref = top;
    }
    const float2 l = make_float2(kLog2e, kLog2e), r = make_float2(-ref, -ref);
#pragma unroll
    for (int e = 0; e < EV; e += 2) {
      float2 t = __fmul2_rn(__fadd2_rn(make_float2(x[e], x[e + 1]), r), l);
      t.x = exp2_fast(t.x);
      t.y = exp2_fast(t.y);
      sum = __fadd2_rn(sum, t);
    }
  }
  // sum of exp(x - top); the product with log2(e) to twice 32 bits, since ref may be far from top
  __device__ __forceinline__ float relative() const {
    const float s = sum.x + sum.y, d = ref - top;
    if (!(d > -1e30f) || !(d < 1e30f)) return s;   // nothing but -inf, or NaN
    const float hi = d * kLog2e, lo = fmaf(d, kLog2e, -hi);
    return s * fmaf(exp2f(hi), lo * 0.6931472f, exp2f(hi));
  }
};

// W: see SelRow::words.  The loop's loads are under no branch but their predicate: with the edges
// among them they would wait for one another (half the rate).  A row that is not to be read is
// left when the first loads are under way: they do not wait for the scores.
template <typename T, int W>
__device__ __forceinline__ void stream_row(SelShare &own, const SelRow<T> &row, int first, int end, bool read) {
  constexpr int EV = SelRow<T>::EV, U = 2;
  typename SelRow<T>::Raw ahead[U];
  const auto fetch = [&](int j) {
#pragma unroll
    for (int n = 0; n < U; ++n)
      if (j + n * kSelThreads < end) ahead[n] = row.template load<W>(j + n * kSelThreads);
  };
  int j = first + (int)threadIdx.x;
  fetch(j);
  if (!read) return;
  for (; j < end; j += U * kSelThreads) {
    uint4 q[U];
#pragma unroll
    for (int n = 0; n < U; ++n) q[n] = row.template vector_of<W>(ahead[n]);
    fetch(j + U * kSelThreads);
#pragma unroll
    for (int n = 0; n < U; ++n)
      if (j + n * kSelThreads < end) {
        float x[EV];
        SelRow<T>::unpack(q[n], x);
        own.template add<EV>(x, SelRow<T>::most_of(q[n], x), j + n * kSelThreads);
      }
  }
}

// An entry of a list: a logit and its symbol, larger logits first and then lower symbols; 0: none.
__device__ __forceinline__ uint64_t entry_of(float x, uint32_t symbol) {
  return (uint64_t)ordered(x) << 32 | (0xffffffffu - symbol);
}
__device__ __forceinline__ uint32_t symbol_of(uint64_t e) { return 0xffffffffu - (uint32_t)e; }
__device__ __forceinline__ float logit_of(uint64_t e) { return unordered((uint32_t)(e >> 32)); }

// The m-th largest of a warp's values (-inf where they are fewer), `each` = m.
__device__ __forceinline__ float mth_of_warp(float own, int each) {
  float most = own;
  for (int n = 0; n < each; ++n) {
    most = warp_max(own);
    if ((threadIdx.x & 31) == __ffs(__ballot_sync(0xffffffffu, own == most)) - 1) own = neg_inf<float>();
  }
  return most;
}

// What the first launch leaves of a row, or of a part of one; its list follows in `entries`.
struct SelSum {
  double sum;   // of exp(x - top)
  float top;
};

struct RowShared {
  uint64_t buffer[kSelBuffer], next[kSelWarps];
  double part_sum[kSelWarps];
  float part_top[kSelWarps];
  uint32_t bound[kSelWarps];
  int column[kSelThreads];
  int found, columns;
};

// a hypothesis: 0 none, 1 finished, 2 its row is read
__device__ __forceinline__ int kind_of(float score, const uint8_t *finished, size_t at) {
  return !(fabsf(score) < INFINITY) ? 0 : finished != nullptr && finished[at] != 0 ? 1 : 2;
}

__device__ __forceinline__ void push_entry(RowShared &sm, uint64_t e) {
  const int n = atomicAdd(&sm.found, 1);
  if (n < kSelBuffer) sm.buffer[n] = e;
}

// `take` for every element of vector j that is `wanted`
template <typename T, typename Wanted, typename Take>
__device__ __forceinline__ void look_at(const SelRow<T> &row, int j, Wanted &&wanted, Take &&take) {
  constexpr int EV = SelRow<T>::EV;
  const uint4 q = load_any(row, j);
  float x[EV];
  SelRow<T>::unpack(q, x);
  unsigned reach = 0;
#pragma unroll
  for (int e = 0; e < EV; ++e) reach |= (unsigned)wanted(x[e]) << e;
  for (; reach != 0; reach &= reach - 1) {   // mostly one
    const int at = __ffs(reach) - 1;
    float v = x[0];
#pragma unroll
    for (int e = 1; e < EV; ++e) v = e == at ? x[e] : v;
    take(entry_of(v, (uint32_t)(j * EV + at)));
  }
}

// Where more reach the bound than the buffer holds: logits in clumps, or many equal ones.  The bound
// again, the `beam`-th largest of all maxima now; what is above it lies in fewer than `beam`
// columns, and of those equal to it only the lowest symbols count.  Returns how many it found,
// still more than the buffer holds where the best ones lie in few columns.  Not inlined: it is
// rare, and the registers it needs would be the kernel's.
template <typename T>
__device__ __noinline__ int crowded_row(RowShared &sm, SelRow<T> row, int first, int end, float top, float column_top,
                                        float edge, int symbol, int beam) {
  constexpr int EV = SelRow<T>::EV;
  const int tid = threadIdx.x;
  const uint32_t mine = ordered(top);
  const auto push = [&](uint64_t e) { push_entry(sm, e); };
  __syncthreads();   // all have seen how many there were
  sm.column[tid] = (int)mine;
  if (tid == 0) sm.found = 0;
  __syncthreads();
  int rank = 0;
  for (int o = 0; o < kSelThreads; ++o) {
    const uint32_t other = (uint32_t)sm.column[o];
    rank += other > mine || (other == mine && o < tid);
  }
  if (rank == beam - 1) sm.bound[0] = mine;
  __syncthreads();
  const float bound = unordered(max(sm.bound[0], ordered(-FLT_MAX)));
  const auto above = [&](float x) { return x > bound; };
  const auto equal = [&](float x) { return x == bound; };
  if (above(edge)) push(entry_of(edge, (uint32_t)symbol));
  if (above(column_top))
    for (int j = first + tid; j < end; j += kSelThreads) look_at(row, j, above, push);
  __syncthreads();
  // The lowest symbols: the first vector's, then some vectors at a time, no more than the buffer has
  // room for, then the last two vectors'.  Everybody reads the count before anybody adds to it.
  constexpr int kSome = (kSelBuffer - 4 * kSelMost) / EV;
  int found = sm.found;
  __syncthreads();
  if (found < beam && equal(edge) && symbol < EV) push(entry_of(edge, (uint32_t)symbol));
  for (int from = first; found < beam && from < end; from += kSome) {
    for (int j = from + tid; j < min(end, from + kSome); j += kSelThreads) look_at(row, j, equal, push);
    __syncthreads();
    found = sm.found;
    __syncthreads();
  }
  if (found < beam && equal(edge) && symbol >= EV) push(entry_of(edge, (uint32_t)symbol));
  __syncthreads();
  return sm.found;
}

template <typename T>
__global__ void __launch_bounds__(kSelThreads, kSelResident)
select_rows_kernel(const T *__restrict__ logits, long long batch, long long row_stride,
                   const float *__restrict__ scores, const uint8_t *__restrict__ finished, int V,
                   SelSum *__restrict__ sums, uint64_t *__restrict__ entries, int beam) {
  __shared__ RowShared sm;
  // the second launch may be set up meanwhile; it waits for this one's end before it reads
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int part = blockIdx.x, parts = gridDim.x, i = blockIdx.y, K = gridDim.y, b = blockIdx.z;
  const size_t at = (size_t)b * K + i, unit = at * parts + part;
  const bool read = kind_of(scores[at], finished, at) == 2;
  const int main_end = max(1, SelRow<T>::vectors(V) - 2), share = (main_end - 1 + parts - 1) / parts;
  const int first = min(main_end, 1 + part * share), end = min(main_end, first + share);
  const bool edges = part == 0;
  const SelRow<T> row(logits + b * batch + i * row_stride, V);
  SelSum *const out = sums + unit;
  uint64_t *const list = entries + unit * beam;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // an edge element for the lanes of the last warp, which have least of the row to read
  const int symbol = edges && warp == kSelWarps - 1 ? row.edge_symbol(lane) : -1;
  float edge = symbol >= 0 ? in_f32(row.row[symbol]) : neg_inf<float>();
  SelShare own;
  switch (row.words()) {
    case -1: stream_row<T, -1>(own, row, first, end, read); break;
    case 0: stream_row<T, 0>(own, row, first, end, read); break;
    case 1: stream_row<T, 1>(own, row, first, end, read); break;
    case 2: stream_row<T, 2>(own, row, first, end, read); break;
    default: stream_row<T, 3>(own, row, first, end, read); break;
  }
  if (!read) return;
  const float column_top = own.top;
  const int column_at = own.at;
  const float column_next = own.next;
  if (symbol >= 0) {
    const float x[2] = {edge, neg_inf<float>()};
    own.template add<2>(x, edge, 0);
  }
  // bound
  const int whole = min(kSelWarps, max(1, (end - first) / 32));   // warps whose lanes all have a share
  uint32_t left = ordered(own.top);
  const uint32_t most = __reduce_max_sync(0xffffffffu, left);
  uint32_t mth = most;
  for (int n = 1; n < (beam + whole - 1) / whole; ++n) {
    if (lane == __ffs(__ballot_sync(0xffffffffu, left == mth)) - 1) left = 0;
    mth = __reduce_max_sync(0xffffffffu, left);
  }
  const float warp_top = unordered(most);
  const float warp_total = warp_sum(own.relative() * exp_below(own.top, warp_top));
  if (lane == 0) {
    sm.part_top[warp] = warp_top;
    sm.part_sum[warp] = warp_total;
    sm.bound[warp] = warp < whole ? mth : 0xffffffffu;
  }
  if (tid == 0) sm.found = sm.columns = 0;
  if (tid < beam) list[tid] = 0;
  __syncthreads();
  uint32_t least = 0xffffffffu;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) least = min(least, sm.bound[w]);
  const float bound = unordered(max(least, ordered(-FLT_MAX)));   // -inf is no candidate
  // collect
  const auto push = [&](uint64_t e) { push_entry(sm, e); };
  const auto look = [&](int j, auto &&wanted, auto &&take) { look_at(row, j, wanted, take); };
  const auto reaches = [&](float x) { return x >= bound; };
  if (column_top >= bound) {
    if (column_next >= bound) sm.column[atomicAdd(&sm.columns, 1)] = tid;
    else look(column_at, reaches, push);
  }
  if (edge >= bound) push(entry_of(edge, (uint32_t)symbol));
  if (warp == kSelWarps - 2 && lane < kSelWarps) {   // the row's maximum and sum
    const unsigned mask = (1u << kSelWarps) - 1;
    const float mine = sm.part_top[lane], m = unordered(__reduce_max_sync(mask, ordered(mine)));
    double sum = sm.part_sum[lane] * (double)exp_below(mine, m);
#pragma unroll
    for (int o = kSelWarps / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
    if (lane == 0) out->top = m, out->sum = sum;
  }
  __syncthreads();
  const int columns = sm.columns, pairs = columns * ((end - first + kSelThreads - 1) / kSelThreads);
  for (int p = tid; p < pairs; p += kSelThreads) {
    const int level = p / columns, j = first + sm.column[p - level * columns] + level * kSelThreads;
    if (j < end && *(volatile int *)&sm.found <= kSelBuffer) look(j, reaches, push);
  }
  if (columns > 0) __syncthreads();
  int found = sm.found;
  if (found > kSelBuffer)
    found = crowded_row(sm, row, first, end, own.top, column_top, edge, symbol, beam);
  if (found <= kSelBuffer) {
    // order
    for (int c = tid; c < found; c += kSelThreads) {
      const uint64_t mine = sm.buffer[c];
      int earlier = 0;
#pragma unroll 8
      for (int o = 0; o < found; ++o) earlier += sm.buffer[o] > mine;
      if (earlier < beam) list[earlier] = mine;
    }
  } else {
    // still more, where the best ones lie in few columns: one at a time
    uint64_t last = ~0ull;
    for (int n = 0; n < beam; ++n) {
      uint64_t best = 0;
      const auto keep = [&](uint64_t e) { best = e < last && e > best ? e : best; };
      if (edge >= bound) keep(entry_of(edge, (uint32_t)symbol));
      if (column_top >= bound)
        for (int j = first + tid; j < end; j += kSelThreads) look(j, reaches, keep);
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
      }
      if (lane == 0) sm.next[warp] = best;
      __syncthreads();
      for (int w = 0; w < kSelWarps; ++w) best = sm.next[w] > best ? sm.next[w] : best;
      if (tid == 0) list[n] = best;
      last = best;
      __syncthreads();
    }
  }
}

// ---- joining an utterance's rows -------------------------------------------------------
// A score as an ordered integer (0: none) and a place in K x V, lower places first.
struct SelEntry {
  uint64_t key;
  uint32_t place;
};
__device__ __forceinline__ bool before(const SelEntry &a, const SelEntry &b) {
  return a.key > b.key || (a.key == b.key && a.place < b.place);
}

__global__ void __launch_bounds__(kSelThreads)
select_join_kernel(const SelSum *__restrict__ sums, const uint64_t *__restrict__ entries,
                   const float *__restrict__ scores, const uint8_t *__restrict__ finished, int blank,
                   float *__restrict__ out_scores, int64_t *__restrict__ out_parents,
                   int64_t *__restrict__ out_tokens, int K, int V, int parts, int beam) {
  __shared__ uint64_t key[kSelBuffer], next_key[kSelWarps];
  __shared__ uint32_t place[kSelBuffer], next_place[kSelWarps];
  __shared__ double row_log[kSelBeams];
  __shared__ float row_top[kSelBeams], row_shift[kSelBeams];   // score less log-sum; -inf: offers nothing
  __shared__ float warp_bound[kSelWarps], warp_widest[kSelWarps];
  __shared__ int found;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const SelSum *const sum = sums + (size_t)b * K * parts;
  const uint64_t *const list = entries + (size_t)b * K * parts * beam;
  // Neighbouring entries go to different warps: every warp then has about the same share of good
  // ones, and the least of their m-th best is a close bound.
  const int each_row = parts * beam, all = K * each_row, own = lane * kSelWarps + warp;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint64_t first_entry = own < all ? list[own] : 0;   // whether it is needed or not
  // a row's log-sum.  A finished row is one whose only entry has logit and log-sum 0.
  float widest = 0;
  for (int i = tid; i < K; i += kSelThreads) {
    const size_t at = (size_t)b * K + i;
    const float score = scores[at];
    const int kind = kind_of(score, finished, at);
    float top = 0, shift = kind == 1 ? score : neg_inf<float>();
    double log_sum = 0;
    if (kind == 2) {
      double total = 0;
      top = neg_inf<float>();
      for (int p = 0; p < parts; ++p) top = fmaxf(top, sum[i * parts + p].top);
      for (int p = 0; p < parts; ++p)
        total += sum[i * parts + p].sum * (double)exp_below(sum[i * parts + p].top, top);
      log_sum = log_of(total);
      if (fabsf(top) < INFINITY && total < (double)INFINITY)   // no NaN either; the row offers something
        shift = fmaxf((float)((double)score - (double)top - log_sum), -FLT_MAX);
    }
    row_log[i] = log_sum;
    row_top[i] = top;
    row_shift[i] = shift;
    if (shift != neg_inf<float>()) widest = fmaxf(widest, fabsf(shift));
  }
  if (tid == 0) found = 0;
  __syncthreads();
  const auto entry = [&](int n, int &i, bool &done) {   // the n-th of K x parts x beam; 0: none
    i = n / each_row;
    if (row_shift[i] == neg_inf<float>()) return (uint64_t)0;
    done = finished != nullptr && finished[(size_t)b * K + i] != 0;
    return !done ? (n < kSelThreads ? first_entry : list[n]) : n == i * each_row ? entry_of(0.0f, (uint32_t)blank) : (uint64_t)0;
  };
  float best = neg_inf<float>();
  for (int n = own; n < all; n += kSelThreads) {
    int i;
    bool done;
    const uint64_t e = entry(n, i, done);
    if (e != 0) best = fmaxf(best, logit_of(e) + row_shift[i]);
  }
  const int whole = min(kSelWarps, all);   // warps that have entries
  const float mth = mth_of_warp(best, (beam + whole - 1) / whole);
  widest = warp_max(widest);
  if (lane == 0) warp_bound[warp] = warp < whole ? mth : INFINITY, warp_widest[warp] = widest;
  __syncthreads();
  float bound = INFINITY;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) bound = fminf(bound, warp_bound[w]), widest = fmaxf(widest, warp_widest[w]);
  // a score in 32 bits, logit + shift, is off by at most 2^-24 of itself and of the shift; beyond
  // 1e30 (rows masked by the lowest numbers there are) all entries are taken
  bound -= 4.0f * 0x1p-23f * (fabsf(bound) + widest);
  if (!(widest < 1e30f)) bound = neg_inf<float>();
  const auto collect = [&](auto &&take) {
    for (int n = own; n < all; n += kSelThreads) {
      int i;
      bool done;
      const uint64_t e = entry(n, i, done);
      if (e == 0 || logit_of(e) + row_shift[i] < bound) continue;
      const double score = scores[(size_t)b * K + i];
      const uint32_t v = symbol_of(e);
      take(SelEntry{ordered(score + (((double)logit_of(e) - (double)row_top[i]) - row_log[i])), (uint32_t)i * (uint32_t)V + v});
    }
  };
  collect([&](const SelEntry &e) {
    const int n = atomicAdd(&found, 1);
    if (n < kSelBuffer) key[n] = e.key, place[n] = e.place;
  });
  __syncthreads();
  const auto write = [&](int n, const SelEntry &e) {
    const size_t o = (size_t)b * beam + n;
    out_scores[o] = (float)unordered(e.key);
    out_parents[o] = (int64_t)(e.place / (uint32_t)V);
    out_tokens[o] = (int64_t)(e.place % (uint32_t)V);
  };
  if (tid >= found && tid < beam) {   // slots left over
    const size_t o = (size_t)b * beam + tid;
    out_scores[o] = neg_inf<float>();
    out_parents[o] = out_tokens[o] = -1;
  }
  if (found <= kSelBuffer) {
    for (int c = tid; c < found; c += kSelThreads) {
      const SelEntry mine = {key[c], place[c]};
      int earlier = 0;
#pragma unroll 4
      for (int o = 0; o < found; ++o) earlier += before({key[o], place[o]}, mine);
      if (earlier < beam) write(earlier, mine);
    }
    return;
  }
  SelEntry last = {~0ull, 0};
  for (int n = 0; n < beam; ++n) {
    SelEntry next = {0, 0xffffffffu};
    collect([&](const SelEntry &e) { next = before(last, e) && before(e, next) ? e : next; });
    for (int o = 16; o > 0; o >>= 1) {
      const SelEntry other = {__shfl_xor_sync(0xffffffffu, next.key, o), __shfl_xor_sync(0xffffffffu, next.place, o)};
      if (before(other, next)) next = other;
    }
    if (lane == 0) next_key[warp] = next.key, next_place[warp] = next.place;
    __syncthreads();
    for (int w = 0; w < kSelWarps; ++w)
      if (before({next_key[w], next_place[w]}, next)) next = {next_key[w], next_place[w]};
    if (tid == 0) write(n, next);
    last = next;
    __syncthreads();
  }
}

// ---- reordering --------------------------------------------------------------------------
// A gather of rows, bound by memory: every thread has several pieces of 16 bytes (or fewer, where
// rows do not begin on such boundaries) under way at once, since each waits for its parent first.
constexpr int kReorderMost = 32;   // tensors of one launch
constexpr int kReorderThreads = 256, kReorderPieces = 4;
struct ReorderList {
  const char *from[kReorderMost];
  char *to[kReorderMost];
  long long batch[kReorderMost], beam[kReorderMost];   // strides of `from` in bytes
  long long bytes[kReorderMost];                       // of one row
  int width[kReorderMost];                             // of a piece, or of what is left beside shifted ones
};

template <typename W>
__device__ __forceinline__ void reorder_pieces(const ReorderList &list, int n, const int64_t *__restrict__ parents,
                                               long long rows, int beams, int K) {
  const long long per = list.bytes[n] / (long long)sizeof(W), all = rows * per;
  const long long first = (long long)blockIdx.x * (kReorderThreads * kReorderPieces) + threadIdx.x;
  W piece[kReorderPieces];
#pragma unroll
  for (int u = 0; u < kReorderPieces; ++u) {
    const long long at = first + u * kReorderThreads;
    if (at >= all) break;
    const long long row = all <= INT_MAX ? (int)at / (int)per : at / per;
    const int64_t p = parents[row];
    piece[u] = W{};
    if (p >= 0 && p < K)
      piece[u] = __ldg(reinterpret_cast<const W *>(list.from[n] + div_rows(row, beams) * list.batch[n] +
                                                   p * list.beam[n]) + (at - row * per));
  }
#pragma unroll
  for (int u = 0; u < kReorderPieces; ++u) {
    const long long at = first + u * kReorderThreads;
    if (at < all) reinterpret_cast<W *>(list.to[n])[at] = piece[u];
  }
}

// Rows that do not begin on 16-byte boundaries, both sides multiples of U apart from them: 16 bytes
// of the destination at a time, shifted together from the two granules of the source that hold
// them; what is left of a row before the first boundary, behind the last, and where a granule
// would reach out of the source row, goes U by U.  (256 x 8 rows of 1001 16-bit values in 12
// tensors: 36 us, U by U alone 96; of 1002, 34 and 50; rows of 8-byte pieces gain nothing.)
template <typename U>
__device__ __forceinline__ void reorder_shifted(const ReorderList &list, int n, const int64_t *__restrict__ parents,
                                                long long rows, int beams, int K) {
  const long long bytes = list.bytes[n], per = bytes / 16 + 2, all = rows * per;   // head, chunks, tail
  const long long first = (long long)blockIdx.x * (kReorderThreads * kReorderPieces) + threadIdx.x;
  uint4 piece[kReorderPieces], *target[kReorderPieces];
#pragma unroll
  for (int u = 0; u < kReorderPieces; ++u) {
    target[u] = nullptr;
    const long long at = first + u * kReorderThreads;
    if (at >= all) continue;   // every target is set
    const long long row = all <= INT_MAX ? (int)at / (int)per : at / per, k = at - row * per;
    const int64_t p = parents[row];
    const char *const from = p >= 0 && p < K ? list.from[n] + div_rows(row, beams) * list.batch[n] + p * list.beam[n]
                                             : nullptr;
    char *const to = list.to[n] + row * bytes;
    const long long head = min(bytes, (long long)(-(uintptr_t)to & 15));
    const long long lo = k == 0 ? 0 : head + 16 * (k - 1), hi = k == 0 ? head : min(bytes, lo + 16);
    const int off = (int)((uintptr_t)(from + lo) & 15);
    if (from == nullptr && hi - lo == 16) {
      piece[u] = uint4{};
      target[u] = reinterpret_cast<uint4 *>(to + lo);
    } else if (from != nullptr && hi - lo == 16 && lo >= off && lo - off + 32 <= bytes) {
      const uint4 *g = reinterpret_cast<const uint4 *>(from + lo - off);
      const uint4 q = __ldg(g), r = __ldg(g + 1);
      uint32_t w[8] = {q.x, q.y, q.z, q.w, r.x, r.y, r.z, r.w};
#pragma unroll
      for (int i = 0; i < 7; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], off % 4 * 8);
      piece[u] = make_uint4(w[0], w[1], w[2], w[3]);
      target[u] = reinterpret_cast<uint4 *>(to + lo);
    } else {
      constexpr int kMost = 16 / (int)sizeof(U);
      U rest[kMost];
#pragma unroll
      for (int i = 0; i < kMost; ++i)
        rest[i] = from != nullptr && lo + i * (int)sizeof(U) < hi ? __ldg(reinterpret_cast<const U *>(from + lo) + i) : U{};
#pragma unroll
      for (int i = 0; i < kMost; ++i)
        if (lo + i * (int)sizeof(U) < hi) reinterpret_cast<U *>(to + lo)[i] = rest[i];
    }
  }
#pragma unroll
  for (int u = 0; u < kReorderPieces; ++u)
    if (target[u] != nullptr) *target[u] = piece[u];
}

__global__ void __launch_bounds__(kReorderThreads)
beam_reorder_kernel(const __grid_constant__ ReorderList list, const int64_t *__restrict__ parents, long long rows,
                    int beams, int K) {
  const int n = blockIdx.y;
  switch (list.width[n]) {
    case 16: reorder_pieces<uint4>(list, n, parents, rows, beams, K); break;
    case 8: reorder_pieces<uint2>(list, n, parents, rows, beams, K); break;
    case 4: reorder_pieces<uint32_t>(list, n, parents, rows, beams, K); break;
    case 2: reorder_pieces<uint16_t>(list, n, parents, rows, beams, K); break;
    default: reorder_pieces<uint8_t>(list, n, parents, rows, beams, K);
  }
}

// a launch of its own: its registers would cost the aligned rows a sixth of their rate
__global__ void __launch_bounds__(kReorderThreads)
beam_reorder_shifted_kernel(const __grid_constant__ ReorderList list, const int64_t *__restrict__ parents,
                            long long rows, int beams, int K) {
  const int n = blockIdx.y;
  switch (list.width[n]) {
    case 4: reorder_shifted<uint32_t>(list, n, parents, rows, beams, K); break;
    case 2: reorder_shifted<uint16_t>(list, n, parents, rows, beams, K); break;
    default: reorder_shifted<uint8_t>(list, n, parents, rows, beams, K);
  }
}

// Parts of a row: as many as give every multiprocessor two CTAs, each with two rounds of the
// stream's loop or more.
static int select_parts(int size, int B, int K, int V) {
  const long long vectors = ((long long)V * size + 15) / 16;
  int parts = 1;
  while (parts < kSelParts && (long long)B * K * (parts + 1) <= 2 * sm_count() && (parts + 1) * 8 * kSelThreads <= vectors)
    ++parts;
  return parts;
}

template <typename T>
static int select_launch(const T *logits, long long batch, long long row, const float *scores,
                         const uint8_t *finished, int blank, float *out_scores, int64_t *out_parents,
                         int64_t *out_tokens, void *scratch, int B, int K, int V, int beam, cudaStream_t st) {
  const int parts = select_parts((int)sizeof(T), B, K, V);
  SelSum *sums = (SelSum *)scratch;
  uint64_t *entries = (uint64_t *)(sums + (size_t)B * K * parts);
  FRNNT_KERNEL(select_rows_kernel<T><<<dim3((unsigned)parts, (unsigned)K, (unsigned)B), kSelThreads, 0, st>>>(
      logits, batch, row, scores, finished, V, sums, entries, beam));
  FRNNT_CUDA(cudaGetLastError());
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)B);
  config.blockDim = dim3(kSelThreads);
  config.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  FRNNT_CUDA(FRNNT_KERNEL(cudaLaunchKernelEx(&config, select_join_kernel, (const SelSum *)sums,
                                             (const uint64_t *)entries, scores, finished, blank, out_scores,
                                             out_parents, out_tokens, K, V, parts, beam)));
  return FRNNT_OK;
}

}  // namespace frnnt

using namespace frnnt;

extern "C" size_t frnnt_beam_select_scratch_bytes(int dtype, int B, int K, int V, int beam) {
  if ((dtype != FRNNT_F32 && !is_half_input(dtype)) || B <= 0 || K <= 0 || V <= 0 || beam <= 0) return 0;
  return (size_t)B * K * select_parts(is_half_input(dtype) ? 2 : 4, B, K, V) * (sizeof(SelSum) + beam * sizeof(uint64_t));
}

extern "C" int frnnt_beam_select(int dtype, const void *logits, long long batch, long long row, const float *scores,
                                 const uint8_t *finished, int blank, float *out_scores, int64_t *out_parents,
                                 int64_t *out_tokens, void *scratch, int B, int K, int V, int beam, void *stream) {
  FRNNT_REQUIRE(dtype == FRNNT_F32 || is_half_input(dtype), FRNNT_EINVAL, "dtype must be FRNNT_F32, _F16 or _BF16");
  FRNNT_REQUIRE(B >= 0 && K >= 1 && V >= 1, FRNNT_EINVAL, "bad sizes");
  FRNNT_REQUIRE(beam >= 1 && beam <= kSelMost, FRNNT_EUNSUPPORTED, "beam must be 1 to %d", kSelMost);
  FRNNT_REQUIRE(K <= kSelBeams, FRNNT_EUNSUPPORTED, "at most %d beams", kSelBeams);
  FRNNT_REQUIRE((long long)K * V < INT_MAX, FRNNT_EUNSUPPORTED, "beams times vocabulary must be below 2^31");
  FRNNT_REQUIRE(finished == nullptr || (blank >= 0 && blank < V), FRNNT_EINVAL, "termination symbol out of range");
  if (B == 0) return FRNNT_OK;
  FRNNT_REQUIRE(logits && scores && out_scores && out_parents && out_tokens && scratch, FRNNT_EINVAL, "NULL argument");
  FRNNT_REQUIRE((uintptr_t)scratch % 16 == 0, FRNNT_EINVAL, "scratch must be 16-byte aligned");
  FRNNT_REQUIRE(B <= 65535, FRNNT_EUNSUPPORTED, "B too large for the grid");
#define FRNNT_SELECT(TYPE)                                                                                \
  return select_launch<TYPE>((const TYPE *)logits, batch, row, scores, finished, blank, out_scores,       \
                             out_parents, out_tokens, scratch, B, K, V, beam, (cudaStream_t)stream)
  if (dtype == FRNNT_F32) FRNNT_SELECT(float);
  if (dtype == FRNNT_F16) FRNNT_SELECT(__half);
  FRNNT_SELECT(__nv_bfloat16);
#undef FRNNT_SELECT
}

extern "C" int frnnt_beam_reorder(int count, const frnnt_rows *tensors, const int64_t *parents, int B, int beams, int K,
                                  void *stream) {
  FRNNT_REQUIRE(count >= 0 && B >= 0 && beams >= 0 && K >= 1, FRNNT_EINVAL, "bad sizes");
  const long long rows = (long long)B * beams;
  if (count == 0 || rows == 0) return FRNNT_OK;
  FRNNT_REQUIRE(tensors && parents, FRNNT_EINVAL, "NULL argument");
  for (int n = 0; n < count; ++n) {
    const frnnt_rows &t = tensors[n];
    FRNNT_REQUIRE(t.bytes >= 0 && (t.bytes == 0 || (t.from && t.to)), FRNNT_EINVAL, "NULL argument");
    FRNNT_REQUIRE(t.bytes == 0 || t.from != t.to, FRNNT_EINVAL, "a tensor cannot be reordered in place");
  }
  cudaStream_t st = (cudaStream_t)stream;
  // two kinds of rows: those moved in pieces of their alignment (8 or 16 bytes, or short), and shifted ones
  for (int shifted = 0; shifted < 2; ++shifted) {
    ReorderList list{};
    int m = 0;
    long long blocks = 1;
    for (int n = 0; n < count; ++n) {
      const frnnt_rows &t = tensors[n];
      const unsigned long long low = (uintptr_t)t.from | (uintptr_t)t.to | (unsigned long long)t.batch |
                                     (unsigned long long)t.beam | (unsigned long long)t.bytes;
      const int width = low % 16 == 0 ? 16 : low % 8 == 0 ? 8 : low % 4 == 0 ? 4 : low % 2 == 0 ? 2 : 1;
      if (t.bytes > 0 && (width <= 4 && t.bytes >= 64) == (shifted == 1)) {
        list.from[m] = (const char *)t.from;
        list.to[m] = (char *)t.to;
        list.batch[m] = t.batch;
        list.beam[m] = t.beam;
        list.bytes[m] = t.bytes;
        list.width[m] = width;
        ++m;
        const long long pieces = rows * (shifted ? t.bytes / 16 + 2 : t.bytes / width);
        const long long need = (pieces + kReorderThreads * kReorderPieces - 1) / (kReorderThreads * kReorderPieces);
        blocks = need > blocks ? need : blocks;
      }
      if (m == kReorderMost || (n + 1 == count && m > 0)) {
        FRNNT_REQUIRE(blocks <= INT_MAX, FRNNT_EUNSUPPORTED, "too many rows for the grid");
        const dim3 grid((unsigned)blocks, (unsigned)m);
        if (shifted)
          FRNNT_KERNEL(beam_reorder_shifted_kernel<<<grid, kReorderThreads, 0, st>>>(list, parents, rows, beams, K));
        else
          FRNNT_KERNEL(beam_reorder_kernel<<<grid, kReorderThreads, 0, st>>>(list, parents, rows, beams, K));
        FRNNT_CUDA(cudaGetLastError());
        m = 0;
        blocks = 1;
      }
    }
  }
  return FRNNT_OK;
}
