// Gated linear recurrence: h_t = f_t h_{t-1} + (1 - f_t) x_t with f = sigmoid(gate), every channel
// on its own; forward, backward, and one token for decoding.
//
// A step is the map h -> f h + u, and maps compose: (A1, B1) then (A2, B2) is (A1 A2, A2 B1 + B2).
// So a CTA takes a tile of 128 steps at once: every thread composes the few consecutive steps
// that it holds in registers (a "piece"), the pieces of a channel are joined through shared
// memory, and every thread then runs its steps again from the state before its piece, which is
// the recurrence itself and all that is rounded to the output's type.  Where there are fewer
// channels than would fill the GPU, a cluster of CTAs takes that many tiles of one sequence at
// once and joins their compositions through distributed shared memory; the order of all sums
// depends on the sizes alone.
//
// backward: lam_t = dh_t + f_{t+1} lam_{t+1} is the same recurrence from the other end, with the
// same products of gates.  h_{t-1} is recomputed from the state that the forward keeps per tile:
// 5 values an element move instead of 6, and h keeps its 32 bits.
//
// Both are bound by memory: 3 values an element forward, 5 backward, in their own type.  Inputs
// go to shared memory with cp.async a tile ahead, each thread fetching just what it reads
// itself, so that no barrier belongs to the copies.
#include <cooperative_groups.h>

#include <climits>

#include "common.cuh"
#include "recurrence.cuh"

namespace frnnt {

constexpr int kRecMostCluster = 8;

// ---- copies to shared memory ---------------------------------------------------------
template <int BYTES> __device__ __forceinline__ void copy_async(void *to, const void *from) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else if constexpr (BYTES == 8)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(at), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// One input's tile: kSteps vectors per thread, at [step][thread], so that a warp's accesses are
// contiguous.  Values of two bytes that no wider vector reaches are loaded and stored instead
// (cp.async moves 4, 8 or 16 bytes).
template <typename S> struct RecTile {
  using T = typename S::T;
  using Pack = RecPack<T, S::VEC>;
  __device__ static void fetch(Pack *tile, const T *from, long long step, int first, int n) {
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      if (first + s >= n) break;
      const T *p = from + (first + s) * step;
      if constexpr (sizeof(Pack) == 2)
        tile[s * kRecThreads] = *reinterpret_cast<const Pack *>(p);
      else
        copy_async<(int)sizeof(Pack)>(&tile[s * kRecThreads], p);
    }
  }
};

// where a thread stands in the tile of its CTA
template <typename S> struct RecPlace {
  int piece, c, channel;     // piece of the tile, channel within the tile, channel
  bool inside;               // the channel exists
  int join_q, join_c;        // as a joiner: run of pieces and channel within the tile
  bool joiner;
  __device__ RecPlace(int tile, int D) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    piece = warp * S::kGroups + lane / S::LC;
    c = lane % S::LC * S::VEC;
    channel = tile * S::kWidth + c;
    inside = channel < D;    // D is a multiple of VEC
    joiner = tid < S::kJoiners;
    join_q = S::kJoin == 1 ? 0 : lane >> 3;
    join_c = S::kJoin == 1 ? tid : warp * 8 + (lane & 7);
  }
};

// VEC values of the exchange, 16 bytes at a time where VEC of them fill that
template <typename real, int VEC> __device__ __forceinline__ void put(real *to, const real (&v)[VEC]) {
#pragma unroll
  for (int k = 0; k < VEC; k += VEC % 4 == 0 ? 4 : VEC % 2 == 0 ? 2 : 1) {
    if constexpr (sizeof(real) == 4 && VEC % 4 == 0)
      *reinterpret_cast<float4 *>(to + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
    else if constexpr (sizeof(real) == 4 && VEC % 2 == 0)
      *reinterpret_cast<float2 *>(to + k) = make_float2(v[k], v[k + 1]);
    else if constexpr (VEC % 2 == 0)
      *reinterpret_cast<double2 *>(to + k) = make_double2(v[k], v[k + 1]);
    else
      to[k] = v[k];
  }
}
template <typename real, int VEC> __device__ __forceinline__ void get(const real *from, real (&v)[VEC]) {
#pragma unroll
  for (int k = 0; k < VEC; k += VEC % 4 == 0 ? 4 : VEC % 2 == 0 ? 2 : 1) {
    if constexpr (sizeof(real) == 4 && VEC % 4 == 0) {
      const float4 q = *reinterpret_cast<const float4 *>(from + k);
      v[k] = q.x, v[k + 1] = q.y, v[k + 2] = q.z, v[k + 3] = q.w;
    } else if constexpr (sizeof(real) == 4 && VEC % 2 == 0) {
      const float2 q = *reinterpret_cast<const float2 *>(from + k);
      v[k] = q.x, v[k + 1] = q.y;
    } else if constexpr (VEC % 2 == 0) {
      const double2 q = *reinterpret_cast<const double2 *>(from + k);
      v[k] = q.x, v[k + 1] = q.y;
    } else {
      v[k] = from[k];
    }
  }
}

// The state that a tile starts from, and the one after all tiles of the cluster's turn: `carry`
// is the state before the turn, (A, B) the composition of this CTA's tile, slots [ranks][2][width]
// where every CTA leaves its own in every CTA.  FORWARD: in the order of the ranks, else against.
template <typename S, bool FORWARD>
__device__ __forceinline__ typename S::real
join_cluster(typename S::real A, typename S::real B, typename S::real &carry, typename S::real *slots, int rank,
             int ranks, const RecPlace<S> &at) {
  using real = typename S::real;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  if (at.joiner) {
    for (int r = at.join_q; r < ranks; r += S::kJoin) {
      real *peer = cluster.map_shared_rank(slots, r) + rank * 2 * S::kWidth + at.join_c;
      peer[0] = A;
      peer[S::kWidth] = B;
    }
  }
  cluster.sync();
  real before = carry;
  if (at.joiner) {
    for (int i = 0; i < ranks; ++i) {
      const int r = FORWARD ? i : ranks - 1 - i;
      if (r == rank) before = carry;
      const real *own = slots + r * 2 * S::kWidth + at.join_c;
      carry = own[0] * carry + own[S::kWidth];
    }
  }
  return before;
}

template <typename S, bool CLUSTER>
__global__ void __launch_bounds__(kRecThreads)
recurrence_forward_kernel(RecTensor x, RecTensor gate, const typename S::real *__restrict__ initial,
                          const int64_t *__restrict__ lengths, typename S::T *__restrict__ h,
                          typename S::real *__restrict__ last, typename S::real *__restrict__ saved, int steps,
                          int D) {
  using T = typename S::T;
  using real = typename S::real;
  using Pack = RecPack<T, S::VEC>;
  constexpr int VEC = S::VEC, STEPS = S::kSteps;
  extern __shared__ __align__(16) unsigned char smem[];
  Pack *const tiles = reinterpret_cast<Pack *>(smem) + threadIdx.x;        // [2][x, gate][STEPS][thread]
  real *const exchange = reinterpret_cast<real *>(smem + 4 * S::kStage);   // [2][A, B][kExchange]
  real *const slots = exchange + 4 * S::kExchange;                         // [2][ranks][2][kWidth]
  const int rank = CLUSTER ? blockIdx.x : 0, ranks = CLUSTER ? gridDim.x : 1;
  const int b = blockIdx.z;
  const RecPlace<S> at(blockIdx.y, D);
  const int n = steps_of(lengths, b, steps), chunks = (steps + kRecChunk - 1) / kRecChunk;
  const T *const X = (const T *)x.data + b * x.batch + at.channel;
  const T *const G = (const T *)gate.data + b * gate.batch + at.channel;
  T *const H = h + (size_t)b * steps * D + at.channel;
  const int join_channel = blockIdx.y * S::kWidth + at.join_c;
  const bool keeper = at.joiner && join_channel < D;
  real carry = keeper && initial != nullptr ? initial[(size_t)b * D + join_channel] : real(0);
  const int turns = (n + kRecChunk * ranks - 1) / (kRecChunk * ranks);
  const int piece_first = at.piece * STEPS;

  const auto fetch = [&](int turn) {
    const int first = (turn * ranks + rank) * kRecChunk + piece_first;
    Pack *tile = tiles + (turn & 1) * 2 * STEPS * kRecThreads;
    if (at.inside && turn < turns) {
      RecTile<S>::fetch(tile, X, x.step, first, n);
      RecTile<S>::fetch(tile + STEPS * kRecThreads, G, gate.step, first, n);
    }
    copy_commit();
  };
  fetch(0);
  if constexpr (CLUSTER) cooperative_groups::this_cluster().sync();   // all have started
  for (int turn = 0; turn < turns; ++turn) {
    fetch(turn + 1);
    copy_wait<1>();
    const int chunk = turn * ranks + rank, first = chunk * kRecChunk + piece_first;
    real *const EA = exchange + (turn & 1) * 2 * S::kExchange, *const EB = EA + S::kExchange;
    real f[STEPS][VEC], u[STEPS][VEC], A[VEC], B[VEC];
    const Pack *tile = tiles + (turn & 1) * 2 * STEPS * kRecThreads;
#pragma unroll
    for (int k = 0; k < VEC; ++k) A[k] = real(1), B[k] = real(0);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const bool live = at.inside && first + s < n;
      real xv[VEC], gv[VEC];
      rec_unpack<T, VEC>(tile[s * kRecThreads], xv);
      rec_unpack<T, VEC>(tile[(STEPS + s) * kRecThreads], gv);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        real keep, take;
        gate_pair<T>(gv[k], keep, take);
        f[s][k] = live ? keep : real(1);
        u[s][k] = live ? take * xv[k] : real(0);
        A[k] *= f[s][k];
        B[k] = f[s][k] * B[k] + u[s][k];
      }
    }
    put<real, VEC>(EA + S::at(at.piece, at.c), A);
    put<real, VEC>(EB + S::at(at.piece, at.c), B);
    __syncthreads();
    // join: kRun pieces a thread, then the runs of a channel by shuffles
    real ra[S::kRun], rb[S::kRun], a = real(1), bb = real(0);
    if (at.joiner) {
#pragma unroll
      for (int j = 0; j < S::kRun; ++j) {
        const int e = S::at(at.join_q * S::kRun + j, at.join_c);
        ra[j] = EA[e];
        rb[j] = EB[e];
        a *= ra[j];
        bb = ra[j] * bb + rb[j];
      }
    }
    real ex_a = real(1), ex_b = real(0);   // the runs before this one
    if constexpr (S::kJoin > 1) {
#pragma unroll
      for (int o = 1; o < S::kJoin; o *= 2) {
        const real pa = __shfl_up_sync(0xffffffffu, a, 8 * o), pb = __shfl_up_sync(0xffffffffu, bb, 8 * o);
        if (at.join_q >= o) {
          bb = a * pb + bb;
          a *= pa;
        }
      }
      const real pa = __shfl_up_sync(0xffffffffu, a, 8), pb = __shfl_up_sync(0xffffffffu, bb, 8);
      if (at.join_q > 0) ex_a = pa, ex_b = pb;
      a = __shfl_sync(0xffffffffu, a, 8 * (S::kJoin - 1) + (threadIdx.x & 7));
      bb = __shfl_sync(0xffffffffu, bb, 8 * (S::kJoin - 1) + (threadIdx.x & 7));
    }
    real start = carry;
    if constexpr (CLUSTER)
      start = join_cluster<S, true>(a, bb, carry, slots + (turn & 1) * ranks * 2 * S::kWidth, rank, ranks, at);
    else
      carry = a * carry + bb;
    if (at.joiner) {
      if (saved != nullptr && at.join_q == 0 && keeper && chunk < chunks)
        saved[((size_t)b * chunks + chunk) * D + join_channel] = start;
      real state = ex_a * start + ex_b;
#pragma unroll
      for (int j = 0; j < S::kRun; ++j) {
        EB[S::at(at.join_q * S::kRun + j, at.join_c)] = state;
        state = ra[j] * state + rb[j];
      }
    }
    __syncthreads();
    real state[VEC];
    get<real, VEC>(EB + S::at(at.piece, at.c), state);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) state[k] = f[s][k] * state[k] + u[s][k];
      if (at.inside && first + s < n)
        *reinterpret_cast<Pack *>(H + (size_t)(first + s) * D) = rec_pack<T, VEC>(state);
    }
  }
  if (at.inside) {   // behind the sequence
    const real zero[VEC] = {};
    for (long long t = (long long)n + rank * S::kPieces + at.piece; t < steps; t += ranks * S::kPieces)
      *reinterpret_cast<Pack *>(H + t * D) = rec_pack<T, VEC>(zero);
  }
  if (keeper && rank == 0 && at.join_q == 0) last[(size_t)b * D + join_channel] = carry;
}

template <typename S, bool CLUSTER>
__global__ void __launch_bounds__(kRecThreads)
recurrence_backward_kernel(RecTensor x, RecTensor gate, const int64_t *__restrict__ lengths,
                           const typename S::real *__restrict__ saved, RecTensor dh,
                           const typename S::real *__restrict__ dlast, typename S::T *__restrict__ dx,
                           typename S::T *__restrict__ dgate, typename S::real *__restrict__ dinitial, int steps,
                           int D) {
  using T = typename S::T;
  using real = typename S::real;
  using Pack = RecPack<T, S::VEC>;
  constexpr int VEC = S::VEC, STEPS = S::kSteps;
  extern __shared__ __align__(16) unsigned char smem[];
  Pack *const tiles = reinterpret_cast<Pack *>(smem) + threadIdx.x;        // [2][x, gate, dh][STEPS][thread]
  real *const exchange = reinterpret_cast<real *>(smem + 6 * S::kStage);   // [2][A, B, M][kExchange]
  real *const slots = exchange + 6 * S::kExchange;                         // [2][ranks][2][kWidth]
  const int rank = CLUSTER ? blockIdx.x : 0, ranks = CLUSTER ? gridDim.x : 1;
  const int b = blockIdx.z;
  const RecPlace<S> at(blockIdx.y, D);
  const int n = steps_of(lengths, b, steps), chunks = (steps + kRecChunk - 1) / kRecChunk;
  const T *const X = (const T *)x.data + b * x.batch + at.channel;
  const T *const G = (const T *)gate.data + b * gate.batch + at.channel;
  const T *const DH = dh.data == nullptr ? nullptr : (const T *)dh.data + b * dh.batch + at.channel;
  T *const DX = dx + (size_t)b * steps * D + at.channel, *const DG = dgate + (size_t)b * steps * D + at.channel;
  const int join_channel = blockIdx.y * S::kWidth + at.join_c;
  const bool keeper = at.joiner && join_channel < D;
  real carry = keeper && dlast != nullptr ? dlast[(size_t)b * D + join_channel] : real(0);
  const int turns = (n + kRecChunk * ranks - 1) / (kRecChunk * ranks);
  const int piece_first = at.piece * STEPS;

  const auto fetch = [&](int turn) {
    const int first = (turn * ranks + rank) * kRecChunk + piece_first;
    Pack *tile = tiles + (turn & 1) * 3 * STEPS * kRecThreads;
    if (at.inside && turn >= 0) {
      RecTile<S>::fetch(tile, X, x.step, first, n);
      RecTile<S>::fetch(tile + STEPS * kRecThreads, G, gate.step, first, n);
      if (DH != nullptr) RecTile<S>::fetch(tile + 2 * STEPS * kRecThreads, DH, dh.step, first, n);
    }
    copy_commit();
  };
  fetch(turns - 1);
  if constexpr (CLUSTER) cooperative_groups::this_cluster().sync();   // all have started
  for (int turn = turns - 1; turn >= 0; --turn) {
    fetch(turn - 1);
    const int chunk = turn * ranks + rank, first = chunk * kRecChunk + piece_first;
    real start = real(0);   // the state before the tile
    if (keeper && chunk * kRecChunk < n) start = saved[((size_t)b * chunks + chunk) * D + join_channel];
    copy_wait<1>();
    real *const EA = exchange + (turn & 1) * 3 * S::kExchange, *const EB = EA + S::kExchange,
               *const EM = EB + S::kExchange;
    real f[STEPS][VEC], take[STEPS][VEC], A[VEC], B[VEC], M[VEC];
    const Pack *tile = tiles + (turn & 1) * 3 * STEPS * kRecThreads;
#pragma unroll
    for (int k = 0; k < VEC; ++k) A[k] = real(1), B[k] = M[k] = real(0);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const bool live = at.inside && first + s < n;
      real xv[VEC], gv[VEC];
      rec_unpack<T, VEC>(tile[s * kRecThreads], xv);
      rec_unpack<T, VEC>(tile[(STEPS + s) * kRecThreads], gv);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        gate_pair<T>(gv[k], f[s][k], take[s][k]);
        f[s][k] = live ? f[s][k] : real(1);
        A[k] *= f[s][k];
        B[k] = f[s][k] * B[k] + (live ? take[s][k] * xv[k] : real(0));
      }
    }
#pragma unroll
    for (int s = STEPS - 1; s >= 0; --s) {
      const bool live = at.inside && first + s < n && DH != nullptr;
      real dv[VEC];
      rec_unpack<T, VEC>(tile[(2 * STEPS + s) * kRecThreads], dv);
#pragma unroll
      for (int k = 0; k < VEC; ++k) M[k] = f[s][k] * (M[k] + (live ? dv[k] : real(0)));
    }
    put<real, VEC>(EA + S::at(at.piece, at.c), A);
    put<real, VEC>(EB + S::at(at.piece, at.c), B);
    put<real, VEC>(EM + S::at(at.piece, at.c), M);
    __syncthreads();
    real ra[S::kRun], rb[S::kRun], rm[S::kRun], a = real(1), bb = real(0), m = real(0);
    if (at.joiner) {
#pragma unroll
      for (int j = 0; j < S::kRun; ++j) {
        const int e = S::at(at.join_q * S::kRun + j, at.join_c);
        ra[j] = EA[e];
        rb[j] = EB[e];
        rm[j] = EM[e];
        a *= ra[j];
        bb = ra[j] * bb + rb[j];
      }
#pragma unroll
      for (int j = S::kRun - 1; j >= 0; --j) m = ra[j] * m + rm[j];
    }
    real ex_a = real(1), ex_b = real(0);   // the runs before this one
    real af_a = real(1), af_m = real(0);   // the runs after it
    if constexpr (S::kJoin > 1) {
      real fa = a, sa = a;
#pragma unroll
      for (int o = 1; o < S::kJoin; o *= 2) {
        const real pa = __shfl_up_sync(0xffffffffu, fa, 8 * o), pb = __shfl_up_sync(0xffffffffu, bb, 8 * o);
        const real na = __shfl_down_sync(0xffffffffu, sa, 8 * o), nm = __shfl_down_sync(0xffffffffu, m, 8 * o);
        if (at.join_q >= o) {
          bb = fa * pb + bb;
          fa *= pa;
        }
        if (at.join_q + o < S::kJoin) {
          m = sa * nm + m;
          sa *= na;
        }
      }
      const real pa = __shfl_up_sync(0xffffffffu, fa, 8), pb = __shfl_up_sync(0xffffffffu, bb, 8);
      const real na = __shfl_down_sync(0xffffffffu, sa, 8), nm = __shfl_down_sync(0xffffffffu, m, 8);
      if (at.join_q > 0) ex_a = pa, ex_b = pb;
      if (at.join_q + 1 < S::kJoin) af_a = na, af_m = nm;
      a = __shfl_sync(0xffffffffu, sa, threadIdx.x & 7);   // of the whole tile
      m = __shfl_sync(0xffffffffu, m, threadIdx.x & 7);
    }
    real flow = carry;
    if constexpr (CLUSTER)
      flow = join_cluster<S, false>(a, m, carry, slots + (turn & 1) * ranks * 2 * S::kWidth, rank, ranks, at);
    else
      carry = a * carry + m;
    if (at.joiner) {
      real state = ex_a * start + ex_b;
      flow = af_a * flow + af_m;
#pragma unroll
      for (int j = 0; j < S::kRun; ++j) {
        EB[S::at(at.join_q * S::kRun + j, at.join_c)] = state;
        state = ra[j] * state + rb[j];
      }
#pragma unroll
      for (int j = S::kRun - 1; j >= 0; --j) {
        EM[S::at(at.join_q * S::kRun + j, at.join_c)] = flow;
        flow = ra[j] * flow + rm[j];
      }
    }
    __syncthreads();
    real before[STEPS][VEC], state[VEC], back[VEC];
    get<real, VEC>(EB + S::at(at.piece, at.c), state);
    get<real, VEC>(EM + S::at(at.piece, at.c), back);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      real xv[VEC];
      rec_unpack<T, VEC>(tile[s * kRecThreads], xv);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        before[s][k] = state[k];
        state[k] = f[s][k] * state[k] + take[s][k] * xv[k];
      }
    }
#pragma unroll
    for (int s = STEPS - 1; s >= 0; --s) {
      if (!at.inside || first + s >= n) continue;
      real xv[VEC], dv[VEC], ox[VEC], og[VEC];
      rec_unpack<T, VEC>(tile[s * kRecThreads], xv);
      rec_unpack<T, VEC>(tile[(2 * STEPS + s) * kRecThreads], dv);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const real lam = back[k] + (DH != nullptr ? dv[k] : real(0));
        ox[k] = take[s][k] * lam;
        og[k] = lam * (before[s][k] - xv[k]) * (f[s][k] * take[s][k]);
        back[k] = f[s][k] * lam;
      }
      *reinterpret_cast<Pack *>(DX + (size_t)(first + s) * D) = rec_pack<T, VEC>(ox);
      *reinterpret_cast<Pack *>(DG + (size_t)(first + s) * D) = rec_pack<T, VEC>(og);
    }
  }
  if (at.inside) {   // behind the sequence
    const real zero[VEC] = {};
    for (long long t = (long long)n + rank * S::kPieces + at.piece; t < steps; t += ranks * S::kPieces) {
      *reinterpret_cast<Pack *>(DX + t * D) = rec_pack<T, VEC>(zero);
      *reinterpret_cast<Pack *>(DG + t * D) = rec_pack<T, VEC>(zero);
    }
  }
  if (dinitial != nullptr && keeper && rank == 0 && at.join_q == 0) dinitial[(size_t)b * D + join_channel] = carry;
}

constexpr int kStepThreads = 128;

// One token: every row reads the state of its parent (its own without parents; zero where the
// parent is not one of the K rows) and writes the new state and its rounding to x's type.
template <typename T>
__global__ void __launch_bounds__(kStepThreads)
recurrence_step_kernel(const T *__restrict__ x, long long x_row, const T *__restrict__ gate, long long gate_row,
                       const RecState<T> *__restrict__ state, const int64_t *__restrict__ parents,
                       T *__restrict__ h, RecState<T> *__restrict__ next, long long rows, int beams, int K, int D) {
  using real = RecState<T>;
  const int d = blockIdx.x * kStepThreads + threadIdx.x;
  if (d >= D) return;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    long long from = row;
    if (parents != nullptr) {
      const int64_t p = parents[row];
      from = p < 0 || p >= K ? -1 : div_rows(row, beams) * K + p;
    }
    real keep, take;
    gate_pair<T>(rec_value<T>(gate[row * gate_row + d]), keep, take);
    const real old = from < 0 ? real(0) : state[from * D + d];
    const real now = keep * old + take * rec_value<T>(x[row * x_row + d]);
    next[row * D + d] = now;
    if (h != nullptr) h[row * D + d] = rec_round<T>(now);
  }
}

// ---- host ----------------------------------------------------------------------------

// CTAs of a cluster: as many tiles of one sequence at once as it takes to give every
// multiprocessor a CTA, no more than the sequence has.
static int ranks_for(long long ctas, int T) {
  int ranks = 1;
  while (ranks < kRecMostCluster && ctas * ranks < sm_count() && 2 * ranks <= (T + kRecChunk - 1) / kRecChunk)
    ranks *= 2;
  return ranks;
}

template <typename S, typename... Params, typename... Args>
static int rec_launch(void (*alone)(Params...), void (*cluster)(Params...), int arrays, int B, int T, int D,
                      cudaStream_t st, Args... args) {
  const int tiles = (D + S::kWidth - 1) / S::kWidth;
  FRNNT_REQUIRE(B <= 65535 && tiles <= 65535, FRNNT_EUNSUPPORTED, "B or D too large for the grid");
  FRNNT_REQUIRE(T <= INT_MAX - kRecMostCluster * kRecChunk, FRNNT_EUNSUPPORTED, "T too large");
  const int ranks = ranks_for((long long)B * tiles, T);
  const size_t smem = 2 * (size_t)arrays * (S::kStage + S::kExchange * sizeof(typename S::real)) +
                      (ranks > 1 ? 4 * ranks * S::kWidth * sizeof(typename S::real) : 0);
  void (*kernel)(Params...) = ranks > 1 ? cluster : alone;
  FRNNT_CUDA(cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)ranks, (unsigned)tiles, (unsigned)B);
  config.blockDim = dim3(kRecThreads);
  config.dynamicSmemBytes = smem;
  config.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = ranks > 1 ? 1 : 0;
  FRNNT_CUDA(FRNNT_KERNEL(cudaLaunchKernelEx(&config, kernel, args...)));
  return FRNNT_OK;
}

// whether rows of D values from `data` on, with these strides, can be read `bytes` at a time
static bool rec_aligned(const RecTensor &t, int size, int D, int bytes) {
  return (uintptr_t)t.data % bytes == 0 && t.batch * size % bytes == 0 && t.step * size % bytes == 0 &&
         (long long)D * size % bytes == 0;
}

template <typename S>
static int forward_as(const RecTensor &x, const RecTensor &gate, const void *initial, const int64_t *lengths, void *h,
                      void *last, void *saved, int B, int T, int D, cudaStream_t st) {
  using real = typename S::real;
  return rec_launch<S>(recurrence_forward_kernel<S, false>, recurrence_forward_kernel<S, true>, 2, B, T, D, st, x, gate,
                       (const real *)initial, lengths, (typename S::T *)h, (real *)last, (real *)saved, T, D);
}
template <typename S>
static int backward_as(const RecTensor &x, const RecTensor &gate, const int64_t *lengths, const void *saved,
                       const RecTensor &dh, const void *dlast, void *dx, void *dgate, void *dinitial, int B, int T,
                       int D, cudaStream_t st) {
  using real = typename S::real;
  return rec_launch<S>(recurrence_backward_kernel<S, false>, recurrence_backward_kernel<S, true>, 3, B, T, D, st, x,
                       gate, lengths, (const real *)saved, dh, (const real *)dlast, (typename S::T *)dx,
                       (typename S::T *)dgate, (real *)dinitial, T, D);
}

// Vectors of 16 bytes where every row allows them, eight lanes to the 128 bytes of a line; else
// of 4 bytes (a float, or a pair of 16-bit values) where they do, else single values, 32 lanes
// side by side.
#define FRNNT_REC_SHAPES(CALL, wide, pairs)                                              \
  switch (dtype) {                                                                       \
    case FRNNT_F32:                                                                      \
      return wide ? CALL(RecShape<float, 4, 8>) : CALL(RecShape<float, 1, 32>);          \
    case FRNNT_F64:                                                                      \
      return wide ? CALL(RecShape<double, 2, 8>) : CALL(RecShape<double, 1, 32>);        \
    case FRNNT_F16:                                                                      \
      return wide ? CALL(RecShape<__half, 8, 8>)                                         \
                  : pairs ? CALL(RecShape<__half, 2, 32>) : CALL(RecShape<__half, 1, 32>); \
    default:                                                                             \
      return wide ? CALL(RecShape<__nv_bfloat16, 8, 8>)                                  \
                  : pairs ? CALL(RecShape<__nv_bfloat16, 2, 32>) : CALL(RecShape<__nv_bfloat16, 1, 32>); \
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
static int rec_size(int dtype) { return dtype == FRNNT_F64 ? 8 : dtype == FRNNT_F32 ? 4 : 2; }
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
  if (B == 0 || D == 0) return FRNNT_OK;
  FRNNT_REQUIRE(last && (T == 0 || (x && gate && h)), FRNNT_EINVAL, "NULL argument");
  const RecTensor X{x, x_batch, x_step}, G{gate, gate_batch, gate_step};
  const int size = rec_size(dtype);
  const auto fits = [&](int bytes) {
    return rec_aligned(X, size, D, bytes) && rec_aligned(G, size, D, bytes) && (uintptr_t)h % bytes == 0;
  };
  const bool wide = fits(16), pairs = fits(4);
#define FRNNT_REC_FORWARD(...) \
  forward_as<__VA_ARGS__>(X, G, initial, lengths, h, last, saved, B, T, D, (cudaStream_t)stream)
  FRNNT_REC_SHAPES(FRNNT_REC_FORWARD, wide, pairs)
#undef FRNNT_REC_FORWARD
}

extern "C" int frnnt_recurrence_backward(int dtype, const void *x, long long x_batch, long long x_step,
                                         const void *gate, long long gate_batch, long long gate_step,
                                         const int64_t *lengths, const void *saved, const void *dh,
                                         long long dh_batch, long long dh_step, const void *dlast, void *dx,
                                         void *dgate, void *dinitial, int B, int T, int D, void *stream) {
  FRNNT_REQUIRE(rec_dtype(dtype), FRNNT_EINVAL, "dtype must be FRNNT_F32, _F64, _F16 or _BF16");
  FRNNT_REQUIRE(rec_sizes(B, T, D), FRNNT_EINVAL, "bad sizes");
  if (B == 0 || D == 0) return FRNNT_OK;
  FRNNT_REQUIRE(T == 0 || (x && gate && saved && dx && dgate), FRNNT_EINVAL, "NULL argument");
  const RecTensor X{x, x_batch, x_step}, G{gate, gate_batch, gate_step}, DH{dh, dh_batch, dh_step};
  const int size = rec_size(dtype);
  const auto fits = [&](int bytes) {
    return rec_aligned(X, size, D, bytes) && rec_aligned(G, size, D, bytes) &&
           (dh == nullptr || rec_aligned(DH, size, D, bytes)) && (uintptr_t)dx % bytes == 0 &&
           (uintptr_t)dgate % bytes == 0;
  };
  const bool wide = fits(16), pairs = fits(4);
#define FRNNT_REC_BACKWARD(...)                                                              \
  backward_as<__VA_ARGS__>(X, G, lengths, saved, DH, dlast, dx, dgate, dinitial, B, T, D,    \
                           (cudaStream_t)stream)
  FRNNT_REC_SHAPES(FRNNT_REC_BACKWARD, wide, pairs)
#undef FRNNT_REC_BACKWARD
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
  const dim3 grid((unsigned)((D + kStepThreads - 1) / kStepThreads), (unsigned)(rows < 65535 ? rows : 65535));
#define FRNNT_REC_STEP(TYPE)                                                                \
  FRNNT_KERNEL(recurrence_step_kernel<TYPE><<<grid, kStepThreads, 0, st>>>(                  \
      (const TYPE *)x, x_row, (const TYPE *)gate, gate_row, (const RecState<TYPE> *)state,  \
      parents, (TYPE *)h, (RecState<TYPE> *)next, rows, beams, K, D))
  FRNNT_REC_TYPES(FRNNT_REC_STEP)
#undef FRNNT_REC_STEP
  FRNNT_CUDA(cudaGetLastError());
  return FRNNT_OK;
}
