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
// depends on the type, the length and the alignment of the tensors, not on the batch or the cluster.
//
// backward: lam_t = dh_t + f_{t+1} lam_{t+1} is the same recurrence from the other end, with the
// same products of gates.  h_{t-1} is recomputed from the state that the forward keeps per tile:
// 5 values an element move instead of 6, and h keeps its 32 bits.
//
// Both are bound by memory where there are channels enough: 3 values an element forward, 5
// backward, in their own type (64 x 500 x 2048 bf16, ragged: 65 and 113 us, 0.9 of the copy rate
// if nothing were padding).  Inputs go to shared memory with cp.async a tile ahead, each thread
// fetching just what it reads itself, so that no barrier belongs to the copies.  Tiles of 32
// channels and 128 threads, four CTAs a multiprocessor forward and three backward, took the place
// of 64 channels and 256 threads (16 x 2000 x 1024 bf16: 47 + 85 -> 38 + 71 us); the backward
// then issues an instruction in two cycles of three, its products and sums two floats at a time.
#include <cooperative_groups.h>

#include <atomic>
#include <climits>

#include "common.cuh"
#include "recurrence.cuh"

namespace frnnt {

constexpr int kRecMostCluster = 16;   // more than the portable eight: long sequences of few channels

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
// contiguous; steps from n on are filled with `pad`.  Values of two bytes that no wider vector
// reaches are loaded and stored instead (cp.async moves 4, 8 or 16 bytes).
template <typename S> struct RecTile {
  using T = typename S::T;
  using Pack = RecPack<T, S::VEC>;
  __device__ static __forceinline__ void fetch(Pack *tile, const T *from, long long step, int first, int n,
                                               const Pack &pad) {
    const T *p = from + first * step;
    if constexpr (sizeof(Pack) == 2) {   // all loads under way before the first is stored
      Pack v[S::kSteps];
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s, p += step) v[s] = first + s < n ? *reinterpret_cast<const Pack *>(p) : pad;
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) tile[s * kRecThreads] = v[s];
    } else if (first + S::kSteps <= n) {   // nearly always: no comparisons per step
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s, p += step) copy_async<(int)sizeof(Pack)>(&tile[s * kRecThreads], p);
    } else {
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s, p += step) {
        if (first + s < n) copy_async<(int)sizeof(Pack)>(&tile[s * kRecThreads], p);
        else tile[s * kRecThreads] = pad;
      }
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
    // eight channels to a segment of lanes, their kJoin runs eight lanes apart
    join_q = lane / 8 % S::kJoin;
    join_c = (warp * (32 / S::kSegment) + lane / S::kSegment) * 8 + lane % 8;
    joiner = join_c < S::kWidth;
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

// ---- the tiles of a cluster --------------------------------------------------------------
// Every CTA sends the composition of its tile to every CTA, straight into its shared memory and
// counted there by an mbarrier (st.async: a cluster barrier would wait for the stores of h or of
// the gradients too, a microsecond a turn).  Two buffers in turn are enough: who sends for turn
// n + 2 has received everybody's composition of turn n + 1, which they sent after they had read
// turn n's.  Waits are bounded; where one runs out the state becomes NaN and the CTA, from the next
// turn on, sends nothing more, so that the waits of the others for it run out in their turn: NaN
// reaches all that depends on what did not arrive, and no message can be taken for one of another turn.
constexpr int kRecTries = 1 << 20;

struct RecMail {
  void *slots;       // [2][ranks][kWidth][2]
  uint64_t *bars;    // [2]
  int *stops;        // [kRecMostCluster] turns that each CTA sent; INT_MAX: all
  int *gave_up;      // 0, or the turns that this CTA had sent when a wait of its ran out
  int rank, ranks, tries;
  bool failed;       // whether one did before this turn
};
constexpr int kRecMailBytes = 2 * 8 + (kRecMostCluster + 4) * 4;   // behind the slots; whole 16 bytes
__device__ __forceinline__ RecMail mail_at(void *slots, size_t slot_bytes, int rank, int ranks, int tries) {
  uint64_t *const bars = reinterpret_cast<uint64_t *>((char *)slots + slot_bytes);
  int *const stops = reinterpret_cast<int *>(bars + 2);
  return {slots, bars, stops, stops + kRecMostCluster, rank, ranks, tries, false};
}
__device__ __forceinline__ uint32_t peer_address(const void *p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void send_pair(uint32_t to, float a, float b, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(to),
               "r"(__float_as_uint(a)), "r"(__float_as_uint(b)), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void send_pair(uint32_t to, double a, double b, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(to),
               "l"(__double_as_longlong(a)), "l"(__double_as_longlong(b)), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool mail_wait(uint32_t bar, int parity, int tries) {
  bool arrived = false;
  for (int i = 0; !arrived && i < tries; ++i) {
    uint32_t done;
    asm volatile("{\n.reg .pred q;\nmbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\n"
                 "selp.u32 %0, 1, 0, q;\n}"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    arrived = done != 0;
  }
  return arrived;
}
__device__ __forceinline__ void mail_expect(uint32_t bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mail_begin(const RecMail &mail) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((uint32_t)__cvta_generic_to_shared(mail.bars + i)) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *mail.gave_up = 0;
  }
  if (threadIdx.x < kRecMostCluster) mail.stops[threadIdx.x] = INT_MAX;
  cooperative_groups::this_cluster().sync();   // all have started, and have their mbarriers
}
// Before a turn's first barrier: waits run out between its two, so that all threads see the same here.
__device__ __forceinline__ void mail_turn(RecMail &mail) { mail.failed = *(volatile int *)mail.gave_up != 0; }
// Nobody leaves before all that was sent to it has arrived.  A CTA that received every turn has seen
// that.  One that gave up in turn n has everything up to turn n - 1, and nobody sends it turn n + 2
// (for which he would need its turn n + 1): what turns n and n + 1 lack of a full one, since others had
// stopped before, is taken from what their mbarriers expect, and then both complete.
template <typename S> __device__ __forceinline__ void mail_end(const RecMail &mail, int turns) {
  __syncthreads();
  const int sent = *(volatile int *)mail.gave_up;
  if (sent != 0 && threadIdx.x < mail.ranks)
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_address(mail.stops + mail.rank, threadIdx.x)), "r"(sent) : "memory");
  cooperative_groups::this_cluster().sync();
  if (sent == 0 || threadIdx.x != 0) return;
  constexpr int kEach = 2 * S::kWidth * (int)sizeof(typename S::real);   // from one CTA
  const int n = sent - 1;
  int now = 0, after = 0;   // CTAs that sent turns n and n + 1
  for (int r = 0; r < mail.ranks; ++r) {
    now += mail.stops[r] > n;
    after += n + 1 < turns && mail.stops[r] > n + 1;
  }
  const uint32_t bar = (uint32_t)__cvta_generic_to_shared(mail.bars + (n & 1)),
                 next = (uint32_t)__cvta_generic_to_shared(mail.bars + ((n + 1) & 1));
  if (now < mail.ranks)
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"((mail.ranks - now) * kEach) : "memory");
  mail_expect(next, after * kEach);
  mail_wait(bar, (n >> 1) & 1, kRecTries);
  mail_wait(next, ((n + 1) >> 1) & 1, kRecTries);
}
// The composition (A, B) of this CTA's tile to all, in the n-th turn.  For joiners.
template <typename S>
__device__ __forceinline__ void mail_send(typename S::real A, typename S::real B, int n, const RecMail &mail,
                                          const RecPlace<S> &at) {
  using real = typename S::real;
  if (mail.failed) return;
  const int buffer = n & 1;
  const real *slots = (const real *)mail.slots + buffer * mail.ranks * 2 * S::kWidth;
  if (threadIdx.x == 0)
    mail_expect((uint32_t)__cvta_generic_to_shared(mail.bars + buffer), mail.ranks * 2 * S::kWidth * (int)sizeof(real));
  for (int r = at.join_q; r < mail.ranks; r += S::kJoin)
    send_pair(peer_address(slots + (mail.rank * S::kWidth + at.join_c) * 2, r), A, B,
              peer_address(mail.bars + buffer, r));
}
// The state that the tile starts from.  `carry`: the state before the n-th turn, and after it on
// return.  FORWARD: in the order of the ranks, else against it.  For joiners.
template <typename S, bool FORWARD>
__device__ __forceinline__ typename S::real mail_join(typename S::real &carry, int n, const RecMail &mail,
                                                      const RecPlace<S> &at) {
  using real = typename S::real;
  const int buffer = n & 1;
  const real *slots = (const real *)mail.slots + buffer * mail.ranks * 2 * S::kWidth;
  const uint32_t bar = (uint32_t)__cvta_generic_to_shared(mail.bars + buffer);
  if (mail.failed) return carry = real(NAN);
  if (!mail_wait(bar, (n >> 1) & 1, mail.tries)) {
    *(volatile int *)mail.gave_up = n + 1;
    return carry = real(NAN);
  }
  real before = carry;
#pragma unroll 4
  for (int i = 0; i < mail.ranks; ++i) {
    const int r = FORWARD ? i : mail.ranks - 1 - i;
    if (r == mail.rank) before = carry;
    const real *own = slots + (r * S::kWidth + at.join_c) * 2;
    carry = own[0] * carry + own[1];
  }
  return before;
}

template <typename S, bool CLUSTER>
__global__ void __launch_bounds__(kRecThreads, 4)
recurrence_forward_kernel(RecTensor x, RecTensor gate, const typename S::real *__restrict__ initial,
                          const int64_t *__restrict__ lengths, typename S::T *__restrict__ h,
                          typename S::real *__restrict__ last, typename S::real *__restrict__ saved, int steps,
                          int D, int tries) {
  using T = typename S::T;
  using real = typename S::real;
  using Pack = RecPack<T, S::VEC>;
  constexpr int VEC = S::VEC, STEPS = S::kSteps;
  extern __shared__ __align__(16) unsigned char smem[];
  Pack *const tiles = reinterpret_cast<Pack *>(smem) + threadIdx.x;        // [2][x, gate][STEPS][thread]
  real *const exchange = reinterpret_cast<real *>(smem + 4 * S::kStage);   // [2][A, B][kExchange]
  const int rank = CLUSTER ? blockIdx.x : 0, ranks = CLUSTER ? gridDim.x : 1;
  real *const slots = exchange + 4 * S::kExchange;
  RecMail mail = mail_at(slots, 4 * ranks * S::kWidth * sizeof(real), rank, ranks, tries);
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
  const int piece_first = at.piece * STEPS, here = at.inside ? n : 0;   // steps that this thread has

  const auto fetch = [&](int turn) {
    const int first = (turn * ranks + rank) * kRecChunk + piece_first;
    Pack *tile = tiles + (turn & 1) * 2 * STEPS * kRecThreads;
    if (turn < turns) {   // behind the sequence, a gate that keeps the state as it is
      RecTile<S>::fetch(tile, X, x.step, first, here, rec_fill<T, VEC>(0.0f));
      RecTile<S>::fetch(tile + STEPS * kRecThreads, G, gate.step, first, here, rec_fill<T, VEC>(INFINITY));
    }
    copy_commit();
  };
  fetch(0);
  if constexpr (CLUSTER) mail_begin(mail);
  for (int turn = 0; turn < turns; ++turn) {
    fetch(turn + 1);
    copy_wait<1>();
    const int chunk = turn * ranks + rank, first = chunk * kRecChunk + piece_first;
    real *const EA = exchange + (turn & 1) * 2 * S::kExchange, *const EB = EA + S::kExchange;
    real f[STEPS][VEC], u[STEPS][VEC], A[VEC], B[VEC];
    const Pack *tile = tiles + (turn & 1) * 2 * STEPS * kRecThreads;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      real xv[VEC], gv[VEC], take[VEC];
      rec_unpack<T, VEC>(tile[s * kRecThreads], xv);
      rec_unpack<T, VEC>(tile[(STEPS + s) * kRecThreads], gv);
#pragma unroll
      for (int k = 0; k < VEC; ++k) gate_pair<T>(gv[k], f[s][k], take[k]);
      vmul(u[s], take, xv);
      if (s == 0) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) A[k] = f[0][k], B[k] = u[0][k];
      } else {
        vmul(A, A, f[s]);
        vfma(B, f[s], B, u[s]);
      }
    }
    put<real, VEC>(EA + S::at(at.piece, at.c), A);
    put<real, VEC>(EB + S::at(at.piece, at.c), B);
    if constexpr (CLUSTER) mail_turn(mail);
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
        const real pa = __shfl_up_sync(0xffffffffu, a, 8 * o, S::kSegment), pb = __shfl_up_sync(0xffffffffu, bb, 8 * o, S::kSegment);
        if (at.join_q >= o) {
          bb = a * pb + bb;
          a *= pa;
        }
      }
      const real pa = __shfl_up_sync(0xffffffffu, a, 8, S::kSegment), pb = __shfl_up_sync(0xffffffffu, bb, 8, S::kSegment);
      if (at.join_q > 0) ex_a = pa, ex_b = pb;
      a = __shfl_sync(0xffffffffu, a, S::kSegment - 8 + (threadIdx.x & 7), S::kSegment);
      bb = __shfl_sync(0xffffffffu, bb, S::kSegment - 8 + (threadIdx.x & 7), S::kSegment);
    }
    if constexpr (CLUSTER)
      if (at.joiner) mail_send(a, bb, turn, mail, at);
    if (at.joiner) {
      real start = carry;
      if constexpr (CLUSTER) start = mail_join<S, true>(carry, turn, mail, at);
      else carry = a * carry + bb;
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
    T *out = H + (size_t)first * D;
    if (first + STEPS <= here) {   // nearly always
#pragma unroll
      for (int s = 0; s < STEPS; ++s, out += D) {
        vfma(state, f[s], state, u[s]);
        *reinterpret_cast<Pack *>(out) = rec_pack<T, VEC>(state);
      }
    } else {
#pragma unroll
      for (int s = 0; s < STEPS; ++s, out += D) {
        vfma(state, f[s], state, u[s]);
        if (first + s < here) *reinterpret_cast<Pack *>(out) = rec_pack<T, VEC>(state);
      }
    }
  }
  if (at.inside) {   // behind the sequence
    const real zero[VEC] = {};
    for (long long t = (long long)n + rank * S::kPieces + at.piece; t < steps; t += ranks * S::kPieces)
      *reinterpret_cast<Pack *>(H + t * D) = rec_pack<T, VEC>(zero);
  }
  if (keeper && rank == 0 && at.join_q == 0) last[(size_t)b * D + join_channel] = carry;
  if constexpr (CLUSTER) mail_end<S>(mail, turns);
}

template <typename S, bool CLUSTER>
__global__ void __launch_bounds__(kRecThreads, 3)
recurrence_backward_kernel(RecTensor x, RecTensor gate, const int64_t *__restrict__ lengths,
                           const typename S::real *__restrict__ saved, RecTensor dh,
                           const typename S::real *__restrict__ dlast, typename S::T *__restrict__ dx,
                           typename S::T *__restrict__ dgate, typename S::real *__restrict__ dinitial, int steps,
                           int D, int tries) {
  using T = typename S::T;
  using real = typename S::real;
  using Pack = RecPack<T, S::VEC>;
  constexpr int VEC = S::VEC, STEPS = S::kSteps;
  extern __shared__ __align__(16) unsigned char smem[];
  Pack *const tiles = reinterpret_cast<Pack *>(smem) + threadIdx.x;        // [2][x, gate, dh][STEPS][thread]
  real *const exchange = reinterpret_cast<real *>(smem + 6 * S::kStage);   // [2][A, B, M][kExchange]
  const int rank = CLUSTER ? blockIdx.x : 0, ranks = CLUSTER ? gridDim.x : 1;
  real *const slots = exchange + 6 * S::kExchange;
  RecMail mail = mail_at(slots, 4 * ranks * S::kWidth * sizeof(real), rank, ranks, tries);
  const int b = blockIdx.z;
  const RecPlace<S> at(blockIdx.y, D);
  const int n = steps_of(lengths, b, steps), chunks = (steps + kRecChunk - 1) / kRecChunk;
  const T *const X = (const T *)x.data + b * x.batch + at.channel;
  const T *const G = (const T *)gate.data + b * gate.batch + at.channel;
  const T *const DH = (const T *)dh.data + b * dh.batch + at.channel;   // not read where there is none
  T *const DX = dx + (size_t)b * steps * D + at.channel, *const DG = dgate + (size_t)b * steps * D + at.channel;
  const int join_channel = blockIdx.y * S::kWidth + at.join_c;
  const bool keeper = at.joiner && join_channel < D;
  real carry = keeper && dlast != nullptr ? dlast[(size_t)b * D + join_channel] : real(0);
  const int turns = (n + kRecChunk * ranks - 1) / (kRecChunk * ranks);
  const int piece_first = at.piece * STEPS, here = at.inside ? n : 0;   // steps that this thread has

  const auto fetch = [&](int turn) {
    const int first = (turn * ranks + rank) * kRecChunk + piece_first;
    Pack *tile = tiles + (turn & 1) * 3 * STEPS * kRecThreads;
    if (turn >= 0) {   // behind the sequence, a gate that keeps the state as it is
      RecTile<S>::fetch(tile, X, x.step, first, here, rec_fill<T, VEC>(0.0f));
      RecTile<S>::fetch(tile + STEPS * kRecThreads, G, gate.step, first, here, rec_fill<T, VEC>(INFINITY));
      RecTile<S>::fetch(tile + 2 * STEPS * kRecThreads, DH, dh.step, first, dh.data == nullptr ? 0 : here,
                        rec_fill<T, VEC>(0.0f));
    }
    copy_commit();
  };
  fetch(turns - 1);
  if constexpr (CLUSTER) mail_begin(mail);
  for (int turn = turns - 1; turn >= 0; --turn) {
    if constexpr (!CLUSTER) fetch(turn - 1);
    const int chunk = turn * ranks + rank, first = chunk * kRecChunk + piece_first;
    real start = real(0);   // the state before the tile
    if (keeper && saved != nullptr && chunk * kRecChunk < n) start = saved[((size_t)b * chunks + chunk) * D + join_channel];
    copy_wait<CLUSTER ? 0 : 1>();
    real *const EA = exchange + (turn & 1) * 3 * S::kExchange, *const EB = EA + S::kExchange,
               *const EM = EB + S::kExchange;
    real f[STEPS][VEC], take[STEPS][VEC], A[VEC], B[VEC], M[VEC];
    const Pack *tile = tiles + (turn & 1) * 3 * STEPS * kRecThreads;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      real xv[VEC], gv[VEC], u[VEC];
      rec_unpack<T, VEC>(tile[s * kRecThreads], xv);
      rec_unpack<T, VEC>(tile[(STEPS + s) * kRecThreads], gv);
#pragma unroll
      for (int k = 0; k < VEC; ++k) gate_pair<T>(gv[k], f[s][k], take[s][k]);
      vmul(u, take[s], xv);
      if (s == 0) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) A[k] = f[0][k], B[k] = u[k];
      } else {
        vmul(A, A, f[s]);
        vfma(B, f[s], B, u);
      }
    }
    vset(M, real(0));
#pragma unroll
    for (int s = STEPS - 1; s >= 0; --s) {
      real dv[VEC];
      rec_unpack<T, VEC>(tile[(2 * STEPS + s) * kRecThreads], dv);
      vadd(M, M, dv);
      vmul(M, M, f[s]);
    }
    put<real, VEC>(EA + S::at(at.piece, at.c), A);
    put<real, VEC>(EB + S::at(at.piece, at.c), B);
    put<real, VEC>(EM + S::at(at.piece, at.c), M);
    if constexpr (CLUSTER) mail_turn(mail);
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
        const real pa = __shfl_up_sync(0xffffffffu, fa, 8 * o, S::kSegment), pb = __shfl_up_sync(0xffffffffu, bb, 8 * o, S::kSegment);
        const real na = __shfl_down_sync(0xffffffffu, sa, 8 * o, S::kSegment), nm = __shfl_down_sync(0xffffffffu, m, 8 * o, S::kSegment);
        if (at.join_q >= o) {
          bb = fa * pb + bb;
          fa *= pa;
        }
        if (at.join_q + o < S::kJoin) {
          m = sa * nm + m;
          sa *= na;
        }
      }
      const real pa = __shfl_up_sync(0xffffffffu, fa, 8, S::kSegment), pb = __shfl_up_sync(0xffffffffu, bb, 8, S::kSegment);
      const real na = __shfl_down_sync(0xffffffffu, sa, 8, S::kSegment), nm = __shfl_down_sync(0xffffffffu, m, 8, S::kSegment);
      if (at.join_q > 0) ex_a = pa, ex_b = pb;
      if (at.join_q + 1 < S::kJoin) af_a = na, af_m = nm;
      a = __shfl_sync(0xffffffffu, sa, threadIdx.x & 7, S::kSegment);   // of the whole tile
      m = __shfl_sync(0xffffffffu, m, threadIdx.x & 7, S::kSegment);
    }
    if constexpr (CLUSTER) {
      if (at.joiner) mail_send(a, m, turns - 1 - turn, mail, at);
      fetch(turn - 1);   // while the compositions are under way
    }
    if (at.joiner) {
      real flow = carry;
      if constexpr (CLUSTER) flow = mail_join<S, false>(carry, turns - 1 - turn, mail, at);
      else carry = a * carry + m;
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
      real xv[VEC], u[VEC];
      rec_unpack<T, VEC>(tile[s * kRecThreads], xv);
      vsub(before[s], state, xv);   // h_{t-1} - x_t
      vmul(u, take[s], xv);
      vfma(state, f[s], state, u);
    }
    const size_t behind = (size_t)(first + STEPS) * D;
    T *out_x = DX + behind, *out_g = DG + behind;
    const auto step_back = [&](int s, bool live) {
      real dv[VEC], lam[VEC], ox[VEC], og[VEC];
      rec_unpack<T, VEC>(tile[(2 * STEPS + s) * kRecThreads], dv);
      vadd(lam, back, dv);
      vmul(back, f[s], lam);
      vmul(ox, take[s], lam);
      vmul(og, before[s], take[s]);
      vmul(og, og, back);           // lam (h - x) f take
      out_x -= D;
      out_g -= D;
      if (live) {
        *reinterpret_cast<Pack *>(out_x) = rec_pack<T, VEC>(ox);
        *reinterpret_cast<Pack *>(out_g) = rec_pack<T, VEC>(og);
      }
    };
    if (first + STEPS <= here) {   // nearly always
#pragma unroll
      for (int s = STEPS - 1; s >= 0; --s) step_back(s, true);
    } else {
#pragma unroll
      for (int s = STEPS - 1; s >= 0; --s) step_back(s, first + s < here);
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
  if constexpr (CLUSTER) mail_end<S>(mail, turns);
}

// One token: every row reads the state of its parent (its own without parents; zero where the
// parent is not one of the K rows) and writes the new state and its rounding to x's type.  A
// thread has VEC channels: 16 bytes of x and of gate where all rows allow that.
constexpr int kStepThreads = 256;

template <typename T, int VEC>
__global__ void __launch_bounds__(kStepThreads)
recurrence_step_kernel(const T *__restrict__ x, long long x_row, const T *__restrict__ gate, long long gate_row,
                       const RecState<T> *__restrict__ state, const int64_t *__restrict__ parents,
                       T *__restrict__ h, RecState<T> *__restrict__ next, long long rows, int beams, int K, int D) {
  using real = RecState<T>;
  using Pack = RecPack<T, VEC>;
  const int per = D / VEC;
  const long long n = (long long)blockIdx.x * kStepThreads + threadIdx.x, row = div_rows(n, per);
  if (row >= rows) return;
  const int d = (int)(n - row * per) * VEC;
  const Pack xp = *reinterpret_cast<const Pack *>(x + row * x_row + d);
  const Pack gp = *reinterpret_cast<const Pack *>(gate + row * gate_row + d);
  long long from = row;
  if (parents != nullptr) {
    const int64_t p = parents[row];
    from = p < 0 || p >= K ? -1 : div_rows(row, beams) * K + p;
  }
  real xv[VEC], gv[VEC], old[VEC], take[VEC], keep[VEC];
  if (from >= 0) get<real, VEC>(state + from * D + d, old);
  else vset(old, real(0));
  rec_unpack<T, VEC>(xp, xv);
  rec_unpack<T, VEC>(gp, gv);
#pragma unroll
  for (int k = 0; k < VEC; ++k) gate_pair<T>(gv[k], keep[k], take[k]);
  vmul(xv, take, xv);
  vfma(old, keep, old, xv);
  put<real, VEC>(next + row * D + d, old);
  if (h != nullptr) *reinterpret_cast<Pack *>(h + row * D + d) = rec_pack<T, VEC>(old);
}

template <typename T, int VEC>
static int step_as(const void *x, long long x_row, const void *gate, long long gate_row, const void *state,
                   const int64_t *parents, void *h, void *next, long long rows, int beams, int K, int D,
                   cudaStream_t st) {
  const long long blocks = (rows * (D / VEC) + kStepThreads - 1) / kStepThreads;
  FRNNT_REQUIRE(blocks <= INT_MAX, FRNNT_EUNSUPPORTED, "too many rows for the grid");
  FRNNT_KERNEL(recurrence_step_kernel<T, VEC><<<(unsigned)blocks, kStepThreads, 0, st>>>(
      (const T *)x, x_row, (const T *)gate, gate_row, (const RecState<T> *)state, parents, (T *)h,
      (RecState<T> *)next, rows, beams, K, D));
  FRNNT_CUDA(cudaGetLastError());
  return FRNNT_OK;
}

// ---- host ----------------------------------------------------------------------------

// CTAs of a cluster: tiles of one sequence at once.  The most for which all clusters are on the GPU
// together, as the runtime counts them (a cluster stays within a GPC, so the multiprocessors' room
// alone does not say: of 16 CTAs at two a multiprocessor only 14 clusters fit, of 12 CTAs 21), and no
// more than the sequence has tiles.  A second round of clusters costs more than idle multiprocessors:
// backward of 1 x 30011 x 512 fp16 58 us with clusters of 12, 76 with 16; 2 x 3000 x 256 fp32 12 us
// with 8, 20 with 16.  Within one round, more are faster: forward of 8 x 4096 x 512 bf16 34, 33, 28 and
// 27 us with 1 to 4.  Above the portable eight that holds up to two CTAs a multiprocessor: 1 x 30011
// x 512 41 us with 16 (256 CTAs), 54 with 8, but 1 x 8000 x 1024 21 us with 12 (384 CTAs), 19 with 8.
constexpr int kRecRanks[] = {16, 12, 8, 6, 4, 3, 2};
constexpr int kRecRankKinds = sizeof(kRecRanks) / sizeof(int);

template <typename S> static size_t rec_smem(int arrays, int ranks) {
  return 2 * (size_t)arrays * (S::kStage + S::kExchange * sizeof(typename S::real)) +
         (ranks > 1 ? 4 * ranks * S::kWidth * sizeof(typename S::real) + kRecMailBytes : 0);
}

template <typename S, typename... Params, typename... Args>
static int rec_launch(void (*alone)(Params...), void (*cluster)(Params...), int arrays, int B, int T, int D,
                      cudaStream_t st, Args... args) {
  const int tiles = (D + S::kWidth - 1) / S::kWidth, chunks = (T + kRecChunk - 1) / kRecChunk;
  FRNNT_REQUIRE(B <= 65535 && tiles <= 65535, FRNNT_EUNSUPPORTED, "B or D too large for the grid");
  FRNNT_REQUIRE(T <= INT_MAX - 4 * kRecMostCluster * kRecChunk, FRNNT_EUNSUPPORTED, "T too large");
  cudaLaunchConfig_t config = {};
  config.blockDim = dim3(kRecThreads);
  config.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  // attributes and room belong to the kernel on a device: asked for once
  static std::atomic<uint64_t> allowed[2];
  static std::atomic<int> room[64][kRecRankKinds];   // clusters at once, and one
  int dev = 0;
  FRNNT_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  const auto allow = [&](bool clusters) {
    if (dev <= 63 && allowed[clusters].load(std::memory_order_relaxed) & bit) return FRNNT_OK;
    const void *kernel = clusters ? (const void *)cluster : (const void *)alone;
    const size_t most = rec_smem<S>(arrays, clusters ? kRecMostCluster : 1);
    FRNNT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    if (clusters) FRNNT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    allowed[clusters].fetch_or(bit, std::memory_order_relaxed);
    return FRNNT_OK;
  };
  const auto shape = [&](int ranks) {
    config.gridDim = dim3((unsigned)ranks, (unsigned)tiles, (unsigned)B);
    config.dynamicSmemBytes = rec_smem<S>(arrays, ranks);
    attr[0].val.clusterDim.x = (unsigned)ranks;
    config.numAttrs = ranks > 1 ? 1 : 0;
  };
  const long long clusters = (long long)B * tiles;
  int ranks = 1;
  for (int i = 0; i < kRecRankKinds && ranks == 1; ++i) {
    const int r = kRecRanks[i];
    if (r > chunks || clusters * r > (r > 8 ? 2 : 4) * sm_count()) continue;   // four at most fit a multiprocessor
    int fit = dev <= 63 ? room[dev][i].load(std::memory_order_relaxed) - 1 : -1;
    if (fit < 0) {
      const int rc = allow(true);
      if (rc != FRNNT_OK) return rc;
      shape(r);
      if (cudaOccupancyMaxActiveClusters(&fit, cluster, &config) != cudaSuccess) {   // no room for one
        fit = 0;
        (void)cudaGetLastError();
      }
      if (dev <= 63) room[dev][i].store(fit + 1, std::memory_order_relaxed);
    }
    if (clusters <= fit) ranks = r;
  }
  const int rc = allow(ranks > 1);
  if (rc != FRNNT_OK) return rc;
  shape(ranks);
  FRNNT_CUDA(FRNNT_KERNEL(cudaLaunchKernelEx(&config, ranks > 1 ? cluster : alone, args...)));
  return FRNNT_OK;
}

// whether rows of D values from `data` on, with these strides, can be read `bytes` at a time
static bool rec_aligned(const RecTensor &t, int size, int D, int bytes) {
  return (uintptr_t)t.data % bytes == 0 && t.batch * size % bytes == 0 && t.step * size % bytes == 0 &&
         (long long)D * size % bytes == 0;
}

template <typename S>
static int forward_as(const RecTensor &x, const RecTensor &gate, const void *initial, const int64_t *lengths, void *h,
                      void *last, void *saved, int B, int T, int D, int tries, cudaStream_t st) {
  using real = typename S::real;
  return rec_launch<S>(recurrence_forward_kernel<S, false>, recurrence_forward_kernel<S, true>, 2, B, T, D, st, x, gate,
                       (const real *)initial, lengths, (typename S::T *)h, (real *)last, (real *)saved, T, D,
                       tries);
}
template <typename S>
static int backward_as(const RecTensor &x, const RecTensor &gate, const int64_t *lengths, const void *saved,
                       const RecTensor &dh, const void *dlast, void *dx, void *dgate, void *dinitial, int B, int T,
                       int D, int tries, cudaStream_t st) {
  using real = typename S::real;
  return rec_launch<S>(recurrence_backward_kernel<S, false>, recurrence_backward_kernel<S, true>, 3, B, T, D, st, x,
                       gate, lengths, (const real *)saved, dh, (const real *)dlast, (typename S::T *)dx,
                       (typename S::T *)dgate, (real *)dinitial, T, D, tries);
}

// Vectors of 16 bytes where every row allows them, else of 4 bytes (a float, or a pair of 16-bit
// values) where they do, else single values; 64 or 128 bytes of a row side by side, and 32 values
// a thread (16 doubles).
#define FRNNT_REC_SHAPES(CALL, wide, pairs)                                              \
  switch (dtype) {                                                                       \
    case FRNNT_F32:                                                                      \
      return wide ? CALL(RecShape<float, 4, 8>) : CALL(RecShape<float, 1, 16>);          \
    case FRNNT_F64:                                                                      \
      return wide ? CALL(RecShape<double, 2, 8>) : CALL(RecShape<double, 1, 16>);        \
    case FRNNT_F16:                                                                      \
      return wide ? CALL(RecShape<__half, 8, 4>)                                         \
                  : pairs ? CALL(RecShape<__half, 2, 16>) : CALL(RecShape<__half, 1, 32>); \
    default:                                                                             \
      return wide ? CALL(RecShape<__nv_bfloat16, 8, 4>)                                  \
                  : pairs ? CALL(RecShape<__nv_bfloat16, 2, 16>) : CALL(RecShape<__nv_bfloat16, 1, 32>); \
  }

}  // namespace frnnt

using namespace frnnt;

static bool rec_dtype(int dtype) {
  return dtype == FRNNT_F32 || dtype == FRNNT_F64 || dtype == FRNNT_F16 || dtype == FRNNT_BF16;
}
static int rec_size(int dtype) { return dtype == FRNNT_F64 ? 8 : dtype == FRNNT_F32 ? 4 : 2; }
static bool rec_sizes(int B, int T, int D) { return B >= 0 && T >= 0 && D >= 0; }

extern "C" size_t frnnt_recurrence_saved_bytes(int dtype, int B, int T, int D) {
  if (!rec_dtype(dtype) || B <= 0 || T <= kRecChunk || D <= 0) return 0;   // one tile starts from `initial`
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
  forward_as<__VA_ARGS__>(X, G, initial, lengths, h, last, saved, B, T, D, kRecTries, (cudaStream_t)stream)
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
  FRNNT_REQUIRE(T == 0 || (x && gate && (saved || T <= kRecChunk) && dx && dgate), FRNNT_EINVAL, "NULL argument");
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
                           kRecTries, (cudaStream_t)stream)
  FRNNT_REC_SHAPES(FRNNT_REC_BACKWARD, wide, pairs)
#undef FRNNT_REC_BACKWARD
}

extern "C" int frnnt_recurrence_limited(const float *x, const float *gate, float *h, float *last, void *saved,
                                        const float *dh, float *dx, float *dgate, int B, int T, int D, int tries,
                                        void *stream) {
  FRNNT_REQUIRE(B >= 1 && T >= 1 && D >= 1, FRNNT_EINVAL, "bad sizes");
  FRNNT_REQUIRE(x && gate && h && last && dh && dx && dgate && (saved || T <= kRecChunk), FRNNT_EINVAL, "NULL argument");
  if (tries < 0) tries = kRecTries;
  using S = RecShape<float, 1, 16>;
  const RecTensor X{x, (long long)T * D, D}, G{gate, (long long)T * D, D}, DH{dh, (long long)T * D, D};
  const int rc = forward_as<S>(X, G, nullptr, nullptr, h, last, saved, B, T, D, tries, (cudaStream_t)stream);
  if (rc != FRNNT_OK) return rc;
  return backward_as<S>(X, G, nullptr, saved, DH, nullptr, dx, dgate, nullptr, B, T, D, tries, (cudaStream_t)stream);
}

extern "C" int frnnt_recurrence_step(int dtype, const void *x, long long x_row, const void *gate,
                                     long long gate_row, const void *state, const int64_t *parents, void *h,
                                     void *next, long long rows, int beams, int K, int D, void *stream) {
  FRNNT_REQUIRE(rec_dtype(dtype), FRNNT_EINVAL, "dtype must be FRNNT_F32, _F64, _F16 or _BF16");
  FRNNT_REQUIRE(rows >= 0 && beams >= 1 && K >= 1 && D >= 0, FRNNT_EINVAL, "bad sizes");
  if (rows == 0 || D == 0) return FRNNT_OK;
  FRNNT_REQUIRE(x && gate && state && next, FRNNT_EINVAL, "NULL argument");
  FRNNT_REQUIRE(state != next, FRNNT_EINVAL, "the new states may not overwrite the old ones");
  const int size = rec_size(dtype);
  const auto aligned = [&](const void *p, long long row) { return (uintptr_t)p % 16 == 0 && row * size % 16 == 0; };
  const bool wide = aligned(x, x_row) && aligned(gate, gate_row) && aligned(h, D) && (uintptr_t)state % 16 == 0 &&
                    (uintptr_t)next % 16 == 0;   // rows of states are as wide or wider
#define FRNNT_REC_STEP(TYPE, VEC) \
  step_as<TYPE, VEC>(x, x_row, gate, gate_row, state, parents, h, next, rows, beams, K, D, (cudaStream_t)stream)
  switch (dtype) {
    case FRNNT_F32: return wide ? FRNNT_REC_STEP(float, 4) : FRNNT_REC_STEP(float, 1);
    case FRNNT_F64: return wide ? FRNNT_REC_STEP(double, 2) : FRNNT_REC_STEP(double, 1);
    case FRNNT_F16: return wide ? FRNNT_REC_STEP(__half, 8) : FRNNT_REC_STEP(__half, 1);
    default: return wide ? FRNNT_REC_STEP(__nv_bfloat16, 8) : FRNNT_REC_STEP(__nv_bfloat16, 1);
  }
#undef FRNNT_REC_STEP
}
