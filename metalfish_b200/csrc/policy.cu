// policy.cu -- operators on policy logits and legal-move lists, on device
// buffers: log-probabilities with their backward pass, the clipped policy
// loss with a KL term, and the preference loss over lines of moves.
//
// All of them read a row of logits for each position at the columns that the
// position's legal-move list names (as priors_kernel does). With
// s_j = logit_j / T over the n = min(count, 256) listed moves,
//     logp_j = s_j - log(sum_i exp s_i),  p_j = exp(logp_j),
// and every gradient with respect to the logits has the form
//     dL/dlogit_c = (1/T) * (something of p, logp at c), zero off the list,
// so a gradient row is a row of zeros with ~30 values in it.
//
// What bounds them. The arithmetic is ~40 operations a move: nothing. The
// log-probabilities read one 32-byte sector of the row for almost every move
// (19 sectors for the 31 moves of an average position, 64 bytes of DRAM each)
// in three dependent steps (offsets, indices, logits), so they are bound by
// load latency and by the instructions of a row, not by its bytes. The gradient
// operators write the whole row (1858 x 4 bytes), 8 times what they need to
// read: they are bound by DRAM writes.
//
// One warp per position: a lane holds two moves in registers, the sums are
// shuffles in a fixed order (results do not depend on timing). CTAs stay on
// their SM and their warps take positions in turn, the lists of the next ones
// loaded ahead. A gradient row is put together in shared memory and written by
// one bulk copy, while the warp goes on. 65536 positions, 1858 fp32 classes, on
// B200: clipped loss with KL 128 us (617 MB of DRAM traffic; the same reads and
// copies without any arithmetic 127-129 us, the copies alone 93), the backward pass
// alone 110 us, log-probabilities 28 us.
#include "policy.cuh"

#include <atomic>
#include <cmath>
#include <cstdio>
#include <type_traits>

#include "../../include/mfb200.h"
#include "gemm_host.h"  // num_sms
#include "pdl.cuh"
#include "sm100_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mfb200 {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kMaxMoves = 256;  // moves of a position that count, as in priors_kernel
constexpr int kMaxWarps = 8;    // of a CTA
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eRest = static_cast<float>(1.4426950408889634 - static_cast<double>(kLog2e));

// Inputs are read with ordinary or volatile loads, never as read-only (__ldg,
// __restrict__ const): a kernel here may start before the one that writes its
// inputs has ended (pdl.cuh), and a read-only load may be moved above pdl_wait.

// The bits of a logit. L2 takes 64 bytes from DRAM for it instead of the 128
// that a plain load takes: 65536 gathers of 16 pairs of logits a row read 88 MB
// instead of 155, in 16-17 instead of 26.6 us.
__device__ __forceinline__ unsigned load_bits(const void *row, int type, int c) {
  if (type == MFB200_TYPE_F32) {
    unsigned v;
    asm volatile("ld.global.L2::64B.u32 %0, [%1];" : "=r"(v) : "l"(static_cast<const float *>(row) + c));
    return v;
  }
  unsigned short u;
  asm volatile("ld.global.L2::64B.u16 %0, [%1];"
               : "=h"(u)
               : "l"(static_cast<const unsigned short *>(row) + c));
  return u;
}
__device__ __forceinline__ float value_of(int type, unsigned bits) {
  return type == MFB200_TYPE_F32    ? __uint_as_float(bits)
         : type == MFB200_TYPE_BF16 ? __uint_as_float(bits << 16)
                                    : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

// The types of a call's matrices are template arguments where they are the same,
// and looked at for every value (kAnyType) where they differ: 16384 bf16
// positions' scores and gradient take 31 us instead of 33, 96 pairs of games 47
// instead of 50.
constexpr int kAnyType = -1;
template <int kType>
__device__ __forceinline__ int type_of(int type) {
  return kType == kAnyType ? type : kType;
}

__device__ __forceinline__ const void *row_of(const void *base, int type, long long stride, int b) {
  return static_cast<const char *>(base) + b * stride * (type == MFB200_TYPE_F32 ? 4 : 2);
}

// One rounding, to nearest even, of the fp32 value to the gradient's type.
__device__ __forceinline__ unsigned bits_of(int type, float v) {
  if (type == MFB200_TYPE_F32) return __float_as_uint(v);
  if (type == MFB200_TYPE_BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  return __half_as_ushort(__float2half_rn(v));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
// The largest value of the warp; NaN is passed over.
__device__ __forceinline__ float warp_max(float v) {
  float top;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(v));
  return top;
}
__device__ __forceinline__ float exp2_fast(float t) {
  float v;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(v) : "f"(t));
  return v;
}
// e^s for s <= 0 as 2^(s log2 e), log2 e in two parts: the rounding of the
// argument is that of one operation and does not lean to one side, which the sum of
// a long list would add up. (Log-probabilities of lines are made in 64 bits instead,
// line_position.)
__device__ __forceinline__ float exp_fast(float s) {
  return exp2_fast(fmaf(s, kLog2e, s * kLog2eRest));
}
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7FC00000); }

// ------------------------------------------------------------------ lists
// What a position's list is read with.
struct ListHead {
  int lo, hi, played;
};
__device__ __forceinline__ ListHead load_head(const PolicyRows &r, int b) {
  return {r.off[b], r.off[b + 1], r.played ? r.played[b] : -1};
}

struct Moves {
  int n;       // moves that count (<= 256)
  int count;   // moves listed
  int lo;      // first entry of the list
  int played;  // edge number, -1 for none
  bool bad;    // offsets or played move out of range
};
// No entry outside [0, num_moves) is ever read. (The offsets are in order
// before their differences are taken, so those are right as unsigned numbers.)
__device__ __forceinline__ Moves resolve(const PolicyRows &r, const ListHead &head, int base) {
  Moves m;
  const unsigned lo = static_cast<unsigned>(head.lo) - static_cast<unsigned>(base);
  const unsigned hi = static_cast<unsigned>(head.hi) - static_cast<unsigned>(base);
  m.bad = head.lo < base || head.hi < head.lo || hi > static_cast<unsigned>(r.num_moves);
  m.lo = static_cast<int>(lo);
  m.count = m.bad ? 0 : static_cast<int>(hi - lo);
  m.n = min(m.count, kMaxMoves);
  // a position with an empty list has no played move, whatever place (>= 0) it is given
  m.bad = m.bad || head.played < -1 || (m.count > 0 && head.played >= m.n);
  m.played = m.bad || m.count == 0 ? -1 : head.played;
  return m;
}

// Lane's entry of the group of 32 moves k of a list, -1 past its end or for a
// column outside the row (whose logit is then 0, without a gradient).
constexpr int kNoMove = -2, kNoColumn = -1;
__device__ __forceinline__ int load_index(const PolicyRows &r, const Moves &m, int k, int lane) {
  const int j = 32 * k + lane;
  return j < m.n ? r.index[m.lo + j] : -32768;
}

// Runs body(b, moves, first, second) for the positions of this CTA, a warp for
// each: `first` and `second` are the lane's entries of the first two groups of
// the list. A CTA has the positions at W = its warps in a row, every grid * W;
// its warps take them in turn from a counter in shared memory. The list of the
// next position and the offsets of the one after are loaded while a position
// is worked on, so of the three loads that follow from one another (offsets,
// list, logits) only the last is waited for.
//
// body may turn a position down by returning true: rare(b, moves) then has it,
// outside the loop that body is in. What is rare and needs many registers
// (lists of more than 64 moves, one in a hundred; 64-bit functions) goes
// there, so that it does not share them with the common path: a spill in that
// path costs more than its bytes, because the fence before a row's copy waits
// for it too (65536 positions of the clipped loss took 330 us with 280 bytes
// of spills). The other warps take the positions that this one is late for.
//
// Where some warps have more than two turns, a long list that comes last would
// keep its CTA waiting (65536 positions: 17 us), so the CTA looks for them first
// and its warps begin with them; body does not see them then.
constexpr unsigned kNone = 0xffffffffu;
constexpr int kLongLists = 64;
struct Turns {
  unsigned next;                    // turn that no warp has taken yet
  int found, taken;                 // long lists
  unsigned long_rows[kLongLists];
};
// Sets the counters; all threads of the CTA. The first three turns of a warp are fixed.
__device__ __forceinline__ void start_turns(Turns *turns) {
  if (threadIdx.x == 0) {
    turns->next = 3 * (blockDim.x >> 5);
    turns->found = turns->taken = 0;
  }
  __syncthreads();
}

template <class Body, class Rare>
__device__ __forceinline__ void for_positions(const PolicyRows &r, unsigned ctas, Turns *turns,
                                              Body body, Rare rare) {
  const int lane = threadIdx.x & 31;
  const unsigned batch = r.batch;
  const unsigned warps = blockDim.x >> 5, shift = __popc(warps - 1);  // a power of two
  const unsigned step = ctas * warps;
  auto row = [&](unsigned turn) {
    return blockIdx.x * warps + (turn & (warps - 1)) + (turn >> shift) * step;
  };
  const int base = r.off[0];
  bool long_first = false;
  if (row(2 * warps) < batch) {
    for (unsigned t = threadIdx.x; row(t) < batch; t += blockDim.x) {
      const long long count = static_cast<long long>(r.off[row(t) + 1]) - r.off[row(t)];
      if (count > 64) {
        const int i = atomicAdd(&turns->found, 1);
        if (i < kLongLists) turns->long_rows[i] = row(t);
      }
    }
    __syncthreads();
    long_first = turns->found <= kLongLists;
  }
  auto take_long = [&] {
    int i = 0;
    if (lane == 0) i = atomicAdd(&turns->taken, 1);
    i = __shfl_sync(kFull, i, 0);
    return long_first && i < turns->found ? turns->long_rows[i] : kNone;
  };
  unsigned todo = long_first ? take_long() : kNone;  // for rare
  // this warp's positions: now, next, after
  unsigned b0 = row(threadIdx.x >> 5), b1 = b0 + step, b2 = b1 + step;
  while (true) {
    if (todo != kNone) {
      rare(static_cast<int>(todo), resolve(r, load_head(r, todo), base));
      todo = long_first ? take_long() : kNone;
      continue;
    }
    if (b0 >= batch) break;
    Moves m = resolve(r, load_head(r, b0), base);
    ListHead next{};
    if (b1 < batch) next = load_head(r, b1);
    int c0 = load_index(r, m, 0, lane), c1 = m.n > 32 ? load_index(r, m, 1, lane) : -32768;
    unsigned b;
    bool turned_down;
    while (true) {
      b = b0;
      Moves mn{};
      int n0 = -32768, n1 = -32768;
      ListHead after{};
      if (b1 < batch) {
        mn = resolve(r, next, base);
        n0 = load_index(r, mn, 0, lane);
        if (mn.n > 32) n1 = load_index(r, mn, 1, lane);
        if (b2 < batch) after = load_head(r, b2);
      }
      unsigned turn = 0;
      if (lane == 0) turn = atomicAdd(&turns->next, 1u);
      turned_down = m.n > 64 ? !long_first : m.bad || body(static_cast<int>(b), m, c0, c1);
      b0 = b1;
      b1 = b2;
      b2 = row(__shfl_sync(kFull, turn, 0));
      if (turned_down || b0 >= batch) break;
      m = mn;
      c0 = n0;
      c1 = n1;
      next = after;
    }
    if (turned_down) todo = b;
  }
}

// ------------------------------------------------------------------ softmax of a list
// The moves of a position, 32 k + lane in group k. Lanes past the list's end
// hold a logit of -inf, which no sum sees.
template <int G>
struct Edges {
  int col[G];
  float z[G];  // logits
  float e[G];  // exp(s - s_top)
};

template <int G>
__device__ __forceinline__ void columns(const PolicyRows &r, const Moves &m, int c0, int c1,
                                        int lane, Edges<G> &v) {
#pragma unroll
  for (int k = 0; k < G; ++k) {
    int c = k == 0 ? c0 : k == 1 ? c1 : -32768;
    if (k > 1 && 32 * k < m.n) c = load_index(r, m, k, lane);
    v.col[k] = c >= 0 && c < r.classes ? c : 32 * k + lane < m.n ? kNoColumn : kNoMove;
  }
}

// Logits of the lane's moves, in two steps: with two groups every lane loads
// (column 0 where it has none, so that no load is in a branch of its own), and
// no load's value is looked at before the last is under way. Eight groups have
// no registers to spare for that. Groups past the list's end are not loaded.
template <int G>
__device__ __forceinline__ void load_logits(int n, const void *row, int type, const int (&col)[G],
                                            unsigned (&bits)[G]) {
#pragma unroll
  for (int k = 0; k < G; ++k)
    if (G <= 2 && 32 * k < n) bits[k] = load_bits(row, type, max(col[k], 0));
}
template <int G>
__device__ __forceinline__ void logits_of(int n, const void *row, int type, const int (&col)[G],
                                          const unsigned (&bits)[G], float (&z)[G]) {
#pragma unroll
  for (int k = 0; k < G; ++k) {
    z[k] = col[k] == kNoMove ? -INFINITY : 0.0f;
    if (32 * k < n && col[k] >= 0) z[k] = value_of(type, G <= 2 ? bits[k] : load_bits(row, type, col[k]));
  }
}

// Softmax statistics. The largest entry is kept out of the sum (S = 1 + rest),
// so that log S and 1 - p of a nearly certain move keep their digits.
struct Norm {
  float top;   // largest logit
  int lead;    // its edge in the lane that has it (the first such lane), else -1
  bool live;   // some move has a logit above -inf (or NaN)
  float rest;  // sum of exp(s - s_top) over the other moves
  float log_s, inv_s;
};

// Sets top and live.
template <int G>
__device__ __forceinline__ void find_top(int n, const float (&z)[G], Norm &q) {
  float top = z[0];
#pragma unroll
  for (int k = 1; k < G; ++k)
    if (32 * k < n) top = fmaxf(top, z[k]);
  q.top = warp_max(top);
  q.live = q.top > -INFINITY;
  if (!q.live) {
    bool nan = false;
#pragma unroll
    for (int k = 0; k < G; ++k) nan |= 32 * k < n && z[k] != z[k];
    q.live = __any_sync(kFull, nan);
  }
}
// Keeps one largest entry out of the sum, `mine` being this lane's lowest edge
// with the largest logit, already kept out, or -1: every lane but the first that
// has one puts it back. Sets lead.
__device__ __forceinline__ void leave_one_out(int mine, int lane, Norm &q) {
  const int first = __ffs(__ballot_sync(kFull, mine >= 0)) - 1;
  if (mine >= 0 && lane != first) q.rest += 1.0f;
  q.lead = lane == first ? mine : -1;
}

// Largest logit, and e[k] = exp(s - s_top) with this lane's part of `rest` and
// of sum e s.
template <int G>
__device__ __forceinline__ Norm softmax_part(int n, const float (&z)[G], float inv_temp,
                                             int lane, float (&e)[G],
                                             float &es) {
  Norm q;
  find_top<G>(n, z, q);
  q.rest = 0.0f;
  es = 0.0f;
  int mine = -1;
#pragma unroll
  for (int k = 0; k < G; ++k) {
    e[k] = 0.0f;
    if (32 * k < n) {
      const float t = (z[k] - q.top) * inv_temp;
      e[k] = exp_fast(t);
      if (e[k] != 0.0f) es += e[k] * t;
      if (mine < 0 && z[k] == q.top)
        mine = 32 * k + lane;
      else
        q.rest += e[k];
    }
  }
  leave_one_out(mine, lane, q);
  return q;
}

__device__ __forceinline__ float reciprocal(float x) {
  float v;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(v) : "f"(x));  // within one step
  return v;
}

// Ends softmax_part for a row: the sums over the warp, their logarithm and
// reciprocal. Returns the entropy -sum p log p = log S - sum(e s) / S, two terms
// that are never negative. With kMore `more` is summed as well, with kSecond the
// sum of a second softmax w over the same list.
//
// The sums share one reduction: after the step over 16 lanes the lower half works
// on one value and the upper on another, after the step over 8 each quarter on
// one, so three take 6 shuffles instead of 15 and two 5 instead of 10, and one
// logarithm and one reciprocal serve both softmaxes.
enum class Sums { kTwo, kMore, kSecond };
template <Sums kSums>
__device__ __forceinline__ float softmax_done(Norm &q, float es, Norm &w, float &more, int lane) {
  constexpr bool kTwo = kSums == Sums::kTwo, kSecond = kSums == Sums::kSecond;
  const bool upper = lane & 16, second = lane & 8;
  if (q.top == INFINITY) q.rest = quiet_nan();  // its own inf - inf is not in the sum
  if (kSecond && w.top == INFINITY) w.rest = quiet_nan();
  const float x = kTwo ? es : kSecond ? w.rest : more;
  float v = (upper ? x : q.rest) + __shfl_xor_sync(kFull, upper ? q.rest : x, 16);
  if (kTwo) {
    v += __shfl_xor_sync(kFull, v, 8);
  } else {
    const float b = es + __shfl_xor_sync(kFull, es, 16);
    v = (second ? b : v) + __shfl_xor_sync(kFull, second ? v : b, 8);
  }
  v += __shfl_xor_sync(kFull, v, 4);
  v += __shfl_xor_sync(kFull, v, 2);
  v += __shfl_xor_sync(kFull, v, 1);
  // lanes 0-7 hold q.rest, 16-23 es of two sums, w.rest or `more`, 8-15 es of three
  const float log_v = log1pf(v), inv_v = reciprocal(1.0f + v);
  q.rest = __shfl_sync(kFull, v, 0);
  q.log_s = __shfl_sync(kFull, log_v, 0);
  q.inv_s = __shfl_sync(kFull, inv_v, 0);
  es = __shfl_sync(kFull, v, kTwo ? 16 : 8);
  if (kSecond) {
    w.log_s = __shfl_sync(kFull, log_v, 16);
    w.inv_s = __shfl_sync(kFull, inv_v, 16);
  } else if (!kTwo) {
    more = __shfl_sync(kFull, v, 16);
  }
  return q.log_s - es * q.inv_s;
}

// The value of move j, which every lane gets. Its lane picks it out with a test
// of every group: a choice among the groups' addresses would put the array into
// local memory.
template <int G>
__device__ __forceinline__ float of_move(const float (&v)[G], int j, int lane) {
  float t = 0.0f;
#pragma unroll
  for (int k = 0; k < G; ++k)
    if (32 * k + lane == j) t = v[k];
  return __shfl_sync(kFull, t, j & 31);
}

// ------------------------------------------------------------------ gradient rows
struct Grad {
  void *base;  // null: no gradient
  long long stride;
  int type;
};

// A warp's gradient row in shared memory, zero between rows. The values of a
// row's moves are put into it, one bulk copy (cp.async.bulk) writes the whole
// row, and the values are taken out again before the next row's go in, by
// which time the copy has read them. The row keeps its place within 16 bytes,
// so that the copy runs from the first to the last 16-byte boundary of the
// row; the elements around them are stored singly.
struct RowImage {
  char *buf;     // 16-byte aligned, a row and 16 bytes long
  bool pending;  // a bulk copy may still be reading it
  int old[2];    // byte offsets of the lane's values, -1 for none
};

__host__ __device__ __forceinline__ int image_bytes(int row_bytes) {
  return ((row_bytes + 15) & ~15) + 16;
}

__device__ __forceinline__ RowImage clear_image(char *buf, int row_bytes, int lane) {
  const int n = image_bytes(row_bytes) >> 4;
  for (int i = lane; i < n; i += 32) reinterpret_cast<uint4 *>(buf)[i] = make_uint4(0, 0, 0, 0);
  __syncwarp();
  return {buf, false, {-1, -1}};
}

__device__ __forceinline__ void put(char *p, int size, unsigned bits) {
  if (size == 4)
    *reinterpret_cast<unsigned *>(p) = bits;
  else
    *reinterpret_cast<unsigned short *>(p) = static_cast<unsigned short>(bits);
}
__device__ __forceinline__ unsigned get(const char *p, int size) {
  return size == 4 ? *reinterpret_cast<const unsigned *>(p) : *reinterpret_cast<const unsigned short *>(p);
}

__device__ __forceinline__ void take_out(RowImage &im, int size, int lane) {
  if (im.pending) {
    if (lane == 0) bulk_wait_read0();
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (im.old[k] >= 0) put(im.buf + im.old[k], size, 0u);
    __syncwarp();
    im.pending = false;
  }
}

// Writes row b: g[k] at the columns of the list, 0 elsewhere. A column that is
// listed more than once gets the sum of its values, in the list's order; the
// moves find that out by leaving their numbers in the image.
template <int G, int kType>
__device__ __forceinline__ void write_row(RowImage &im, const Grad &out, int classes, int b, int n,
                                          int lane, const int (&col)[G], float (&g)[G]) {
  const int type = type_of<kType>(out.type), size = type == MFB200_TYPE_F32 ? 4 : 2;
  char *dst = static_cast<char *>(out.base) + b * out.stride * size;
  const int shift = static_cast<int>(reinterpret_cast<unsigned long long>(dst) & 15);
  int at[G];
  take_out(im, size, lane);
#pragma unroll
  for (int k = 0; k < G; ++k) {
    at[k] = -1;
    if (32 * k < n && col[k] >= 0) {
      at[k] = shift + col[k] * size;
      put(im.buf + at[k], size, 32 * k + lane + 1);
    }
  }
  __syncwarp();
  bool again = false;
#pragma unroll
  for (int k = 0; k < G; ++k)
    if (32 * k < n && at[k] >= 0) again |= get(im.buf + at[k], size) != 32u * k + lane + 1;
  if (__any_sync(kFull, again)) {
    float sum[G];
    bool first[G];
#pragma unroll
    for (int k = 0; k < G; ++k) sum[k] = 0.0f, first[k] = true;
#pragma unroll
    for (int k2 = 0; k2 < G; ++k2) {
      for (int src = 0; src < 32 && 32 * k2 + src < n; ++src) {
        const int c = __shfl_sync(kFull, col[k2], src);
        const float v = __shfl_sync(kFull, g[k2], src);
#pragma unroll
        for (int k = 0; k < G; ++k) {
          if (col[k] == c) {
            sum[k] += v;
            if (32 * k2 + src < 32 * k + lane) first[k] = false;
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < G; ++k) {
      g[k] = sum[k];
      if (!first[k]) at[k] = -1;
    }
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < G; ++k)
    if (32 * k < n && at[k] >= 0) put(im.buf + at[k], size, bits_of(type, g[k]));
  fence_proxy_async_smem();
  __syncwarp();
  // [shift, end) of the image is the row; [lo, hi) of it lies between 16-byte boundaries
  const int end = shift + classes * size;
  const int lo = (shift + 15) & ~15, hi = end & ~15;
  if (lane == 0 && hi > lo) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst - shift + lo),
                 "r"(smem_u32(im.buf + lo)), "r"(hi - lo)
                 : "memory");
    bulk_commit();
  }
  const int head = hi > lo ? (lo - shift) / size : classes;  // elements before the copy, and after
  const int tail = hi > lo ? (end - hi) / size : 0;
  if (lane < head + tail) {
    const int p = lane < head ? shift + lane * size : hi + (lane - head) * size;
    put(dst - shift + p, size, get(im.buf + p, size));
  }
  im.pending = true;
  if (G == 2) {
    im.old[0] = at[0];
    im.old[1] = at[1];
  } else {  // too many values to remember: take them out at once
    if (lane == 0) bulk_wait_read0();
    __syncwarp();
#pragma unroll
    for (int k = 0; k < G; ++k)
      if (32 * k < n && at[k] >= 0) put(im.buf + at[k], size, 0u);
    __syncwarp();
    im.pending = false;
  }
}

// A row of NaN, for a malformed position.
__device__ __forceinline__ void write_nan_row(const Grad &out, int classes, int b, int lane) {
  const int size = out.type == MFB200_TYPE_F32 ? 4 : 2;
  char *dst = static_cast<char *>(out.base) + b * out.stride * size;
  for (int i = lane; i < classes; i += 32) put(dst + static_cast<long long>(i) * size, size, bits_of(out.type, quiet_nan()));
}

// ------------------------------------------------------------------ log-probabilities
template <int G, int kType>
__device__ __forceinline__ void score_position(const PolicyRows &r, int b,
                                               const Moves &m, int c0, int c1, int lane,
                                               float *move_logp, float *played_logp,
                                               float *entropy) {
  Edges<G> v;
  columns<G>(r, m, c0, c1, lane, v);
  unsigned bits[G];
  const int type = type_of<kType>(r.type);
  const void *row = row_of(r.logits, type, r.stride, b);
  load_logits<G>(m.n, row, type, v.col, bits);
  logits_of<G>(m.n, row, type, v.col, bits, v.z);
  float es;
  Norm q = softmax_part<G>(m.n, v.z, r.inv_temp, lane, v.e, es);
  const float h = softmax_done<Sums::kTwo>(q, es, q, es, lane);
  if (move_logp) {
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const int j = 32 * k + lane;
      if (j < m.n)
        move_logp[m.lo + j] = q.live ? (v.z[k] - q.top) * r.inv_temp - q.log_s : -INFINITY;
    }
    if (G > 2)
      for (int j = m.n + lane; j < m.count; j += 32) move_logp[m.lo + j] = -INFINITY;
  }
  const bool takes = q.live && m.played >= 0;
  const float z = of_move<G>(v.z, m.played < 0 ? 0 : m.played, lane);
  const float logp = (z - q.top) * r.inv_temp - q.log_s;
  if (lane == 0) {
    if (played_logp) played_logp[b] = m.bad ? quiet_nan() : takes ? logp : 0.0f;
    if (entropy) entropy[b] = m.bad ? quiet_nan() : q.live ? h : 0.0f;
  }
}

// The played move's log-probability for sums over lines, whose difference is
// small: made in 64 bits and given in two parts, the rounded value and the rest.
// (From 32-bit exponentials the margin of a pair of 6-ply lines was 6e-7 of itself
// off in the middle of 150 cases and 1e-5 in the worst.) The first part
// tells whether the position takes part: +0 for one without a move, a set sign bit
// or NaN for the others (takes_part). row_grad gets the zero of a position in no line.
__device__ __forceinline__ bool takes_part(float logp) { return signbit(logp) || logp != logp; }

template <int G, int kType>
__device__ __forceinline__ void line_position(const PolicyRows &r, int b, const Moves &m, int c0,
                                              int c1, int lane, float *played_logp,
                                              float *logp_rest, float *row_grad) {
  Edges<G> v;
  columns<G>(r, m, c0, c1, lane, v);
  unsigned bits[G];
  const int type = type_of<kType>(r.type);
  const void *row = row_of(r.logits, type, r.stride, b);
  load_logits<G>(m.n, row, type, v.col, bits);
  logits_of<G>(m.n, row, type, v.col, bits, v.z);
  Norm q;
  find_top<G>(m.n, v.z, q);
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < G; ++k)
    if (32 * k < m.n) sum += exp((static_cast<double>(v.z[k]) - q.top) * r.inv_temp64);
  sum = warp_sum(sum);
  const float z = of_move<G>(v.z, m.played < 0 ? 0 : m.played, lane);
  const double logp = (static_cast<double>(z) - q.top) * r.inv_temp64 - log(sum);
  if (lane == 0) {
    const bool takes = m.bad || (q.live && m.played >= 0);
    const float value = m.bad ? quiet_nan() : static_cast<float>(logp);
    played_logp[b] = takes ? copysignf(value, -1.0f) : 0.0f;  // never above 0
    logp_rest[b] = takes && fabsf(value) < INFINITY ? static_cast<float>(logp - value) : 0.0f;
    row_grad[b] = 0.0f;
  }
}

// CTAs on an SM. 40 warps with 48 registers: 50021 bf16 positions take 21 us; with
// 48 warps and 40 registers 22, with 32 warps and 64 registers 27. The same for
// lines: 96 pairs of games 42 us, 43 with 32 warps.
constexpr int kScoreCtas = 5;
template <int kType>
__global__ void __launch_bounds__(32 * kMaxWarps, kScoreCtas)
    move_logprobs_kernel(const __grid_constant__ PolicyRows r, float *move_logp,
                         float *played_logp, float *entropy) {
  __shared__ Turns turns;
  start_turns(&turns);
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31;
  for_positions(
      r, gridDim.x, &turns,
      [&](int b, const Moves &m, int c0, int c1) {
        score_position<2, kType>(r, b, m, c0, c1, lane, move_logp, played_logp, entropy);
        return false;
      },
      [&](int b, const Moves &m) {
        score_position<8, kType>(r, b, m, load_index(r, m, 0, lane), load_index(r, m, 1, lane),
                                 lane, move_logp, played_logp, entropy);
      });
}

template <int kType>
__global__ void __launch_bounds__(32 * kMaxWarps, kScoreCtas)
    line_logprobs_kernel(const __grid_constant__ PolicyRows r, float *played_logp, float *logp_rest,
                         float *row_grad) {
  __shared__ Turns turns;
  start_turns(&turns);
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31;
  for_positions(
      r, gridDim.x, &turns,
      [&](int b, const Moves &m, int c0, int c1) {
        line_position<2, kType>(r, b, m, c0, c1, lane, played_logp, logp_rest, row_grad);
        return false;
      },
      [&](int b, const Moves &m) {
        line_position<8, kType>(r, b, m, load_index(r, m, 0, lane), load_index(r, m, 1, lane),
                                lane, played_logp, logp_rest, row_grad);
      });
}

// [c = a] - p_c for move j; 1 - p of the largest entry is rest / S
__device__ __forceinline__ float played_term(const Moves &m, const Norm &q, int j, float p) {
  return j != m.played ? -p : j == q.lead ? q.rest * q.inv_s : 1.0f - p;
}

// dL/dlogit_c = (1/T) [ G_c + [c = a] g - p_c (sum G + g) - g_H p_c (logp_c + H) ]
// for upstream gradients G of the moves' log-probabilities, g of the played
// move's and g_H of the entropy, each of which may be null.
struct BackArgs {
  const float *moves, *played, *entropy;
  bool parts_only;  // a row whose upstream gradient is 0 takes no part: a zero row, whatever its logits are
  Grad out;
  // the sum of n losses, by one more CTA, where `total` is set
  const float *loss;
  int n;
  float *total;
};

template <int G, int kType>
__device__ __forceinline__ void back_position(const PolicyRows &r, const BackArgs &a,
                                              int b, const Moves &m, int c0,
                                              int c1, int lane, RowImage &im) {
  Edges<G> v;
  columns<G>(r, m, c0, c1, lane, v);
  unsigned bits[G];
  const int type = type_of<kType>(r.type);
  const void *row = row_of(r.logits, type, r.stride, b);
  load_logits<G>(m.n, row, type, v.col, bits);
  float g[G], total = 0.0f;
#pragma unroll
  for (int k = 0; k < G; ++k) {
    g[k] = a.moves && 32 * k + lane < m.n ? a.moves[m.lo + 32 * k + lane] : 0.0f;
    total += g[k];
  }
  const float ga = a.played && m.played >= 0 ? a.played[b] : 0.0f;
  const float gh = a.entropy ? a.entropy[b] : 0.0f;
  logits_of<G>(m.n, row, type, v.col, bits, v.z);
  float es;
  Norm q = softmax_part<G>(m.n, v.z, r.inv_temp, lane, v.e, es);
  const float h = softmax_done<Sums::kMore>(q, es, q, total, lane);
  const bool takes = q.live && !(a.parts_only && ga == 0.0f);
#pragma unroll
  for (int k = 0; k < G; ++k) {
    if (32 * k >= m.n) continue;
    const int j = 32 * k + lane;
    const float p = v.e[k] * q.inv_s;
    float t = g[k] - p * total + ga * played_term(m, q, j, p);
    if (a.entropy && p != 0.0f) t -= gh * p * ((v.z[k] - q.top) * r.inv_temp - q.log_s + h);
    g[k] = t * r.inv_temp;
    if (!takes) v.col[k] = kNoColumn;
  }
  write_row<G, kType>(im, a.out, r.classes, b, m.n, lane, v.col, g);
}

// The sum of n losses by the `ctas` CTAs of a cluster (or one CTA), in 64 bits
// and in one order.
__device__ void sum_losses(const float *loss, int n, float *total, unsigned ctas) {
  __shared__ double part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned rank = ctas > 1 ? blockIdx.x : 0;
  double v = 0.0;
  const long long step = static_cast<long long>(blockDim.x) * ctas;
  long long i = static_cast<long long>(rank) * blockDim.x + threadIdx.x;
  for (; n - i > 15 * step; i += 16 * step) {  // sixteen loads under way at once
    float x[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = loss[i + k * step];
#pragma unroll
    for (int k = 0; k < 16; ++k) v += x[k];
  }
  float x[15];
#pragma unroll
  for (int k = 0; k < 15; ++k) x[k] = i + k * step < n ? loss[i + k * step] : 0.0f;
#pragma unroll
  for (int k = 0; k < 15; ++k) v += x[k];
  v = warp_sum(v);
  if (lane == 0) part[warp] = v;
  __syncthreads();
  if (warp == 0) {
    v = lane < static_cast<int>(blockDim.x >> 5) ? part[lane] : 0.0;
    v = warp_sum(v);
    if (ctas == 1) {
      if (lane == 0) *total = static_cast<float>(v);
      return;
    }
    if (lane == 0) part[0] = v;
  }
  if (ctas == 1) return;
  cluster_sync();
  if (rank == 0 && warp == 0) {
    double w = 0.0;
    if (lane < static_cast<int>(ctas)) {
      unsigned at;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(part)), "r"(lane));
      asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(w) : "r"(at));
    }
    w = warp_sum(w);
    if (lane == 0) *total = static_cast<float>(w);
  }
  cluster_sync();  // no CTA leaves while its part is read
}

template <int kType>
__global__ void __launch_bounds__(32 * kMaxWarps, 3)
    move_logprobs_backward_kernel(const __grid_constant__ PolicyRows r,
                                  const __grid_constant__ BackArgs a) {
  extern __shared__ __align__(16) char images[];
  const int lane = threadIdx.x & 31;
  const int row_bytes = r.classes * (type_of<kType>(a.out.type) == MFB200_TYPE_F32 ? 4 : 2);
  const unsigned ctas = gridDim.x - (a.total ? 1 : 0);
  RowImage im = clear_image(images + (threadIdx.x >> 5) * image_bytes(row_bytes), row_bytes, lane);
  __shared__ Turns turns;
  start_turns(&turns);
  pdl_wait();
  pdl_launch();
  if (blockIdx.x == ctas) {
    sum_losses(a.loss, a.n, a.total, 1);
    return;
  }
  for_positions(
      r, ctas, &turns,
      [&](int b, const Moves &m, int c0, int c1) {
        back_position<2, kType>(r, a, b, m, c0, c1, lane, im);
        return false;
      },
      [&](int b, const Moves &m) {
        if (m.bad)
          write_nan_row(a.out, r.classes, b, lane);
        else
          back_position<8, kType>(r, a, b, m, load_index(r, m, 0, lane),
                                  load_index(r, m, 1, lane), lane, im);
      });
  if (lane == 0) bulk_wait0();
}

// ------------------------------------------------------------------ clipped policy loss
struct ClipArgs {
  const float *old_logp, *advantage, *weight;  // weight may be null (1)
  const void *ref;                             // reference logits, or null
  long long ref_stride;
  int ref_type;
  double low, high;  // 1 - clip_low, 1 + clip_high
  float kl_coef, entropy_coef, scale;
  float *loss, *logp, *kl, *entropy;  // each may be null
  Grad grad;
};

// KL = sum p (e^-d - 1 + d) with d = log p - log q (sum p e^-d = sum q = 1):
// every term is >= 0 and an error common to all d cancels, so the KL of two
// near policies keeps its digits. For |d| < 1/2 by the series d^2/2 - d^3/6 +
// ... + d^8/8!, whose next term is at most 5e-8 of it; else from p, q and d themselves.
__device__ __forceinline__ float kl_term(float p, float pr, float d) {
  float t = 1.0f / 40320;
  t = fmaf(t, -d, 1.0f / 5040);
  t = fmaf(t, -d, 1.0f / 720);
  t = fmaf(t, -d, 1.0f / 120);
  t = fmaf(t, -d, 1.0f / 24);
  t = fmaf(t, -d, 1.0f / 6);
  t = fmaf(t, -d, 1.0f / 2);
  const float near = p * (d * d * t), far = pr - p + p * d;
  return p == 0.0f ? pr : fabsf(d) < 0.5f ? near : far;
}

// What the rounding of d = a - b leaves (the exact difference is d plus it); NaN
// where one is infinite.
__device__ __forceinline__ float difference_rest(float a, float b, float d) {
  const float t = d - a;
  return (a - (d - t)) - (b + t);
}

// Returns true, with nothing written, for a ratio too near the clip's border
// to be decided in 32 bits, unless kExact.
template <int G, bool kExact, int kType>
__device__ __forceinline__ bool clip_position(const PolicyRows &r, const ClipArgs &a,
                                              int b, const Moves &m, int c0,
                                              int c1, int lane, RowImage &im) {
  Edges<G> v;
  columns<G>(r, m, c0, c1, lane, v);
  float d[G];  // the reference's logits, then d = log p - log q
  unsigned bits[G], ref_bits[G];
  const int type = type_of<kType>(r.type);
  const void *row = row_of(r.logits, type, r.stride, b);
  load_logits<G>(m.n, row, type, v.col, bits);
  const int ref_type = type_of<kType>(a.ref_type);
  const void *ref = a.ref ? row_of(a.ref, ref_type, a.ref_stride, b) : nullptr;
  if (a.ref) load_logits<G>(m.n, ref, ref_type, v.col, ref_bits);
  const float old = a.old_logp[b], adv = a.advantage[b];
  const float c = a.scale * (a.weight ? a.weight[b] : 1.0f);
  logits_of<G>(m.n, row, type, v.col, bits, v.z);
  if (a.ref) logits_of<G>(m.n, ref, ref_type, v.col, ref_bits, d);
  float es;
  Norm q = softmax_part<G>(m.n, v.z, r.inv_temp, lane, v.e, es);
  float h, kl = 0.0f;
  if (a.ref) {
    float er[G], es_r;
    Norm w = softmax_part<G>(m.n, d, r.inv_temp, lane, er, es_r);
    h = softmax_done<Sums::kSecond>(q, es, w, kl, lane);
    const float tops = q.top - w.top;
    const float tops_rest = difference_rest(q.top, w.top, tops);
#pragma unroll
    for (int k = 0; k < G; ++k) {
      if (32 * k < m.n) {
        // z - z' minus the difference of the tops, with what either rounding leaves: exact, for near
        // policies and for logits with a number of their own added to each row
        const float x = v.z[k] - d[k], low = difference_rest(v.z[k], d[k], x) - tops_rest;
        const float apart = (x - tops) + (low == low ? low : 0.0f);
        d[k] = apart * r.inv_temp + (w.log_s - q.log_s);
        kl += kl_term(v.e[k] * q.inv_s, er[k] * w.inv_s, d[k]);
      }
    }
    kl = warp_sum(kl);
  } else {
    h = softmax_done<Sums::kTwo>(q, es, q, kl, lane);
  }
  const bool takes = q.live && m.played >= 0;
  const float za = of_move<G>(v.z, m.played < 0 ? 0 : m.played, lane);
  const float sa = (za - q.top) * r.inv_temp;
  const float ratio = exp_fast((sa - old) - q.log_s);
  // The gradient jumps where the ratio crosses the clip's border, so a ratio
  // within the rounding of the border is computed again in 64 bits.
  const float border = static_cast<float>(adv > 0.0f ? a.high : a.low);
  bool active = adv > 0.0f ? !(ratio > border) : !(ratio < border);
  if (takes && fabsf(ratio - border) <=
                   border * (4e-6f + 3e-7f * (fabsf(sa) + q.log_s + fabsf(old)))) {
    if (!kExact) return true;
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < G; ++k)
      if (32 * k < m.n) sum += exp((static_cast<double>(v.z[k]) - q.top) / r.temp);
    sum = warp_sum(sum);
    const double exact =
        exp((static_cast<double>(za) - q.top) / r.temp - log(sum) - static_cast<double>(old));
    active = adv > 0.0f ? !(exact > a.high) : !(exact < a.low);
  }
  // A term whose coefficient is 0 (advantage, kl_coef) is left out: the ratio and the
  // KL may be infinite. kl_coef is 0 without a reference.
  if (a.grad.base) {
    const float slope = active && adv != 0.0f ? -adv * ratio : 0.0f;
    float g[G];
#pragma unroll
    for (int k = 0; k < G; ++k) {
      if (32 * k >= m.n) continue;
      const float p = v.e[k] * q.inv_s;
      float t = slope * played_term(m, q, 32 * k + lane, p);
      if (p != 0.0f) {
        if (a.kl_coef != 0.0f) t += a.kl_coef * p * (d[k] - kl);
        t += a.entropy_coef * p * ((v.z[k] - q.top) * r.inv_temp - q.log_s + h);
      }
      g[k] = c * r.inv_temp * t;
      if (!takes) v.col[k] = kNoColumn;
    }
    write_row<G, kType>(im, a.grad, r.classes, b, m.n, lane, v.col, g);
  }
  // after the row: the fence before its copy would wait for these stores
  if (lane == 0) {
    float loss = adv != 0.0f ? -adv * (active ? ratio : border) : 0.0f;
    if (a.kl_coef != 0.0f) loss += a.kl_coef * kl;
    loss -= a.entropy_coef * h;
    if (a.loss) a.loss[b] = takes ? c * loss : 0.0f;
    if (a.logp) a.logp[b] = takes ? sa - q.log_s : 0.0f;
    if (a.kl) a.kl[b] = q.live ? kl : 0.0f;
    if (a.entropy) a.entropy[b] = q.live ? h : 0.0f;
  }
  return false;
}

template <int kType>
__global__ void __launch_bounds__(32 * kMaxWarps, 3)
    clipped_policy_loss_kernel(const __grid_constant__ PolicyRows r,
                               const __grid_constant__ ClipArgs a) {
  extern __shared__ __align__(16) char images[];
  const int lane = threadIdx.x & 31;
  RowImage im{};
  if (a.grad.base) {
    const int row_bytes = r.classes * (type_of<kType>(a.grad.type) == MFB200_TYPE_F32 ? 4 : 2);
    im = clear_image(images + (threadIdx.x >> 5) * image_bytes(row_bytes), row_bytes, lane);
  }
  __shared__ Turns turns;
  start_turns(&turns);
  pdl_wait();
  pdl_launch();
  for_positions(
      r, gridDim.x, &turns,
      [&](int b, const Moves &m, int c0, int c1) {
        return clip_position<2, false, kType>(r, a, b, m, c0, c1, lane, im);
      },
      [&](int b, const Moves &m) {
        if (!m.bad) {
          clip_position<8, true, kType>(r, a, b, m, load_index(r, m, 0, lane),
                                        load_index(r, m, 1, lane), lane, im);
          return;
        }
        if (lane == 0) {
          if (a.loss) a.loss[b] = quiet_nan();
          if (a.logp) a.logp[b] = quiet_nan();
          if (a.kl) a.kl[b] = quiet_nan();
          if (a.entropy) a.entropy[b] = quiet_nan();
        }
        if (a.grad.base) write_nan_row(a.grad, r.classes, b, lane);
      });
  if (lane == 0) bulk_wait0();
}

// ------------------------------------------------------------------ preference loss
// One warp per pair of lines. With D = the sum over a line's rows of
// (logp - ref) and m = beta (D_preferred - D_rejected):
//     L = scale w ( -(1 - eps) log sigma(m) - eps log sigma(-m) ),
// and dL/dlogp of a row is +-beta dL/dm. A row that takes no part has its reference
// value left out and a zero gradient. Rows in no line
// keep the zero they have. The sums run in 64 bits, in an order fixed by the rows.
__global__ void __launch_bounds__(256)
    preference_pair_kernel(int pairs, int batch, const int32_t *lines,
                           const float *logp, const float *rest, const float *ref,
                           const float *weight, float beta, float eps, float scale,
                           float *row_grad, float *line_logp,
                           float *margin, float *loss) {
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31;
  const int i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (i >= pairs) return;
  const int at[3] = {lines[2 * i], lines[2 * i + 1], lines[2 * i + 2]};
  if (at[0] < 0 || at[1] < at[0] || at[2] < at[1] || at[2] > batch) {
    if (lane == 0) {
      line_logp[2 * i] = line_logp[2 * i + 1] = quiet_nan();
      margin[i] = loss[i] = quiet_nan();
    }
    return;
  }
  const float w = scale * (weight ? weight[i] : 1.0f);
  const unsigned first = at[0], cut = at[1], end = at[2];  // (unsigned: a step may pass 2^31)
  double sum[2] = {0.0, 0.0}, gain[2] = {0.0, 0.0};
  for (unsigned from = first; from < end; from += 256) {  // 24 loads under way at once
    float lp[8], low[8], frozen[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned b = from + 32 * k + lane;
      lp[k] = b < end ? logp[b] : 0.0f;
      low[k] = b < end ? rest[b] : 0.0f;
      frozen[k] = b < end ? ref[b] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (from + 32 * k >= end) break;
      const int side = from + 32 * k + lane < cut ? 0 : 1;
      const double value = static_cast<double>(lp[k]) + low[k];
      const double up = takes_part(lp[k]) ? value - frozen[k] : 0.0;
      sum[0] += side ? 0.0 : value;
      sum[1] += side ? value : 0.0;
      gain[0] += side ? 0.0 : up;
      gain[1] += side ? up : 0.0;
    }
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    sum[side] = warp_sum(sum[side]);
    gain[side] = warp_sum(gain[side]);
  }
  // A term whose coefficient is 0 is left out, so that it is 0 where the margin is infinite.
  const float mg = beta == 0.0f ? 0.0f : static_cast<float>(static_cast<double>(beta) * (gain[0] - gain[1]));
  // -log sigma(m) = max(-m, 0) + log(1 + e^-|m|); sigma(-|m|) = e^-|m| / (1 + e^-|m|)
  const float tail = expf(-fabsf(mg));
  const float less = fmaxf(-mg, 0.0f) + log1pf(tail), more = fmaxf(mg, 0.0f) + log1pf(tail);
  const float small = tail / (1.0f + tail), large = 1.0f / (1.0f + tail);
  const float up = mg < 0.0f ? small : large, down = mg < 0.0f ? large : small;  // sigma(m), sigma(-m)
  const float slope = w * beta * (eps * up - (1.0f - eps) * down);
  if (lane == 0) {
    line_logp[2 * i] = static_cast<float>(sum[0]);
    line_logp[2 * i + 1] = static_cast<float>(sum[1]);
    margin[i] = mg;
    // fmaxf drops a NaN margin: it is added back
    loss[i] = mg != mg ? mg : w * ((eps < 1.0f ? (1.0f - eps) * less : 0.0f) + (eps > 0.0f ? eps * more : 0.0f));
  }
  for (unsigned from = first; from < end; from += 256) {
    float lp[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned b = from + 32 * k + lane;
      lp[k] = b < end ? logp[b] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned b = from + 32 * k + lane;
      if (b < end) row_grad[b] = !takes_part(lp[k]) ? 0.0f : b < cut ? slope : -slope;
    }
  }
}

// ------------------------------------------------------------------ total
__global__ void __launch_bounds__(1024) loss_total_kernel(const float *loss, int n, float *total) {
  pdl_wait();
  pdl_launch();
  sum_losses(loss, n, total, gridDim.x);
}

// ------------------------------------------------------------------ launches
struct Shape {
  int warps, ctas;
  size_t smem;
};

// Positions are spread over the SMs before they share a CTA; a CTA's warps
// then take `per_sm` CTAs' worth of positions in turn.
Shape shape_for(int batch, int max_warps, int per_sm, size_t bytes_per_warp) {
  const int sms = num_sms();
  int w = 1;
  while (w < max_warps && batch > sms * w) w *= 2;
  const long long need = (static_cast<long long>(batch) + w - 1) / w;
  const long long most = static_cast<long long>(sms) * per_sm;
  return {w, static_cast<int>(need < most ? need : most), w * bytes_per_warp};
}

// With a row image per warp: as many warps as keep three CTAs on an SM.
Shape shape_with_images(const PolicyRows &r, const Grad &g) {
  constexpr size_t kPerSm = 225 * 1024, kReserved = 1024;
  const size_t bytes = image_bytes(r.classes * (g.type == MFB200_TYPE_F32 ? 4 : 2));
  int w = kMaxWarps;
  while (w > 1 && 3 * (w * bytes + kReserved) > kPerSm) w /= 2;
  const Shape s = shape_for(r.batch, w, 1, bytes);
  int per_sm = static_cast<int>(kPerSm / (s.smem + kReserved));
  per_sm = per_sm > 3 ? 3 : per_sm < 1 ? 1 : per_sm;
  return shape_for(r.batch, w, per_sm, bytes);
}

// Raises a kernel's shared-memory limit once per device to what the largest row needs.
template <class K>
cudaError_t allow_images(K *kernel, std::atomic<unsigned long long> &done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
  if (e == cudaSuccess) done.fetch_or(bit);
  return e;
}

// launch(type) with the type as a constant.
template <class Launch>
cudaError_t with_type(int type, Launch launch) {
  switch (type) {
    case MFB200_TYPE_F32: return launch(std::integral_constant<int, MFB200_TYPE_F32>());
    case MFB200_TYPE_BF16: return launch(std::integral_constant<int, MFB200_TYPE_BF16>());
    default: return launch(std::integral_constant<int, MFB200_TYPE_F16>());
  }
}

cudaError_t launch_backward(const PolicyRows &r, const BackArgs &a, cudaStream_t s) {
  const Shape t = shape_with_images(r, a.out);
  const auto launch = [&](auto type) {
    static std::atomic<unsigned long long> done{0};
    constexpr auto *kernel = move_logprobs_backward_kernel<decltype(type)::value>;
    if (cudaError_t e = allow_images(kernel, done)) return e;
    return launch_k(kernel, dim3(t.ctas + (a.total ? 1 : 0)), dim3(32 * t.warps), t.smem, s, 1, r, a);
  };
  return a.out.type == r.type ? with_type(r.type, launch)
                              : launch(std::integral_constant<int, kAnyType>());
}

cudaError_t launch_clip(const PolicyRows &r, const ClipArgs &a, cudaStream_t s) {
  const Shape t = a.grad.base ? shape_with_images(r, a.grad) : shape_for(r.batch, kMaxWarps, 3, 0);
  const bool same = (!a.ref || a.ref_type == r.type) && (!a.grad.base || a.grad.type == r.type);
  const auto launch = [&](auto type) {
    static std::atomic<unsigned long long> done{0};
    constexpr auto *kernel = clipped_policy_loss_kernel<decltype(type)::value>;
    if (cudaError_t e = allow_images(kernel, done)) return e;
    return launch_k(kernel, dim3(t.ctas), dim3(32 * t.warps), t.smem, s, 1, r, a);
  };
  return same ? with_type(r.type, launch) : launch(std::integral_constant<int, kAnyType>());
}

cudaError_t launch_lines(const PolicyRows &r, float *played_logp, float *logp_rest, float *row_grad,
                         cudaStream_t s) {
  const Shape t = shape_for(r.batch, kMaxWarps, kScoreCtas, 0);
  return with_type(r.type, [&](auto type) {
    return launch_k(line_logprobs_kernel<decltype(type)::value>, dim3(t.ctas), dim3(32 * t.warps), 0,
                    s, 1, r, played_logp, logp_rest, row_grad);
  });
}

cudaError_t launch_pairs(int pairs, int batch, const int32_t *lines, const float *logp,
                         const float *rest, const float *ref, const float *weight, float beta, float eps, float scale,
                         float *row_grad, float *line_logp, float *margin, float *loss,
                         cudaStream_t s) {
  int w = 1;
  while (w < 8 && pairs > num_sms() * w) w *= 2;
  return launch_k(preference_pair_kernel, dim3((static_cast<unsigned>(pairs) + w - 1) / w),
                  dim3(32 * w), 0, s, 1, pairs, batch, lines, logp, rest, ref, weight, beta, eps, scale,
                  row_grad, line_logp, margin, loss);
}

cudaError_t launch_total(const float *loss, int n, float *total, cudaStream_t s) {
  const int threads = n >= 1024 ? 1024 : n > 0 ? (n + 31) / 32 * 32 : 32;
  const int ctas = n > 16384 ? 8 : 1;  // more than 16 losses a thread: a cluster
  return launch_k(loss_total_kernel, dim3(ctas), dim3(threads), 0, s, ctas, loss, n, total);
}

}  // namespace

cudaError_t launch_move_logprobs(const PolicyRows &r, float *move_logp, float *played_logp,
                                 float *entropy, cudaStream_t s) {
  const Shape t = shape_for(r.batch, kMaxWarps, kScoreCtas, 0);
  return with_type(r.type, [&](auto type) {
    return launch_k(move_logprobs_kernel<decltype(type)::value>, dim3(t.ctas), dim3(32 * t.warps), 0,
                    s, 1, r, move_logp, played_logp, entropy);
  });
}

}  // namespace mfb200

// ------------------------------------------------------------------ C ABI
namespace {

using namespace mfb200;

thread_local char t_err[256];

int fail(const char *fn, const char *msg) {
  std::snprintf(t_err, sizeof(t_err), "%s: %s", fn, msg);
  return 1;
}

int type_size(int type) {
  return type == MFB200_TYPE_F32 ? 4 : type == MFB200_TYPE_BF16 || type == MFB200_TYPE_F16 ? 2 : 0;
}

bool aligned(const void *p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// Bytes of an array, or of a [batch, classes] matrix whose rows are `stride`
// elements apart. Matrices of one pitch may lie in one another's gaps (columns of
// one wide buffer): they meet where their columns do.
struct Range {
  uintptr_t lo, hi;
  uintptr_t pitch, width;  // of a matrix, else 0
  bool meets(const Range &o) const {
    if (lo >= o.hi || o.lo >= hi) return false;
    if (!pitch || pitch != o.pitch) return true;
    const uintptr_t past = lo <= o.lo ? (o.lo - lo) % pitch : (pitch - (lo - o.lo) % pitch) % pitch;
    return past < width || pitch - past < o.width;
  }
};
Range matrix(const void *p, long long stride, int type, int batch, int classes) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p), pitch = static_cast<uintptr_t>(stride) * type_size(type),
                  width = static_cast<uintptr_t>(classes) * type_size(type);
  return {lo, lo + (batch - 1) * pitch + width, pitch, width};
}
Range array(const void *p, long long n, int size) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  return {lo, p ? lo + static_cast<uintptr_t>(n) * size : lo, 0, 0};
}

const char *check_matrix(const void *p, long long stride, int type, int classes, int batch) {
  if (!p) return "null logits";
  const int size = type_size(type);
  if (!size) return "unknown element type";
  if (!aligned(p, size)) return "a matrix is not aligned to its element type";
  if (stride < classes) return "a row stride is smaller than the number of classes";
  if (stride > (1LL << 46) / batch) return "a row stride is too large";
  return nullptr;
}

// Everything that can be checked without reading device memory. batch > 0.
const char *check_rows(const mfb200_policy_rows &r, bool needs_played) {
  if (r.classes < 1 || r.classes > 32767) return "classes must be between 1 and 32767";
  if (const char *e = check_matrix(r.logits, r.logits_stride, r.logits_type, r.classes, r.batch)) return e;
  if (!r.move_offsets) return "null move_offsets";
  if (r.num_moves < 0 || r.num_moves > INT32_MAX) return "num_moves must be between 0 and 2^31 - 1";
  if (!r.move_index && r.num_moves > 0) return "null move_index";
  if (needs_played && !r.played) return "null played";
  if (!aligned(r.move_offsets, 4) || !aligned(r.move_index, 2) || !aligned(r.played, 4))
    return "a list is not aligned to its element type";
  if (!(r.softmax_temp >= 1e-30 && r.softmax_temp <= 1e30))
    return "softmax_temp must be positive (between 1e-30 and 1e30)";
  return nullptr;
}

const char *check_grad(const mfb200_policy_rows &r, const void *grad, long long stride, int type) {
  if (const char *e = check_matrix(grad, stride, type, r.classes, r.batch)) return e;
  return nullptr;
}

// The device the buffers live on must be the current one: a launch on another
// would read them through peer mappings, or fault.
const char *check_device(const void *p) {
  cudaPointerAttributes at{};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return "no current CUDA device";
  }
  if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
    cudaGetLastError();
    return "the data are not behind a device pointer";
  }
  if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
    return "the data are not in device memory";
  if (at.type == cudaMemoryTypeDevice && at.device != dev)
    return "the data are on another device than the current one";
  return nullptr;
}

PolicyRows rows_of(const mfb200_policy_rows &r) {
  PolicyRows o{};
  o.logits = r.logits;
  o.stride = r.logits_stride;
  o.type = r.logits_type;
  o.batch = r.batch;
  o.classes = r.classes;
  o.off = r.move_offsets;
  o.index = r.move_index;
  o.num_moves = r.num_moves;
  o.played = r.played;
  o.temp = r.softmax_temp;
  o.inv_temp64 = 1.0 / r.softmax_temp;
  o.inv_temp = static_cast<float>(o.inv_temp64);
  return o;
}

int launched(const char *fn, cudaError_t e) {
  if (e == cudaSuccess) return 0;
  cudaGetLastError();
  std::snprintf(t_err, sizeof(t_err), "%s: launch failed: %s", fn, cudaGetErrorString(e));
  return 1;
}

}  // namespace

extern "C" MFB200_API const char *mfb200_policy_last_error(void) { return t_err; }

extern "C" MFB200_API int mfb200_move_logprobs(const mfb200_policy_rows *rows, float *d_move_logp,
                                               float *d_played_logp, float *d_entropy,
                                               void *stream) {
  const char *fn = "mfb200_move_logprobs";
  if (!rows) return fail(fn, "null rows");
  if (rows->batch < 0) return fail(fn, "negative batch");
  if (rows->batch == 0) return 0;
  if (const char *e = check_rows(*rows, d_played_logp != nullptr)) return fail(fn, e);
  if (!aligned(d_move_logp, 4) || !aligned(d_played_logp, 4) || !aligned(d_entropy, 4))
    return fail(fn, "an output is not aligned to its element type");
  if (!d_move_logp && !d_played_logp && !d_entropy) return fail(fn, "no output");
  if (const char *e = check_device(rows->logits)) return fail(fn, e);
  return launched(fn, launch_move_logprobs(rows_of(*rows), d_move_logp, d_played_logp, d_entropy,
                                           static_cast<cudaStream_t>(stream)));
}

extern "C" MFB200_API int mfb200_move_logprobs_backward(
    const mfb200_policy_rows *rows, const float *d_grad_moves, const float *d_grad_played,
    const float *d_grad_entropy, void *d_grad_logits, int64_t grad_stride, int grad_type,
    void *stream) {
  const char *fn = "mfb200_move_logprobs_backward";
  if (!rows) return fail(fn, "null rows");
  if (rows->batch < 0) return fail(fn, "negative batch");
  if (rows->batch == 0) return 0;
  if (const char *e = check_rows(*rows, d_grad_played != nullptr)) return fail(fn, e);
  if (const char *e = check_grad(*rows, d_grad_logits, grad_stride, grad_type)) return fail(fn, e);
  if (!aligned(d_grad_moves, 4) || !aligned(d_grad_played, 4) || !aligned(d_grad_entropy, 4))
    return fail(fn, "a gradient is not aligned to its element type");
  const int n = rows->batch;
  const Range g = matrix(d_grad_logits, grad_stride, grad_type, n, rows->classes);
  if (g.meets(matrix(rows->logits, rows->logits_stride, rows->logits_type, n, rows->classes)) ||
      g.meets(array(d_grad_moves, rows->num_moves, 4)) || g.meets(array(d_grad_played, n, 4)) ||
      g.meets(array(d_grad_entropy, n, 4)) || g.meets(array(rows->move_offsets, n + 1LL, 4)) ||
      g.meets(array(rows->move_index, rows->num_moves, 2)) || g.meets(array(rows->played, n, 4)))
    return fail(fn, "the gradient overlaps an input");
  if (const char *e = check_device(rows->logits)) return fail(fn, e);
  BackArgs a{};
  a.moves = d_grad_moves;
  a.played = d_grad_played;
  a.entropy = d_grad_entropy;
  a.out = Grad{d_grad_logits, grad_stride, grad_type};
  return launched(fn, launch_backward(rows_of(*rows), a, static_cast<cudaStream_t>(stream)));
}

extern "C" MFB200_API int mfb200_clipped_policy_loss(
    const mfb200_policy_rows *rows, const mfb200_clip_config *cfg, const float *d_old_logp,
    const float *d_advantage, const float *d_weight, const void *d_ref_logits, int64_t ref_stride,
    int ref_type, float *d_loss, float *d_logp, float *d_kl, float *d_entropy, float *d_total,
    void *d_grad_logits, int64_t grad_stride, int grad_type, void *stream) {
  const char *fn = "mfb200_clipped_policy_loss";
  if (!rows || !cfg) return fail(fn, "null rows or config");
  if (rows->batch < 0) return fail(fn, "negative batch");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows->batch == 0)
    return d_total ? launched(fn, cudaMemsetAsync(d_total, 0, sizeof(float), s)) : 0;
  if (const char *e = check_rows(*rows, true)) return fail(fn, e);
  if (!d_old_logp || !d_advantage) return fail(fn, "null old_logp or advantage");
  if (!(cfg->clip_low >= 0.0 && cfg->clip_low <= 1.0) || !(cfg->clip_high >= 0.0 && cfg->clip_high <= 1e30))
    return fail(fn, "clip_low must be between 0 and 1 and clip_high not negative");
  if (!std::isfinite(cfg->kl_coef) || !std::isfinite(cfg->entropy_coef) || !std::isfinite(cfg->scale))
    return fail(fn, "a coefficient is not finite");
  if (!d_ref_logits && (cfg->kl_coef != 0.0f || d_kl))
    return fail(fn, "the KL term needs reference logits");
  if (d_ref_logits)
    if (const char *e = check_matrix(d_ref_logits, ref_stride, ref_type, rows->classes, rows->batch))
      return fail(fn, e);
  if (d_total && !d_loss) return fail(fn, "the total needs the losses");
  if (!d_loss && !d_logp && !d_kl && !d_entropy && !d_grad_logits) return fail(fn, "no output");
  const void *words[] = {d_old_logp, d_advantage, d_weight, d_loss, d_logp, d_kl, d_entropy, d_total};
  for (const void *p : words)
    if (!aligned(p, 4)) return fail(fn, "an array is not aligned to its element type");
  const int n = rows->batch;
  if (d_grad_logits) {
    if (const char *e = check_grad(*rows, d_grad_logits, grad_stride, grad_type)) return fail(fn, e);
    const Range g = matrix(d_grad_logits, grad_stride, grad_type, n, rows->classes);
    bool meets =
        g.meets(matrix(rows->logits, rows->logits_stride, rows->logits_type, n, rows->classes)) ||
        g.meets(array(rows->move_offsets, n + 1LL, 4)) ||
        g.meets(array(rows->move_index, rows->num_moves, 2)) || g.meets(array(rows->played, n, 4));
    if (d_ref_logits) meets = meets || g.meets(matrix(d_ref_logits, ref_stride, ref_type, n, rows->classes));
    for (const void *p : words) meets = meets || g.meets(array(p, p == d_total ? 1 : n, 4));
    if (meets) return fail(fn, "the gradient overlaps another array");
  }
  if (const char *e = check_device(rows->logits)) return fail(fn, e);
  ClipArgs a{};
  a.old_logp = d_old_logp;
  a.advantage = d_advantage;
  a.weight = d_weight;
  a.ref = d_ref_logits;
  a.ref_stride = ref_stride;
  a.ref_type = ref_type;
  a.low = 1.0 - cfg->clip_low;
  a.high = 1.0 + cfg->clip_high;
  a.kl_coef = cfg->kl_coef;
  a.entropy_coef = cfg->entropy_coef;
  a.scale = cfg->scale;
  a.loss = d_loss;
  a.logp = d_logp;
  a.kl = d_kl;
  a.entropy = d_entropy;
  a.grad = Grad{d_grad_logits, grad_stride, grad_type};
  const cudaError_t e = launch_clip(rows_of(*rows), a, s);
  if (e != cudaSuccess || !d_total) return launched(fn, e);
  return launched(fn, launch_total(d_loss, n, d_total, s));
}

extern "C" MFB200_API int mfb200_preference_loss(
    const mfb200_policy_rows *rows, const mfb200_preference_config *cfg,
    const int32_t *d_line_offsets, int pairs, const float *d_ref_logp, const float *d_weight,
    float *d_logp, float *d_logp_rest, float *d_row_grad, float *d_line_logp, float *d_margin,
    float *d_loss, float *d_total, void *d_grad_logits, int64_t grad_stride, int grad_type,
    void *stream) {
  const char *fn = "mfb200_preference_loss";
  if (!rows || !cfg) return fail(fn, "null rows or config");
  if (rows->batch < 0 || pairs < 0) return fail(fn, "negative batch or number of pairs");
  if (pairs > (INT32_MAX - 1) / 2) return fail(fn, "too many pairs");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows->batch > 0)
    if (const char *e = check_rows(*rows, true)) return fail(fn, e);
  if (!std::isfinite(cfg->beta) || !std::isfinite(cfg->scale))
    return fail(fn, "a coefficient is not finite");
  if (!(cfg->label_smoothing >= 0.0f && cfg->label_smoothing <= 1.0f))
    return fail(fn, "label_smoothing must be between 0 and 1");
  if (pairs > 0 && (!d_line_offsets || !d_line_logp || !d_margin || !d_loss))
    return fail(fn, "null line_offsets, line_logp, margin or loss");
  if (rows->batch > 0 && (!d_ref_logp || !d_logp || !d_logp_rest || !d_row_grad))
    return fail(fn, "null ref_logp, logp, logp_rest or row_grad");
  const int n = rows->batch;
  const void *per_row[] = {d_ref_logp, d_logp, d_logp_rest, d_row_grad};
  const void *per_pair[] = {d_weight, d_margin, d_loss};
  for (const void *p : per_row)
    if (!aligned(p, 4)) return fail(fn, "an array is not aligned to its element type");
  for (const void *p : per_pair)
    if (!aligned(p, 4)) return fail(fn, "an array is not aligned to its element type");
  if (!aligned(d_line_offsets, 4) || !aligned(d_line_logp, 4) || !aligned(d_total, 4))
    return fail(fn, "an array is not aligned to its element type");
  if (n > 0 && d_grad_logits) {
    if (const char *e = check_grad(*rows, d_grad_logits, grad_stride, grad_type)) return fail(fn, e);
    const Range g = matrix(d_grad_logits, grad_stride, grad_type, n, rows->classes);
    bool meets =
        g.meets(matrix(rows->logits, rows->logits_stride, rows->logits_type, n, rows->classes)) ||
        g.meets(array(rows->move_offsets, n + 1LL, 4)) ||
        g.meets(array(rows->move_index, rows->num_moves, 2)) || g.meets(array(rows->played, n, 4)) ||
        g.meets(array(d_line_offsets, 2LL * pairs + 1, 4)) ||
        g.meets(array(d_line_logp, 2LL * pairs, 4)) || g.meets(array(d_total, 1, 4));
    for (const void *p : per_row) meets = meets || g.meets(array(p, n, 4));
    for (const void *p : per_pair) meets = meets || g.meets(array(p, pairs, 4));
    if (meets) return fail(fn, "the gradient overlaps another array");
  }
  if (n > 0 || pairs > 0)
    if (const char *e = check_device(n > 0 ? rows->logits : d_line_offsets)) return fail(fn, e);
  const PolicyRows r = rows_of(*rows);
  cudaError_t e = cudaSuccess;
  if (n > 0) e = launch_lines(r, d_logp, d_logp_rest, d_row_grad, s);
  if (e == cudaSuccess && pairs > 0)
    e = launch_pairs(pairs, n, d_line_offsets, d_logp, d_logp_rest, d_ref_logp, d_weight, cfg->beta,
                     cfg->label_smoothing, cfg->scale, d_row_grad, d_line_logp, d_margin, d_loss, s);
  const bool with_grad = n > 0 && d_grad_logits;
  if (e == cudaSuccess && with_grad) {
    BackArgs a{};
    a.played = d_row_grad;
    a.parts_only = true;
    a.out = Grad{d_grad_logits, grad_stride, grad_type};
    if (pairs > 0 && d_total) {
      a.loss = d_loss;
      a.n = pairs;
      a.total = d_total;
    }
    e = launch_backward(r, a, s);
  }
  if (e == cudaSuccess && d_total) {
    if (pairs == 0)
      e = cudaMemsetAsync(d_total, 0, sizeof(float), s);
    else if (!with_grad)
      e = launch_total(d_loss, pairs, d_total, s);
  }
  return launched(fn, e);
}
