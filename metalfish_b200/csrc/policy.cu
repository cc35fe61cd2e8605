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
// (19 sectors for the 31 moves of an average position) in three dependent
// steps (offsets, indices, logits), so they are bound by load latency until
// the sectors' bandwidth. The gradient operators are bound by writing the
// whole row (1858 x 4 bytes), 8 times what they read.
//
// One warp per position: a lane holds up to eight moves in registers, the
// sums are shuffles in a fixed order (results do not depend on timing), and
// nothing goes through shared memory but the test for repeated indices. The
// zeros of a gradient row are stored first, as 16-byte pieces, so that they
// drain while the warp waits for its three loads; the ~30 values follow after
// a __syncwarp and meet the zeros in L2.
#include "policy.cuh"

#include <cmath>
#include <cstdio>

#include "../../include/mfb200.h"
#include "pdl.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mfb200 {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kMaxMoves = 256;  // moves of a position that count, as in priors_kernel
constexpr int kPerLane = kMaxMoves / 32;
constexpr int kMaxWarps = 8;  // positions per CTA

// One iteration for each group of 32 moves that the position has; n is the
// same in every lane, so the groups past it are skipped by the whole warp.
// Inputs are read with ordinary loads, never as read-only (__ldg, __restrict__
// const): a kernel here may start before the one that writes its inputs has
// ended (pdl.cuh), and a read-only load may be moved above pdl_wait.
#define FOR_GROUPS(k, n) _Pragma("unroll") for (int k = 0; k < kPerLane; ++k) if (32 * k < (n))

__device__ __forceinline__ float load_as_float(const void *base, int type, long long i) {
  if (type == MFB200_TYPE_F32) return static_cast<const float *>(base)[i];
  const unsigned short u = static_cast<const unsigned short *>(base)[i];
  return type == MFB200_TYPE_BF16 ? __uint_as_float(static_cast<unsigned>(u) << 16)
                                  : __half2float(__ushort_as_half(u));
}

// One rounding, to nearest even, of the fp32 value to the gradient's type.
__device__ __forceinline__ void store_as(void *base, int type, long long i, float v) {
  if (type == MFB200_TYPE_F32)
    static_cast<float *>(base)[i] = v;
  else if (type == MFB200_TYPE_BF16)
    static_cast<__nv_bfloat16 *>(base)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half *>(base)[i] = __float2half_rn(v);
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
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// A position's legal moves, spread over the warp: move 32 k + lane.
struct Moves {
  int n;        // moves that count (<= 256)
  int count;    // moves listed
  long long lo; // first entry of the list
  int played;   // edge number, -1 for none
  bool bad;     // offsets or played move out of range
  int col[kPerLane];  // column, -1 for none (the logit is then 0, without a gradient)
};

// What a list is read with. Loaded first; the zeros of a gradient row are
// stored between this and the list itself, while these loads are under way.
struct ListHead {
  int base, lo, hi, played;
};
__device__ __forceinline__ ListHead load_head(const PolicyRows &r, int b) {
  return {r.off[0], r.off[b], r.off[b + 1], r.played ? r.played[b] : -1};
}

// The list itself. No entry outside [0, num_moves) is read.
__device__ __forceinline__ Moves load_moves(const PolicyRows &r, const ListHead &head, int lane) {
  Moves m;
  const long long lo = static_cast<long long>(head.lo) - head.base;
  const long long hi = static_cast<long long>(head.hi) - head.base;
  m.bad = lo < 0 || hi < lo || hi > r.num_moves;
  m.count = m.bad ? 0 : static_cast<int>(hi - lo);
  m.n = m.count < kMaxMoves ? m.count : kMaxMoves;
  m.lo = lo;
  // a position with an empty list has no played move, whatever it is given
  m.bad = m.bad || head.played < -1 || (m.count > 0 && head.played >= m.n);
  m.played = m.bad || m.count == 0 ? -1 : head.played;
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) m.col[k] = -1;
  FOR_GROUPS(k, m.n) {
    const int j = 32 * k + lane;
    if (j < m.n) {
      const int c = r.index[m.lo + j];
      m.col[k] = c >= 0 && c < r.classes ? c : -1;
    }
  }
  return m;
}

// Softmax statistics of a row over its list. The largest entry is kept out of
// the sum (S = 1 + rest), so that log S and 1 - p of a nearly certain move
// keep their digits.
struct Norm {
  float top;    // largest logit
  float rest;   // sum of exp(s - s_top) over the other moves
  float log_s, inv_s;
  int lead;     // lowest edge with the largest logit
  bool live;    // some move has a logit above -inf (or NaN)
};

// z[k]: the logits of the lane's moves. On return e[k] = exp(s - s_top).
__device__ __forceinline__ Norm normalise(const Moves &m, const float (&z)[kPerLane],
                                          float inv_temp, int lane, float (&e)[kPerLane]) {
  Norm q;
  float top = -INFINITY;
  bool some = false;
  FOR_GROUPS(k, m.n) {
    if (32 * k + lane < m.n) {
      top = fmaxf(top, z[k]);
      some |= !(z[k] == -INFINITY);
    }
  }
  q.top = warp_max(top);
  q.live = __any_sync(kFull, some);
  q.lead = -1;
  float rest = 0.0f;
  FOR_GROUPS(k, m.n) {
    const bool mine = 32 * k + lane < m.n;
    const unsigned at = __ballot_sync(kFull, mine && z[k] == q.top);
    if (q.lead < 0 && at) q.lead = 32 * k + __ffs(at) - 1;
    e[k] = mine ? expf((z[k] - q.top) * inv_temp) : 0.0f;
    if (32 * k + lane != q.lead) rest += e[k];
  }
  // the largest entry's own inf - inf is not in the sum
  q.rest = q.top == INFINITY ? __int_as_float(0x7FC00000) : warp_sum(rest);
  q.log_s = log1pf(q.rest);
  q.inv_s = 1.0f / (1.0f + q.rest);
  return q;
}

__device__ __forceinline__ void load_logits(const PolicyRows &r, const Moves &m, const void *base,
                                            long long stride, int type, int b,
                                            float (&z)[kPerLane]) {
  const long long row = static_cast<long long>(b) * stride;
  FOR_GROUPS(k, m.n) z[k] = m.col[k] >= 0 ? load_as_float(base, type, row + m.col[k]) : 0.0f;
}

// The value that move j's lane holds in group v[j / 32].
__device__ __forceinline__ float of_move(const float (&v)[kPerLane], int n, int j) {
  float got = 0.0f;
  FOR_GROUPS(k, n) {
    const float t = __shfl_sync(kFull, v[k], j & 31);
    if (j >> 5 == k) got = t;
  }
  return got;
}

struct Grad {
  void *base;  // null: no gradient
  long long stride;
  int type;
};

// The row's bytes, all the same element: 16-byte stores between the first and
// last 16-byte boundary, single elements around them.
__device__ __forceinline__ void fill_row(const Grad &g, int classes, int b, int lane,
                                         unsigned word) {
  const int size = g.type == MFB200_TYPE_F32 ? 4 : 2;
  char *p = static_cast<char *>(g.base) + static_cast<long long>(b) * g.stride * size;
  const int bytes = classes * size;
  int head = static_cast<int>((16 - (reinterpret_cast<unsigned long long>(p) & 15)) & 15);
  if (head > bytes) head = bytes;
  const int body = (bytes - head) >> 4;
  const int tail = head + (body << 4);
  uint4 v = make_uint4(word, word, word, word);
  uint4 *q = reinterpret_cast<uint4 *>(p + head);
  for (int i = lane; i < body; i += 32) q[i] = v;
  const int around = (head + bytes - tail) / size;
  if (lane < around) {
    const int at = lane * size < head ? lane * size : tail + lane * size - head;
    if (size == 4)
      *reinterpret_cast<unsigned *>(p + at) = word;
    else
      *reinterpret_cast<unsigned short *>(p + at) = static_cast<unsigned short>(word);
  }
}

__device__ __forceinline__ unsigned nan_word(int type) {
  return type == MFB200_TYPE_F32 ? 0x7FC00000u : type == MFB200_TYPE_BF16 ? 0x7FC07FC0u : 0x7E007E00u;
}

// Writes g[k] to the columns of the list, over the zeros that fill_row wrote.
// A column that is listed more than once gets the sum of its values, in the
// list's order. `seen`: one bit per column, shared memory of this warp.
__device__ __forceinline__ void scatter_row(const Grad &out, const Moves &m, int classes, int b,
                                            int lane, const float (&g)[kPerLane], unsigned *seen) {
  const long long row = static_cast<long long>(b) * out.stride;
  const int words = (classes + 31) >> 5;
  for (int i = lane; i < words; i += 32) seen[i] = 0u;
  __syncwarp();
  bool again = false;
  FOR_GROUPS(k, m.n) {
    if (m.col[k] >= 0) {
      const unsigned bit = 1u << (m.col[k] & 31);
      again |= (atomicOr(seen + (m.col[k] >> 5), bit) & bit) != 0u;
    }
  }
  if (!__any_sync(kFull, again)) {
    FOR_GROUPS(k, m.n) if (m.col[k] >= 0) store_as(out.base, out.type, row + m.col[k], g[k]);
    return;
  }
  float sum[kPerLane];
  bool first[kPerLane];
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) sum[k] = 0.0f, first[k] = true;
  FOR_GROUPS(k2, m.n) {
    for (int src = 0; src < 32 && 32 * k2 + src < m.n; ++src) {
      const int c = __shfl_sync(kFull, m.col[k2], src);
      const float v = __shfl_sync(kFull, g[k2], src);
      FOR_GROUPS(k, m.n) {
        if (m.col[k] == c) {
          sum[k] += v;
          if (32 * k2 + src < 32 * k + lane) first[k] = false;
        }
      }
    }
  }
  FOR_GROUPS(k, m.n)
  if (m.col[k] >= 0 && first[k]) store_as(out.base, out.type, row + m.col[k], sum[k]);
}

__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7FC00000); }

// ------------------------------------------------------------------ log-probabilities
__global__ void __launch_bounds__(32 * kMaxWarps)
    move_logprobs_kernel(PolicyRows r, float *move_logp,
                         float *played_logp, float *entropy,
                         float *row_state) {
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31;
  const unsigned at_row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (at_row >= static_cast<unsigned>(r.batch)) return;
  const int b = static_cast<int>(at_row);
  const Moves m = load_moves(r, load_head(r, b), lane);
  float z[kPerLane], e[kPerLane];
  load_logits(r, m, r.logits, r.stride, r.type, b, z);
  const Norm q = normalise(m, z, r.inv_temp, lane, e);
  float h = 0.0f;
  FOR_GROUPS(k, m.n) {
    const int j = 32 * k + lane;
    if (j < m.n) {
      const float logp = q.live ? (z[k] - q.top) * r.inv_temp - q.log_s : -INFINITY;
      const float p = e[k] * q.inv_s;
      if (p != 0.0f) h -= p * logp;  // 0 log 0 = 0; NaN passes
      if (move_logp) move_logp[m.lo + j] = logp;
    }
  }
  if (move_logp)
    for (int j = m.n + lane; j < m.count; j += 32) move_logp[m.lo + j] = -INFINITY;
  h = warp_sum(h);
  const bool takes = q.live && m.played >= 0;
  const float at = (of_move(z, m.n, m.played < 0 ? 0 : m.played) - q.top) * r.inv_temp - q.log_s;
  if (lane == 0) {
    if (played_logp) played_logp[b] = m.bad ? quiet_nan() : takes ? at : 0.0f;
    if (entropy) entropy[b] = m.bad ? quiet_nan() : q.live ? h : 0.0f;
    if (row_state) row_state[b] = takes || m.bad ? 0.0f : -0.0f;
  }
}

// dL/dlogit_c = (1/T) [ G_c + [c = a] g - p_c (sum G + g) - g_H p_c (logp_c + H) ]
// for upstream gradients G of the moves' log-probabilities, g of the played
// move's and g_H of the entropy, each of which may be null.
__global__ void __launch_bounds__(32 * kMaxWarps)
    move_logprobs_backward_kernel(PolicyRows r, const float *grad_moves,
                                  const float *grad_played,
                                  const float *grad_entropy, Grad out) {
  extern __shared__ unsigned seen_all[];
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned at_row = blockIdx.x * (blockDim.x >> 5) + warp;
  if (at_row >= static_cast<unsigned>(r.batch)) return;
  const int b = static_cast<int>(at_row);
  const ListHead head = load_head(r, b);
  fill_row(out, r.classes, b, lane, 0u);
  const Moves m = load_moves(r, head, lane);
  if (m.bad) {
    __syncwarp();
    fill_row(out, r.classes, b, lane, nan_word(out.type));
    return;
  }
  float z[kPerLane], e[kPerLane], g[kPerLane];
  load_logits(r, m, r.logits, r.stride, r.type, b, z);
  float total = 0.0f;
  FOR_GROUPS(k, m.n) {
    const int j = 32 * k + lane;
    g[k] = grad_moves && j < m.n ? grad_moves[m.lo + j] : 0.0f;
    total += g[k];
  }
  const float ga = grad_played && m.played >= 0 ? grad_played[b] : 0.0f;
  const float gh = grad_entropy ? grad_entropy[b] : 0.0f;
  const Norm q = normalise(m, z, r.inv_temp, lane, e);
  if (!q.live) return;
  total = warp_sum(total);
  float h = 0.0f;
  if (grad_entropy) {
    FOR_GROUPS(k, m.n) {
      const float p = e[k] * q.inv_s;
      if (p != 0.0f) h -= p * ((z[k] - q.top) * r.inv_temp - q.log_s);
    }
    h = warp_sum(h);
  }
  FOR_GROUPS(k, m.n) {
    const int j = 32 * k + lane;
    const float p = e[k] * q.inv_s;
    float v = g[k] - p * total;
    // ([c = a] - p_c) g; 1 - p of the largest entry is rest / S
    v += ga * (j != m.played ? -p : j == q.lead ? q.rest * q.inv_s : 1.0f - p);
    if (grad_entropy && p != 0.0f)
      v -= gh * p * ((z[k] - q.top) * r.inv_temp - q.log_s + h);
    g[k] = v * r.inv_temp;
  }
  scatter_row(out, m, r.classes, b, lane, g, seen_all + warp * ((r.classes + 31) >> 5));
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

// e^-d - 1 + d, the contribution of a move to KL = sum p (e^-d - 1 + d) with
// d = log p - log q (sum p e^-d = sum q = 1). Every term is >= 0 and an error
// common to all d cancels, so the KL of two near policies keeps its digits.
// Taylor series for |d| < 1, where the exponential would cancel.
__device__ __forceinline__ float kl_term(float d) {
  float t = 1.0f;
#pragma unroll
  for (int i = 13; i >= 3; --i) t = 1.0f - d * (1.0f / i) * t;
  return 0.5f * d * d * t;
}

__global__ void __launch_bounds__(32 * kMaxWarps)
    clipped_policy_loss_kernel(PolicyRows r, ClipArgs a) {
  extern __shared__ unsigned seen_all[];
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned at_row = blockIdx.x * (blockDim.x >> 5) + warp;
  if (at_row >= static_cast<unsigned>(r.batch)) return;
  const int b = static_cast<int>(at_row);
  const ListHead head = load_head(r, b);
  const float old = a.old_logp[b], adv = a.advantage[b];
  const float c0 = a.scale * (a.weight ? a.weight[b] : 1.0f);
  if (a.grad.base) fill_row(a.grad, r.classes, b, lane, 0u);
  const Moves m = load_moves(r, head, lane);
  float z[kPerLane], e[kPerLane], zr[kPerLane], d[kPerLane];
  load_logits(r, m, r.logits, r.stride, r.type, b, z);
  if (a.ref) load_logits(r, m, a.ref, a.ref_stride, a.ref_type, b, zr);
  const Norm q = normalise(m, z, r.inv_temp, lane, e);
  const bool takes = q.live && m.played >= 0;

  float h = 0.0f;
  FOR_GROUPS(k, m.n) {
    const float p = e[k] * q.inv_s;
    if (p != 0.0f) h -= p * ((z[k] - q.top) * r.inv_temp - q.log_s);
  }
  h = q.live ? warp_sum(h) : 0.0f;
  float kl = 0.0f;
  if (a.ref) {
    const Norm w = normalise(m, zr, r.inv_temp, lane, d);  // d: exp(s - s_top) of the reference
    FOR_GROUPS(k, m.n) {
      const float p = e[k] * q.inv_s, pr = d[k] * w.inv_s;
      // d = log p - log q: the near logits are subtracted first
      d[k] = ((z[k] - zr[k]) - (q.top - w.top)) * r.inv_temp + (w.log_s - q.log_s);
      if (32 * k + lane < m.n)
        kl += p == 0.0f ? pr : fabsf(d[k]) < 1.0f ? p * kl_term(d[k]) : pr - p + p * d[k];
    }
    kl = q.live ? warp_sum(kl) : 0.0f;
  }

  const float sa = (of_move(z, m.n, m.played < 0 ? 0 : m.played) - q.top) * r.inv_temp;
  const float ratio = expf((sa - old) - q.log_s);
  // The gradient jumps where the ratio crosses the clip's border, so a ratio
  // within the rounding of the border is computed again in 64 bits.
  const float border = static_cast<float>(adv > 0.0f ? a.high : a.low);
  bool active = adv > 0.0f ? !(ratio > border) : !(ratio < border);
  if (takes && fabsf(ratio - border) <= border * (2e-6f + 1e-6f * (fabsf(sa) + q.log_s + fabsf(old)))) {
    double sum = 0.0;
    FOR_GROUPS(k, m.n)
    if (32 * k + lane < m.n)
      sum += exp((static_cast<double>(z[k]) - q.top) / r.temp);
    sum = warp_sum(sum);
    const double za = of_move(z, m.n, m.played);
    const double exact = exp((za - q.top) / r.temp - log(sum) - static_cast<double>(old));
    active = adv > 0.0f ? !(exact > a.high) : !(exact < a.low);
  }
  if (lane == 0) {
    const float bad = quiet_nan();
    float loss = -adv * (active ? ratio : border);
    if (a.ref) loss += a.kl_coef * kl;
    loss -= a.entropy_coef * h;
    if (a.loss) a.loss[b] = m.bad ? bad : takes ? c0 * loss : 0.0f;
    if (a.logp) a.logp[b] = m.bad ? bad : takes ? sa - q.log_s : 0.0f;
    if (a.kl) a.kl[b] = m.bad ? bad : kl;
    if (a.entropy) a.entropy[b] = m.bad ? bad : h;
  }
  if (!a.grad.base) return;
  if (m.bad) {
    __syncwarp();
    fill_row(a.grad, r.classes, b, lane, nan_word(a.grad.type));
    return;
  }
  if (!takes) return;
  const float c = c0 * r.inv_temp;
  const float slope = active ? -adv * ratio : 0.0f;
  float g[kPerLane];
  FOR_GROUPS(k, m.n) {
    const int j = 32 * k + lane;
    const float p = e[k] * q.inv_s;
    float v = slope * (j != m.played ? -p : j == q.lead ? q.rest * q.inv_s : 1.0f - p);
    if (p != 0.0f) {
      if (a.ref) v += a.kl_coef * p * (d[k] - kl);
      v += a.entropy_coef * p * ((z[k] - q.top) * r.inv_temp - q.log_s + h);
    }
    g[k] = c * v;
  }
  scatter_row(a.grad, m, r.classes, b, lane, g, seen_all + warp * ((r.classes + 31) >> 5));
}

// ------------------------------------------------------------------ preference loss
// One warp per pair of lines. With D = the sum over a line's rows of
// (logp - ref) and m = beta (D_preferred - D_rejected):
//     L = scale w ( -(1 - eps) log sigma(m) - eps log sigma(-m) ),
// and dL/dlogp of a row is +-beta dL/dm, written over the row's state (+0: the
// row takes part; -0: it does not, its reference value is left out). Rows in no
// line keep a zero. The sums run in 64 bits, in an order fixed by the rows.
__global__ void __launch_bounds__(256)
    preference_pair_kernel(int pairs, int batch, const int32_t *lines,
                           const float *logp, const float *ref,
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
  double sum[2] = {0.0, 0.0}, gain[2] = {0.0, 0.0};
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    for (int b = at[side] + lane; b < at[side + 1]; b += 32) {
      if (signbit(row_grad[b])) continue;
      const double lp = logp[b];
      sum[side] += lp;
      gain[side] += lp - static_cast<double>(ref[b]);
    }
    sum[side] = warp_sum(sum[side]);
    gain[side] = warp_sum(gain[side]);
  }
  const float mg = static_cast<float>(static_cast<double>(beta) * (gain[0] - gain[1]));
  const float w = scale * (weight ? weight[i] : 1.0f);
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
    loss[i] = mg != mg ? mg : w * ((1.0f - eps) * less + eps * more);
  }
#pragma unroll
  for (int side = 0; side < 2; ++side)
    for (int b = at[side] + lane; b < at[side + 1]; b += 32)
      row_grad[b] = signbit(row_grad[b]) ? 0.0f : side ? -slope : slope;
}

// ------------------------------------------------------------------ total
// The sum of the losses, in 64 bits and in one order.
__global__ void __launch_bounds__(1024)
    loss_total_kernel(const float *loss, int n, float *total) {
  __shared__ double part[32];
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) v += loss[i];
  v = warp_sum(v);
  if (lane == 0) part[warp] = v;
  __syncthreads();
  if (warp == 0) {
    v = lane < static_cast<int>(blockDim.x >> 5) ? part[lane] : 0.0;
    v = warp_sum(v);
    if (lane == 0) *total = static_cast<float>(v);
  }
}

// ------------------------------------------------------------------ launches
// Warps (positions) per CTA: one while the positions fit one per SM, so that
// each has an SM's load units to itself, up to eight.
int warps_for(int batch) {
  int w = 1;
  while (w < kMaxWarps && batch > 148 * w) w *= 2;
  return w;
}

size_t seen_bytes(const PolicyRows &r, int warps) {
  return static_cast<size_t>(warps) * ((r.classes + 31) / 32) * sizeof(unsigned);
}

cudaError_t launch_backward(const PolicyRows &r, const float *grad_moves, const float *grad_played,
                            const float *grad_entropy, const Grad &g, cudaStream_t s) {
  const int w = warps_for(r.batch);
  return launch_k(move_logprobs_backward_kernel, dim3((r.batch + w - 1) / w), dim3(32 * w),
                  seen_bytes(r, w), s, 1, r, grad_moves, grad_played, grad_entropy, g);
}

cudaError_t launch_total(const float *loss, int n, float *total, cudaStream_t s) {
  const int threads = n >= 1024 ? 1024 : (n + 31) / 32 * 32;
  return launch_k(loss_total_kernel, dim3(1), dim3(threads ? threads : 32), 0, s, 1, loss, n, total);
}

}  // namespace

cudaError_t launch_move_logprobs(const PolicyRows &r, float *move_logp, float *played_logp,
                                 float *entropy, float *row_state, cudaStream_t s) {
  const int w = warps_for(r.batch);
  return launch_k(move_logprobs_kernel, dim3((r.batch + w - 1) / w), dim3(32 * w), 0, s, 1, r,
                  move_logp, played_logp, entropy, row_state);
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

// Byte range of a [batch, classes] matrix whose rows are `stride` elements apart.
struct Range {
  uintptr_t lo, hi;
  bool meets(const Range &o) const { return lo < o.hi && o.lo < hi; }
};
Range matrix(const void *p, long long stride, int type, int batch, int classes) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  return {lo, lo + (static_cast<uintptr_t>(batch - 1) * stride + classes) * type_size(type)};
}
Range array(const void *p, long long n, int size) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  return {lo, p ? lo + static_cast<uintptr_t>(n) * size : lo};
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
    return "the logits are not a device pointer";
  }
  if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
    return "the logits are not in device memory";
  if (at.type == cudaMemoryTypeDevice && at.device != dev)
    return "the logits are on another device than the current one";
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
  o.inv_temp = static_cast<float>(1.0 / r.softmax_temp);
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
                                           nullptr, static_cast<cudaStream_t>(stream)));
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
  return launched(fn, launch_backward(rows_of(*rows), d_grad_moves, d_grad_played, d_grad_entropy,
                                      Grad{d_grad_logits, grad_stride, grad_type},
                                      static_cast<cudaStream_t>(stream)));
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
  const PolicyRows r = rows_of(*rows);
  const int w = warps_for(n);
  const cudaError_t e = launch_k(clipped_policy_loss_kernel, dim3((n + w - 1) / w), dim3(32 * w),
                                 seen_bytes(r, w), s, 1, r, a);
  if (e != cudaSuccess || !d_total) return launched(fn, e);
  return launched(fn, launch_total(d_loss, n, d_total, s));
}

extern "C" MFB200_API int mfb200_preference_loss(
    const mfb200_policy_rows *rows, const mfb200_preference_config *cfg,
    const int32_t *d_line_offsets, int pairs, const float *d_ref_logp, const float *d_weight,
    float *d_logp, float *d_row_grad, float *d_line_logp, float *d_margin, float *d_loss,
    float *d_total, void *d_grad_logits, int64_t grad_stride, int grad_type, void *stream) {
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
  if (rows->batch > 0 && (!d_ref_logp || !d_logp || !d_row_grad))
    return fail(fn, "null ref_logp, logp or row_grad");
  const int n = rows->batch;
  const void *per_row[] = {d_ref_logp, d_logp, d_row_grad};
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
  if (n > 0)
    if (const char *e = check_device(rows->logits)) return fail(fn, e);
  const PolicyRows r = rows_of(*rows);
  cudaError_t e = cudaSuccess;
  if (n > 0) e = launch_move_logprobs(r, nullptr, d_logp, nullptr, d_row_grad, s);
  if (e == cudaSuccess && pairs > 0) {
    const int w = warps_for(pairs);
    e = launch_k(preference_pair_kernel, dim3((pairs + w - 1) / w), dim3(32 * w), 0, s, 1, pairs, n,
                 d_line_offsets, static_cast<const float *>(d_logp), d_ref_logp, d_weight, cfg->beta,
                 cfg->label_smoothing, cfg->scale, d_row_grad, d_line_logp, d_margin, d_loss);
  }
  if (e == cudaSuccess && n > 0 && d_grad_logits)
    e = launch_backward(r, nullptr, d_row_grad, nullptr, Grad{d_grad_logits, grad_stride, grad_type}, s);
  if (e == cudaSuccess && d_total) {
    if (pairs > 0)
      e = launch_total(d_loss, pairs, d_total, s);
    else
      e = cudaMemsetAsync(d_total, 0, sizeof(float), s);
  }
  return launched(fn, e);
}
