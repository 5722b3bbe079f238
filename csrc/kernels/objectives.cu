// Fine-tuning objectives over the language-model head: log-probabilities of tokens, the clipped policy loss with a KL term, the paired
// log-ratio loss.  All three are functions of logp_i = z_it - log sum_j exp(z_ij), z = x w^T, of the tokens that count, and have the gradient
// dz_ij = h_i (1[j = t] - p_ij) with one number h_i = dloss / dlogp_i per token, dx = dz w, dw = dz^T x.
//
// Of a fine-tuning batch only the answers' tokens count, a third to two thirds of it.  So the counted rows are gathered first, in their order
// (rows_count, rows_gather), and the GEMMs behind read from device memory how many there are (Live in gemm_common.cuh): masked tokens cost
// nothing, whatever they hold, and the host does not wait for the number.  Then as for the cross entropy (xent.cu): the head's GEMM leaves
// (max, sum of exponentials) per row and part of the columns, rows_finish makes logp and h of them, and for the gradient a second GEMM
// computes the logits again or, above a width of 512, rows_dlogits takes what the first has kept of them in 16 bits.  Everything per token is
// computed in 64 bits: e^d - d - 1 of two nearly equal log-probabilities and the sums over long answers need it, and there are few tokens.
// Every sum has a fixed order: a call repeats bit for bit.
#include <cuda_fp16.h>
#include "common.cuh"
#include "gemm_common.cuh"
#include "host_utils.h"

namespace cpb {

struct Rows {                // the gathered rows, kept from the forward pass to the backward pass
  int* live;                 // [0] how many, [1] a ticket, [2] 2 x half
  int half;                  // see FEW_ROWS; 0 where there are more
  int* ranges;               // [chunks] into how many ranges of K the product for dx is split
  int* from;                 // [N] gathered row -> row
  int* place;                // [N] row -> gathered row, or -1
  int64_t* targets;          // [N] gathered
  float2* norm;              // [N] gathered: (max, 1 / sum of exponentials)
  float* h;                  // [N] gathered: dloss / dlogp, written by the policy loss
  float* target_p;           // [N] gathered: the target's probability
  __nv_bfloat16* x;          // [N, d] gathered, zero from the last row to the next multiple of 64; [2 x half, d] twice, zero to `half`
  float2* stats;             // [chunks][parts][rows of the chunk] (max, sum of exponentials), or null
  __half* logits;            // [N, V] gathered: distances to the part's max, or null
};

// Up to FEW_ROWS rows the products of the backward pass wait for the weights, not for the tensor core, and dlogits are given to them as a sum of
// two bf16 numbers: `half` rows of rounded ones, and behind them as many of what the rounding has left, to which the gathered rows of x
// stand a second time.  So the gradients of a short call, where no average over many rows makes up for it, are rounded once.  Error of dx and
// dw against 64 bits over that of results rounded once: 136 rows 1.3 to 1.5, now 1.00.
// keep: 0 logits are computed again, 1 kept, 2 kept and dlogits in two parts.
constexpr int FEW_ROWS = 256;
enum : int { KEEP_NONE = 0, KEEP_LOGITS = 1, KEEP_FEW = 2 };
static int half_rows(long N, int keep) { return keep == KEEP_FEW ? (int)((N + 63) / 64 * 64) : 0; }

__device__ __forceinline__ bool row_counts(const int64_t* targets, const float* weights, int row, int n_valid) {
  const int64_t t = targets[row];
  return t >= 0 && t < n_valid && (weights == nullptr || weights[row] != 0.f);
}

// Counted rows of every 32; the rows that do not count have a log-probability of 0.
__global__ void __launch_bounds__(256)
rows_count_kernel(const int64_t* __restrict__ targets, const float* __restrict__ weights, int* __restrict__ counts, float* __restrict__ logp,
                  int* __restrict__ live, int N, int n_valid, int* status) {
  pdl_release();
  pdl_wait();
  const int row = blockIdx.x * 256 + threadIdx.x;
  bool on = false;
  if (row < N) {
    on = row_counts(targets, weights, row, n_valid);
    if (targets[row] >= n_valid) report(status, ST_BAD_INDEX, 1300, (int)targets[row]);
    logp[row] = 0.f;
  }
  const unsigned mask = __ballot_sync(0xffffffffu, on);
  if ((threadIdx.x & 31) == 0 && row < N) counts[row >> 5] = __popc(mask);
  if (row == 0) live[1] = 0;
}

// Into how many ranges of K the product dz w is split: its K is the vocabulary, its tiles are few, and how many there are the host does not
// know.  The time of the pair with the most work, nanoseconds as in gemm.cu: `t64` for 64 of K, and a write and a read of the partial
// results in L2 at 16 TB/s.  4600 of 8192 rows, width 384: planned for 8192 rows 222 us, like this 128.
struct Ranges { int n_blocks, k_blocks, t64, most, pairs, d; };
// A whole warp, a candidate per lane (most <= 32).
__device__ __forceinline__ int ranges_of(const Ranges& q, int rows) {
  const int tiles = (rows + 2 * GEMM_BM - 1) / (2 * GEMM_BM) * q.n_blocks, s = 1 + (threadIdx.x & 31);
  const int each = (q.k_blocks + s - 1) / s;
  float t = 3e38f;
  if (s <= q.most && (q.k_blocks + each - 1) / each == s)          // no range is empty
    t = (float)((tiles * s + q.pairs - 1) / q.pairs) * (float)(each * q.t64) + (float)s * (200.f + (float)rows * (float)q.d * (8.f / 16000.f));
  int at = s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t2 = __shfl_xor_sync(0xffffffffu, t, o);
    const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
    if (t2 < t || (t2 == t && at2 < at)) { t = t2; at = at2; }
  }
  return t < 3e38f ? at : 1;
}

// Gathers 32 rows per block: x[b, t] has strides sb and st.  Bound by memory, 2 d bytes in and out per row.  COUNT: every block counts the
// rows in front of its own by itself and there is no rows_count, up to COUNT_ROWS rows; eight rows per block, one for each warp: 136 rows of
// 768 11 us for both kernels, 8 for this one.
constexpr int COUNT_ROWS = 4096;
constexpr int gather_rows(bool count) { return count ? 8 : 32; }
template <bool COUNT>
__global__ void __launch_bounds__(256)
rows_gather_kernel(const __nv_bfloat16* __restrict__ x, long sb, long st, int T, int d, const int64_t* __restrict__ targets,
                   const float* __restrict__ weights, const int* __restrict__ counts, float* __restrict__ logp, Rows r, Ranges q, int chunk, int N, int n_valid,
                   int* status) {
  pdl_release();
  pdl_wait();
  constexpr int EACH = gather_rows(COUNT);
  __shared__ int part[8], s_base, s_n, s_from[EACH];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = blockIdx.x;
  int before = 0;
  if (COUNT) {
    for (int i = threadIdx.x; i < group * EACH; i += 256) before += row_counts(targets, weights, i, n_valid);
  } else {
    for (int i = threadIdx.x; i < group; i += 256) before += counts[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) part[warp] = before;
  __syncthreads();
  if (warp == 0) {
    int base = 0;
    for (int i = 0; i < 8; ++i) base += part[i];
    const int row = lane < EACH ? group * EACH + lane : N;
    const bool on = row < N && row_counts(targets, weights, row, n_valid);
    const unsigned mask = __ballot_sync(0xffffffffu, on);
    const int rank = __popc(mask & ((1u << lane) - 1u));
    if (on) {
      s_from[rank] = row;
      r.from[base + rank] = row;
      r.targets[base + rank] = targets[row];
    }
    if (row < N) r.place[row] = on ? base + rank : -1;
    if (COUNT && row < N) {
      logp[row] = 0.f;
      if (targets[row] >= n_valid) report(status, ST_BAD_INDEX, 1300, (int)targets[row]);
    }
    if (lane == 0) { s_base = base; s_n = __popc(mask); }
    if (group == (int)gridDim.x - 1) {
      const int live = base + __popc(mask);
      if (lane == 0) { r.live[0] = live; r.live[2] = 2 * r.half; if (COUNT) r.live[1] = 0; }
      for (int c = 0; c * chunk < N; ++c) {
        const int s = ranges_of(q, r.half ? 2 * r.half : max(0, min(chunk, live - c * chunk)));
        if (lane == 0) r.ranges[c] = s;
      }
    }
  }
  __syncthreads();
  const int nvec = d >> 3;
  for (int i = warp; i < s_n; i += 8) {
    const int row = s_from[i], b = row / T;
    const uint4* src = (const uint4*)(x + b * sb + (row - b * T) * st);
    uint4* dst = (uint4*)(r.x + (size_t)(s_base + i) * d);
    for (int c = lane; c < nvec; c += 128) {
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) if (c + 32 * k < nvec) v[k] = src[c + 32 * k];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (c + 32 * k >= nvec) continue;
        dst[c + 32 * k] = v[k];
        if (r.half) dst[(size_t)r.half * nvec + c + 32 * k] = v[k];
      }
    }
  }
  if (group == (int)gridDim.x - 1) {                               // K of the weight gradient is taken 64 rows at a time
    const int total = s_base + s_n, end = r.half ? r.half : min(N, (total + 63) & ~63);
    for (int i = total + warp; i < end; i += 8)
      for (int c = lane; c < nvec; c += 32) {
        ((uint4*)(r.x + (size_t)i * d))[c] = make_uint4(0, 0, 0, 0);
        if (r.half) ((uint4*)(r.x + (size_t)(r.half + i) * d))[c] = make_uint4(0, 0, 0, 0);
      }
  }
}

struct Policy {
  const float *old_logp, *advantages, *weights, *ref_logp;         // [N] by row; weights and ref_logp may be null
  double low, high, kl;                                            // the ratio is clipped to [low, high]
  double* part;                                                    // [blocks][4]
  float *loss, *terms;                                             // [1], and [4] sums of weight x (surrogate, KL, clipped, 1)
};

// The tensor core cuts off what an accumulator has no bits for after every 16 of K, so a logit comes out too small in size: half a last place a
// step, for a sum that grows evenly K 2^-30 of it.  Measured at logits above 8 (spread 4, 50304 and 128256 columns), relative: K 384
// -3.4e-7, 768 -7.0e-7, 2048 -1.97e-6, 4096 -4.05e-6; this factor takes it back.  A sum that has its size early is off by
// up to twice that, one that gets it late by next to nothing, so it is nowhere further off with the factor than without.
// `l2e` is it times log2 e, rounded to fp32, and `all` what that comes to: a target's logit has to take the same as the exponentials, or
// log-probabilities are up to 2e-7 off on average.
struct LogitScale { float l2e; double all; };
static LogitScale logit_scale(int d) {
  const float l2e = (float)((1. + (double)d / 1073741824.) * 1.4426950408889634);
  return LogitScale{l2e, (double)l2e * 0.6931471805599453};
}

// Between the two passes of the head's GEMM: logp and (max, 1 / sum) of 32 gathered rows per block, and for a policy loss its terms and h.
// A warp takes every sixteenth part of the columns (the lanes' pairs are adjacent in memory), warp 0 adds the warps', always in the same order.
// A target's logit is the tensor core's, like those in the sum: computed exactly, logp deviates a third as much from token to token (K 4096
// 3e-6 for 1e-5), but what the factor above does not meet then stays in every one of them (2.4e-6 there), and sums over answers are worse.
// ex2.approx is 4.8e-8 too low on average where it is not exact, as it is for the maximum itself: the sum gets that back (logp 1e-7 too high on
// average without, 1e-8 to 5e-8 with it).
constexpr int RF_WARPS = 16;
constexpr double EX2_LOW = 4.8e-8;
template <bool POLICY>
__global__ void __launch_bounds__(RF_WARPS * 32)
rows_finish_kernel(const float2* __restrict__ stats, const float* __restrict__ target_logit, Rows r, float* __restrict__ logp, int before, int rows,
                   int tiles, LogitScale scale, Policy q, int blocks_before, int blocks) {
  pdl_release();
  pdl_wait();
  __shared__ double2 part[RF_WARPS][32];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;                          // in this launch
  const int at = before + row;                                     // gathered
  const bool on = row < rows && at < r.live[0];
  float m = -INFINITY;
  double s = 0.;
  // a part without a finite maximum contributes its sum as it is: zero, or NaN
  const auto below = [&](float v, float top) { return v == top || v == -INFINITY ? 1. : (1. + EX2_LOW) * (double)ex2f((v - top) * scale.l2e); };
  const auto given = [&](float2 v, float top) { return v.x == -INFINITY ? (double)v.y : ((double)v.y + EX2_LOW * ((double)v.y - 1.)) * below(v.x, top); };
  if (on) {
    int t = warp;
    for (; t + 7 * RF_WARPS < tiles; t += 8 * RF_WARPS) {
      float2 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = stats[(size_t)(t + k * RF_WARPS) * rows + row];
      float top = m;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, v[k].x);
      s *= below(m, top);
#pragma unroll
      for (int k = 0; k < 8; ++k) s += given(v[k], top);
      m = top;
    }
    for (; t < tiles; t += RF_WARPS) {
      const float2 v = stats[(size_t)t * rows + row];
      const float top = fmaxf(m, v.x);
      s = s * below(m, top) + given(v, top);
      m = top;
    }
  }
  part[warp][lane] = make_double2((double)m, s);
  __syncthreads();
  if (warp == 0) {
    float top = m;
#pragma unroll
    for (int k = 1; k < RF_WARPS; ++k) top = fmaxf(top, (float)part[k][lane].x);
    s *= below(m, top);
#pragma unroll
    for (int k = 1; k < RF_WARPS; ++k) s += part[k][lane].y * below((float)part[k][lane].x, top);
    m = top;
    double sur = 0., kl = 0., cut = 0., wt = 0.;
    if (on) {
      const double lp = scale.all * ((double)target_logit[row] - (double)m) - log(s);
      r.norm[at] = make_float2(m, (float)(1. / s));
      r.target_p[at] = (float)exp(lp);
      const int from = r.from[at];
      logp[from] = (float)lp;
      if (POLICY) {
        const double a = q.advantages[from], ratio = exp(lp - (double)q.old_logp[from]);
        wt = q.weights ? (double)q.weights[from] : 1.;
        const bool c = (a > 0. && ratio > q.high) || (a < 0. && ratio < q.low);
        // an advantage of nothing has no surrogate, however far the ratio is
        sur = a == 0. ? 0. : -a * (c ? (a > 0. ? q.high : q.low) : ratio);
        double h = a == 0. || c ? 0. : sur;                        // d(-a r) / dlogp = -a r
        if (q.ref_logp) {
          const double delta = (double)q.ref_logp[from] - lp, e = expm1(delta);
          kl = e - delta;
          if (q.kl != 0.) h -= q.kl * e;
        }
        r.h[at] = (float)(wt * h);
        sur *= wt; kl *= wt; cut = c ? wt : 0.;
      }
    }
    if (POLICY) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        sur += __shfl_xor_sync(0xffffffffu, sur, o); kl += __shfl_xor_sync(0xffffffffu, kl, o);
        cut += __shfl_xor_sync(0xffffffffu, cut, o); wt += __shfl_xor_sync(0xffffffffu, wt, o);
      }
      if (lane == 0) {
        double* out = q.part + 4 * (size_t)(blocks_before + blockIdx.x);
        out[0] = sur; out[1] = kl; out[2] = cut; out[3] = wt;
        __threadfence();
        s_last = atomicAdd(r.live + 1, 1) == blocks - 1;           // of all launches of the call
      }
    }
  }
  if (!POLICY) return;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  // the last block adds all parts: thread by thread, then the threads in order
  __shared__ double total[RF_WARPS][4];
  double v[4] = {0., 0., 0., 0.};
  for (int i = threadIdx.x; i < blocks; i += RF_WARPS * 32)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += __ldcg(q.part + 4 * (size_t)i + k);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if (lane == 0)
    for (int k = 0; k < 4; ++k) total[warp][k] = v[k];
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < RF_WARPS; ++w)
    for (int k = 0; k < 4; ++k) total[0][k] += total[w][k];
  *q.loss = (float)(q.kl != 0. ? total[0][0] + q.kl * total[0][1] : total[0][0]);
  for (int k = 0; k < 4; ++k) q.terms[k] = (float)total[0][k];
}

// Sums of 256 threads in a fixed order; thread 0 has the result.
__device__ __forceinline__ double block_sum(double v, double* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 1; i < 8; ++i) v += scratch[i];
  return v;
}

// sums[b][s] = sum over the s-th part of sequence b of logp - ref, of the tokens that count.
__global__ void __launch_bounds__(256)
sequence_sums_kernel(const float* __restrict__ logp, const float* __restrict__ ref, const int64_t* __restrict__ targets, double* __restrict__ sums,
                     int T, int part, int n_valid) {
  pdl_release();
  pdl_wait();
  __shared__ double scratch[8];
  const int b = blockIdx.y, t0 = blockIdx.x * part, t1 = min(T, t0 + part);
  double v = 0.;
  for (int t = t0 + threadIdx.x; t < t1; t += 256) {
    const size_t i = (size_t)b * T + t;
    if (targets[i] >= 0 && targets[i] < n_valid) v += (double)logp[i] - (double)ref[i];
  }
  v = block_sum(v, scratch);
  if (threadIdx.x == 0) sums[(size_t)b * gridDim.x + blockIdx.x] = v;
}

// Pairs (i, pairs + i): the loss, the log-ratio of every sequence and dloss / dlogp of its tokens, behind the last the largest size of one.
__global__ void __launch_bounds__(256)
preference_kernel(const double* __restrict__ sums, int parts, int pairs, const float* __restrict__ weights, double beta, double smoothing,
                  float* __restrict__ loss, float* __restrict__ ratios, float* __restrict__ h) {
  pdl_release();
  pdl_wait();
  __shared__ double scratch[8];
  __shared__ float top[8];
  double l = 0.;
  float most = 0.f;
  for (int i = threadIdx.x; i < pairs; i += 256) {
    double c = 0., r = 0.;
    for (int k = 0; k < parts; ++k) {
      c += sums[(size_t)i * parts + k];
      r += sums[(size_t)(pairs + i) * parts + k];
    }
    ratios[i] = (float)c; ratios[pairs + i] = (float)r;
    const double wt = weights ? (double)weights[i] : 1.;
    double g = 0.;
    if (wt != 0.) {
      // softplus(-z) = max(-z, 0) + log1p(e^-|z|); its derivative -sigma(-z)
      const double z = beta * (c - r), e = exp(-fabs(z)), small = log1p(e), pos = 1. / (1. + e), neg = e / (1. + e);
      const double up = z > 0. ? pos : z <= 0. ? neg : z, down = z > 0. ? neg : z <= 0. ? pos : z;      // sigma(z), sigma(-z); NaN stays
      // a side that counts nothing is left out, infinite or not
      l += wt * ((smoothing < 1. ? (1. - smoothing) * (fmax(-z, 0.) + small) : 0.) + (smoothing > 0. ? smoothing * (fmax(z, 0.) + small) : 0.));
      g = wt * beta * (smoothing * up - (1. - smoothing) * down);
    }
    h[i] = (float)g; h[pairs + i] = (float)-g;
    most = fmaxf(most, fabsf((float)g));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = most;
  l = block_sum(l, scratch);                                       // with a barrier
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 8; ++i) most = fmaxf(most, top[i]);
  *loss = (float)l;
  h[2 * pairs] = most;
}

// The tokens of an answer all have the same dloss / dlogp, and bf16 of it may be off by 2^-8 in all of them at once.  So a gradient whose largest h
// is known is taken at 2^e in the place of g h, a number that bf16 holds and below which (1 - p) loses least, and the products are multiplied
// with m, g h = m 2^e.  Error of dx and dw of one pair against 64 bits: 1.27 to 1.64 times that of results rounded once without, 1.22 to 1.29 with it.
struct Even { const float* most; float* back; };                   // the largest |h|, or null; where m goes
__device__ __forceinline__ float even_factor(const Even& q, const float* __restrict__ g, float& back) {
  back = 1.f;
  if (q.most == nullptr) return 1.f;
  const float v = fabsf(*q.most * (g ? *g : 1.f));
  if (!(v > 0.f && v < INFINITY)) return 1.f;
  int e;
  back = frexpf(v, &e);
  return 1.f / back;
}

// scale = -g dloss/dlogp of the gathered rows, 0 behind the last: what xent.cu calls grad_scale, row by row.  h is by gathered row (each ==
// 0) or by row / each.
__device__ __forceinline__ float row_scale(const Rows& r, const float* __restrict__ h, int each, const float* __restrict__ g, int i) {
  const float v = -(each == 0 ? h[i] : h[r.from[i] / each]);
  return g ? v * *g : v;
}
__global__ void __launch_bounds__(256)
rows_scale_kernel(Rows r, const float* __restrict__ h, int each, const float* __restrict__ g, Even even, float* __restrict__ scale, int N) {
  pdl_release();
  pdl_wait();
  const int i = blockIdx.x * 256 + threadIdx.x;
  float back;
  const float factor = even_factor(even, g, back);
  if (i == 0) *even.back = back;
  if (i < N) scale[i] = i < r.live[0] ? row_scale(r, h, each, g, i) * factor : 0.f;
}

// dlogits of gathered rows from what was kept of the logits.  Bound by memory: 2 bytes in and 2 out per logit; four 16-byte loads per
// thread before the first use.  Rows behind the last one are zero up to the next multiple of 64, see Live.
constexpr int RD_COLS = 256 * 32;
__global__ void __launch_bounds__(256)
rows_dlogits_kernel(Rows r, const float* __restrict__ h, int each, const float* __restrict__ g, Even even, int before, int rows, __nv_bfloat16* __restrict__ dlogits, int n_valid, int V, float l2e) {
  pdl_release();
  pdl_wait();
  const int row = blockIdx.y, at = before + row, live = r.live[0];
  float back;
  const float factor = even_factor(even, g, back);
  if (at == 0 && blockIdx.x == 0 && threadIdx.x == 0) *even.back = back;
  if (at >= (r.half ? r.half : (live + 63) & ~63)) return;
  const float s = at < live ? row_scale(r, h, each, g, at) * factor : 0.f;
  const bool on = s != 0.f;                                        // a row of gradient 0 is zero, whatever its logits are
  const int c0 = blockIdx.x * RD_COLS + 8 * threadIdx.x;
  uint4 v[4];
  float f[4];
  const float2* stats = r.stats + (size_t)((V + 255) / 256) * before + row;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = c0 + 2048 * k;
    v[k] = make_uint4(0, 0, 0, 0);
    f[k] = 0.f;
    if (on && c < V) {
      v[k] = *(const uint4*)(r.logits + (size_t)at * V + c);
      f[k] = stats[(size_t)(c >> 8) * rows].x;
    }
  }
  float top = 0.f, inv = 0.f;
  int tgt = -1;
  if (on) { top = r.norm[at].x; inv = r.norm[at].y * s; tgt = (int)r.targets[at]; }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = c0 + 2048 * k;
    if (c >= V) break;
    const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
    const float far = f[k] == -INFINITY ? 0.f : ex2f((f[k] - top) * l2e) * inv;      // a tile of nothing but -inf
    float p[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 d2 = __half22float2(*(const __half2*)&u[e]);
      p[2 * e] = ex2f(d2.x * l2e) * far;
      p[2 * e + 1] = ex2f(d2.y * l2e) * far;
    }
    if (!on || c + 8 > n_valid) {
#pragma unroll
      for (int e = 0; e < 8; ++e) if (!on || c + e >= n_valid) p[e] = 0.f;
    }
    if (tgt >= c && tgt < c + 8) {
      const float one = s * (r.target_p[at] - 1.f);
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = tgt == c + e ? one : p[e];
    }
    const uint4 out = make_uint4(pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]), pack_bf16(p[4], p[5]), pack_bf16(p[6], p[7]));
    *(uint4*)(dlogits + (size_t)row * V + c) = out;
    if (r.half) {
      const uint32_t o[4] = {out.x, out.y, out.z, out.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) { p[2 * e] -= bf16_lo(o[e]); p[2 * e + 1] -= bf16_hi(o[e]); }
      *(uint4*)(dlogits + (size_t)(r.half + row) * V + c) = make_uint4(pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]), pack_bf16(p[4], p[5]), pack_bf16(p[6], p[7]));
    }
  }
}

// dx of the rows of one chunk: the gathered row's, the sum of its parts in their order; with the first chunk the rows that do not count, 0.
// Four columns per thread and eight parts on their way, bound by the parts' way through L2.
__global__ void __launch_bounds__(256)
rows_scatter_kernel(const float* __restrict__ parts, const int* __restrict__ ranges, const int* __restrict__ place, __nv_bfloat16* __restrict__ out,
                    int N, int d, int before, int rows, int half, size_t total) {
  pdl_release();
  pdl_wait();
  const int nvec = d >> 2, count = *ranges, all = half ? 2 * count : count;        // few rows: the rounded rows' parts, then the others'
  const size_t step = (size_t)rows * nvec, low = (size_t)half * nvec;
  for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const int row = (int)(i / nvec), c = (int)(i - (size_t)row * nvec), to = place[row], at = to - before;
    if (to < 0 ? before > 0 : at < 0 || at >= rows) continue;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (to >= 0) {
      const float4* src = (const float4*)parts + (size_t)at * nvec + c;
      for (int s = 0; s < all; s += 8) {
        float4 u[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          u[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (s + k < all) u[k] = s + k < count ? src[(s + k) * step] : src[(s + k - count) * step + low];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) { a.x += u[k].x; a.y += u[k].y; a.z += u[k].z; a.w += u[k].w; }
      }
    }
    *(uint2*)(out + (size_t)row * d + 4 * c) = make_uint2(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w));
  }
}

// fp32 gradient of the weights, added up over chunks of rows, as bf16
__global__ void __launch_bounds__(256)
weight_cast_kernel(const float4* __restrict__ in, uint4* __restrict__ out, size_t n8) {
  pdl_release();
  pdl_wait();
  for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < n8; i += (size_t)gridDim.x * 256) {
    const float4 a = in[2 * i], b = in[2 * i + 1];
    out[i] = make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
  }
}

// ------------------------------------------------------------------ layout of the buffers
static size_t take(size_t& at, size_t bytes) {
  const size_t here = at;
  at = (at + bytes + 255) & ~(size_t)255;
  return here;
}
// `base` may be null: the size alone
static Rows rows_layout(char* base, long N, int d, long V, int chunk, int keep, size_t& bytes) {
  size_t at = 0;
  Rows r;
  r.half = half_rows(N, keep);
  r.live = (int*)(base + take(at, 256));
  r.ranges = (int*)(base + take(at, (N / chunk + 1) * 4));
  r.from = (int*)(base + take(at, N * 4));
  r.place = (int*)(base + take(at, N * 4));
  r.targets = (int64_t*)(base + take(at, N * 8));
  r.norm = (float2*)(base + take(at, N * 8));
  r.h = (float*)(base + take(at, N * 4));
  r.target_p = (float*)(base + take(at, N * 4));
  r.x = (__nv_bfloat16*)(base + take(at, (size_t)(r.half ? 2 * r.half : N) * d * 2));
  r.stats = keep ? (float2*)(base + take(at, (size_t)((V + 255) / 256) * N * 8)) : nullptr;
  r.logits = keep ? (__half*)(base + take(at, (size_t)N * V * 2)) : nullptr;
  bytes = at;
  return r;
}
// What the forward pass alone needs stands behind the rows, in the same buffer: it is small, and an allocation costs the host 3 us.
struct FwdScratch { int* counts; float2* stats; float* target_logit; double* part; };
static FwdScratch fwd_layout(char* base, long N, int d, long V, int chunk, int keep, size_t& bytes) {
  size_t at = bytes;
  const long rows = N < chunk ? N : chunk, parts = (V + 255) / 256 * head_parts(d);
  FwdScratch s;
  s.counts = (int*)(base + take(at, (N + 31) / 32 * 4));
  s.stats = (float2*)(base + take(at, keep ? 0 : (size_t)parts * rows * 8));
  s.target_logit = (float*)(base + take(at, rows * 4));
  s.part = (double*)(base + take(at, ((N + 31) / 32 + N / chunk + 1) * 32));
  bytes = at;
  return s;
}
// Where dw goes: nowhere, added to an fp32 buffer, or as bf16 (through an fp32 buffer where there are several chunks of rows).
enum : int { DW_NONE = 0, DW_ADD = 1, DW_BF16 = 2 };
// Tiles of the product dz w: the width that covers d in the least time.  At most 512 MB of partial results, or one of them.
static Ranges dx_ranges(int rows, int d, int V) {
  Ranges q{};
  long best = 0;
  for (const int bn : {256, 192, 128}) {
    const int n = (d + bn - 1) / bn, t64 = bn == 256 ? 370 : bn == 192 ? 300 : 240;
    if (best == 0 || (long)n * t64 < best) { best = (long)n * t64; q.n_blocks = n; q.t64 = t64; }
  }
  q.k_blocks = (V + GEMM_BK - 1) / GEMM_BK;
  const long most = (128L << 20) / ((long)rows * d);
  q.most = (int)(most < 1 ? 1 : most > 32 ? 32 : most);
  q.pairs = sm_count() > 1 ? sm_count() / 2 : 1;
  q.d = d;
  return q;
}
struct BwdScratch { float *scale, *back; __nv_bfloat16* dlogits; float *dx, *dw, *partials; };
static BwdScratch bwd_layout(char* base, long N, int d, long V, int chunk, int keep, int dw, int want_dx, size_t& bytes) {
  size_t at = 0;
  const int half = half_rows(N, keep);
  const long rows = half ? 2 * half : N < chunk ? N : chunk;
  const bool one = N <= chunk;
  BwdScratch s;
  s.scale = (float*)(base + take(at, N * 4));
  s.back = (float*)(base + take(at, 4));
  s.dlogits = (__nv_bfloat16*)(base + take(at, (size_t)rows * V * 2));
  s.dw = (float*)(base + take(at, dw == DW_BF16 && !one ? (size_t)V * d * 4 : 0));
  size_t parts = 0, most = 0;
  for (long r0 = 0; r0 < N; r0 += chunk) {                         // the last chunk has a plan of its own
    const long n = half ? 2 * half : N - r0 < chunk ? N - r0 : chunk;
    if (r0 > 0 && n == chunk) continue;
    if (want_dx) {
      const size_t m = (size_t)dx_ranges((int)n, d, (int)V).most * n * d;
      if (m > parts) parts = m;
    }
    if (dw != DW_NONE) {
      const int epi = dw == DW_BF16 && one ? EPI_BF16 : EPI_F32_ACC, k = gemm_splits((int)V, d, (int)n, epi);
      const size_t m = (size_t)(epi == EPI_BF16 ? k : k - 1) * V * d;
      if (k > 1 && m > most) most = m;
    }
  }
  s.dx = (float*)(base + take(at, parts * 4));
  s.partials = (float*)(base + take(at, most * 4));
  bytes = at;
  return s;
}

}  // namespace cpb

using namespace cpb;

// Bytes of the buffers of an objective over N rows of width d and V columns: kept between the passes, and of the backward pass.
extern "C" int cpb_objective_plan(int N, int d, int V, int chunk, int keep, int dw, int want_dx, int64_t* bytes) {
  if (keep == KEEP_FEW && N > FEW_ROWS) return set_error(CPB_ERR_ARG, "objective: %d rows are not few", N);
  if (N <= 0 || d <= 0 || V <= 0 || chunk <= 0 || chunk % 256) return set_error(CPB_ERR_ARG, "objective: %d rows of %d, %d columns, chunks of %d", N, d, V, chunk);
  size_t kept, bwd;
  rows_layout(nullptr, N, d, V, chunk, keep, kept);
  fwd_layout(nullptr, N, d, V, chunk, keep, kept);
  bwd_layout(nullptr, N, d, V, chunk, keep, dw, want_dx, bwd);
  bytes[0] = (int64_t)kept; bytes[1] = (int64_t)bwd;
  return CPB_OK;
}

static int objective_args(int N, int d, int V, int n_valid, int ldw, int chunk, int keep) {
  if (keep < KEEP_NONE || keep > KEEP_FEW || (keep == KEEP_FEW && N > FEW_ROWS)) return set_error(CPB_ERR_ARG, "objective: %d rows kept as %d", N, keep);
  if (N <= 0 || d <= 0 || V <= 0) return set_error(CPB_ERR_ARG, "objective: empty problem, %d rows of %d, %d columns", N, d, V);
  if ((d % 8) || (V % 8) || (ldw % 8)) return set_error(CPB_ERR_ARG, "objective: widths and row strides must be multiples of 8 (got d=%d V=%d ldw=%d)", d, V, ldw);
  if (n_valid <= 0 || n_valid > V) return set_error(CPB_ERR_ARG, "objective: n_valid=%d outside 1..%d", n_valid, V);
  if (chunk <= 0 || chunk % 256 || chunk > 65280) return set_error(CPB_ERR_ARG, "objective: chunks of %d rows", chunk);
  return CPB_OK;
}

// x bf16 [B, T, d] (strides sb, st, rows 16-byte aligned), w bf16 [V, d], targets [B, T]; a row counts where 0 <= target < n_valid and, with
// `weights`, its weight is not 0.  logp [B, T].  With `advantages`, the policy loss: old_logp, advantages, weights, ref_logp [B, T] (the
// last two may be null), loss [1] and terms [4], see Policy.  kept: cpb_objective_plan.
extern "C" int cpb_objective_fwd(const void* x, long sb, long st, int N, int T, int d, const void* w, int ldw, int V, int n_valid, const int64_t* targets,
                                 const float* old_logp, const float* advantages, const float* weights, const float* ref_logp, double low, double high,
                                 double kl, float* logp, float* loss, float* terms, void* kept, int keep, int chunk, int* status, cudaStream_t stream) {
  int rc = objective_args(N, d, V, n_valid, ldw, chunk, keep);
  if (rc != CPB_OK) return rc;
  if (T <= 0 || N % T || (sb % 8) || (st % 8) || ((uintptr_t)x & 15)) return set_error(CPB_ERR_ARG, "objective: hidden states need 16-byte aligned rows");
  size_t bytes;
  const Rows r = rows_layout((char*)kept, N, d, V, chunk, keep, bytes);
  const FwdScratch s = fwd_layout((char*)kept, N, d, V, chunk, keep, bytes);
  const int tiles = (V + 255) / 256 * (keep ? 1 : head_parts(d));
  const bool count = N <= COUNT_ROWS;
  if (!count) CPB_CUDA_OK(launch_pdl(rows_count_kernel, (N + 255) / 256, 256, 0, stream, targets, weights, s.counts, logp, r.live, N, n_valid, status));
  const int groups = (N + gather_rows(count) - 1) / gather_rows(count);
  auto gather = count ? rows_gather_kernel<true> : rows_gather_kernel<false>;
  CPB_CUDA_OK(launch_pdl(gather, groups, 256, 0, stream, (const __nv_bfloat16*)x, sb, st, T, d, targets, weights, s.counts, logp, r, dx_ranges(r.half ? 2 * r.half : N < chunk ? N : chunk, d, V),
                         chunk, N, n_valid, status));
  int blocks = 0;
  for (int r0 = 0; r0 < N; r0 += chunk) blocks += ((N - r0 < chunk ? N - r0 : chunk) + 31) / 32;
  const LogitScale scale = logit_scale(d);
  const Policy q{old_logp, advantages, weights, ref_logp, low, high, kl, s.part, loss, terms};
  for (int r0 = 0, done = 0; r0 < N; r0 += chunk) {
    const int n = N - r0 < chunk ? N - r0 : chunk;
    float2* stats = keep ? r.stats + (size_t)tiles * r0 : s.stats;
    const HeadParams head{r.targets + r0, stats, s.target_logit, nullptr, n_valid, 0.f, nullptr, scale.l2e};
    if ((rc = gemm_head_live(r.x + (size_t)r0 * d, w, keep ? r.logits + (size_t)r0 * V : nullptr, n, V, d, d, ldw, V, keep ? 2 : 0, head, Live{r.live, r0, 0, nullptr}, status, stream)) != CPB_OK) return rc;
    auto kern = advantages ? rows_finish_kernel<true> : rows_finish_kernel<false>;
    CPB_CUDA_OK(launch_pdl(kern, (n + 31) / 32, RF_WARPS * 32, 0, stream, stats, s.target_logit, r, logp, r0, n, tiles, scale, q, done, blocks));
    done += (n + 31) / 32;
  }
  return check_launch("objective_fwd");
}

// sums fp64 [2 pairs][parts] of logp - ref over the counted tokens of every sequence of T tokens, part by part.
static int sequence_sums(const float* logp, const float* ref, const int64_t* targets, double* sums, int seqs, int T, int parts, int n_valid,
                         cudaStream_t stream) {
  if (seqs <= 0 || T <= 0 || parts <= 0 || seqs > 65535) return set_error(CPB_ERR_ARG, "sequence_sums: %d sequences of %d in %d parts", seqs, T, parts);
  CPB_CUDA_OK(launch_pdl(sequence_sums_kernel, dim3(parts, seqs), 256, 0, stream, logp, ref, targets, sums, T, (T + parts - 1) / parts, n_valid));
  return check_launch("sequence_sums");
}
extern "C" int cpb_sequence_sums(const float* logp, const float* ref, const int64_t* targets, double* sums, int seqs, int T, int parts, int n_valid,
                                 cudaStream_t stream) {
  return sequence_sums(logp, ref, targets, sums, seqs, T, parts, n_valid, stream);
}

// loss [1], ratios [2 pairs] and h [2 pairs + 1] from the sums, which with `logp` are taken first; weights [pairs] or null.
extern "C" int cpb_preference(const float* logp, const float* ref, const int64_t* targets, int T, int n_valid, double* sums, int parts, int pairs,
                              const float* weights, double beta, double smoothing, float* loss, float* ratios, float* h, cudaStream_t stream) {
  if (logp != nullptr) {
    const int rc = sequence_sums(logp, ref, targets, sums, 2 * pairs, T, parts, n_valid, stream);
    if (rc != CPB_OK) return rc;
  }
  if (pairs <= 0 || parts <= 0) return set_error(CPB_ERR_ARG, "preference: %d pairs in %d parts", pairs, parts);
  CPB_CUDA_OK(launch_pdl(preference_kernel, 1, 256, 0, stream, sums, parts, pairs, weights, beta, smoothing, loss, ratios, h));
  return check_launch("preference");
}

// Gradients: h is dloss / dlogp of row i at h[i / each] (h null: the policy loss's, as the forward pass has left it), most the largest size of
// one or null, g a factor in device memory or null.  dx bf16 [N, d] or null.  dw: DW_ADD fp32 [V, d], added to; DW_BF16 bf16 [V, d].
extern "C" int cpb_objective_bwd(int N, int d, const void* w, int ldw, int V, int n_valid, const float* h, int each, const float* most, const float* g, void* dx, void* dw,
                                 int dw_kind, const void* kept, int keep, void* scratch, int chunk, int* status, cudaStream_t stream) {
  int rc = objective_args(N, d, V, n_valid, ldw, chunk, keep);
  if (rc != CPB_OK) return rc;
  if ((h != nullptr && each <= 0) || dw_kind < DW_NONE || dw_kind > DW_BF16 || (dw_kind != DW_NONE && dw == nullptr))
    return set_error(CPB_ERR_ARG, "objective: gradients of %d rows each, weights' gradient of kind %d", each, dw_kind);
  size_t bytes;
  const Rows r = rows_layout((char*)kept, N, d, V, chunk, keep, bytes);
  const BwdScratch s = bwd_layout((char*)scratch, N, d, V, chunk, keep, dw_kind, dx != nullptr, bytes);
  const bool one = N <= chunk;
  const float l2e = logit_scale(d).l2e;
  const Ranges q = dx_ranges(r.half ? 2 * r.half : one ? N : chunk, d, V);
  if (h == nullptr) { h = r.h; each = 0; }
  const Even even{most, s.back};
  const float* back = most ? s.back : nullptr;
  if (!keep) CPB_CUDA_OK(launch_pdl(rows_scale_kernel, (N + 255) / 256, 256, 0, stream, r, h, each, g, even, s.scale, N));
  for (int r0 = 0, c = 0; r0 < N; r0 += chunk, ++c) {
    const int n = N - r0 < chunk ? N - r0 : chunk, m = r.half ? 2 * r.half : n;        // rows of x, of dlogits
    const int* live = r.half ? r.live + 2 : r.live;
    if (keep) {
      CPB_CUDA_OK(launch_pdl(rows_dlogits_kernel, dim3((V + RD_COLS - 1) / RD_COLS, r.half ? r.half : n), 256, 0, stream, r, h, each, g, even, r0, n, s.dlogits, n_valid, V, l2e));
    } else {
      const HeadParams head{r.targets + r0, nullptr, nullptr, r.norm + r0, n_valid, 0.f, s.scale + r0, l2e};
      if ((rc = gemm_head_live(r.x + (size_t)r0 * d, w, s.dlogits, n, V, d, d, ldw, V, 1, head, Live{r.live, r0, 0, nullptr}, status, stream)) != CPB_OK) return rc;
    }
    if (dx != nullptr) {
      const int bn = q.t64 == 370 ? 256 : q.t64 == 300 ? 192 : 128;
      if ((rc = gemm_live_parts(s.dlogits, w, s.dx, m, d, V, ldw, bn, q.most, back, Live{live, r0, 0, r.ranges + c}, status, stream)) != CPB_OK) return rc;
      const size_t total = (size_t)N * (d / 4), blocks = (total + 255) / 256, cap = (size_t)sm_count() * 8;
      CPB_CUDA_OK(launch_pdl(rows_scatter_kernel, (unsigned)(blocks < cap ? blocks : cap), 256, 0, stream, s.dx, r.ranges + c, r.place, (__nv_bfloat16*)dx, N, d, r0, m, r.half, total));
    }
    if (dw_kind != DW_NONE) {
      const bool direct = dw_kind == DW_BF16 && one;
      const int epi = direct ? EPI_BF16 : dw_kind == DW_BF16 && r0 == 0 ? EPI_F32 : EPI_F32_ACC;
      GemmLive p{s.dlogits, r.x + (size_t)r0 * d, dw_kind == DW_BF16 && !one ? (void*)s.dw : dw, V, d, m, V, d, d, 1, 1, epi, back, s.partials,
                 epi == EPI_F32 ? 1 : gemm_splits(V, d, m, epi)};
      if ((rc = gemm_live(p, Live{live, r0, 1, nullptr}, status, stream)) != CPB_OK) return rc;
    }
  }
  if (dw_kind == DW_BF16 && !one) {
    const size_t n8 = (size_t)V * d / 8, blocks = (n8 + 255) / 256, cap = (size_t)sm_count() * 8;
    CPB_CUDA_OK(launch_pdl(weight_cast_kernel, (unsigned)(blocks < cap ? blocks : cap), 256, 0, stream, (const float4*)s.dw, (uint4*)dw, n8));
  }
  return check_launch("objective_bwd");
}
