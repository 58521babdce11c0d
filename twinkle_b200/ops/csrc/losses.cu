// Losses of a policy step on per-token log-probabilities, forward and backward: the clipped policy loss with its KL and entropy terms, and losses on pairs of rows.
//
// What bounds them: launches for a micro-batch (torch takes 20 to 40), memory for a batch: 16 to 32 bytes read per token, the labels 8 of them, and 4
// written.  A forward pass reads every input once: a row is summed by a cluster of up to 8 CTAs, a second launch of one CTA joins the rows.  The policy
// loss writes each token's derivative without the row's weight, which is known only when all rows are; its backward pass reads that one number
// per token.  Paired losses have one derivative per row: their backward pass reads the labels.
//
// Measured, us on the device: 64 x 4095 tokens with reference, entropies and advantages per token 5.9 + 2.5 (joining) and 3.6 (backward); sequence ratios of 256 x 16384 27 (84 MB read, 17 written:
// 3.7 TB/s) and 7.1; 512 x 8192 pairs 14 (67 MB: 4.8 TB/s) and 8.4.  A token's inputs behind a branch on its label made each batch of loads wait for the one before (53 and 28 us); with every
// thread of a cluster reading the others' sums those reads took longer than the tokens (95 and 40).  On the host a step with its gradient takes 85 to 110 us, 50 of them torch's engine.  Exact
// exponentials and quotients cost nothing here (5.9 and 27 us as with fast ones, whose results were two to three times as far from 64 bits).
//
// Precision: per token in fp32, sums over tokens and rows in fp64 (a loss is a small difference of sums of advantages).  Differences of log-probs are formed in fp64 and compared
// with the logarithms of the bounds, so that a token at a bound falls on the right side; e^d − 1 and e^d − d − 1 of small d come from a series.  The file is compiled
// without fast math.
// Masked tokens are not read into any sum: infinities and NaN there have no effect.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>
#include <torch/types.h>

#include <cmath>

#include "common.cuh"
#include "host.h"
#include "vec.cuh"

namespace tk {

namespace ls {
constexpr int THREADS = 256, UNROLL = 4, HOLD = 32, CTAS = 4;      // tokens of a batch, tokens whose terms a thread keeps, CTAs of an SM
}

// e^x − 1 and, without cancellation, e^x − 1 − x.  Where |x| ≤ 1 the latter is its series up to x^11 (the next term is below 2^-27 of the sum), three and a half roundings; beyond, the
// difference costs at most a rounding of e^x − 1 over a third of it: both are within 2^-21.5, and the former stays finite where x is −∞.
struct Exp {
  float less_one, rest;
};
__device__ __forceinline__ Exp exp_parts(float x) {
  if (!(fabsf(x) <= 1.f)) {
    const float e = expm1f(x);
    return {e, e - x};
  }
  float r = 1.f / 39916800.f;
  r = fmaf(r, x, 1.f / 3628800.f);
  r = fmaf(r, x, 1.f / 362880.f);
  r = fmaf(r, x, 1.f / 40320.f);
  r = fmaf(r, x, 1.f / 5040.f);
  r = fmaf(r, x, 1.f / 720.f);
  r = fmaf(r, x, 1.f / 120.f);
  r = fmaf(r, x, 1.f / 24.f);
  r = fmaf(r, x, 1.f / 6.f);
  r = fmaf(r, x, 0.5f);
  r *= x * x;
  return {r + x, r};
}

// Which tokens count: labels other than `ignore`, or a mask of bytes (ignore: 0).
struct Tokens {
  const void* p;
  long ld;
  int64_t ignore;
  bool bytes;
  // What stands at U tokens, `step` apart; those from S on read the last one.  Loads only, without a branch between them: nothing waits for the first before the last is asked for.
  template <int U>
  __device__ __forceinline__ void load(int64_t (&x)[U], long b, int t0, int step, int S) const {
    if (bytes) {
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = reinterpret_cast<const uint8_t*>(p)[b * ld + min(t0 + u * step, S - 1)];
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = reinterpret_cast<const int64_t*>(p)[b * ld + min(t0 + u * step, S - 1)];
    }
  }
};
// A row per sequence with unit stride, or (one) a number per row; null: none.
struct Rows {
  const float* p;
  long ld;
  bool one;
  template <int U>
  __device__ __forceinline__ void load(float (&x)[U], long b, int t0, int step, int S) const {
    if (p == nullptr) return;
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = p[b * ld + (one ? 0 : min(t0 + u * step, S - 1))];
  }
};

// Sums of N numbers over the threads of a cluster; every thread gets them.  `sh`: [warps + 2][N] of shared memory, which a second call may use again.
template <int N>
__device__ __forceinline__ void cluster_sums(double (&x)[N], double (*sh)[N], int ctas) {
  namespace cg = cooperative_groups;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int WARPS = ls::THREADS / 32;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
  __syncthreads();
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) sh[warp][i] = x[i];
  __syncthreads();
  if (threadIdx.x < N) {
    double s = 0.0;
    for (int w = 0; w < WARPS; ++w) s += sh[w][threadIdx.x];
    sh[WARPS][threadIdx.x] = s;
  }
  if (ctas > 1) {
    const cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (threadIdx.x < N) {          // a thread per number: from every thread these reads cost more than the tokens
      double s = 0.0;
#pragma unroll
      for (int r = 0; r < 8; ++r) s += r < ctas ? cluster.map_shared_rank(&sh[WARPS][0], r)[threadIdx.x] : 0.0;
      sh[WARPS + 1][threadIdx.x] = s;
    }
    cluster.sync();                 // nobody leaves, and nothing is overwritten, while it is read
  } else {
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = sh[ctas > 1 ? WARPS + 1 : WARPS][i];
}

// ---------------------------------------------------------------- policy loss
enum { RATIO_TOKEN = 0, RATIO_SEQUENCE = 1 };
enum { CLIP = 0, SOFT = 1, WEIGHT = 2 };
enum { REDUCE_SEQUENCE = 0, REDUCE_TOKEN = 1, REDUCE_SUM = 2 };

struct Policy {
  Tokens tokens;
  Rows logps, old, ref, ent, adv;      // old null: the log-probs themselves
  float* deriv;                        // [B, S] derivative by the log-prob without the row's weight
  double* sums;                        // [B, 5] loss, tokens, KL to the old policy, tokens below and above the bounds
  int B, S;
  float lo, hi, beta, entropy, tau_pos, tau_neg, top;      // bounds of the ratio; WEIGHT: largest ratio
  double log_lo, log_hi, log_top;
};

struct Ratio {
  float r, r1, rest;      // ratio, ratio − 1, ratio − 1 − its logarithm
  bool below, above, over;
};
__device__ __forceinline__ Ratio ratio_of(const Policy& p, double l) {
  Ratio x;
  const float lr = static_cast<float>(l);
  const Exp e = exp_parts(lr);
  x.r = expf(lr);
  x.r1 = e.less_one;
  x.rest = e.rest;
  x.below = l < p.log_lo;
  x.above = l > p.log_hi;
  x.over = l > p.log_top;
  return x;
}
// Loss of a token and its derivatives by the logarithm of the ratio and, directly, by the log-prob.
template <int KIND>
__device__ __forceinline__ void surrogate(const Policy& p, const Ratio& x, float a, float logp, float& f, float& by_ratio, float& by_logp) {
  by_logp = 0.f;
  if constexpr (KIND == CLIP) {
    const float bounded = x.below ? p.lo : x.above ? p.hi : x.r;
    const bool bound = a >= 0.f ? x.above : x.below;         // the other bound is never the smaller product
    f = -(bound ? bounded : x.r) * a;
    by_ratio = bound ? 0.f : -x.r * a;
  } else if constexpr (KIND == SOFT) {
    const float tau = a > 0.f ? p.tau_pos : p.tau_neg;
    const float z = tau * x.r1, e = expf(-fabsf(z)), high = 1.f / (1.f + e), low = e * high;      // the gate and what it leaves of one, neither by a difference
    f = -(z >= 0.f ? high : low) * 4.f / tau * a;
    by_ratio = -4.f * high * low * x.r * a;
  } else {
    const float w = (x.over ? p.top : x.r) * a;
    f = -w * logp;
    by_ratio = 0.f;
    by_logp = -w;
  }
}

// Inputs of a thread's next tokens, all asked for before the first is used.
template <int U>
struct Batch {
  float logp[U], old[U], ref[U], ent[U], adv[U];
  bool on[U];
  __device__ __forceinline__ void load(const Policy& p, long b, int t0, int step) {
    int64_t label[U];
    p.tokens.load(label, b, t0, step, p.S);
    p.logps.load(logp, b, t0, step, p.S);
    p.old.load(old, b, t0, step, p.S);
    p.ref.load(ref, b, t0, step, p.S);
    p.ent.load(ent, b, t0, step, p.S);
    p.adv.load(adv, b, t0, step, p.S);
    if (p.old.p == nullptr) {
#pragma unroll
      for (int u = 0; u < U; ++u) old[u] = logp[u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) on[u] = t0 + u * step < p.S && label[u] != p.tokens.ignore;
  }
  __device__ __forceinline__ double log_ratio(int u, bool& inside) const {
    const double d = static_cast<double>(logp[u]) - static_cast<double>(old[u]);
    inside = d >= -20.0 && d <= 20.0;
    return d < -20.0 ? -20.0 : d > 20.0 ? 20.0 : d;
  }
  // terms that do not come from the ratio: their loss, and the derivative by the log-prob
  __device__ __forceinline__ void others(const Policy& p, int u, float& f, float& by_logp) const {
    if (p.ref.p != nullptr) {
      const float d = static_cast<float>(static_cast<double>(ref[u]) - static_cast<double>(logp[u]));
      const Exp e = exp_parts(d);
      f += p.beta * e.rest;
      by_logp -= p.beta * e.less_one;
    }
    if (p.ent.p != nullptr) f -= p.entropy * ent[u];
  }
};

__device__ __forceinline__ void put_sums(const Policy& p, long b, const double (&s)[5]) {
  if (blockIdx.x == 0 && threadIdx.x < 5) {
    double v = s[0];
#pragma unroll
    for (int i = 1; i < 5; ++i) v = threadIdx.x == i ? s[i] : v;
    p.sums[b * 5 + threadIdx.x] = v;
  }
}

// Ratios of tokens; one row per cluster.
template <int KIND>
__global__ void __launch_bounds__(ls::THREADS, ls::CTAS) policy_token_kernel(const Policy p) {
  using namespace ls;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ double sh[THREADS / 32 + 2][5];
  const int ctas = gridDim.x, step = ctas * THREADS;
  const long b = blockIdx.y;
  double loss = 0.0, kl = 0.0;
  int n = 0, below = 0, above = 0;
  for (int t0 = blockIdx.x * THREADS + threadIdx.x; t0 < p.S; t0 += step * UNROLL) {
    Batch<UNROLL> x;
    x.load(p, b, t0, step);
    float f4 = 0.f, kl4 = 0.f;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float g = 0.f;
      if (x.on[u]) {
        bool inside;
        const Ratio r = ratio_of(p, x.log_ratio(u, inside));
        float f, by_ratio, by_logp;
        surrogate<KIND>(p, r, x.adv[u], x.logp[u], f, by_ratio, by_logp);
        x.others(p, u, f, by_logp);
        g = (inside ? by_ratio : 0.f) + by_logp;
        f4 += f;
        kl4 += r.rest;
        ++n;
        below += r.below;
        above += r.above;
      }
      if (p.deriv != nullptr && t0 + u * step < p.S) p.deriv[b * p.S + t0 + u * step] = g;
    }
    loss += f4;
    kl += kl4;
  }
  double s[5] = {loss, static_cast<double>(n), kl, static_cast<double>(below), static_cast<double>(above)};
  cluster_sums(s, sh, ctas);
  put_sums(p, b, s);
}

// One ratio per row.  The row's loss and its derivative by the logarithm of the ratio are sums over the advantages of either sign, so one pass over the inputs is enough; what a token's
// own derivative needs beside them stays in shared memory for rows of up to HOLD tokens per thread of the cluster, and comes from the inputs again, then in L2, for longer ones.
template <int KIND>
__global__ void __launch_bounds__(ls::THREADS, ls::CTAS) policy_sequence_kernel(const Policy p) {
  using namespace ls;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ double sh[THREADS / 32 + 2][6];
  const int ctas = gridDim.x, step = ctas * THREADS, first = blockIdx.x * THREADS + threadIdx.x;
  const long b = blockIdx.y;
  const bool held = KIND != WEIGHT && p.S <= step * HOLD;
  __shared__ float keep[HOLD][THREADS];
  uint32_t on = 0, inner = 0;
  double s[6] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0};      // other terms, tokens, log ratios, advantages from 0 on, below 0, advantage · log-prob
  auto sum = [&](int t0, int at) {
    Batch<UNROLL> x;
    x.load(p, b, t0, step);
    float f4 = 0.f;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (x.on[u]) {
        bool inside;
        s[2] += x.log_ratio(u, inside);
        float by_logp = 0.f;
        x.others(p, u, f4, by_logp);
        s[1] += 1.0;
        if (x.adv[u] >= 0.f) s[3] += x.adv[u]; else s[4] += x.adv[u];
        if constexpr (KIND == WEIGHT) s[5] += static_cast<double>(x.adv[u]) * x.logp[u];
        if (held) {
          keep[at + u][threadIdx.x] = by_logp;
          on |= 1u << (at + u);
          inner |= (inside ? 1u : 0u) << (at + u);
        }
      }
    s[0] += f4;
  };
  for (int t0 = first, at = 0; t0 < p.S; t0 += step * UNROLL, at += UNROLL) sum(t0, at);
  cluster_sums(s, sh, ctas);
  const double n = s[1] > 0.0 ? s[1] : 1.0;
  const Ratio r = ratio_of(p, s[2] / n);
  // the surrogate is proportional to the size of the advantage
  float f_up, d_up, f_down, d_down, by_logp;
  surrogate<KIND>(p, r, 1.f, 0.f, f_up, d_up, by_logp);
  surrogate<KIND>(p, r, -1.f, 0.f, f_down, d_down, by_logp);
  const float weight = r.over ? p.top : r.r;
  const double loss = s[0] + (KIND == WEIGHT ? -weight * s[5] : f_up * s[3] - f_down * s[4]);
  const float by_each = KIND == WEIGHT ? 0.f : static_cast<float>((d_up * s[3] - d_down * s[4]) / n);
  if (p.deriv != nullptr) {
    if (held) {
#pragma unroll 4
      for (int t = first, i = 0; t < p.S; t += step, ++i) p.deriv[b * p.S + t] = on >> i & 1u ? (inner >> i & 1u ? by_each : 0.f) + keep[i][threadIdx.x] : 0.f;
    } else {
      for (int t0 = first; t0 < p.S; t0 += step * UNROLL) {
        Batch<UNROLL> x;
        x.load(p, b, t0, step);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          float g = 0.f;
          if (x.on[u]) {
            bool inside;
            x.log_ratio(u, inside);
            float f = 0.f, direct = KIND == WEIGHT ? -weight * x.adv[u] : 0.f;
            x.others(p, u, f, direct);
            g = (inside ? by_each : 0.f) + direct;
          }
          if (t0 + u * step < p.S) p.deriv[b * p.S + t0 + u * step] = g;
        }
      }
    }
  }
  const double out[5] = {loss, s[1], s[1] * static_cast<double>(r.rest), r.below ? s[1] : 0.0, r.above ? s[1] : 0.0};
  put_sums(p, b, out);
}

// Joins the rows: loss, weight of every row, figures.  One CTA; threads take rows in turn, so the order of the sums is that of the rows' numbers.
__global__ void __launch_bounds__(ls::THREADS) policy_join_kernel(const double* __restrict__ sums, float* __restrict__ weight, float* __restrict__ loss, float* __restrict__ stats, int B,
                                                                  int reduce, double denominator) {
  __shared__ double sh[ls::THREADS / 32 + 2][5];
  double s[5] = {0.0, 0.0, 0.0, 0.0, 0.0};
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int b = threadIdx.x; b < B; b += ls::THREADS) {
    const double n = sums[b * 5L + 1] > 0.0 ? sums[b * 5L + 1] : 1.0;
    s[0] += reduce == REDUCE_SEQUENCE ? sums[b * 5L] / n : sums[b * 5L];
#pragma unroll
    for (int i = 1; i < 5; ++i) s[i] += sums[b * 5L + i];
  }
  cluster_sums(s, sh, 1);
  const double many = s[1] > 0.0 ? s[1] : 1.0, over = reduce == REDUCE_SEQUENCE ? static_cast<double>(B) : reduce == REDUCE_TOKEN ? many : denominator;
  for (int b = threadIdx.x; b < B; b += ls::THREADS) {
    const double n = sums[b * 5L + 1] > 0.0 ? sums[b * 5L + 1] : 1.0;
    weight[b] = static_cast<float>(reduce == REDUCE_SEQUENCE ? 1.0 / (over * n) : 1.0 / over);
  }
  if (threadIdx.x == 0) {
    *loss = static_cast<float>(s[0] / over);
    stats[0] = static_cast<float>(s[2] / many);
    stats[1] = static_cast<float>(s[3] / many);
    stats[2] = static_cast<float>(s[4] / many);
    stats[3] = static_cast<float>(s[1]);
  }
}

// grad = derivative · weight of the row · gradient of the loss; entropies: −c · weight · gradient of the loss on tokens that count
__global__ void __launch_bounds__(ls::THREADS) policy_grad_kernel(const float* __restrict__ deriv, const float* __restrict__ weight, const float* __restrict__ up, const Tokens tokens,
                                                                  float entropy, float* __restrict__ grad, float* __restrict__ grad_ent, int S) {
  using namespace ls;
  const long b = blockIdx.y;
  const float w = weight[b] * *up;
  const int step = gridDim.x * THREADS;
  for (int t0 = blockIdx.x * THREADS + threadIdx.x; t0 < S; t0 += step * UNROLL) {
    float d[UNROLL];
    int64_t label[UNROLL];
    if (grad != nullptr) Rows{deriv, S, false}.load(d, b, t0, step, S);
    if (grad_ent != nullptr) tokens.load(label, b, t0, step, S);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int t = t0 + u * step;
      if (t >= S) break;
      if (grad != nullptr) grad[b * S + t] = d[u] == 0.f ? 0.f : d[u] * w;      // masked tokens have none, whatever the gradient of the loss is
      if (grad_ent != nullptr) grad_ent[b * S + t] = label[u] != tokens.ignore ? -entropy * w : 0.f;
    }
  }
}

// ------------------------------------------------------------ preference loss
enum { SIGMOID = 0, HINGE = 1, IPO = 2, KTO_PAIR = 3, SIMPO = 4, ORPO = 5 };

struct Preference {
  Tokens tokens;
  Rows logps, ref;
  double* sums;          // [B, 3] log-probs, tokens, reference log-probs
  int S;
};

__global__ void __launch_bounds__(ls::THREADS, ls::CTAS) preference_rows_kernel(const Preference p) {
  using namespace ls;
  __shared__ double sh[THREADS / 32 + 2][3];
  const int ctas = gridDim.x;
  const long b = blockIdx.y;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int step = ctas * THREADS;
  const bool each = p.ref.p != nullptr && !p.ref.one;
  double s[3] = {0.0, 0.0, 0.0};
  int n = 0;
  for (int t0 = blockIdx.x * THREADS + threadIdx.x; t0 < p.S; t0 += step * UNROLL) {
    float x[UNROLL], y[UNROLL] = {};
    int64_t label[UNROLL];
    p.tokens.load(label, b, t0, step, p.S);
    p.logps.load(x, b, t0, step, p.S);
    if (each) p.ref.load(y, b, t0, step, p.S);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (t0 + u * step < p.S && label[u] != p.tokens.ignore) {
        s[0] += x[u];
        s[2] += y[u];
        ++n;
      }
  }
  s[1] = n;
  cluster_sums(s, sh, ctas);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.sums[b * 3] = s[0];
    p.sums[b * 3 + 1] = s[1];
    p.sums[b * 3 + 2] = p.ref.p != nullptr && p.ref.one ? static_cast<double>(p.ref.p[b * p.ref.ld]) : s[2];
  }
}

struct PairArgs {
  int form, pairs;
  double beta, gamma, smoothing, nll;
};

__device__ __forceinline__ double softplus64(double z) { return fmax(z, 0.0) + log1p(exp(-fabs(z))); }
__device__ __forceinline__ double sigmoid64(double z) { return 1.0 / (1.0 + exp(-z)); }

__global__ void __launch_bounds__(ls::THREADS) preference_join_kernel(const double* __restrict__ sums, PairArgs a, float* __restrict__ coef, float* __restrict__ loss,
                                                                      float* __restrict__ stats) {
  __shared__ double sh[ls::THREADS / 32 + 2][7];
  double s[7] = {};     // losses, chosen and rejected levels, chosen above rejected, log-probs of both, chosen tokens
  const bool mean = a.form == SIMPO || a.form == ORPO;
  double chosen_tokens = 0.0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // the likelihood term's denominator is a sum over all pairs: it comes first
  if (a.nll != 0.0) {
    double n[1] = {0.0};
    for (int i = threadIdx.x; i < a.pairs; i += ls::THREADS) n[0] += sums[6L * i + 1];
    cluster_sums(n, reinterpret_cast<double(*)[1]>(&sh[0][0]), 1);
    chosen_tokens = n[0] > 0.0 ? n[0] : 1.0;
  }
  for (int i = threadIdx.x; i < a.pairs; i += ls::THREADS) {
    const double *x = sums + 6L * i, *y = x + 3;
    const double px = mean ? 1.0 / fmax(x[1], 1.0) : 1.0, py = mean ? 1.0 / fmax(y[1], 1.0) : 1.0;
    const double c = mean ? x[0] * px : x[0] - x[2], j = mean ? y[0] * py : y[0] - y[2];
    const double z = a.beta * (c - j) - a.gamma;
    double f, dc, dj;
    if (a.form == SIGMOID || a.form == SIMPO) {
      f = softplus64(-z) * (1.0 - a.smoothing) + (a.smoothing != 0.0 ? softplus64(z) * a.smoothing : 0.0);
      dc = a.beta * (-sigmoid64(-z) * (1.0 - a.smoothing) + sigmoid64(z) * a.smoothing);
      dj = -dc;
    } else if (a.form == HINGE) {
      f = z < 1.0 ? 1.0 - z : z >= 1.0 ? 0.0 : z;      // not a number stays one
      dc = z < 1.0 ? -a.beta : 0.0;
      dj = -dc;
    } else if (a.form == IPO) {
      const double u = z - 1.0 / (2.0 * a.beta);
      f = u * u;
      dc = 2.0 * a.beta * u;
      dj = -dc;
    } else if (a.form == KTO_PAIR) {
      const double p = sigmoid64(a.beta * c), q = sigmoid64(a.beta * j);
      f = 1.0 - p + q;
      dc = -a.beta * p * (1.0 - p);
      dj = a.beta * q * (1.0 - q);
    } else {
      // log odds; a probability above 1 − 1e-6 counts as that
      const double most = -1.000000500000333e-6;        // log(1 − 1e-6)
      const double rc = -expm1(fmin(c, most)), rj = -expm1(fmin(j, most));
      const double odds = c - j - (log(rc) - log(rj)), d = -a.beta * sigmoid64(-odds);
      f = a.beta * softplus64(-odds);
      dc = d * (c <= most ? 1.0 / rc : 1.0);
      dj = -d * (j <= most ? 1.0 / rj : 1.0);
    }
    coef[2 * i] = static_cast<float>(dc * px / a.pairs - (a.nll != 0.0 ? a.nll / chosen_tokens : 0.0));
    coef[2 * i + 1] = static_cast<float>(dj * py / a.pairs);
    s[0] += f;
    s[1] += c;
    s[2] += j;
    s[3] += c > j;
    s[4] += x[0];
    s[5] += y[0];
  }
  cluster_sums(s, sh, 1);
  if (threadIdx.x == 0) {
    *loss = static_cast<float>(s[0] / a.pairs - (a.nll != 0.0 ? a.nll * s[4] / chosen_tokens : 0.0));
    stats[0] = static_cast<float>(a.beta * s[1] / a.pairs);
    stats[1] = static_cast<float>(a.beta * s[2] / a.pairs);
    stats[2] = static_cast<float>(a.beta * (s[1] - s[2]) / a.pairs);
    stats[3] = static_cast<float>(s[3] / a.pairs);
    stats[4] = static_cast<float>(s[4] / a.pairs);
    stats[5] = static_cast<float>(s[5] / a.pairs);
  }
}

__global__ void __launch_bounds__(ls::THREADS) preference_grad_kernel(const float* __restrict__ coef, const float* __restrict__ up, const Tokens tokens, float* __restrict__ grad, int S) {
  using namespace ls;
  const long b = blockIdx.y;
  const float c = coef[b] * *up;
  const int step = gridDim.x * THREADS;
  for (int t0 = blockIdx.x * THREADS + threadIdx.x; t0 < S; t0 += step * UNROLL) {
    int64_t label[UNROLL];
    tokens.load(label, b, t0, step, S);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (t0 + u * step < S) grad[b * S + t0 + u * step] = label[u] != tokens.ignore ? c : 0.f;
  }
}

// -------------------------------------------------------------------- host side
static Tokens tokens_of(const torch::Tensor& labels, const torch::Tensor& like, int64_t ignore) {
  TORCH_CHECK(labels.is_cuda() && labels.device() == like.device() && labels.sizes() == like.sizes() && (labels.scalar_type() == torch::kInt64 || labels.scalar_type() == torch::kBool) &&
                  (labels.size(1) <= 1 || labels.stride(1) == 1), "labels int64 or a boolean mask [rows, tokens] like the log-probs, tokens side by side");
  const bool bytes = labels.scalar_type() == torch::kBool;
  return {labels.data_ptr(), labels.stride(0), bytes ? 0 : ignore, bytes};
}
static Rows rows_of(const OptT& t, const torch::Tensor& like, bool per_row, const char* what) {
  if (!has(t)) return {nullptr, 0, false};
  TORCH_CHECK(t->is_cuda() && t->device() == like.device() && t->scalar_type() == torch::kFloat32, what, ": fp32 on the device of the log-probs");
  if (per_row && t->dim() == 1) {
    TORCH_CHECK(t->size(0) == like.size(0), what, ": one number per row");
    return {t->data_ptr<float>(), t->stride(0), true};
  }
  TORCH_CHECK(t->sizes() == like.sizes() && (t->size(1) <= 1 || t->stride(1) == 1), what, " [rows, tokens] like the log-probs, tokens side by side");
  return {t->data_ptr<float>(), t->stride(0), false};
}
static void check_logps(const torch::Tensor& logps) {
  TORCH_CHECK(logps.is_cuda() && logps.dim() == 2 && logps.scalar_type() == torch::kFloat32 && logps.numel() > 0 && (logps.size(1) <= 1 || logps.stride(1) == 1),
              "log-probs [rows, tokens] fp32, not empty, tokens side by side");
  TORCH_CHECK(logps.size(0) <= 65535 && logps.size(1) < (int64_t(1) << 30), "up to 65535 rows of 2^30 tokens");
}

// CTAs per row: down to a batch of tokens per thread, while all are resident at once (more of them, each with less to do, wait for one another's latencies: 256 rows of 16k tokens
// took 80 us on 8 CTAs a row).
static int row_ctas(int64_t B, int64_t S) {
  int c = 1;
  while (c < 8 && 2 * B * c <= ls::CTAS * num_sms() && S > static_cast<int64_t>(c) * ls::THREADS * ls::UNROLL) c *= 2;
  return c;
}

template <typename F, typename P>
static void launch_rows(F kernel, const P& p, int64_t B, int64_t S, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(row_ctas(B, S), B);
  cfg.blockDim = dim3(ls::THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cfg.gridDim.x;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  count_launch();
}
// Joins the rows: begins while they are summed and waits for them.
template <typename... A>
static void launch_join(void (*kernel)(A...), cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(ls::THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
  count_launch();
}
static dim3 grad_grid(int64_t B, int64_t S) {
  const int64_t most = (8 * num_sms() + B - 1) / B, want = (S + ls::THREADS * ls::UNROLL - 1) / (ls::THREADS * ls::UNROLL);
  return dim3(static_cast<unsigned>(std::max<int64_t>(1, std::min(want, most))), static_cast<unsigned>(B));
}

// {loss [], stats [4], derivative [B, S] (empty unless wanted), weight [B]}
std::vector<torch::Tensor> policy_loss_fwd(const torch::Tensor& logps, const torch::Tensor& labels, const torch::Tensor& adv, const OptT& old, const OptT& ref, const OptT& ent, int64_t ratio,
                                           int64_t kind, int64_t reduce, double eps_low, double eps_high, double beta, double entropy, double tau_pos, double tau_neg, double denominator,
                                           int64_t ignore, bool want_grad) {
  check_logps(logps);
  TORCH_CHECK(ratio >= 0 && ratio <= 1 && kind >= 0 && kind <= 2 && reduce >= 0 && reduce <= 2, "policy_loss: ratio, surrogate, reduction");
  c10::cuda::CUDAGuard guard(logps.device());
  const int64_t B = logps.size(0), S = logps.size(1);
  Policy p{};
  p.tokens = tokens_of(labels, logps, ignore);
  p.logps = rows_of(logps, logps, false, "log-probs");
  p.old = rows_of(old, logps, false, "old log-probs");
  p.ref = rows_of(ref, logps, false, "reference log-probs");
  p.ent = rows_of(ent, logps, false, "entropies");
  p.adv = rows_of(adv, logps, true, "advantages");
  const auto f32 = logps.options();
  auto sums = torch::empty({B, 5}, f32.dtype(torch::kFloat64)), weight = torch::empty({B}, f32), loss = torch::empty({}, f32), stats = torch::empty({4}, f32);
  auto deriv = want_grad ? torch::empty({B, S}, f32) : torch::empty({0}, f32);
  p.deriv = want_grad ? deriv.data_ptr<float>() : nullptr;
  p.sums = sums.data_ptr<double>();
  p.B = B; p.S = S;
  p.lo = static_cast<float>(1.0 - eps_low); p.hi = static_cast<float>(1.0 + eps_high); p.top = static_cast<float>(1.0 + eps_low);
  p.log_lo = eps_low < 1.0 ? std::log1p(-eps_low) : -INFINITY; p.log_hi = std::log1p(eps_high); p.log_top = std::log1p(eps_low);
  p.beta = static_cast<float>(beta); p.entropy = static_cast<float>(entropy); p.tau_pos = static_cast<float>(tau_pos); p.tau_neg = static_cast<float>(tau_neg);
  auto stream = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto kernel) { launch_rows(kernel, p, B, S, stream); };
  if (ratio == RATIO_TOKEN) {
    if (kind == CLIP) go(policy_token_kernel<CLIP>); else if (kind == SOFT) go(policy_token_kernel<SOFT>); else go(policy_token_kernel<WEIGHT>);
  } else {
    if (kind == CLIP) go(policy_sequence_kernel<CLIP>); else if (kind == SOFT) go(policy_sequence_kernel<SOFT>); else go(policy_sequence_kernel<WEIGHT>);
  }
  launch_join(policy_join_kernel, stream, static_cast<const double*>(p.sums), weight.data_ptr<float>(), loss.data_ptr<float>(), stats.data_ptr<float>(), static_cast<int>(B), static_cast<int>(reduce),
              denominator);
  return {loss, stats, deriv, weight};
}

// {gradient by the log-probs, by the entropies} (empty where not wanted)
std::vector<torch::Tensor> policy_loss_bwd(const torch::Tensor& up, const OptT& deriv, const torch::Tensor& weight, const torch::Tensor& labels, double entropy, int64_t ignore, bool want_ent) {
  TORCH_CHECK(up.is_cuda() && up.scalar_type() == torch::kFloat32 && up.numel() == 1, "gradient of the loss: one fp32 number");
  c10::cuda::CUDAGuard guard(weight.device());
  const int64_t B = labels.size(0), S = labels.size(1);
  const auto f32 = weight.options();
  auto grad = has(deriv) ? torch::empty({B, S}, f32) : torch::empty({0}, f32), grad_ent = want_ent ? torch::empty({B, S}, f32) : torch::empty({0}, f32);
  const Tokens tokens = tokens_of(labels, labels, ignore);
  policy_grad_kernel<<<grad_grid(B, S), ls::THREADS, 0, at::cuda::getCurrentCUDAStream()>>>(has(deriv) ? deriv->data_ptr<float>() : nullptr, weight.data_ptr<float>(), up.data_ptr<float>(), tokens,
      static_cast<float>(entropy), has(deriv) ? grad.data_ptr<float>() : nullptr, want_ent ? grad_ent.data_ptr<float>() : nullptr, static_cast<int>(S));
  count_launch();
  TK_CUDA_CHECK(cudaGetLastError());
  return {grad, grad_ent};
}

// {loss [], stats [6], coefficient [B]}
std::vector<torch::Tensor> preference_loss_fwd(const torch::Tensor& logps, const torch::Tensor& labels, const OptT& ref, int64_t form, double beta, double gamma, double smoothing, double nll,
                                               int64_t ignore) {
  check_logps(logps);
  TORCH_CHECK(logps.size(0) % 2 == 0 && form >= 0 && form <= 5, "preference_loss: rows in pairs, one of six forms");
  c10::cuda::CUDAGuard guard(logps.device());
  const int64_t B = logps.size(0), S = logps.size(1);
  Preference p{};
  p.tokens = tokens_of(labels, logps, ignore);
  p.logps = rows_of(logps, logps, false, "log-probs");
  p.ref = rows_of(ref, logps, true, "reference log-probs");
  const auto f32 = logps.options();
  auto sums = torch::empty({B, 3}, f32.dtype(torch::kFloat64)), coef = torch::empty({B}, f32), loss = torch::empty({}, f32), stats = torch::empty({6}, f32);
  p.sums = sums.data_ptr<double>();
  p.S = S;
  auto stream = at::cuda::getCurrentCUDAStream();
  launch_rows(preference_rows_kernel, p, B, S, stream);
  const PairArgs a{static_cast<int>(form), static_cast<int>(B / 2), beta, gamma, smoothing, nll};
  launch_join(preference_join_kernel, stream, static_cast<const double*>(p.sums), a, coef.data_ptr<float>(), loss.data_ptr<float>(), stats.data_ptr<float>());
  return {loss, stats, coef};
}

torch::Tensor preference_loss_bwd(const torch::Tensor& up, const torch::Tensor& coef, const torch::Tensor& labels, int64_t ignore) {
  TORCH_CHECK(up.is_cuda() && up.scalar_type() == torch::kFloat32 && up.numel() == 1, "gradient of the loss: one fp32 number");
  c10::cuda::CUDAGuard guard(coef.device());
  const int64_t B = labels.size(0), S = labels.size(1);
  auto grad = torch::empty({B, S}, coef.options());
  const Tokens tokens = tokens_of(labels, labels, ignore);
  preference_grad_kernel<<<grad_grid(B, S), ls::THREADS, 0, at::cuda::getCurrentCUDAStream()>>>(coef.data_ptr<float>(), up.data_ptr<float>(), tokens, grad.data_ptr<float>(), static_cast<int>(S));
  count_launch();
  TK_CUDA_CHECK(cudaGetLastError());
  return grad;
}

}  // namespace tk
