// Losses on choices: the log-probability that a network gives to a label, the clipped policy loss with a KL term, the
// preference loss on pairs of texts, and their gradients. A network's outputs are spike values z, its logits are -z, as in the
// cross-entropy of snntc_train.cu.
//
//   top = max_j -z_j, total = sum_j exp(-z_j - top), lp = (-z_a - top) - log(total), p_j = exp(-z_j - top) / total
//   every gradient is  dz_j = factor * (p_j - [j = a])  with factor = dloss / dlp, one number per row.
//
// A row whose label is outside [0, J) does not count: its logits are not read, its gradient is zero.
// (top, total) are kept for the backward, never their log-sum: beside a |top| of 1e5 (no output spiked) it would lose total.
// What is one number per row (lp, ratios, the KL term, sums over texts) is formed in 64 bits: the clip decides by comparing, and a
// text's sum of hundreds of lp is taken from another one of the same size.
#include "../../include/snntc_b200.h"
#include "snntc_launch.cuh"

#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

namespace snntc { void count_launch(int n = 1); void note_cuda_error(cudaError_t e); }

namespace {

using snntc::chain_next;
using snntc::chain_wait;
using snntc::launch_chained;
using snntc::ld_plain;

constexpr int kRowThreads = 256;

// (running maximum, sum of exp(x - maximum)) of the logits x that a lane has seen. The maximum starts at the lowest finite value,
// not at -inf, whose difference from itself is no number.
struct Online {
  float top = -FLT_MAX, total = 0.f;
  __device__ __forceinline__ void add(float x) {
    const float t = fmaxf(top, x);
    total = total * expf(top - t) + expf(x - t);
    top = t;
  }
  __device__ __forceinline__ void join(float t2, float s2) {
    const float t = fmaxf(top, t2);
    total = total * expf(top - t) + s2 * expf(t2 - t);
    top = t;
  }
};

__device__ __forceinline__ bool counts(long long label, int J) { return label >= 0 && label < J; }

__device__ __forceinline__ double label_logp(float z_label, float2 st) {
  return (-(double)z_label - (double)st.x) - log((double)st.y);
}

// One warp per row: (top, total) and lp
__global__ void __launch_bounds__(kRowThreads)
choice_rows_kernel(const float* z, const long long* labels, float* __restrict__ logp, double* __restrict__ logp64,
                   float2* __restrict__ stats, float* __restrict__ factor, long long R, int J) {
  chain_wait();
  chain_next();
  const long long r = ((long long)blockIdx.x * kRowThreads + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (r >= R) return;
  const long long label = ld_plain(labels + r);
  Online o;
  double lp = 0.0;
  if (counts(label, J)) {
    const float* row = z + r * J;
    for (int j = lane; j < J; j += 32) o.add(-ld_plain(row + j));
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
      const float t = __shfl_xor_sync(0xffffffffu, o.top, d), s = __shfl_xor_sync(0xffffffffu, o.total, d);
      o.join(t, s);
    }
    lp = label_logp(ld_plain(row + label), make_float2(o.top, o.total));
  }
  if (lane == 0) {
    if (logp) logp[r] = (float)lp;
    if (logp64) logp64[r] = lp;
    if (stats) stats[r] = make_float2(o.top, o.total);
    if (factor) factor[r] = 0.f;
  }
}

// dz = factor * (p - onehot), one warp per row
__global__ void __launch_bounds__(kRowThreads)
choice_grad_kernel(const float* z, const long long* labels, const float2* stats, const float* factor, const float* gout,
                   float* __restrict__ dz, long long R, int J) {
  chain_wait();
  chain_next();
  const long long r = ((long long)blockIdx.x * kRowThreads + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (r >= R) return;
  const long long label = ld_plain(labels + r);
  const float f = ld_plain(factor + r) * (gout ? ld_plain(gout) : 1.f);
  const float* row = z + r * J;
  float* to = dz + r * J;
  if (!counts(label, J) || f == 0.f) {
    for (int j = lane; j < J; j += 32) to[j] = 0.f;
    return;
  }
  const float2 st = ld_plain(stats + r);
  const float inv = 1.f / st.y;
  for (int j = lane; j < J; j += 32) to[j] = f * (expf(-ld_plain(row + j) - st.x) * inv - (j == label ? 1.f : 0.f));
}

struct PolicyParams { double lower, upper, kl_coef; };

// loss term, KL term, clipped or not, and dterm/dlp of one row
struct PolicyRow {
  double loss, kl, slope;
  bool clipped;
};
__device__ __forceinline__ PolicyRow policy_row(double lp, double old, double adv, bool has_ref, double ref, const PolicyParams& q) {
  PolicyRow p;
  const double ratio = exp(lp - old);
  p.clipped = (adv > 0 && ratio > q.upper) || (adv < 0 && ratio < q.lower);
  const double gain = (p.clipped ? (adv > 0 ? q.upper : q.lower) : ratio) * adv;
  p.kl = 0;
  p.slope = p.clipped ? 0 : -ratio * adv;
  if (has_ref) {
    const double away = ref - lp, e = expm1(away);
    p.kl = e - away;
    p.slope -= q.kl_coef * e;
  }
  p.loss = q.kl_coef * p.kl - gain;
  return p;
}

// Sum of three numbers over a CTA in a fixed order, valid in thread 0
__device__ __forceinline__ double3 block_sum(double3 v) {
  __shared__ double part[3][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, d);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, d);
    v.z += __shfl_xor_sync(0xffffffffu, v.z, d);
  }
  __syncthreads();
  if (lane == 0) { part[0][warp] = v.x; part[1][warp] = v.y; part[2][warp] = v.z; }
  __syncthreads();
  double3 t = make_double3(0, 0, 0);
  if (threadIdx.x == 0)
    for (int k = 0; k < warps; ++k) { t.x += part[0][k]; t.y += part[1][k]; t.z += part[2][k]; }
  return t;
}

// One CTA: the terms of all rows, the mean over those that count, and the factors of the gradient.
__global__ void __launch_bounds__(1024)
policy_rows_kernel(const double* lp, const long long* labels, const float* old, const float* adv, const float* ref,
                   float* __restrict__ factor, float* __restrict__ loss, float* __restrict__ out2, long long R, int J,
                   PolicyParams q) {
  chain_wait();
  chain_next();
  __shared__ double inv_n;
  double3 n = make_double3(0, 0, 0);
  for (long long r = threadIdx.x; r < R; r += blockDim.x) n.x += counts(ld_plain(labels + r), J) ? 1.0 : 0.0;
  n = block_sum(n);
  if (threadIdx.x == 0) inv_n = n.x > 0 ? 1.0 / n.x : 0.0;
  __syncthreads();
  double3 sum = make_double3(0, 0, 0);
  for (long long r = threadIdx.x; r < R; r += blockDim.x) {
    if (!counts(ld_plain(labels + r), J)) continue;
    const PolicyRow p = policy_row(ld_plain(lp + r), ld_plain(old + r), ld_plain(adv + r), ref != nullptr, ref ? ld_plain(ref + r) : 0.f, q);
    sum.x += p.loss;
    sum.y += p.kl;
    sum.z += p.clipped ? 1.0 : 0.0;
    factor[r] = (float)(p.slope * inv_n);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) {
    *loss = (float)(sum.x * inv_n);
    out2[0] = (float)(sum.y * inv_n);
    out2[1] = (float)(sum.z * inv_n);
  }
}

// rows [first, last) of a text; whatever the caller's numbers are, inside [0, R)
__device__ __forceinline__ void text_rows(const long long* starts, long long rows_per_text, int text, long long R, long long& first,
                                          long long& last) {
  first = starts ? ld_plain(starts + text) : text * rows_per_text;
  last = starts ? ld_plain(starts + text + 1) : first + rows_per_text;
  first = first < 0 ? 0 : first > R ? R : first;
  last = last < first ? first : last > R ? R : last;
}

// One CTA per pair: the sums of its two texts, the margin, its loss, and the factors of the texts' rows.
__global__ void __launch_bounds__(512)
preference_pairs_kernel(const double* lp, const long long* starts, const float* ref, float* __restrict__ margins,
                        float* __restrict__ factor, double* __restrict__ terms, long long R, int P, long long rows_per_text,
                        double beta, double smoothing) {
  chain_wait();
  chain_next();
  __shared__ double slope;
  const int k = blockIdx.x;
  long long f0, l0, f1, l1;
  text_rows(starts, rows_per_text, k, R, f0, l0);
  text_rows(starts, rows_per_text, P + k, R, f1, l1);
  double3 sum = make_double3(0, 0, 0);
  for (long long r = f0 + threadIdx.x; r < l0; r += blockDim.x) sum.x += ld_plain(lp + r);
  for (long long r = f1 + threadIdx.x; r < l1; r += blockDim.x) sum.y += ld_plain(lp + r);
  sum = block_sum(sum);
  if (threadIdx.x == 0) {
    double good = sum.x, bad = sum.y;
    if (ref) { good -= ld_plain(ref + k); bad -= ld_plain(ref + P + k); }
    const double m = beta * (good - bad);
    const double tail = log1p(exp(-fabs(m)));                  // -log sigma(|m|)
    terms[k] = (1 - smoothing) * (tail + fmax(-m, 0.0)) + smoothing * (tail + fmax(m, 0.0));
    margins[k] = (float)m;
    slope = beta / P * (1 / (1 + exp(-m)) - (1 - smoothing));
  }
  __syncthreads();
  const float f = (float)slope;
  for (long long r = f0 + threadIdx.x; r < l0; r += blockDim.x) factor[r] = f;
  for (long long r = f1 + threadIdx.x; r < l1; r += blockDim.x) factor[r] = -f;
}

__global__ void __launch_bounds__(512) mean_kernel(const double* terms, int n, float* __restrict__ mean) {
  chain_wait();
  chain_next();
  double3 s = make_double3(0, 0, 0);
  for (int k = threadIdx.x; k < n; k += blockDim.x) s.x += ld_plain(terms + k);
  s = block_sum(s);
  if (threadIdx.x == 0) *mean = (float)(s.x / n);
}

int done() {
  snntc::count_launch();
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return SNNTC_OK;
  snntc::note_cuda_error(e);
  return SNNTC_E_CUDA;
}

int check_rows(long long R, int J) {
  if (R <= 0 || J <= 0) return SNNTC_E_SHAPE;
  return R > 0x7fffffffLL ? SNNTC_E_TOO_LARGE : SNNTC_OK;
}

int launch_rows(const float* z, const long long* labels, float* logp, double* logp64, float* stats, float* factor, long long R, int J,
                cudaStream_t s) {
  const unsigned grid = (unsigned)((R * 32 + kRowThreads - 1) / kRowThreads);
  (void)launch_chained(choice_rows_kernel, grid, kRowThreads, 0, s, 0, z, labels, logp, logp64, (float2*)stats, factor, R, J);
  return done();
}

}  // namespace

extern "C" {

int snntc_label_logp_forward(const float* z, const long long* labels, float* logp, float* stats_2R, long long R, int J, void* stream) {
  if (!z || !labels || !logp) return SNNTC_E_NULL;
  if (const int rc = check_rows(R, J)) return rc;
  return launch_rows(z, labels, logp, nullptr, stats_2R, nullptr, R, J, (cudaStream_t)stream);
}

int snntc_choice_backward(const float* z, const long long* labels, const float* stats_2R, const float* factor, const float* gout,
                          float* dz, long long R, int J, void* stream) {
  if (!z || !labels || !stats_2R || !factor || !dz) return SNNTC_E_NULL;
  if (const int rc = check_rows(R, J)) return rc;
  const unsigned grid = (unsigned)((R * 32 + kRowThreads - 1) / kRowThreads);
  (void)launch_chained(choice_grad_kernel, grid, kRowThreads, 0, (cudaStream_t)stream, 0, z, labels, (const float2*)stats_2R, factor, gout,
                       dz, R, J);
  return done();
}

size_t snntc_policy_loss_workspace_bytes(long long R) { return R <= 0 ? 0 : (size_t)R * sizeof(double); }

int snntc_policy_loss(const float* z, const long long* labels, const float* old_logp, const float* advantage, const float* ref_logp,
                      float* loss, float* kl_and_clipped, float* stats_2R, float* factor, long long R, int J, double clip_low,
                      double clip_high, double kl_coef, void* workspace, size_t workspace_bytes, void* stream) {
  if (!z || !labels || !old_logp || !advantage || !loss || !kl_and_clipped || !stats_2R || !factor) return SNNTC_E_NULL;
  if (const int rc = check_rows(R, J)) return rc;
  if (!(clip_low >= 0 && clip_low <= 1 && clip_high >= 0 && kl_coef - kl_coef == 0) || (kl_coef != 0 && !ref_logp)) return SNNTC_E_PARAMS;
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < snntc_policy_loss_workspace_bytes(R)) return SNNTC_E_WORKSPACE;
  double* lp = (double*)workspace;
  cudaStream_t s = (cudaStream_t)stream;
  if (const int rc = launch_rows(z, labels, nullptr, lp, stats_2R, factor, R, J, s)) return rc;
  const PolicyParams q{1 - clip_low, 1 + clip_high, kl_coef};
  (void)launch_chained(policy_rows_kernel, 1, 1024, 0, s, 0, lp, labels, old_logp, advantage, ref_logp, factor, loss, kl_and_clipped, R, J, q);
  return done();
}

size_t snntc_preference_loss_workspace_bytes(long long R, int P) {
  return R <= 0 || P <= 0 ? 0 : ((size_t)R + (size_t)P) * sizeof(double);
}

int snntc_preference_loss(const float* z, const long long* labels, const long long* starts, const float* ref_logp, float* loss,
                          float* margins, float* stats_2R, float* factor, long long R, int J, int P, double beta, double smoothing,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (!z || !labels || !loss || !margins || !stats_2R || !factor) return SNNTC_E_NULL;
  if (const int rc = check_rows(R, J)) return rc;
  if (P <= 0 || (!starts && R % (2LL * P) != 0)) return SNNTC_E_SHAPE;
  if (!(beta - beta == 0) || !(smoothing >= 0 && smoothing <= 1)) return SNNTC_E_PARAMS;
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < snntc_preference_loss_workspace_bytes(R, P)) return SNNTC_E_WORKSPACE;
  double* lp = (double*)workspace;
  double* terms = lp + R;
  cudaStream_t s = (cudaStream_t)stream;
  if (const int rc = launch_rows(z, labels, nullptr, lp, stats_2R, factor, R, J, s)) return rc;
  (void)launch_chained(preference_pairs_kernel, (unsigned)P, 512, 0, s, 0, lp, starts, ref_logp, margins, factor, terms, R, P,
                       R / (2LL * P), beta, smoothing);
  if (const int rc = done()) return rc;
  (void)launch_chained(mean_kernel, 1, 512, 0, s, 0, terms, P, loss);
  return done();
}

}  // extern "C"
