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

#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math_constants.h>
#include <stdint.h>

#include <utility>

namespace {

namespace cg = cooperative_groups;
using snntc::chain_next;
using snntc::chain_wait;
using snntc::done;
using snntc::launch_chained;
using snntc::ld_plain;
using snntc::ld_stream_at;
using snntc::streaming;

__device__ __forceinline__ bool counts(long long label, int J) { return label >= 0 && label < J; }

// exp(d) for d <= 0 as 2^(d log2 e), one product and one instruction: off by 2^-22 + |d| 2^-23 relative, and by some -5e-8 in the mean.
// With expf in its place the gradients' largest relative errors fall from 23 half steps of float32 to 14 (spike values up to some 13
// apart), their norm's stays at one, and it is the dearer one: policy loss with gradient of 8192 rows of 50 021 598 us instead of 577, of
// 32 768 of 1500 95, 87; log-probabilities with gradient of 4096 of 16 384 131, 125.
__device__ __forceinline__ float exp_term(float d) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * 1.44269504f));
  return e;
}
// A term of a row's sum. Where log-probabilities are what is wanted, expf, whose mean is off by 5e-9: those of a text's rows are added
// up, and what they have in common adds up with them (margins of 8192 rows in 32 texts: 1.3e-6 off with the short form, relative). It is
// the dearer one: 4096 rows of 32 768 93 us, 84 with the short form, which a single row's ratio and probabilities are served by.
template <bool SHORT>
__device__ __forceinline__ float sum_term(float d) { return SHORT ? exp_term(d) : expf(d); }

constexpr int kSumThreads = 1024;
constexpr int kFewPairs = 8;         // one for each CTA of a cluster (8 pairs: 7 us against 8.5 with a launch for the mean, 12: 9.4, 8.3)
constexpr int kSmallBlocks = 16;     // CTAs' worth of rows for a policy loss by one cluster

__device__ __forceinline__ double label_logp(float z_label, float2 st) {
  return (-(double)z_label - (double)st.x) - log((double)st.y);
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
  const double unclipped = adv == 0 && isinf(ratio) ? 0 : ratio * adv;      // (an advantage of 0 has no part, whatever the ratio)
  p.kl = 0;
  p.slope = p.clipped ? 0 : -unclipped;
  p.loss = -(p.clipped ? (adv > 0 ? q.upper : q.lower) * adv : unclipped);
  if (has_ref) {
    const double away = ref - lp, e = expm1(away);
    p.kl = isinf(e) ? e : e - away;              // (away is infinite, too, where an output at +inf rules the label out)
    if (q.kl_coef != 0) {        // (a label that does not spike overflows e: without a weight that stays out of the loss)
      p.slope -= q.kl_coef * e;
      p.loss += q.kl_coef * p.kl;
    }
  }
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

// Sum of three numbers over a cluster in a fixed order, the same value in all threads
__device__ __forceinline__ double3 cluster_sum(double3 v) {
  __shared__ double3 mine;
  cg::cluster_group cl = cg::this_cluster();
  v = block_sum(v);
  if (threadIdx.x == 0) mine = v;
  if (cl.num_blocks() == 1) {
    __syncthreads();
    const double3 t = mine;
    __syncthreads();
    return t;
  }
  cl.sync();
  double3 t = make_double3(0, 0, 0);
  for (unsigned k = 0; k < cl.num_blocks(); ++k) {
    const double3 o = *cl.map_shared_rank(&mine, k);
    t.x += o.x;
    t.y += o.y;
    t.z += o.z;
  }
  cl.sync();                                   // no CTA leaves, or comes back, while its number may still be read
  return t;
}

// How many rows count, over a cluster, the same number in all threads
__device__ __forceinline__ unsigned cluster_count(const long long* labels, long long R, int J) {
  __shared__ unsigned part[32], mine;
  cg::cluster_group cl = cg::this_cluster();
  unsigned n = 0;
#pragma unroll 8
  for (long long r = (long long)blockIdx.x * blockDim.x + threadIdx.x; r < R; r += (long long)gridDim.x * blockDim.x)
    n += counts(ld_plain(labels + r), J) ? 1u : 0u;
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x < 32) {
    n = __reduce_add_sync(0xffffffffu, threadIdx.x < blockDim.x / 32 ? part[threadIdx.x] : 0u);
    if (threadIdx.x == 0) mine = n;
  }
  cl.sync();
  n = 0;
  for (unsigned k = 0; k < cl.num_blocks(); ++k) n += *cl.map_shared_rank(&mine, k);
  cl.sync();
  return n;
}

// One cluster: 65 536 labels are eight loads a thread.
__global__ void __launch_bounds__(kSumThreads)
policy_count_kernel(const long long* labels, double* __restrict__ inv_n, long long R, int J) {
  chain_wait();
  chain_next();
  const unsigned n = cluster_count(labels, R, J);
  if (blockIdx.x == 0 && threadIdx.x == 0) *inv_n = n > 0 ? 1.0 / n : 0.0;
}

__global__ void __launch_bounds__(kSumThreads)
policy_mean_kernel(const double3* terms, const double* inv_n, float* __restrict__ loss, float* __restrict__ out2, long long n) {
  chain_wait();
  chain_next();
  double3 sum = make_double3(0, 0, 0);
  for (long long r = (long long)blockIdx.x * kSumThreads + threadIdx.x; r < n; r += (long long)gridDim.x * kSumThreads) {
    const double3 t = ld_plain(terms + r);
    sum.x += t.x;
    sum.y += t.y;
    sum.z += t.z;
  }
  sum = cluster_sum(sum);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const double inv = ld_plain(inv_n);
    *loss = (float)(sum.x * inv);
    out2[0] = (float)(sum.y * inv);
    out2[1] = (float)(sum.z * inv);
  }
}

// ---- rows. What bounds them is memory: 4 bytes read per logit, and 4 written where the gradient is formed. Where the loss's factor follows
// from the row alone (the policy loss) the gradient is written in the pass that reads the row. Rows of any length start anywhere, so
// a row is seen through the 16-byte vectors that cover it; those that stick out at its ends are loaded and stored by element.
// Short rows stay in registers, NV vectors of four a lane, all loads in flight at once; long ones are streamed. Maxima are a lane's or a
// warp's own: it sums exp(x - its maximum), and one exchange joins (maximum, sum) pairs.
template <int NV>
struct RowValues { float x[4 * NV]; };

// x = -z of the vectors first, first + stride, ...; -inf outside the row
template <int NV>
__device__ __forceinline__ RowValues<NV> load_row(const float* row, int J, bool live, int first, int stride) {
  RowValues<NV> v;
  const int lead = (int)(((uintptr_t)row >> 2) & 3);
  const float4* base = (const float4*)(row - lead);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int at = first + k * stride, j0 = 4 * at - lead;
    float4 q = make_float4(CUDART_INF_F, CUDART_INF_F, CUDART_INF_F, CUDART_INF_F);
    if (live && j0 >= 0 && j0 + 4 <= J) q = ld_plain(base + at);
    v.x[4 * k] = -q.x;
    v.x[4 * k + 1] = -q.y;
    v.x[4 * k + 2] = -q.z;
    v.x[4 * k + 3] = -q.w;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int j0 = 4 * (first + k * stride) - lead;
    if (live && (j0 < 0 || j0 + 4 > J) && j0 < J) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (j0 + c >= 0 && j0 + c < J) v.x[4 * k + c] = -ld_plain(row + j0 + c);
    }
  }
  return v;
}

// to[j] = x, less `hot` at the label; the values are where load_row of `row` has put them, and `to` may lie otherwise to 16 bytes
template <int NV>
__device__ __forceinline__ void store_row(float* to, const float* row, const RowValues<NV>& v, int J, long long label, float hot, int first,
                                          int stride) {
  const int lead = (int)(((uintptr_t)row >> 2) & 3);
  const bool alike = (((uintptr_t)to ^ (uintptr_t)row) & 15) == 0;
  float4* base = (float4*)(to - lead);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int at = first + k * stride, j0 = 4 * at - lead;
    float q[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) q[c] = v.x[4 * k + c] - (j0 + c == label ? hot : 0.f);
    if (alike && j0 >= 0 && j0 + 4 <= J) {
      base[at] = make_float4(q[0], q[1], q[2], q[3]);
    } else if (j0 < J) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (j0 + c >= 0 && j0 + c < J) to[j0 + c] = q[c];
    }
  }
}

// A row as its whole 16-byte vectors and the up to six elements at its ends, of which the first lanes of a group take one each
struct Ends {
  const float4* body;
  int head, vectors, at;
  bool mine;
  __device__ __forceinline__ Ends(const float* row, int J, int gl) {
    head = min(J, (int)((4 - ((uintptr_t)row >> 2)) & 3));
    vectors = (J - head) / 4;
    const int tail = head + 4 * vectors;
    body = (const float4*)(row + head);
    at = gl < head ? gl : tail + gl - head;
    mine = gl < head + J - tail;
  }
};

// to = scale * exp(-row - top), less f at the label; zeros where f is 0. By LANES lanes, U vectors at a time, from the row's end to its
// beginning. `to` is `apart` bytes behind the row.
struct RowGradient {
  const float* row;
  ptrdiff_t apart;
  Ends e;
  float top, scale, f;
  int hot;
  __device__ __forceinline__ void put(const float4* from, float4 q) const {
    float* to = (float*)((char*)from + apart);
    if ((apart & 15) == 0) {
      __stcs((float4*)to, q);
    } else {
      to[0] = q.x;
      to[1] = q.y;
      to[2] = q.z;
      to[3] = q.w;
    }
  }
  // the vectors v, v - LANES, ...: all of the K, or as many as there are down to the first
  template <int LANES, bool ALL, int... K>
  __device__ __forceinline__ void some(int v, std::integer_sequence<int, K...>) const {
    const float4* at = e.body + v;
    float4 q[sizeof...(K)] = {(ALL || v - K * LANES >= 0 ? ld_stream_at<-K * LANES * 16>(at, scale) : make_float4(0.f, 0.f, 0.f, 0.f))...};
#pragma unroll
    for (int k = 0; k < (int)sizeof...(K); ++k) {
      if (!ALL && v - k * LANES < 0) break;
      q[k].x = exp_term(-q[k].x - top) * scale;
      q[k].y = exp_term(-q[k].y - top) * scale;
      q[k].z = exp_term(-q[k].z - top) * scale;
      q[k].w = exp_term(-q[k].w - top) * scale;
      if (v - k * LANES == (hot - e.head) >> 2) {
        const int c = (hot - e.head) & 3;
        q[k].x -= c == 0 ? f : 0.f;
        q[k].y -= c == 1 ? f : 0.f;
        q[k].z -= c == 2 ? f : 0.f;
        q[k].w -= c == 3 ? f : 0.f;
      }
      put(at - k * LANES, q[k]);
    }
  }
  template <int LANES, int U>
  __device__ __forceinline__ void all(int gl) const {
    if (e.mine) *(float*)((char*)(row + e.at) + apart) = f == 0.f ? 0.f : exp_term(-ld_plain(row + e.at) - top) * scale - (e.at == hot ? f : 0.f);
    if (f == 0.f) {
      for (int v = gl; v < e.vectors; v += LANES) put(e.body + v, make_float4(0.f, 0.f, 0.f, 0.f));
      return;
    }
    int v = e.vectors - 1 - gl;
    if (U > 2)
      for (; v - (U - 1) * LANES >= 0; v -= U * LANES) some<LANES, true>(v, std::make_integer_sequence<int, U>());
    for (; v >= 0; v -= 2 * LANES) some<LANES, false>(v, std::make_integer_sequence<int, 2>());
  }
};

template <int W>
__device__ __forceinline__ float lanes_max(float m) {
#pragma unroll
  for (int d = W / 2; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  return m;
}
template <int W>
__device__ __forceinline__ float lanes_sum(float s) {
#pragma unroll
  for (int d = W / 2; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  return s;
}

// The vectors at, at + stride, ... into a lane's running (maximum, sum): N of them, or as many as lie less than `left` behind the first
template <int N, bool SHORT>
__device__ __forceinline__ void absorb(const float4* at, int stride, int left, float& top, float& total) {
  float x[4 * N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    float4 q = make_float4(CUDART_INF_F, CUDART_INF_F, CUDART_INF_F, CUDART_INF_F);
    if (k * stride < left) q = ld_plain(at + k * stride);
    x[4 * k] = -q.x;
    x[4 * k + 1] = -q.y;
    x[4 * k + 2] = -q.z;
    x[4 * k + 3] = -q.w;
  }
  float m[4] = {top, -FLT_MAX, -FLT_MAX, -FLT_MAX}, s[4] = {};
#pragma unroll
  for (int k = 0; k < 4 * N; ++k) m[k % 4] = fmaxf(m[k % 4], x[k]);
  const float t = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
#pragma unroll
  for (int k = 0; k < 4 * N; ++k) s[k % 4] += sum_term<SHORT>(x[k] - t);
  total = fmaf(total, expf(top - t), (s[0] + s[1]) + (s[2] + s[3]));
  top = t;
}

struct RowOut {
  float* logp;
  double* logp64;
  float2* stats;
  float* factor;
};
struct Policy {
  const float *old, *adv, *ref;
  const double* inv_n;
  double3* terms;
  float* dz;           // null: no gradient wanted
  PolicyParams q;
};

// What a row's numbers are formed from besides its sums: asked for when the row is, into L1, and loaded when they are needed -- in
// registers meanwhile they would cost the row's loop its place (32 a thread at 2048 threads an SM).
struct RowIn { float z_label, old, adv, ref; double inv_n; };
__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(__cvta_generic_to_global(p))); }
template <bool POLICY>
__device__ __forceinline__ void prefetch_inputs(long long r, const float* row, long long label, const Policy& pol) {
  prefetch(row + label);
  if (POLICY) {
    prefetch(pol.old + r);
    prefetch(pol.adv + r);
    if (pol.ref) prefetch(pol.ref + r);
  }
}
template <bool POLICY>
__device__ __forceinline__ RowIn row_inputs(long long r, bool live, const float* row, long long label, const Policy& pol) {
  RowIn in = {};
  if (live) {
    in.z_label = ld_plain(row + label);
    if (POLICY) {
      in.old = ld_plain(pol.old + r);
      in.adv = ld_plain(pol.adv + r);
      if (pol.ref) in.ref = ld_plain(pol.ref + r);
      in.inv_n = ld_plain(pol.inv_n);
    }
  }
  return in;
}

// The numbers of a row, by one thread; returns the gradient's factor. ROWS rows of a CTA together: their terms of the loss are added in
// a fixed order and leave as one (threads without a row take part in that).
template <bool POLICY, int ROWS>
__device__ __forceinline__ float row_numbers(const float* z, const long long* labels, long long r, bool ok, int J, float2 st, const RowOut& out,
                                             const Policy& pol, double3* sum) {
  const long long label = ok ? ld_plain(labels + r) : -1;
  const bool live = counts(label, J);
  const RowIn in = row_inputs<POLICY>(r, live, z + (ok ? r : 0) * J, label, pol);
  double lp = 0.0;
  float f = 0.f;
  double3 term = make_double3(0, 0, 0);
  if (live) {
    lp = label_logp(in.z_label, st);
    if (POLICY) {
      const PolicyRow p = policy_row(lp, in.old, in.adv, pol.ref != nullptr, in.ref, pol.q);
      f = (float)(p.slope * in.inv_n);
      term = make_double3(p.loss, p.kl, p.clipped ? 1.0 : 0.0);
    }
  }
  if (ok) {
    if (out.logp) out.logp[r] = (float)lp;
    if (out.logp64) out.logp64[r] = lp;
    if (out.stats) out.stats[r] = st;
    if (out.factor) out.factor[r] = f;
  }
  if (POLICY) {
    if (ROWS > 32) {
      term = block_sum(term);
    } else if (ROWS > 1) {
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) {
        term.x += __shfl_xor_sync(0xffffffffu, term.x, d);
        term.y += __shfl_xor_sync(0xffffffffu, term.y, d);
        term.z += __shfl_xor_sync(0xffffffffu, term.z, d);
      }
    }
    if (threadIdx.x == 0) *sum = term;
  }
  return f;
}

// T threads with T / G rows, G lanes to a row: part of a warp, a warp, or the whole CTA.
// HOLD: the row stays in the lanes' registers, NV vectors each; else the lanes go through it NV vectors at a time with a running
// (maximum, sum) each, and for the policy loss once more, from the row's end to its beginning, for the gradient: what was read last is
// still in L1 and L2.
// The rows' numbers are formed together, by one thread a row: in 64 bits they are some 300 instructions at half rate, whether one lane
// of a warp runs them or all (65 536 rows of 1000, a warp each: 35 of 141 us).
// blk: which T / G rows; term: their part of the loss, in thread 0.
template <int T, int G, int NV, bool HOLD, bool POLICY>
__device__ __forceinline__ void rows_of_cta(const float* z, const long long* labels, const RowOut& out, const Policy& pol, long long R, int J,
                                            long long blk, double3* term) {
  static_assert(G <= 32 || (G == T && !HOLD), "a row belongs to part of a warp, a warp or, streamed, the CTA");
  constexpr int kRows = T / G, W = G < 32 ? G : 32, kGradAhead = NV == 8 ? 8 : 2;
  __shared__ float2 stats[kRows > T / 32 ? kRows : T / 32];   // (top, total): of rows, or of a row's warps
  __shared__ float factors[kRows];
  const int tid = threadIdx.x, lane = tid & 31, gl = tid % G, own = tid / G;
  const long long r0 = blk * kRows, r = r0 + own;
  const bool ok = r < R;                       // (of whole groups; all lanes run the shuffles)
  const long long label = ok ? ld_plain(labels + r) : -1;
  const bool live = counts(label, J);
  const float* row = z + (ok ? r : r0) * J;
  // thread t < kRows forms the numbers of row r0 + t
  const long long mine = r0 + tid;
  const bool mine_ok = tid < kRows && mine < R;
  if (mine_ok) {
    const long long l = G == T ? label : ld_plain(labels + mine);
    if (counts(l, J)) prefetch_inputs<POLICY>(mine, z + mine * J, l, pol);
  }

  RowValues<NV> v;
  Ends e(row, J, gl);
  float top = -FLT_MAX, total = 0.f, over = 0.f;
  if constexpr (HOLD) {
    v = load_row<NV>(row, J, live, gl, G);
    float m[4] = {-FLT_MAX, -FLT_MAX, -FLT_MAX, -FLT_MAX}, s[4] = {};
#pragma unroll
    for (int k = 0; k < 4 * NV; ++k) m[k % 4] = fmaxf(m[k % 4], v.x[k]);
    top = lanes_max<W>(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
#pragma unroll
    for (int k = 0; k < 4 * NV; ++k) {
      v.x[k] = sum_term<POLICY>(v.x[k] - top);
      s[k % 4] += v.x[k];
    }
    total = lanes_sum<W>((s[0] + s[1]) + (s[2] + s[3]));
    over = 1.f / total;                        // (here, not behind the barrier: 16 384 rows of 1000 41.0 us, 42.3)
  } else {
    if (live) {
      int v0 = gl;
      if (NV == 8) {
        for (; v0 + (NV - 1) * G < e.vectors; v0 += NV * G) absorb<NV, POLICY>(e.body + v0, G, NV * G, top, total);
        for (; v0 < e.vectors; v0 += 2 * G) absorb<2, POLICY>(e.body + v0, G, e.vectors - v0, top, total);
      } else {
        for (; v0 < e.vectors; v0 += NV * G) absorb<NV, POLICY>(e.body + v0, G, e.vectors - v0, top, total);
      }
      if (e.mine) {
        const float x = -ld_plain(row + e.at), t = fmaxf(top, x);
        total = fmaf(total, expf(top - t), expf(x - t));
        top = t;
      }
    }
    const float t = lanes_max<W>(top);
    total = lanes_sum<W>(total * expf(top - t));
    top = t;
  }
  if (G == T) {
    if (lane == 0) stats[tid >> 5] = make_float2(top, total);
    __syncthreads();
    const float2 p = lane < T / 32 ? stats[lane] : make_float2(-FLT_MAX, 0.f);
    top = lanes_max<32>(p.x);
    total = lanes_sum<32>(p.y * expf(p.x - top));
    if (tid == 0) factors[0] = row_numbers<POLICY, 1>(z, labels, mine, true, J, make_float2(top, total), out, pol, term);
    if (!POLICY) return;
    __syncthreads();
  } else {
    if (gl == 0) stats[own] = make_float2(top, total);
    if (T > 32) __syncthreads(); else __syncwarp();
    if (kRows > 32 || tid < 32) {
      const float f = row_numbers<POLICY, kRows>(z, labels, mine, mine_ok, J, stats[tid < kRows ? tid : 0], out, pol, term);
      if (tid < kRows) factors[tid] = f;
    }
    if (!POLICY) return;
    if (T > 32) __syncthreads(); else __syncwarp();
  }
  if (pol.dz == nullptr || !ok) return;
  const float f = factors[own];
  if constexpr (HOLD) {
    float* to = pol.dz + r * J;
    const float scale = f * over;
#pragma unroll
    for (int k = 0; k < 4 * NV; ++k) v.x[k] = f == 0.f ? 0.f : v.x[k] * scale;
    store_row<NV>(to, row, v, J, label, f, gl, G);
  } else {
    RowGradient{row, (char*)pol.dz - (char*)z, e, top, f == 0.f ? 0.f : f / total, f, (int)label}.template all<G, kGradAhead>(gl);
  }
}

template <int T, int G, int NV, bool HOLD, bool POLICY>
__global__ void __launch_bounds__(T, HOLD || NV == 8 ? 1024 / T : 2048 / T)
choice_rows_kernel(const float* z, const long long* labels, RowOut out, Policy pol, long long R, int J) {
  chain_wait();
  chain_next();
  rows_of_cta<T, G, NV, HOLD, POLICY>(z, labels, out, pol, R, J, blockIdx.x, POLICY ? &pol.terms[blockIdx.x] : nullptr);
}

// The whole policy loss of a few rows: one cluster counts them, takes them in turn and adds their terms. One launch instead of three: 7 us
// instead of 10 to 14 (1024 rows of 10; 128 of 1000: 10.5, 13.7; 4096 of 10, two rounds of the cluster: 10.5, 14.5).
template <int T, int G, int NV>
__global__ void __launch_bounds__(T)
policy_small_kernel(const float* z, const long long* labels, RowOut out, Policy pol, float* __restrict__ loss, float* __restrict__ out2,
                    long long R, int J) {
  chain_wait();
  chain_next();
  __shared__ double inv_n;
  __shared__ double3 term;
  double3 sum = make_double3(0, 0, 0);
  const unsigned n = cluster_count(labels, R, J);
  const double inv = n > 0 ? 1.0 / n : 0.0;
  if (threadIdx.x == 0) inv_n = inv;
  __syncthreads();
  pol.inv_n = &inv_n;
  for (long long blk = blockIdx.x; blk * (T / G) < R; blk += gridDim.x) {
    rows_of_cta<T, G, NV, true, true>(z, labels, out, pol, R, J, blk, &term);
    if (threadIdx.x == 0) {                    // (who has written it)
      sum.x += term.x;
      sum.y += term.y;
      sum.z += term.z;
    }
    __syncthreads();
  }
  sum = cluster_sum(sum);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *loss = (float)(sum.x * inv);
    out2[0] = (float)(sum.y * inv);
    out2[1] = (float)(sum.z * inv);
  }
}

// dz = factor * (p - onehot), from the kept (top, total): no sums, so a row is cut into chunks of a CTA where it is long. From the last
// row to the first: the forward has gone the other way, and what it read last may still be in L2.
template <int T, int G, int NV, bool HOLD>
__global__ void __launch_bounds__(T)
choice_grad_kernel(const float* z, const long long* labels, const float2* stats, const float* factor, const float* gout,
                   float* __restrict__ dz, long long R, int J, int chunks) {
  chain_wait();
  chain_next();
  const int gl = threadIdx.x % G;
  const long long back = G == T ? (long long)(blockIdx.x / chunks) : (long long)blockIdx.x * (T / G) + threadIdx.x / G;
  if (back >= R) return;
  const long long r = R - 1 - back;
  const long long label = ld_plain(labels + r);
  float f = ld_plain(factor + r) * (gout ? ld_plain(gout) : 1.f);
  if (!counts(label, J)) f = 0.f;
  const float2 st = ld_plain(stats + r);
  const float scale = f == 0.f ? 0.f : f / st.y;
  const float* row = z + r * J;
  if constexpr (HOLD) {
    float* to = dz + r * J;
    const int first = G == T ? (int)(blockIdx.x % chunks) * G * NV + gl : gl;
    RowValues<NV> v = load_row<NV>(row, J, f != 0.f, first, G);
#pragma unroll
    for (int k = 0; k < 4 * NV; ++k) v.x[k] = f == 0.f ? 0.f : exp_term(v.x[k] - st.x) * scale;
    store_row<NV>(to, row, v, J, label, f, first, G);
  } else {
    const Ends e(row, J, gl);
    RowGradient{row, (char*)dz - (char*)z, e, st.x, scale, f, (int)label}.template all<G, NV>(gl);
  }
}

// dz *= *gout, unless that is 1 (the loss is the whole objective): then there is nothing to do
__global__ void __launch_bounds__(256) scale_kernel(float* dz, const float* gout, size_t n) {
  chain_wait();
  chain_next();
  const float g = ld_plain(gout);
  if (g == 1.f) return;
  const size_t stride = (size_t)gridDim.x * 256;
  for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < n; e += stride) dz[e] *= g;
}

// rows [first, last) of a text; whatever the caller's numbers are, inside [0, R)
__device__ __forceinline__ void text_rows(const long long* starts, long long rows_per_text, int text, long long R, long long& first,
                                          long long& last) {
  first = starts ? ld_plain(starts + text) : text * rows_per_text;
  last = starts ? ld_plain(starts + text + 1) : first + rows_per_text;
  first = first < 0 ? 0 : first > R ? R : first;
  last = last < first ? first : last > R ? R : last;
}

// A CTA takes a pair at a time: the sums of its two texts, the margin, its loss, and the factors of the texts' rows. A few pairs by one
// cluster, which leaves their mean, too; else one CTA each and their terms.
template <bool FEW>
__global__ void __launch_bounds__(512)
preference_pairs_kernel(const double* lp, const long long* starts, const float* ref, float* __restrict__ margins, float* __restrict__ factor,
                        double* __restrict__ terms, float* __restrict__ loss, long long R, int P, long long rows_per_text, double beta,
                        double smoothing) {
  chain_wait();
  chain_next();
  __shared__ double slope;
  double3 total = make_double3(0, 0, 0);
  for (int k = blockIdx.x; k < P; k += gridDim.x) {
    long long f0, l0, f1, l1;
    text_rows(starts, rows_per_text, k, R, f0, l0);
    text_rows(starts, rows_per_text, P + k, R, f1, l1);
    double3 sum = make_double3(0, 0, 0);
#pragma unroll 4
    for (long long r = f0 + threadIdx.x; r < l0; r += blockDim.x) sum.x += ld_plain(lp + r);
#pragma unroll 4
    for (long long r = f1 + threadIdx.x; r < l1; r += blockDim.x) sum.y += ld_plain(lp + r);
    sum = block_sum(sum);
    if (threadIdx.x == 0) {
      double good = sum.x, bad = sum.y;
      if (ref) { good -= ld_plain(ref + k); bad -= ld_plain(ref + P + k); }
      const double m = beta * (good - bad);
      const double far = log1p(exp(-fabs(m)));                 // -log sigma(|m|)
      // (a margin is infinite where an output at +inf rules a text's label out: a side without weight has no part then, either)
      const double term = (smoothing < 1 ? (1 - smoothing) * (far + fmax(-m, 0.0)) : 0.0) + (smoothing > 0 ? smoothing * (far + fmax(m, 0.0)) : 0.0);
      if (FEW) total.x += term;
      else terms[k] = term;
      margins[k] = (float)m;
      slope = beta / P * (1 / (1 + exp(-m)) - (1 - smoothing));
    }
    __syncthreads();
    const float f = (float)slope;
    for (long long r = f0 + threadIdx.x; r < l0; r += blockDim.x) factor[r] = f;
    for (long long r = f1 + threadIdx.x; r < l1; r += blockDim.x) factor[r] = -f;
    __syncthreads();
  }
  if (FEW) {
    total = cluster_sum(total);
    if (blockIdx.x == 0 && threadIdx.x == 0) *loss = (float)(total.x / P);
  }
}

__global__ void __launch_bounds__(512) mean_kernel(const double* terms, int n, float* __restrict__ mean) {
  chain_wait();
  chain_next();
  double3 s = make_double3(0, 0, 0);
  for (int k = threadIdx.x; k < n; k += blockDim.x) s.x += ld_plain(terms + k);
  s = block_sum(s);
  if (threadIdx.x == 0) *mean = (float)(s.x / n);
}

int check_rows(long long R, int J) {
  if (R <= 0 || J <= 0) return SNNTC_E_SHAPE;
  return R > 0x7fffffffLL || J > (1 << 30) ? SNNTC_E_TOO_LARGE : SNNTC_OK;   // (places in a row are 32-bit numbers)
}

// Longest row whose covering vectors fit `lanes` lanes of nv: rows that all start on 16 bytes fill them, others may begin three
// elements into the first
struct RowShape {
  int J, slack;
  RowShape(const float* z, int J) : J(J), slack((uintptr_t)z % 16 == 0 && J % 4 == 0 ? 0 : 3) {}
  bool fits(int lanes, int nv) const { return J + slack <= 4 * lanes * nv; }
};

template <int T_, int G_, int NV_, bool HOLD_>
struct Lanes {
  static constexpr int T = T_, G = G_, NV = NV_;
  static constexpr bool HOLD = HOLD_;
};
// Calls as() with the kernel's shape for rows of this length.
// Up to 1024 elements: the fewest lanes that hold a row in eight vectors each, as every lane less shares the row's numbers and shuffles
// among more rows (131 072 rows of 125: 37 us with a warp each, 14.6 with four lanes).
// Up to warp_row: a warp that streams. Sums: 16 384 rows of 3001 39 us, 49 by CTAs of 128; of 5000 59, 66. With gradient: 32 768 rows of
// 1500 85 (eight vectors in flight; 90 with four), 111; of 3001 113, 85.
// Then a CTA, the larger the longer the row: what follows a row's last load -- joins, its numbers -- takes a CTA's time whatever its
// size, and the CTAs of an SM should be in different phases. With gradient, 128, 256 and 512 threads: 16 384 rows of 5000 124, 132, 163;
// 8192 of 8000 111, 97, 107; 4096 of 12 000 93, 82, 82.
// Beyond 12 000 eight vectors in flight on half an SM's threads instead of four on all of them, which leaves those 32 registers each:
// 4096 rows of 16 384 46 and 98 us (sums, with gradient), 50 and 102; but 8192 of 9000 64 and 124, 61 and 115.
// With gradient, what the CTAs of all SMs read must still be in L2 when it is read again, so from long_row on they are few and large:
// 4096 rows of 26 000 160 us with 256 threads, 178 with 512; of 32 768 202, 182.
template <int WARP_NV, typename As>
auto by_length(const RowShape& w, int warp_row, int long_row, As as) {
  if (w.fits(1, 4)) return as(Lanes<256, 1, 4, true>{});
  if (w.fits(1, 8)) return as(Lanes<128, 1, 8, true>{});
  if (w.fits(2, 8)) return as(Lanes<128, 2, 8, true>{});
  if (w.fits(4, 8)) return as(Lanes<128, 4, 8, true>{});
  if (w.fits(8, 8)) return as(Lanes<128, 8, 8, true>{});
  if (w.fits(16, 8)) return as(Lanes<128, 16, 8, true>{});
  if (w.fits(32, 8)) return as(Lanes<128, 32, 8, true>{});
  if (w.J <= warp_row) return as(Lanes<256, 32, WARP_NV, false>{});
  if (w.J <= 6000) return as(Lanes<128, 128, 4, false>{});
  if (w.J <= 12000) return as(Lanes<256, 256, 4, false>{});
  if (w.J <= long_row) return as(Lanes<256, 256, 8, false>{});
  return as(Lanes<512, 512, 8, false>{});
}

template <bool POLICY>
int launch_rows(const float* z, const long long* labels, const RowOut& out, const Policy& pol, long long R, int J, cudaStream_t s,
                unsigned* ctas = nullptr) {
  return by_length<(POLICY ? 8 : 4)>(RowShape(z, J), POLICY ? 1800 : 6000, POLICY ? 28000 : 1 << 30, [&](auto lanes) {
    using L = decltype(lanes);
    constexpr int T = L::T, G = L::G;
    const unsigned grid = (unsigned)((R + T / G - 1) / (T / G));
    if (ctas) *ctas = grid;
    (void)launch_chained(choice_rows_kernel<T, G, L::NV, L::HOLD, POLICY>, streaming(grid), T, 0, s, 0, z, labels, out, pol, R, J);
    return done();
  });
}

template <int T, int G, int NV, bool HOLD>
int launch_grad_as(const float* z, const long long* labels, const float* stats, const float* factor, const float* gout, float* dz,
                   long long R, int J, cudaStream_t s) {
  const int chunks = G == T ? (J + RowShape(z, J).slack + 4 * T * NV - 1) / (4 * T * NV) : 1;
  const long long grid = G == T ? R * chunks : (R + T / G - 1) / (T / G);
  if (grid > 0x7fffffffLL) return SNNTC_E_TOO_LARGE;
  (void)launch_chained(choice_grad_kernel<T, G, NV, HOLD>, streaming((unsigned)grid), T, 0, s, 0, z, labels, (const float2*)stats, factor, gout, dz, R, J, chunks);
  return done();
}

// One cluster of up to eight CTAs
unsigned sum_ctas(long long n) { return n >= 8LL * kSumThreads ? 8 : (unsigned)((n + kSumThreads - 1) / kSumThreads); }

}  // namespace

extern "C" {

int snntc_label_logp_forward(const float* z, const long long* labels, float* logp, float* stats_2R, long long R, int J, void* stream) {
  if (!z || !labels || !logp) return SNNTC_E_NULL;
  if (const int rc = check_rows(R, J)) return rc;
  return launch_rows<false>(z, labels, RowOut{logp, nullptr, (float2*)stats_2R, nullptr}, Policy{}, R, J, (cudaStream_t)stream);
}

int snntc_choice_backward(const float* z, const long long* labels, const float* stats_2R, const float* factor, const float* gout,
                          float* dz, long long R, int J, void* stream) {
  if (!z || !labels || !stats_2R || !factor || !dz) return SNNTC_E_NULL;
  if (const int rc = check_rows(R, J)) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  return by_length<4>(RowShape(z, J), 1800, 0, [&](auto lanes) {
    using L = decltype(lanes);
    if constexpr (L::G == L::T) return launch_grad_as<128, 128, 4, true>(z, labels, stats_2R, factor, gout, dz, R, J, s);
    else return launch_grad_as<L::T, L::G, L::NV, L::HOLD>(z, labels, stats_2R, factor, gout, dz, R, J, s);
  });
}

size_t snntc_policy_loss_workspace_bytes(long long R) { return R <= 0 ? 0 : (size_t)R * sizeof(double3) + 256; }

int snntc_policy_loss(const float* z, const long long* labels, const float* old_logp, const float* advantage, const float* ref_logp,
                      float* loss, float* kl_and_clipped, float* stats_2R, float* factor, float* dz, long long R, int J,
                      double clip_low, double clip_high, double kl_coef, void* workspace, size_t workspace_bytes, void* stream) {
  if (!z || !labels || !old_logp || !advantage || !loss || !kl_and_clipped) return SNNTC_E_NULL;
  if (const int rc = check_rows(R, J)) return rc;
  if (!(clip_low >= 0 && clip_low <= 1 && clip_high >= 0 && kl_coef - kl_coef == 0) || (kl_coef != 0 && !ref_logp)) return SNNTC_E_PARAMS;
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < snntc_policy_loss_workspace_bytes(R)) return SNNTC_E_WORKSPACE;
  double* inv_n = (double*)workspace;
  double3* terms = (double3*)((char*)workspace + 256);
  cudaStream_t s = (cudaStream_t)stream;
  Policy pol{old_logp, advantage, ref_logp, inv_n, terms, dz, PolicyParams{1 - clip_low, 1 + clip_high, kl_coef}};
  const RowOut out{nullptr, nullptr, (float2*)stats_2R, factor};
  int rc = SNNTC_OK;
  const bool small = by_length<4>(RowShape(z, J), 0, 0, [&](auto lanes) {
    using L = decltype(lanes);
    if constexpr (L::HOLD) {
      const long long blocks = (R + L::T / L::G - 1) / (L::T / L::G);
      if (blocks > kSmallBlocks) return false;
      const unsigned ctas = blocks < 8 ? (unsigned)blocks : 8;
      (void)launch_chained(policy_small_kernel<L::T, L::G, L::NV>, ctas, L::T, 0, s, ctas, z, labels, out, pol, loss, kl_and_clipped, R, J);
      rc = done();
      return true;
    }
    return false;
  });
  if (small) return rc;
  const unsigned ctas = sum_ctas(R);
  (void)launch_chained(policy_count_kernel, ctas, kSumThreads, 0, s, ctas, labels, inv_n, R, J);
  if ((rc = done())) return rc;
  unsigned n = 0;                              // CTAs, and so terms
  if ((rc = launch_rows<true>(z, labels, out, pol, R, J, s, &n))) return rc;
  (void)launch_chained(policy_mean_kernel, sum_ctas(n), kSumThreads, 0, s, sum_ctas(n), terms, inv_n, loss, kl_and_clipped, (long long)n);
  return done();
}

int snntc_scale_gradient(float* dz, const float* gout, size_t n, void* stream) {
  if (!dz || !gout) return SNNTC_E_NULL;
  if (n == 0) return SNNTC_OK;
  const size_t ctas = (n + 1023) / 1024;
  (void)launch_chained(scale_kernel, (unsigned)(ctas < 1184 ? ctas : 1184), 256, 0, (cudaStream_t)stream, 0, dz, gout, n);
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
  if (const int rc = launch_rows<false>(z, labels, RowOut{nullptr, lp, (float2*)stats_2R, factor}, Policy{}, R, J, s)) return rc;
  const long long each = R / (2LL * P);
  if (P <= kFewPairs) {
    const unsigned ctas = P < 8 ? P : 8;
    (void)launch_chained(preference_pairs_kernel<true>, ctas, 512, 0, s, ctas, lp, starts, ref_logp, margins, factor, terms, loss, R, P, each,
                         beta, smoothing);
    return done();
  }
  (void)launch_chained(preference_pairs_kernel<false>, (unsigned)P, 512, 0, s, 0, lp, starts, ref_logp, margins, factor, terms, loss, R, P, each,
                       beta, smoothing);
  if (const int rc = done()) return rc;
  (void)launch_chained(mean_kernel, 1, 512, 0, s, 0, terms, P, loss);
  return done();
}

}  // extern "C"
