// Embedding of token ids, the input end of a network on tokens, and the gradient of its table.
//
//   forward   y[t,:] = scale * E[id_t,:], or exp(scale * E[id_t,:]) where the rows hold spike times (as the input encoding of
//             snntc_train.cu does for pixels); no_spike where the id is the padding id or outside the table
//   gradient  dE[v,:] = f * sum over the t with id_t = v of g[t,:], in the order of t; f = scale, or scale * exp(scale * E[v,:])
//
// The gradient sorts (id, position) pairs by id -- a least-significant-digit radix sort, stable, so that every id's positions
// stay in order -- and sums runs of equal ids. No atomics on floats: the same bits every run.
#include "../../include/snntc_b200.h"
#include "snntc_launch.cuh"

#include <cuda_runtime.h>
#include <stdint.h>

namespace snntc { void count_launch(int n = 1); void note_cuda_error(cudaError_t e); }

namespace {

using snntc::chain_next;
using snntc::chain_wait;
using snntc::launch_chained;
using snntc::ld_plain;

// Ids of 32 or 64 bits; what is no token of the table becomes V, the largest key.
struct Ids {
  const void* p;
  int wide;
  long long V, padding;
};
__device__ __forceinline__ unsigned key_of(const Ids& ids, long long t) {
  const long long id = ids.wide ? ld_plain((const long long*)ids.p + t) : (long long)ld_plain((const int*)ids.p + t);
  return id < 0 || id >= ids.V || id == ids.padding ? (unsigned)ids.V : (unsigned)id;
}

__device__ __forceinline__ float value_of(float e, float scale, int spikes) { return spikes ? expf(scale * e) : scale * e; }

constexpr int kThreads = 256;

// One CTA per token
__global__ void __launch_bounds__(kThreads)
embed_forward_kernel(Ids ids, const float* table, float* __restrict__ y, int D, float scale, int spikes, float no_spike) {
  chain_wait();
  chain_next();
  const long long t = blockIdx.x;
  const unsigned key = key_of(ids, t);
  float* to = y + t * D;
  const float* row = table + (long long)key * D;
  for (int d = threadIdx.x; d < D; d += kThreads) to[d] = key == (unsigned)ids.V ? no_spike : value_of(ld_plain(row + d), scale, spikes);
}

// ---- sort. Tiles of consecutive keys, one CTA each; a pass is the count of every digit in every tile, then the scatter, whose
// CTAs add up the counts in front of their own.
constexpr int kDigits = 256;
constexpr int kTiles = 148;

struct Keys {                 // the first pass reads the ids, the later ones pairs
  Ids ids;
  const uint2* pairs;         // (key, position)
};
__device__ __forceinline__ uint2 pair_at(const Keys& k, long long t) {
  return k.pairs ? ld_plain(k.pairs + t) : make_uint2(key_of(k.ids, t), (unsigned)t);
}

__global__ void __launch_bounds__(kThreads)
sort_count_kernel(Keys keys, int* __restrict__ counts, long long N, long long tile, int shift) {
  chain_wait();
  chain_next();
  __shared__ int here[kDigits];
  here[threadIdx.x] = 0;
  __syncthreads();
  const long long t0 = blockIdx.x * tile, t1 = min(N, t0 + tile);
  for (long long t = t0 + threadIdx.x; t < t1; t += kThreads) atomicAdd(&here[(pair_at(keys, t).x >> shift) & (kDigits - 1)], 1);
  __syncthreads();
  counts[blockIdx.x * kDigits + threadIdx.x] = here[threadIdx.x];
}

__global__ void __launch_bounds__(kThreads)
sort_scatter_kernel(Keys keys, const int* counts, uint2* __restrict__ out, long long N, long long tile, int tiles, int shift) {
  chain_wait();
  chain_next();
  constexpr int kWarps = kThreads / 32;
  __shared__ int next[kDigits];             // where the next key of a digit goes
  __shared__ int of_warp[kWarps][kDigits];  // keys of a digit in a warp's 32, then those of the warps in front
  __shared__ int warp_sum[kWarps];
  const int d = threadIdx.x, lane = d & 31, warp = d >> 5;
  int before = 0, total = 0;
  for (int k = 0; k < tiles; ++k) {
    const int c = ld_plain(counts + k * kDigits + d);
    if (k < (int)blockIdx.x) before += c;
    total += c;
  }
  int upto = total;                          // inclusive sums of the digits' totals
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, upto, s);
    if (lane >= s) upto += o;
  }
  if (lane == 31) warp_sum[warp] = upto;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) of_warp[w][d] = 0;
  __syncthreads();
  for (int w = 0; w < warp; ++w) upto += warp_sum[w];
  next[d] = upto - total + before;
  const long long t0 = blockIdx.x * tile, t1 = min(N, t0 + tile);
  for (long long t = t0; t < t1; t += kThreads) {
    const bool ok = t + d < t1;
    const uint2 p = ok ? pair_at(keys, t + d) : make_uint2(0, 0);
    const unsigned digit = ok ? (p.x >> shift) & (kDigits - 1) : kDigits;
    const unsigned same = __match_any_sync(0xffffffffu, digit);
    const int rank = __popc(same & ((1u << lane) - 1));
    if (ok && rank == 0) of_warp[warp][digit] = __popc(same);
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int c = of_warp[w][d];
      of_warp[w][d] = sum;
      sum += c;
    }
    __syncthreads();
    if (ok) out[next[digit] + of_warp[warp][digit] + rank] = p;
    __syncthreads();
    next[d] += sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) of_warp[w][d] = 0;
    __syncthreads();
  }
}

// ---- sums of runs: one CTA per place of the sorted pairs; the one at a run's head sums the run
__global__ void __launch_bounds__(kThreads)
embed_run_sums_kernel(const uint2* pairs, const float* g, const float* table, float* __restrict__ dtable, long long N, long long V, int D,
                      float scale, int spikes) {
  chain_wait();
  chain_next();
  const long long i = blockIdx.x;
  const unsigned key = ld_plain(pairs + i).x;
  if (key >= V || (i > 0 && ld_plain(pairs + i - 1).x == key)) return;
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float sum = 0.f;
    for (long long k = i; k < N; ++k) {
      const uint2 p = ld_plain(pairs + k);
      if (p.x != key) break;
      sum += ld_plain(g + (long long)p.y * D + d);
    }
    const float f = spikes ? scale * expf(scale * ld_plain(table + (long long)key * D + d)) : scale;
    dtable[(long long)key * D + d] = f * sum;
  }
}

int done() {
  snntc::count_launch();
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return SNNTC_OK;
  snntc::note_cuda_error(e);
  return SNNTC_E_CUDA;
}

int check_sizes(int id_bytes, long long N, long long V, int D) {
  if (N < 0 || V <= 0 || D <= 0) return SNNTC_E_SHAPE;
  if (id_bytes != 4 && id_bytes != 8) return SNNTC_E_PARAMS;
  return N > 0x7fffffffLL || V >= 0x7fffffffLL ? SNNTC_E_TOO_LARGE : SNNTC_OK;
}

struct SortPlan {
  int tiles, passes;
  long long tile;
};
SortPlan sort_plan(long long N, long long V) {
  SortPlan p;
  p.tile = (N + kTiles - 1) / kTiles;
  p.tile = (p.tile + kThreads - 1) / kThreads * kThreads;
  p.tiles = (int)((N + p.tile - 1) / p.tile);
  p.passes = 1;
  while (p.passes < 4 && (V >> (8 * p.passes)) != 0) ++p.passes;    // keys are 0 .. V
  return p;
}
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

extern "C" {

int snntc_embedding_forward(const void* ids, int id_bytes, const float* table, float* y, long long N, long long V, int D, float scale,
                            int spikes, long long padding, float no_spike, void* stream) {
  if (const int rc = check_sizes(id_bytes, N, V, D)) return rc;
  if (N == 0) return SNNTC_OK;
  if (!ids || !table || !y) return SNNTC_E_NULL;
  (void)launch_chained(embed_forward_kernel, (unsigned)N, kThreads, 0, (cudaStream_t)stream, 0, Ids{ids, id_bytes == 8, V, padding}, table,
                       y, D, scale, spikes, no_spike);
  return done();
}

size_t snntc_embedding_backward_workspace_bytes(long long N, long long V, int D) {
  if (N <= 0 || V <= 0 || D <= 0) return 0;
  return 2 * round256((size_t)N * sizeof(uint2)) + (size_t)kTiles * kDigits * sizeof(int);
}

int snntc_embedding_backward(const void* ids, int id_bytes, const float* g, const float* table, float* dtable, long long N, long long V,
                             int D, float scale, int spikes, long long padding, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check_sizes(id_bytes, N, V, D)) return rc;
  if (!dtable || (N > 0 && (!ids || !g || (spikes && !table)))) return SNNTC_E_NULL;
  if (N > 0 && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < snntc_embedding_backward_workspace_bytes(N, V, D)))
    return SNNTC_E_WORKSPACE;
  cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = cudaMemsetAsync(dtable, 0, (size_t)V * D * sizeof(float), s);
  if (e != cudaSuccess) {
    snntc::note_cuda_error(e);
    return SNNTC_E_CUDA;
  }
  if (N == 0) return SNNTC_OK;
  uint2* pairs[2];
  pairs[0] = (uint2*)workspace;
  pairs[1] = (uint2*)((char*)workspace + round256((size_t)N * sizeof(uint2)));
  int* counts = (int*)((char*)workspace + 2 * round256((size_t)N * sizeof(uint2)));
  const SortPlan p = sort_plan(N, V);
  Keys keys{Ids{ids, id_bytes == 8, V, padding}, nullptr};
  for (int k = 0; k < p.passes; ++k) {
    (void)launch_chained(sort_count_kernel, (unsigned)p.tiles, kThreads, 0, s, 0, keys, counts, N, p.tile, 8 * k);
    if (const int rc = done()) return rc;
    (void)launch_chained(sort_scatter_kernel, (unsigned)p.tiles, kThreads, 0, s, 0, keys, counts, pairs[k & 1], N, p.tile, p.tiles, 8 * k);
    if (const int rc = done()) return rc;
    keys.pairs = pairs[k & 1];
  }
  (void)launch_chained(embed_run_sums_kernel, (unsigned)N, kThreads, 0, s, 0, keys.pairs, g, table, dtable, N, V, D, scale, spikes);
  return done();
}

}  // extern "C"
