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

// ---- vectors of VEC floats: 4 where rows and pointers allow it, else 1
template <int VEC> struct Vec;
template <> struct Vec<1> {
  float v[1];
  static __device__ __forceinline__ Vec load(const float* p) { return {{ld_plain(p)}}; }
  static __device__ __forceinline__ Vec load_once(const float* p) { return {{__ldcs(p)}}; }
  __device__ __forceinline__ void store(float* p) const { *p = v[0]; }
};
template <> struct Vec<4> {
  float v[4];
  static __device__ __forceinline__ Vec of(float4 q) { return {{q.x, q.y, q.z, q.w}}; }
  static __device__ __forceinline__ Vec load(const float* p) { return of(ld_plain((const float4*)p)); }
  static __device__ __forceinline__ Vec load_once(const float* p) { return of(__ldcs((const float4*)p)); }
  __device__ __forceinline__ void store(float* p) const { *(float4*)p = make_float4(v[0], v[1], v[2], v[3]); }
};

constexpr int kThreads = 256;
constexpr int kRowsAhead = 4;

// L lanes to a row of `vectors` vectors, kRowsAhead rows of a lane in flight: the id and then its row are two loads one behind the other.
template <int VEC>
__global__ void __launch_bounds__(kThreads)
embed_forward_kernel(Ids ids, const float* table, float* __restrict__ y, long long N, int D, int vectors, int L, float scale, int spikes,
                     float no_spike) {
  chain_wait();
  chain_next();
  const int rows = kThreads / L, gl = threadIdx.x % L;
  const long long t0 = (long long)blockIdx.x * rows * kRowsAhead + threadIdx.x / L;
  unsigned key[kRowsAhead];
#pragma unroll
  for (int k = 0; k < kRowsAhead; ++k) key[k] = t0 + k * rows < N ? key_of(ids, t0 + k * rows) : (unsigned)ids.V;
  for (int c = gl; c < vectors; c += L) {
    Vec<VEC> q[kRowsAhead];
#pragma unroll
    for (int k = 0; k < kRowsAhead; ++k)
      if (key[k] != (unsigned)ids.V) q[k] = Vec<VEC>::load(table + (long long)key[k] * D + c * VEC);
#pragma unroll
    for (int k = 0; k < kRowsAhead; ++k) {
      if (t0 + k * rows >= N) break;
      const bool token = key[k] != (unsigned)ids.V;
#pragma unroll
      for (int j = 0; j < VEC; ++j) q[k].v[j] = token ? value_of(q[k].v[j], scale, spikes) : no_spike;
      q[k].store(y + (t0 + k * rows) * D + c * VEC);
    }
  }
}

// ---- sort. Up to kSmallSort pairs by one CTA in shared memory. More: tiles of consecutive keys, one CTA each; a pass is the count of every
// digit in every tile, then the scatter, whose CTAs add up the counts in front of their own.
constexpr int kSmallSort = 4096;
constexpr int kSortThreads = 512;
constexpr int kDigits = 512;              // of nine bits
constexpr int kTiles = 148;
constexpr int kTileKeys = 2048;           // at least

struct Keys {                 // the first pass reads the ids, the later ones pairs
  Ids ids;
  const uint2* pairs;         // (key, position)
};
__device__ __forceinline__ uint2 pair_at(const Keys& k, long long t) {
  return k.pairs ? ld_plain(k.pairs + t) : make_uint2(key_of(k.ids, t), (unsigned)t);
}

// A bitonic network over (key << 32 | position): keys in order, equal ones by position.
__global__ void __launch_bounds__(1024) sort_small_kernel(Ids ids, uint2* __restrict__ out, int N, int size) {
  chain_wait();
  chain_next();
  __shared__ unsigned long long s[kSmallSort];
  for (int t = threadIdx.x; t < size; t += 1024) s[t] = t < N ? (unsigned long long)key_of(ids, t) << 32 | (unsigned)t : ~0ull;
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < size / 2; i += 1024) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const unsigned long long x = s[a], y = s[b];
        if ((x > y) == ((a & k) == 0)) { s[a] = y; s[b] = x; }
      }
    }
  __syncthreads();
  for (int t = threadIdx.x; t < N; t += 1024) out[t] = make_uint2((unsigned)(s[t] >> 32), (unsigned)s[t]);
}

__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(Keys keys, int* __restrict__ counts, long long N, long long tile, int shift, int digits) {
  chain_wait();
  chain_next();
  __shared__ int here[kDigits];
  here[threadIdx.x] = 0;
  __syncthreads();
  const long long t0 = blockIdx.x * tile, t1 = min(N, t0 + tile);
  for (long long t = t0 + threadIdx.x; t < t1; t += kSortThreads) atomicAdd(&here[(pair_at(keys, t).x >> shift) & (digits - 1)], 1);
  __syncthreads();
  counts[blockIdx.x * kDigits + threadIdx.x] = here[threadIdx.x];
}

__global__ void __launch_bounds__(kSortThreads)
sort_scatter_kernel(Keys keys, const int* counts, uint2* __restrict__ out, long long N, long long tile, int tiles, int shift, int digits) {
  chain_wait();
  chain_next();
  constexpr int kWarps = kSortThreads / 32;
  __shared__ int next[kDigits];             // where the next key of a digit goes
  __shared__ int of_warp[kWarps][kDigits];  // keys of a digit in a warp's 32, then those of the warps in front
  __shared__ int warp_sum[kWarps];
  const int d = threadIdx.x, lane = d & 31, warp = d >> 5;
  int before = 0, total = 0;
#pragma unroll 16
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
  for (long long t = t0; t < t1; t += kSortThreads) {
    const bool ok = t + d < t1;
    const uint2 p = ok ? pair_at(keys, t + d) : make_uint2(0, 0);
    const unsigned digit = ok ? (p.x >> shift) & (digits - 1) : kDigits;
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

// ---- sums of runs of equal keys. The sorted pairs are cut into tiles of M; a group of L lanes takes a tile and L vectors of the rows,
// kTermsAhead rows of g in flight. Runs inside a tile are done there and then; of one that crosses a border the first tile leaves its
// part in `tail`, the others theirs in `head`, and the joining kernel adds those in order. So a token that every second place holds is
// summed by as many CTAs as its share, and the order of summation depends on the sizes alone.
// Rows that no token names are zeroed by further CTAs of the same launch, a warp for 32 rows: each lane looks its row up in the sorted keys.
constexpr int kTermsAhead = 8;
constexpr int kSumTiles = 2048;           // at most

struct RunSums {
  const uint2* pairs;
  const float *g, *table;
  float *dtable, *head, *tail;            // parts: [tiles][D]
  long long N, V;
  int D, vectors, L, slices, M, tiles, sum_ctas;
  float scale;
  int spikes;
};

template <int VEC>
__device__ __forceinline__ void write_row(const RunSums& q, unsigned key, int c, Vec<VEC> sum) {
  const long long at = (long long)key * q.D + (long long)c * VEC;
  if (q.spikes) {
    const Vec<VEC> e = Vec<VEC>::load(q.table + at);
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum.v[j] *= q.scale * expf(q.scale * e.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum.v[j] *= q.scale;
  }
  sum.store(q.dtable + at);
}

template <int VEC>
__device__ void zero_rows(const RunSums& q) {
  const int lane = threadIdx.x & 31;
  const long long v0 = ((long long)(blockIdx.x - q.sum_ctas) * (kThreads / 32) + (threadIdx.x >> 5)) * 32;
  if (v0 >= q.V) return;
  long long lo = 0, hi = q.N;             // the first place whose key is not below the lane's row
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if (ld_plain(&q.pairs[mid].x) < v0 + lane) lo = mid + 1;
    else hi = mid;
  }
  const bool empty = v0 + lane < q.V && !(lo < q.N && ld_plain(&q.pairs[lo].x) == v0 + lane);
  const unsigned todo = __ballot_sync(0xffffffffu, empty);
  const Vec<VEC> zero = {};
  if (q.vectors >= 32) {
    for (unsigned m = todo; m; m &= m - 1) {
      float* row = q.dtable + (v0 + __ffs(m) - 1) * q.D;
      for (int c = lane; c < q.vectors; c += 32) zero.store(row + c * VEC);
    }
  } else if (todo) {                      // short rows: the 32 of them are one stretch
    float* rows = q.dtable + v0 * q.D;
    for (int e = lane; e < 32 * q.vectors; e += 32)
      if (todo >> (e / q.vectors) & 1) zero.store(rows + e * VEC);
  }
}

template <int VEC>
__global__ void __launch_bounds__(kThreads) embed_run_sums_kernel(RunSums q) {
  chain_wait();
  chain_next();
  if ((int)blockIdx.x >= q.sum_ctas) return zero_rows<VEC>(q);
  const long long unit = ((long long)blockIdx.x * kThreads + threadIdx.x) / q.L;
  const int tile = (int)(unit / q.slices), c = (int)(unit % q.slices) * q.L + threadIdx.x % q.L;
  if (tile >= q.tiles || c >= q.vectors) return;
  const long long i0 = (long long)tile * q.M, i1 = min(q.N, i0 + q.M);
  const unsigned none = 0xffffffffu;
  unsigned key = ld_plain(&q.pairs[i0].x);
  const unsigned after = i1 < q.N ? ld_plain(&q.pairs[i1].x) : none;
  bool from_before = i0 > 0 && ld_plain(&q.pairs[i0 - 1].x) == key;
  Vec<VEC> sum = {};
  for (long long i = i0; i < i1; i += kTermsAhead) {
    uint2 p[kTermsAhead];
    Vec<VEC> x[kTermsAhead];
#pragma unroll
    for (int k = 0; k < kTermsAhead; ++k) p[k] = i + k < i1 ? ld_plain(q.pairs + i + k) : make_uint2(none, 0);
#pragma unroll
    for (int k = 0; k < kTermsAhead; ++k)
      if (p[k].x < q.V) x[k] = Vec<VEC>::load_once(q.g + (long long)p[k].y * q.D + c * VEC);
#pragma unroll
    for (int k = 0; k < kTermsAhead; ++k) {
      if (p[k].x == none) break;
      if (p[k].x != key) {
        if (from_before) sum.store(q.head + (long long)tile * q.D + c * VEC);
        else write_row<VEC>(q, key, c, sum);
        key = p[k].x;
        from_before = false;
        sum = {};
      }
      if (key >= q.V) return;             // what is no token sorts behind all tokens
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum.v[j] += x[k].v[j];
    }
  }
  if (from_before) sum.store(q.head + (long long)tile * q.D + c * VEC);
  else if (key == after) sum.store(q.tail + (long long)tile * q.D + c * VEC);
  else write_row<VEC>(q, key, c, sum);
}

// One CTA per tile; it has work where a run begins in the tile and goes on behind it.
template <int VEC>
__global__ void __launch_bounds__(kThreads) embed_join_kernel(RunSums q) {
  chain_wait();
  chain_next();
  constexpr int kWarps = kThreads / 32;
  __shared__ Vec<VEC> part[kWarps][32];
  const int tile = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long i0 = (long long)tile * q.M, i1 = i0 + q.M;
  if (i1 >= q.N) return;
  const unsigned key = ld_plain(&q.pairs[i1 - 1].x);
  if (key >= q.V || ld_plain(&q.pairs[i1].x) != key || (i0 > 0 && ld_plain(&q.pairs[i0 - 1].x) == key)) return;
  int lo = tile + 1, hi = q.tiles - 1;     // the last tile that begins with this key
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (ld_plain(&q.pairs[(long long)mid * q.M].x) == key) lo = mid;
    else hi = mid - 1;
  }
  for (int c0 = 0; c0 < q.vectors; c0 += 32) {
    const int c = c0 + lane;
    Vec<VEC> sum = {};
    if (c < q.vectors)
#pragma unroll 8
      for (int t = tile + 1 + warp; t <= lo; t += kWarps) {
        const Vec<VEC> x = Vec<VEC>::load(q.head + (long long)t * q.D + c * VEC);
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum.v[j] += x.v[j];
      }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < q.vectors) {
      sum = Vec<VEC>::load(q.tail + (long long)tile * q.D + c * VEC);
      for (int w = 0; w < kWarps; ++w)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum.v[j] += part[w][lane].v[j];
      write_row<VEC>(q, key, c, sum);
    }
    __syncthreads();
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

bool by_four(int D, const void* a, const void* b, const void* c) {
  return D % 4 == 0 && ((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) % 16 == 0;
}

struct SortPlan {
  int tiles, passes, bits;
  long long tile;
};
SortPlan sort_plan(long long N, long long V) {
  SortPlan p;
  int bits = 1;
  while (V >> bits) ++bits;                 // keys are 0 .. V
  p.passes = (bits + 8) / 9;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.tile = (N + kTiles - 1) / kTiles;
  if (p.tile < kTileKeys) p.tile = kTileKeys;
  p.tile = (p.tile + kSortThreads - 1) / kSortThreads * kSortThreads;
  p.tiles = (int)((N + p.tile - 1) / p.tile);
  return p;
}

// Places per tile of the sums: 32, or as many as make kSumTiles tiles
int sum_tile(long long N) {
  const long long m = (N + kSumTiles - 1) / kSumTiles;
  return (int)(m < 32 ? 32 : (m + 7) / 8 * 8);
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

struct BackwardSpace {
  size_t pairs[2], counts, head, tail, bytes;
  BackwardSpace(long long N, int D) {
    const size_t tiles = (size_t)((N + sum_tile(N) - 1) / sum_tile(N)), parts = round256(tiles * D * sizeof(float));
    pairs[0] = 0;
    pairs[1] = round256((size_t)N * sizeof(uint2));
    counts = 2 * pairs[1];
    head = counts + (size_t)kTiles * kDigits * sizeof(int);
    tail = head + parts;
    bytes = tail + parts;
  }
};

template <int VEC>
int launch_sums(RunSums q, cudaStream_t s) {
  q.vectors = q.D / VEC;
  q.L = 1;
  while (q.L < 32 && q.L < q.vectors) q.L *= 2;
  q.slices = (q.vectors + q.L - 1) / q.L;
  q.sum_ctas = (int)(((long long)q.tiles * q.slices * q.L + kThreads - 1) / kThreads);
  const long long zero_ctas = (q.V + kThreads - 1) / kThreads;
  (void)launch_chained(embed_run_sums_kernel<VEC>, (unsigned)(q.sum_ctas + zero_ctas), kThreads, 0, s, 0, q);
  if (const int rc = done()) return rc;
  if (q.tiles == 1) return SNNTC_OK;
  (void)launch_chained(embed_join_kernel<VEC>, (unsigned)q.tiles, kThreads, 0, s, 0, q);
  return done();
}

}  // namespace

extern "C" {

int snntc_embedding_forward(const void* ids, int id_bytes, const float* table, float* y, long long N, long long V, int D, float scale,
                            int spikes, long long padding, float no_spike, void* stream) {
  if (const int rc = check_sizes(id_bytes, N, V, D)) return rc;
  if (N == 0) return SNNTC_OK;
  if (!ids || !table || !y) return SNNTC_E_NULL;
  const bool four = by_four(D, table, y, nullptr);
  const int vectors = four ? D / 4 : D;
  int L = 1;                                // lanes to a row: the power of two that leaves the fewest of them idle, a warp's width at least
  for (int l = 2; l <= kThreads; l *= 2) {
    const auto lanes = [&](int n) { return (vectors + n - 1) / n * n; };
    if (L < 32 ? L < vectors : lanes(l) <= lanes(L)) L = l;
  }
  const long long rows = (long long)kThreads / L * kRowsAhead, ctas = (N + rows - 1) / rows;
  const Ids in{ids, id_bytes == 8, V, padding};
  if (four) (void)launch_chained(embed_forward_kernel<4>, (unsigned)ctas, kThreads, 0, (cudaStream_t)stream, 0, in, table, y, N, D, vectors, L, scale, spikes, no_spike);
  else (void)launch_chained(embed_forward_kernel<1>, (unsigned)ctas, kThreads, 0, (cudaStream_t)stream, 0, in, table, y, N, D, vectors, L, scale, spikes, no_spike);
  return done();
}

size_t snntc_embedding_backward_workspace_bytes(long long N, long long V, int D) {
  if (N <= 0 || V <= 0 || D <= 0) return 0;
  return BackwardSpace(N, D).bytes;
}

int snntc_embedding_backward(const void* ids, int id_bytes, const float* g, const float* table, float* dtable, long long N, long long V,
                             int D, float scale, int spikes, long long padding, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check_sizes(id_bytes, N, V, D)) return rc;
  if (!dtable || (N > 0 && (!ids || !g || (spikes && !table)))) return SNNTC_E_NULL;
  if (N > 0 && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < snntc_embedding_backward_workspace_bytes(N, V, D)))
    return SNNTC_E_WORKSPACE;
  cudaStream_t s = (cudaStream_t)stream;
  if (N == 0) {
    const cudaError_t e = cudaMemsetAsync(dtable, 0, (size_t)V * D * sizeof(float), s);
    if (e != cudaSuccess) snntc::note_cuda_error(e);
    return e == cudaSuccess ? SNNTC_OK : SNNTC_E_CUDA;
  }
  const BackwardSpace w(N, D);
  char* base = (char*)workspace;
  uint2* pairs[2] = {(uint2*)(base + w.pairs[0]), (uint2*)(base + w.pairs[1])};
  const Ids in{ids, id_bytes == 8, V, padding};
  Keys keys{in, nullptr};
  if (N <= kSmallSort) {
    int size = 2;
    while (size < N) size *= 2;
    (void)launch_chained(sort_small_kernel, 1, 1024, 0, s, 0, in, pairs[0], (int)N, size);
    if (const int rc = done()) return rc;
    keys.pairs = pairs[0];
  } else {
    const SortPlan p = sort_plan(N, V);
    int* counts = (int*)(base + w.counts);
    for (int k = 0; k < p.passes; ++k) {
      (void)launch_chained(sort_count_kernel, (unsigned)p.tiles, kSortThreads, 0, s, 0, keys, counts, N, p.tile, p.bits * k, 1 << p.bits);
      if (const int rc = done()) return rc;
      (void)launch_chained(sort_scatter_kernel, (unsigned)p.tiles, kSortThreads, 0, s, 0, keys, counts, pairs[k & 1], N, p.tile, p.tiles, p.bits * k, 1 << p.bits);
      if (const int rc = done()) return rc;
      keys.pairs = pairs[k & 1];
    }
  }
  RunSums q = {};
  q.pairs = keys.pairs;
  q.g = g;
  q.table = table;
  q.dtable = dtable;
  q.head = (float*)(base + w.head);
  q.tail = (float*)(base + w.tail);
  q.N = N;
  q.V = V;
  q.D = D;
  q.M = sum_tile(N);
  q.tiles = (int)((N + q.M - 1) / q.M);
  q.scale = scale;
  q.spikes = spikes;
  return by_four(D, g, dtable, spikes ? table : nullptr) ? launch_sums<4>(q, s) : launch_sums<1>(q, s);
}

}  // extern "C"
