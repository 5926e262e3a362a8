// Embedding of token ids, the input end of a network on tokens, and the gradient of its table.
//
//   forward   y[t,:] = scale * E[id_t,:], or exp(scale * E[id_t,:]) where the rows hold spike times (as the input encoding of
//             snntc_train.cu does for pixels); no_spike where the id is the padding id or outside the table
//   gradient  dE[v,:] = f * sum over the t with id_t = v of g[t,:]; f = scale, or scale * exp(scale * E[v,:])
//
// The gradient sorts (id, position) pairs by id -- a least-significant-digit radix sort, stable, so that every id's positions
// stay in order -- and sums runs of equal ids, cut at places that the ids of the call fix. No atomics on floats: the same bits every run.
#include "../../include/snntc_b200.h"
#include "snntc_common.cuh"
#include "snntc_launch.cuh"

#include <cuda_runtime.h>
#include <stdint.h>

namespace {

using snntc::chain_next;
using snntc::chain_wait;
using snntc::done;
using snntc::launch_chained;
using snntc::ld_plain;
using snntc::ld_stream;
using snntc::streaming;

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

// ---- what a lane takes of a row of D as its c-th part: FOUR, four floats loaded as one, where rows and pointers lie on 16 bytes; else ONE,
// or in long rows APART, four that are a warp's width apart, so that the loads of neighbouring lanes are of neighbours and as much is in
// flight (lookup and gradient of 65 536 tokens of 511 values: ONE 55 and 121 us, APART 43 and 108; 131 072 of 129: 35 and 73, 39 and 79).
enum Kind { ONE, FOUR, APART };
constexpr int kApart = 256;              // from this length on
__host__ __device__ constexpr int parts_of(Kind kind, int D) { return kind == FOUR ? D / 4 : kind == ONE ? D : (D + 127) / 128 * 32; }

template <Kind KIND>
struct Part {
  static constexpr int N = KIND == ONE ? 1 : 4;
  float v[N];
};
template <Kind KIND>
__device__ __forceinline__ Part<KIND> load_part(const float* row, int c, int D) {
  if constexpr (KIND == ONE) {
    return {{ld_plain(row + c)}};
  } else if constexpr (KIND == FOUR) {
    const float4 q = ld_plain((const float4*)row + c);
    return {{q.x, q.y, q.z, q.w}};
  } else {
    Part<KIND> q = {};
    const int at = c + (c >> 5) * 96;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + 32 * k < D) q.v[k] = ld_plain(row + at + 32 * k);
    return q;
  }
}
template <Kind KIND>
__device__ __forceinline__ Part<KIND> load_part_once(const float* row, int c, int D) {
  if constexpr (KIND == ONE) {
    return {{ld_stream(row + c)}};
  } else if constexpr (KIND == FOUR) {
    const float4 q = ld_stream((const float4*)row + c);
    return {{q.x, q.y, q.z, q.w}};
  } else {
    Part<KIND> q = {};
    const int at = c + (c >> 5) * 96;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + 32 * k < D) q.v[k] = ld_stream(row + at + 32 * k);
    return q;
  }
}
template <Kind KIND>
__device__ __forceinline__ void store_part(float* row, int c, int D, const Part<KIND>& q) {
  if constexpr (KIND == ONE) {
    row[c] = q.v[0];
  } else if constexpr (KIND == FOUR) {
    ((float4*)row)[c] = make_float4(q.v[0], q.v[1], q.v[2], q.v[3]);
  } else {
    const int at = c + (c >> 5) * 96;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + 32 * k < D) row[at + 32 * k] = q.v[k];
  }
}
template <Kind KIND>
__device__ __forceinline__ void store_part_once(float* row, int c, int D, const Part<KIND>& q) {
  if constexpr (KIND == ONE) {
    __stcs(row + c, q.v[0]);
  } else if constexpr (KIND == FOUR) {
    __stcs((float4*)row + c, make_float4(q.v[0], q.v[1], q.v[2], q.v[3]));
  } else {
    const int at = c + (c >> 5) * 96;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + 32 * k < D) __stcs(row + at + 32 * k, q.v[k]);
  }
}

constexpr int kThreads = 256;
// L lanes to a row of `vectors` parts. A lane has AHEAD rows in flight -- an id and then its row are two loads one behind the other -- and
// of each COLUMNS parts, so that what a row's read opens in memory is read at once. us, (AHEAD, COLUMNS) = (4, 1), (2, 2), (1, 4): 131 072
// rows of 512 values 65.6, 59.6, 61.7; 10^6 of 64 67.8, 92, 123 (one part a lane: the second is never there).
// Of single places (4, 4): 131 072 rows of 201 41 us, 45 with (2, 2).
template <Kind KIND, int AHEAD, int COLUMNS>
__global__ void __launch_bounds__(kThreads)
embed_forward_kernel(Ids ids, const float* table, float* __restrict__ y, long long N, int D, int vectors, int L, float scale, int spikes,
                     float no_spike) {
  chain_wait();
  chain_next();
  const int rows = kThreads / L, gl = threadIdx.x % L;
  const long long t0 = (long long)blockIdx.x * rows * AHEAD + threadIdx.x / L;
  unsigned key[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) key[k] = t0 + k * rows < N ? key_of(ids, t0 + k * rows) : (unsigned)ids.V;
  for (int c0 = gl; c0 < vectors; c0 += COLUMNS * L) {
    Part<KIND> q[AHEAD][COLUMNS];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
      for (int m = 0; m < COLUMNS; ++m)
        if (key[k] != (unsigned)ids.V && c0 + m * L < vectors) q[k][m] = load_part<KIND>(table + (long long)key[k] * D, c0 + m * L, D);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (t0 + k * rows >= N) break;
      const bool token = key[k] != (unsigned)ids.V;
#pragma unroll
      for (int m = 0; m < COLUMNS; ++m) {
        if (c0 + m * L >= vectors) break;
#pragma unroll
        for (int j = 0; j < Part<KIND>::N; ++j) q[k][m].v[j] = token ? value_of(q[k][m].v[j], scale, spikes) : no_spike;
        store_part_once<KIND>(y + (t0 + k * rows) * D, c0 + m * L, D, q[k][m]);
      }
    }
  }
}

// ---- sort. Up to kSmallSort pairs: every pair's place is the number of pairs in front of it, counted by comparison with all. More: tiles
// of consecutive keys, one CTA each; a pass is the count of every digit in every tile, then the scatter, whose CTAs add up the counts in
// front of their own.
constexpr int kSmallSort = 8192;
constexpr int kSortThreads = 512;
constexpr int kDigits = 512;              // of nine bits
constexpr int kTiles = 148;
constexpr int kTileKeys = 2048;           // of a tile at a time

struct Keys {                 // the first pass reads the ids, the later ones pairs
  Ids ids;
  const uint2* pairs;         // (key, position)
};
__device__ __forceinline__ uint2 pair_at(const Keys& k, long long t) {
  return k.pairs ? ld_plain(k.pairs + t) : make_uint2(key_of(k.ids, t), (unsigned)t);
}

// 32 pairs to a CTA, a lane each; a warp counts in its share of the keys, four to a load that all lanes share. An equal key counts
// where its position is lower. One launch against four: the gradient of 300 tokens of 100 values takes 11.4 us so and 17 by the passes, of
// 4000 22.8 and 28, of 8000 33 and 31 -- but three launches less for the host, whose time that is at these sizes (a step of 7007 60, 66).
constexpr int kRankThreads = 512;
__global__ void __launch_bounds__(kRankThreads) sort_small_kernel(Ids ids, uint2* __restrict__ out, int N) {
  chain_wait();
  chain_next();
  constexpr int kWarps = kRankThreads / 32;
  __shared__ __align__(16) unsigned keys[kSmallSort];
  __shared__ int counted[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i0 = blockIdx.x * 32, i = i0 + lane;
  const unsigned key = i < N ? key_of(ids, i) : 0;
  const int share = ((N + kWarps - 1) / kWarps + 3) / 4 * 4, j0 = warp * share, j1 = min(N, j0 + share), end = j0 < N ? (j1 + 3) / 4 * 4 : j0;
#pragma unroll 8
  for (int j = j0 + lane; j < end; j += 32) keys[j] = j < j1 ? key_of(ids, j) : 0xffffffffu;
  __syncwarp();
  int n = 0, m = 0;
  // keys in front of the CTA's own, its own, and those behind (i0 and the shares are multiples of four)
  const int own0 = min(max(i0, j0), end), own1 = min(max(i0 + 32, j0), end);
#pragma unroll 8
  for (int j = j0; j < own0; j += 4) {
    const uint4 q = *(const uint4*)&keys[j];
    n += (q.x <= key) + (q.y <= key);
    m += (q.z <= key) + (q.w <= key);
  }
  for (int j = own0; j < own1; ++j) n += keys[j] < key || (keys[j] == key && j < i);
#pragma unroll 8
  for (int j = own1; j < end; j += 4) {
    const uint4 q = *(const uint4*)&keys[j];
    n += (q.x < key) + (q.y < key);
    m += (q.z < key) + (q.w < key);
  }
  counted[warp][lane] = n + m;
  __syncthreads();
  if (warp == 0 && i < N) {
    int place = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) place += counted[w][lane];
    out[place] = make_uint2(key, (unsigned)i);
  }
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
  constexpr int kWarps = kSortThreads / 32, kEach = kTileKeys / kSortThreads, kOfWarp = 32 * kEach;
  __shared__ int next[kDigits];             // where the next key of a digit goes
  __shared__ int of_warp[kWarps][kDigits];  // keys of a digit in a warp's stretch, then those of the warps in front
  __shared__ int warp_sum[kWarps];
  const int d = threadIdx.x, lane = d & 31, warp = d >> 5;
  const long long t0 = blockIdx.x * tile, t1 = min(N, t0 + tile);
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
  for (long long t = t0; t < t1; t += kTileKeys) {
    // every warp ranks a stretch of its own, 32 keys at a time, against the counts of its earlier ones
    uint2 p[kEach];
    int digit[kEach], rank[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const long long at = t + warp * kOfWarp + k * 32 + lane;
      digit[k] = -1;
      if (at < t1) {
        p[k] = pair_at(keys, at);
        digit[k] = (int)((p[k].x >> shift) & (digits - 1));
      }
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const unsigned same = __match_any_sync(0xffffffffu, digit[k]);
      const int in_front = digit[k] >= 0 ? of_warp[warp][digit[k]] : 0;
      rank[k] = in_front + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (digit[k] >= 0 && (same >> lane) == 1) of_warp[warp][digit[k]] = rank[k] + 1;    // the last lane of its digit
      __syncwarp();
    }
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int c = of_warp[w][d];
      of_warp[w][d] = sum;
      sum += c;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kEach; ++k)
      if (digit[k] >= 0) out[next[digit[k]] + of_warp[warp][digit[k]] + rank[k]] = p[k];
    if (t + kTileKeys >= t1) break;
    __syncthreads();
    next[d] += sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) of_warp[w][d] = 0;
    __syncthreads();
  }
}

// ---- sums of runs of equal keys. What bounds them is memory: g read once, the table's gradient written once (131 072 tokens of 512
// values on as many rows: 537 MB in 92 us, 5.8 TB/s, behind 26 us of sort and before 8 us of joins).
// The sorted pairs are cut into tiles of M; a group of L lanes takes a tile and L parts of the rows, kTermsAhead rows of g in flight.
// Runs inside a tile are done there and then, in the order of t; of one that crosses a border the first tile leaves its part in `tail`, the
// others theirs in `head`, and the joining kernel adds those: one after the other, or in eight interleaved sums where there are more than
// eight. So a token that every second place holds is summed by as many CTAs as its share, in an order that the sorted ids fix: the tokens
// below it move its borders, and with them its last bits. (One CTA for each run: 8.3 ms, most of it the most frequent token's.)
// The sums have 32 bits. In 64, parts and joins included, the error of 131 072 tokens of 512 values falls from 1.1e-7 to 2.3e-8 of the
// gradient's norm (float32's own step is 6e-8), and lookup and gradient take 174 us instead of 167; of 10^6 of 16 on 4096 rows 1.8e-7,
// 2.6e-8, 141 and 128 us.
// Rows that no token names are zeroed by further CTAs of the same launch, a warp for 32 rows or a share of them: each lane looks a row up
// in the sorted keys. (A clearing of the whole table in front would write the named rows twice.)
constexpr int kTermsAhead = 8;
constexpr int kSumTiles = 2048;           // at most, of rows that take a warp

struct RunSums {
  const uint2* pairs;
  const float *g, *table;
  float *dtable, *head, *tail;            // parts: [tiles][D]
  long long N, V;
  int D, vectors, L, slices, M, tiles, sum_ctas, zero_shares;
  float scale;
  int spikes;
};

template <Kind KIND>
__device__ __forceinline__ void write_row(const RunSums& q, unsigned key, int c, Part<KIND> sum) {
  const long long row = (long long)key * q.D;
  if (q.spikes) {
    const Part<KIND> e = load_part<KIND>(q.table + row, c, q.D);
#pragma unroll
    for (int j = 0; j < Part<KIND>::N; ++j) sum.v[j] *= q.scale * expf(q.scale * e.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < Part<KIND>::N; ++j) sum.v[j] *= q.scale;
  }
  store_part<KIND>(q.dtable + row, c, q.D, sum);
}

__device__ void zero_rows(const RunSums& q) {
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)(blockIdx.x - q.sum_ctas) * (kThreads / 32) + (threadIdx.x >> 5), v0 = unit / q.zero_shares * 32;
  const int share = (int)(unit % q.zero_shares);
  if (v0 >= q.V) return;
  // the places [lo, hi) whose keys are of these 32 rows, by 32 probes at a time for each end; then every lane looks for its own in there
  long long lo = 0, hi = 0, step = (q.N + 33) / 33;
  for (long long left = q.N; left > 0; left = step - 1, step = (left + 33) / 33) {
    const long long a = lo + (lane + 1) * step - 1, b = hi + (lane + 1) * step - 1;
    const bool below = a < min(q.N, lo + left) && ld_plain(&q.pairs[a].x) < v0, under = b < min(q.N, hi + left) && ld_plain(&q.pairs[b].x) < v0 + 32;
    lo += __popc(__ballot_sync(0xffffffffu, below)) * step;
    hi += __popc(__ballot_sync(0xffffffffu, under)) * step;
  }
  const long long end = hi;
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if (ld_plain(&q.pairs[mid].x) < v0 + lane) lo = mid + 1;
    else hi = mid;
  }
  const bool empty = v0 + lane < q.V && !(lo < end && ld_plain(&q.pairs[lo].x) == v0 + lane);
  unsigned todo = __ballot_sync(0xffffffffu, empty);
  while (todo) {                          // rows behind one another are one stretch of floats; this warp's share of it, in whole vectors
    const int first = __ffs(todo) - 1, behind = __ffs(~(todo >> first)) - 1, rows = behind < 0 ? 32 : behind;   // (all 32: no bit behind them)
    todo &= rows == 32 ? 0u : ~(((1u << rows) - 1) << first);
    float* at = q.dtable + (v0 + first) * q.D;
    const long long n = (long long)rows * q.D;
    const long long head = min(n, (long long)((4 - ((uintptr_t)at >> 2)) & 3)), vectors = (n - head) / 4, tail = head + 4 * vectors;
    const long long each = (vectors + q.zero_shares - 1) / q.zero_shares, a = share * each, b = min(vectors, a + each);
    for (long long k = a + lane; k < b; k += 32) __stcs((float4*)(at + head) + k, make_float4(0.f, 0.f, 0.f, 0.f));
    if (share == 0) {
      if (lane < head) at[lane] = 0.f;
      if (lane < n - tail) at[tail + lane] = 0.f;
    }
  }
}

template <Kind KIND>
__global__ void __launch_bounds__(kThreads) embed_run_sums_kernel(RunSums q) {
  chain_wait();
  chain_next();
  if ((int)blockIdx.x >= q.sum_ctas) return zero_rows(q);
  const long long unit = ((long long)blockIdx.x * kThreads + threadIdx.x) / q.L;
  const int tile = (int)(unit / q.slices), c = (int)(unit % q.slices) * q.L + threadIdx.x % q.L;
  if (tile >= q.tiles || c >= q.vectors) return;
  const long long i0 = (long long)tile * q.M, i1 = min(q.N, i0 + q.M);
  const unsigned none = 0xffffffffu;
  unsigned key = ld_plain(&q.pairs[i0].x);
  const unsigned after = i1 < q.N ? ld_plain(&q.pairs[i1].x) : none;
  bool from_before = i0 > 0 && ld_plain(&q.pairs[i0 - 1].x) == key;
  Part<KIND> sum = {};
  for (long long i = i0; i < i1; i += kTermsAhead) {
    uint2 p[kTermsAhead];
    Part<KIND> x[kTermsAhead];
#pragma unroll
    for (int k = 0; k < kTermsAhead; ++k) p[k] = i + k < i1 ? ld_plain(q.pairs + i + k) : make_uint2(none, 0);
#pragma unroll
    for (int k = 0; k < kTermsAhead; ++k)
      if (p[k].x < q.V) x[k] = load_part_once<KIND>(q.g + (long long)p[k].y * q.D, c, q.D);
#pragma unroll
    for (int k = 0; k < kTermsAhead; ++k) {
      if (p[k].x == none) break;
      if (p[k].x != key) {
        if (from_before) store_part<KIND>(q.head + (long long)tile * q.D, c, q.D, sum);
        else write_row<KIND>(q, key, c, sum);
        key = p[k].x;
        from_before = false;
        sum = {};
      }
      if (key >= q.V) return;             // what is no token sorts behind all tokens
#pragma unroll
      for (int j = 0; j < Part<KIND>::N; ++j) sum.v[j] += x[k].v[j];
    }
  }
  if (from_before) store_part<KIND>(q.head + (long long)tile * q.D, c, q.D, sum);
  else if (key == after) store_part<KIND>(q.tail + (long long)tile * q.D, c, q.D, sum);
  else write_row<KIND>(q, key, c, sum);
}

// Runs that go on behind the tile in which they begin: a warp looks at a tile and 32 parts, adds a run of a few tiles itself and leaves
// a longer one to all warps of its CTA, every eighth of the tiles each, whose sums are then added in the order of the warps.
template <Kind KIND>
__global__ void __launch_bounds__(kThreads) embed_join_kernel(RunSums q) {
  chain_wait();
  chain_next();
  constexpr int kWarps = kThreads / 32, kFew = 8;
  __shared__ Part<KIND> part[kWarps][32];
  __shared__ int last_tile[kWarps];        // of a run that is left to all; 0: none (a run's last tile is behind its first)
  const int columns = (q.vectors + 31) / 32, tile0 = (int)(blockIdx.x / columns) * kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = (int)(blockIdx.x % columns) * 32 + lane;
  const auto head_of = [&](int t) { return load_part<KIND>(q.head + (long long)t * q.D, c, q.D); };
  const auto add = [](Part<KIND>& sum, const Part<KIND>& x) {
#pragma unroll
    for (int j = 0; j < Part<KIND>::N; ++j) sum.v[j] += x.v[j];
  };
  {
    const int tile = tile0 + warp;
    const long long i0 = (long long)tile * q.M, i1 = i0 + q.M;
    int last = 0;
    unsigned key = 0;
    if (i1 < q.N) {
      key = ld_plain(&q.pairs[i1 - 1].x);
      const unsigned after = ld_plain(&q.pairs[i1].x), before = i0 > 0 ? ld_plain(&q.pairs[i0 - 1].x) : 0xffffffffu;
      if (key < q.V && after == key && before != key) {
        last = tile + 1;                   // the last tile that begins with this key, by 32 probes at a time
        for (int left = q.tiles - 1 - last, step = (left + 33) / 33; left > 0; left = step - 1, step = (left + 33) / 33) {
          const int t = last + (lane + 1) * step;
          const bool same = t <= last + left && t < q.tiles && ld_plain(&q.pairs[(long long)t * q.M].x) == key;
          last += __popc(__ballot_sync(0xffffffffu, same)) * step;
        }
      }
    }
    if (last && last - tile <= kFew) {
      if (c < q.vectors) {
        Part<KIND> sum = load_part<KIND>(q.tail + (long long)tile * q.D, c, q.D);
#pragma unroll 4
        for (int t = tile + 1; t <= last; ++t) add(sum, head_of(t));
        write_row<KIND>(q, key, c, sum);
      }
      last = 0;
    }
    if (lane == 0) last_tile[warp] = last;
  }
  __syncthreads();
  for (int k = 0; k < kWarps; ++k) {
    const int last = last_tile[k], tile = tile0 + k;
    if (last == 0) continue;
    Part<KIND> sum = {};
    if (c < q.vectors)
#pragma unroll 8
      for (int t = tile + 1 + warp; t <= last; t += kWarps) add(sum, head_of(t));
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < q.vectors) {
      sum = load_part<KIND>(q.tail + (long long)tile * q.D, c, q.D);
      for (int w = 0; w < kWarps; ++w) add(sum, part[w][lane]);
      write_row<KIND>(q, ld_plain(&q.pairs[(long long)tile * q.M + q.M - 1].x), c, sum);
    }
    __syncthreads();
  }
}

int check_sizes(int id_bytes, long long N, long long V, int D) {
  if (N < 0 || V <= 0 || D <= 0) return SNNTC_E_SHAPE;
  if (id_bytes != 4 && id_bytes != 8) return SNNTC_E_PARAMS;
  return N > 0x7fffffffLL || V >= 0x7fffffffLL || D > (1 << 30) ? SNNTC_E_TOO_LARGE : SNNTC_OK;   // (places in a row are 32-bit numbers)
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
  p.tile = (p.tile + kTileKeys - 1) / kTileKeys * kTileKeys;
  p.tiles = (int)((N + p.tile - 1) / p.tile);
  return p;
}

// Places per tile of the sums: eight, one round of loads, or as many as make kSumTiles tiles; narrow rows, a few lanes each, take more tiles
// (131 072 tokens of 4 values 54 us, 63 with as many as wide ones; of 64 52, 58)
int sum_tile(long long N, int D) {
  int lanes = 1;
  while (lanes < 32 && lanes < parts_of(D % 4 == 0 ? FOUR : D >= kApart ? APART : ONE, D)) lanes *= 2;
  const long long tiles = (long long)kSumTiles * (lanes < 4 ? 8 : 32 / lanes), m = (N + tiles - 1) / tiles;
  return (int)((m + kTermsAhead - 1) / kTermsAhead * kTermsAhead);
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

struct SortSpace {                      // of the radix sort, besides the sorted pairs
  size_t other, counts, bytes;
  explicit SortSpace(long long N, size_t at = 0) {
    other = at;
    counts = other + round256((size_t)N * sizeof(uint2));
    bytes = counts + (size_t)kTiles * kDigits * sizeof(int);
  }
};

struct BackwardSpace {
  size_t pairs, head, tail, bytes;
  SortSpace sort;
  BackwardSpace(long long N, int D) : pairs(0), sort(N, round256((size_t)N * sizeof(uint2))) {
    const size_t tiles = (size_t)((N + sum_tile(N, D) - 1) / sum_tile(N, D)), parts = round256(tiles * D * sizeof(float));
    head = sort.bytes;
    tail = head + parts;
    bytes = tail + parts;
  }
};

// The radix sort of the pairs: `sorted` receives them, `other` and `counts` are scratch. urgent: beside a kernel that fills the GPU, whose
// CTAs still to come would otherwise all go first.
int launch_sort(const Ids& ids, long long N, long long V, uint2* sorted, uint2* other, int* counts, bool urgent, cudaStream_t s) {
  const SortPlan p = sort_plan(N, V);
  int least = 0, greatest = 0;
  if (urgent) (void)cudaDeviceGetStreamPriorityRange(&least, &greatest);
  bool first = true;
  const auto launch = [&](auto kernel, auto... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.tiles);
    cfg.blockDim = dim3(kSortThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // (the kernels are written for it, see launch_chained)
    attr[0].val.programmaticStreamSerializationAllowed = (long)p.tiles * kSortThreads <= snntc::kChainThreads && !(urgent && first);
    first = false;                          // (what the first one on a stream of the library's waits for is an event)
    attr[1].id = cudaLaunchAttributePriority;
    attr[1].val.priority = greatest;
    cfg.attrs = attr;
    cfg.numAttrs = urgent ? 2 : 1;
    (void)cudaLaunchKernelEx(&cfg, kernel, args...);
    return done();
  };
  Keys keys{ids, nullptr};
  for (int k = 0; k < p.passes; ++k) {
    uint2* to = (p.passes - 1 - k) % 2 ? other : sorted;                  // the last pass's is `sorted`
    if (const int rc = launch(sort_count_kernel, keys, counts, N, p.tile, p.bits * k, 1 << p.bits)) return rc;
    if (const int rc = launch(sort_scatter_kernel, keys, (const int*)counts, to, N, p.tile, p.tiles, p.bits * k, 1 << p.bits)) return rc;
    keys.pairs = to;
  }
  return SNNTC_OK;
}

template <Kind KIND>
int launch_sums(RunSums q, cudaStream_t s) {
  q.vectors = parts_of(KIND, q.D);
  q.L = 1;
  while (q.L < 32 && q.L < q.vectors) q.L *= 2;
  q.slices = (q.vectors + q.L - 1) / q.L;
  q.sum_ctas = (int)(((long long)q.tiles * q.slices * q.L + kThreads - 1) / kThreads);
  // a warp zeroes up to 32 KB: 32 rows, or a share of them (8 KB: 131 072 tokens of 512 145 us instead of 131, each share looks its rows up)
  q.zero_shares = (q.D + 255) / 256;
  const long long zero_ctas = ((q.V + 31) / 32 * q.zero_shares + kThreads / 32 - 1) / (kThreads / 32);
  (void)launch_chained(embed_run_sums_kernel<KIND>, (unsigned)(q.sum_ctas + zero_ctas), kThreads, 0, s, 0, q);
  if (const int rc = done()) return rc;
  if (q.tiles == 1) return SNNTC_OK;
  (void)launch_chained(embed_join_kernel<KIND>, (unsigned)((q.tiles + 7) / 8 * ((q.vectors + 31) / 32)), kThreads, 0, s, 0, q);
  return done();
}

// Whether the sort goes beside the lookup: that has to last for some time to hide it. us, lookup and gradient together, beside and one
// after the other: 131 072 tokens of 512 values 173, 193, 20 000 of 1024 98, 102; 131 072 of 30 73, 69, 9000 of 64 73, 69 (the events).
bool sorts_beside(long long N, int D) { return N > kSmallSort && N * D >= (4LL << 20); }

int launch_lookup(const Ids& in, const float* table, float* y, long long N, int D, float scale, int spikes, float no_spike, cudaStream_t s) {
  const Kind kind = by_four(D, table, y, nullptr) ? FOUR : D >= kApart ? APART : ONE;
  const int vectors = parts_of(kind, D);
  int L = 1;                                // lanes to a row: up to a warp
  while (L < 32 && L < vectors) L *= 2;
  const auto launch = [&](auto kernel, int ahead) {
    const long long rows = (long long)kThreads / L * ahead;
    (void)launch_chained(kernel, streaming((unsigned)((N + rows - 1) / rows)), kThreads, 0, s, 0, in, table, y, N, D, vectors, L, scale, spikes, no_spike);
    return done();
  };
  if (vectors <= 32) return kind == FOUR ? launch(embed_forward_kernel<FOUR, 4, 1>, 4) : launch(embed_forward_kernel<ONE, 4, 1>, 4);
  return kind == FOUR  ? launch(embed_forward_kernel<FOUR, 2, 2>, 2)
         : kind == ONE ? launch(embed_forward_kernel<ONE, 4, 4>, 4)
                       : launch(embed_forward_kernel<APART, 2, 2>, 2);
}

}  // namespace

extern "C" {

int snntc_embedding_forward(const void* ids, int id_bytes, const float* table, float* y, long long N, long long V, int D, float scale,
                            int spikes, long long padding, float no_spike, void* stream) {
  if (const int rc = check_sizes(id_bytes, N, V, D)) return rc;
  if (N == 0) return SNNTC_OK;
  if (!ids || !table || !y) return SNNTC_E_NULL;
  return launch_lookup(Ids{ids, id_bytes == 8, V, padding}, table, y, N, D, scale, spikes, no_spike, (cudaStream_t)stream);
}

size_t snntc_embedding_sorted_bytes(long long N, int D) { return sorts_beside(N, D) ? (size_t)N * sizeof(uint2) : 0; }
size_t snntc_embedding_sort_workspace_bytes(long long N, int D) { return sorts_beside(N, D) ? SortSpace(N).bytes : 0; }

int snntc_embedding_forward_sort(const void* ids, int id_bytes, const float* table, float* y, long long N, long long V, int D, float scale,
                                 int spikes, long long padding, float no_spike, void* sorted, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (!sorts_beside(N, D)) return snntc_embedding_forward(ids, id_bytes, table, y, N, V, D, scale, spikes, padding, no_spike, stream);
  if (const int rc = check_sizes(id_bytes, N, V, D)) return rc;
  if (!ids || !table || !y || !sorted) return SNNTC_E_NULL;
  if (!workspace || (uintptr_t)workspace % 256 || (uintptr_t)sorted % 256 || workspace_bytes < snntc_embedding_sort_workspace_bytes(N, D))
    return SNNTC_E_WORKSPACE;
  cudaStream_t s = (cudaStream_t)stream, side = s;
  const Ids in{ids, id_bytes == 8, V, padding};
  const SortSpace w(N);
  snntc::AuxSlot* aux = snntc::aux_acquire(-1, s);
  if (aux) {
    const cudaError_t e = snntc::aux_fork(aux, s);
    if (e != cudaSuccess) {
      snntc::note_cuda_error(e);
      return SNNTC_E_CUDA;
    }
    side = aux->stream;
  }
  int rc = launch_sort(in, N, V, (uint2*)sorted, (uint2*)((char*)workspace + w.other), (int*)((char*)workspace + w.counts), aux != nullptr, side);
  if (rc == SNNTC_OK) rc = launch_lookup(in, table, y, N, D, scale, spikes, no_spike, s);
  if (aux) {                                // on every path: a stream under capture must not be left forked
    const cudaError_t e = snntc::aux_join(aux, s);
    if (e != cudaSuccess && rc == SNNTC_OK) {
      snntc::note_cuda_error(e);
      rc = SNNTC_E_CUDA;
    }
  }
  return rc;
}

size_t snntc_embedding_backward_workspace_bytes(long long N, long long V, int D) {
  if (N <= 0 || V <= 0 || D <= 0) return 0;
  return BackwardSpace(N, D).bytes;
}

int snntc_embedding_backward(const void* ids, int id_bytes, const void* sorted, const float* g, const float* table, float* dtable,
                             long long N, long long V, int D, float scale, int spikes, long long padding, void* workspace,
                             size_t workspace_bytes, void* stream) {
  if (const int rc = check_sizes(id_bytes, N, V, D)) return rc;
  if (!dtable || (N > 0 && ((!ids && !sorted) || !g || (spikes && !table)))) return SNNTC_E_NULL;
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
  uint2* pairs = (uint2*)(base + w.pairs);
  const Ids in{ids, id_bytes == 8, V, padding};
  if (sorted) {
    pairs = (uint2*)sorted;
  } else if (N <= kSmallSort) {
    (void)launch_chained(sort_small_kernel, (unsigned)((N + 31) / 32), kRankThreads, 0, s, 0, in, pairs, (int)N);
    if (const int rc = done()) return rc;
  } else if (const int rc = launch_sort(in, N, V, pairs, (uint2*)(base + w.sort.other), (int*)(base + w.sort.counts), false, s)) {
    return rc;
  }
  RunSums q = {};
  q.pairs = pairs;
  q.g = g;
  q.table = table;
  q.dtable = dtable;
  q.head = (float*)(base + w.head);
  q.tail = (float*)(base + w.tail);
  q.N = N;
  q.V = V;
  q.D = D;
  q.M = sum_tile(N, D);
  q.tiles = (int)((N + q.M - 1) / q.M);
  q.scale = scale;
  q.spikes = spikes;
  if (by_four(D, g, dtable, spikes ? table : nullptr)) return launch_sums<FOUR>(q, s);
  return D >= kApart ? launch_sums<APART>(q, s) : launch_sums<ONE>(q, s);
}

}  // extern "C"
