// g2v_embed.hip -- embedding lookup with scaling, and its gradient.
//
//   y[i]  = scale * W[ids[i]]                       (zero row: ids[i] not in [0, V))
//   dW[v] = scale * sum over i with ids[i] == v of dy[i]
//
// GGIPNN's lookup (src/GGIPNN.py:19-25) and, for train_embedding=True there, the
// gradient of its table.
#include <type_traits>

#include "g2v_counts.h"
#include "g2v_ops.h"

namespace {

using g2v::bf16;
using g2v::f16;

constexpr int kThreads = 256;

// workgroups are numbered over two grid dimensions: one holds 2^32 threads
inline dim3 grid_of(int64_t blocks) {
  const int64_t x = blocks < 1 << 20 ? blocks : 1 << 20;
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
__device__ __forceinline__ int64_t block_number() {
  return (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
}

constexpr int kUnits = 4;  // vectors a thread of the lookup moves

// Rows are moved in vectors of VEC elements, 16 bytes of one of the types.  A
// row of D elements is ceil(D / VEC) vectors; the last one ends with the row and
// overlaps the one before where VEC does not divide D (the same values are
// written twice), so that no width needs a scalar tail.  Rows narrower than a
// vector go element by element.
//
// Memory bound: a row read and a row written per token, no reuse.  Vectors of
// all rows are numbered through and dealt out 1024 to a workgroup, so every
// width fills the lanes and one row is spread over as many threads as it has
// vectors; kUnits independent id -> row chains per thread cover the latency.
// The result goes past the caches, which keep the table's rows instead:
// 262,144 rows of 512 fp32 from 60,000 take 114 us, with ordinary stores 174;
// 65,536 of 4,096 bf16 from 131,072 148 us (4.7 TB/s), 159 with ordinary ones.
template <class TW, class TY, class I, int VEC>
__global__ __launch_bounds__(kThreads) void k_embed_lookup(
    const TW* __restrict__ W, int64_t V, int D, int64_t ld, const I* __restrict__ ids,
    int64_t units, int nv, float scale, TY* __restrict__ out) {
  const int64_t u0 = block_number() * (kThreads * kUnits);
  const int64_t row0 = units <= UINT32_MAX ? (uint32_t)u0 / (uint32_t)nv : u0 / nv;
  const uint32_t r0 = (uint32_t)(u0 - row0 * nv) + threadIdx.x;  // < nv + 1024
  const int64_t left = units - u0;
  int64_t id[kUnits], at[kUnits];
  int col[kUnits];
  float x[kUnits][VEC];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const uint32_t l = r0 + k * kThreads, q = l / (uint32_t)nv;
    const int c = (int)(l - q * nv) * VEC;
    col[k] = c + VEC <= D ? c : D - VEC;
    at[k] = row0 + q;
    id[k] = (int)threadIdx.x + k * kThreads < left ? (int64_t)ids[at[k]] : -1;
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[k][i] = 0.f;
    if (id[k] >= 0 && id[k] < V) {
      g2v::load_vec<TW, VEC>(W + id[k] * ld + col[k], x[k]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[k][i] *= scale;
    }
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k)
    if ((int)threadIdx.x + k * kThreads < left)
      g2v::store_vec_nt<TY, VEC>(out + at[k] * D + col[k], x[k]);
}

// ---- the gradient: tokens sorted by row, then one sum per row --------------------
//
// The sort is stable (tokens of a row stay in token order) and uses no atomics
// on memory, so the order of every sum, and with it the result, is fixed.
// Rows are dealt to kBuckets buckets by their low bits: frequent rows, mostly
// neighbours in a vocabulary sorted by count, fall into different buckets.
// Inside a bucket a workgroup counts its rows in LDS, wave by wave over
// consecutive slices of the tokens, scans the counts and places the tokens.
//
// Up to kScanTokens tokens every bucket's workgroup reads all ids itself: it
// lists its own in LDS and counts those of lower buckets, which is where its
// part of the sorted list begins.  One launch, no exchange between workgroups
// (16,384 tokens: 23 us for the gradient, 30 the other way).
// Beyond that the tokens are split into buckets first (tile counts, then a
// stable scatter), and every workgroup reads its bucket alone; a bucket of more
// than kHotTokens, as a very frequent row makes it, is cut into parts that are
// counted first and then placed by workgroups of their own (262,144 tokens of
// one row: 117 us for the gradient of 24,447 x 200, 245 without).

constexpr int kBuckets = 256;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kKeys = 1024;         // rows a bucket counts at a time (64 KB of LDS)
constexpr int kListBits = 10;       // tokens a wave lists: 2^10 (64 KB of LDS in all, what
                                    // the counts leave room for; 20,000 tokens the other
                                    // way take 31 us where 16,384 take 22)
constexpr int kScanTokens = kSortWaves << kListBits;
constexpr int64_t kScanRows = (int64_t)kBuckets << (32 - kListBits);  // a list entry's row
constexpr int kTileTokens = 1024;   // 65,536 tokens: 42 us, 45 with 4096
constexpr int kMaxTiles = 256;      // larger calls take larger tiles
constexpr int kHotTokens = 4096;    // of a bucket for one workgroup; n / 1024 if more
constexpr int kPer = 2;             // G vectors of a row that one group takes
constexpr int kJoinBlocks = 512;

struct Sorted {
  int32_t* perm;    // [n] token positions, row by row
  int2* rows;       // first place in perm and tokens of every row, bucket by bucket
  int32_t* at;      // [n / L + 1] row at every L-th place of perm
  int32_t* longs;   // [n / L + 1] rows of more than L tokens, bucket by bucket
  int32_t* nlong;   // [kBuckets] how many of them
  int32_t* lfirst;  // [kBuckets] where the bucket's begin
  int32_t* total;   // tokens that name a row
  int log2L;
  int per_bucket;   // rows of a bucket: the stride of `rows`
  // a bucket's workgroup writes one stretch; by row it would write 8 bytes of
  // every 256th line that other workgroups write too
  __device__ __forceinline__ int64_t slot(int v) const {
    return (int64_t)(v % kBuckets) * per_bucket + v / kBuckets;
  }
  __device__ __forceinline__ int2 row(int v) const { return rows[slot(v)]; }
};

// the lanes of the wave whose key equals this lane's, among those that have one
__device__ __forceinline__ uint64_t peers(int key, bool has, int bits) {
  uint64_t m = __ballot(has);
  for (int b = 0; b < bits; ++b) {
    const bool one = (key >> b) & 1;
    const uint64_t o = __ballot(one);
    m &= one ? o : ~o;
  }
  return m;
}

// f(i, key(i)) for the tokens [i0, i1) in order, 64 at a time by a whole wave,
// -1 past the end; four loads in flight
template <class K, class F>
__device__ __forceinline__ void for_slice(int64_t i0, int64_t i1, K key, F f) {
  const int lane = threadIdx.x & 63;
  for (int64_t i = i0; i < i1; i += 256) {
    int k[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t j = i + u * 64 + lane;
      k[u] = j < i1 ? key(j) : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) f(i + u * 64 + lane, k[u]);
  }
}

// the slice of n tokens that this wave takes: whole groups of 64, in wave order
__device__ __forceinline__ void my_slice(int64_t n, int64_t& i0, int64_t& i1) {
  const int64_t per = (n + kSortThreads - 1) / kSortThreads * 64;
  i0 = (int64_t)(threadIdx.x / 64) * per;
  i0 = i0 < n ? i0 : n;
  i1 = i0 + per < n ? i0 + per : n;
}

// exclusive sum over the workgroup, and the sum in all
__device__ __forceinline__ int block_scan(int x, int& all) {
  __shared__ int wsum[kSortWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  int s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int t = __shfl_up(s, d);
    if (lane >= d) s += t;
  }
  if (lane == 63) wsum[wave] = s;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    if (w < wave) before += wsum[w];
    all += wsum[w];
  }
  __syncthreads();
  return before + s - x;
}

// Where one key is most of the wave (a bucket with a very frequent row) it is
// cheaper to take whole keys out one by one than to compare bit by bit: taken
// by the lowest lane left, first once, then while few lanes are left.
constexpr int kFewLanes = 6;

__device__ __forceinline__ uint64_t peers_skewed(int key, bool has, int bits) {
  uint64_t left = __ballot(has), mine = 0;
  bool first = true;
  while (left && (first || __popcll(left) <= kFewLanes)) {
    const int k = __builtin_amdgcn_readlane(key, __builtin_ctzll(left));
    const bool in = has && key == k;
    const uint64_t same = __ballot(in);
    mine = in ? same : mine;
    left &= ~same;
    first = false;
  }
  if (left) {
    const bool rest = left >> (threadIdx.x & 63) & 1;
    const uint64_t m = peers(key, rest, bits);
    mine = rest ? m : mine;
  }
  return mine;
}

// next[key] += the wave's tokens of that key; the most frequent key, often
// that of the first lane, with one access
__device__ __forceinline__ void count_keys(uint32_t* next, int key, bool has) {
  const uint64_t m = __ballot(has);
  if (!m) return;
  const int lead = __builtin_ctzll(m), k = __builtin_amdgcn_readlane(key, lead);
  const uint64_t same = __ballot(has && key == k);
  if ((int)(threadIdx.x & 63) == lead) atomicAdd(&next[key], (uint32_t)__popcll(same));
  else if (has && key != k) atomicAdd(&next[key], 1u);
}

// the place of this lane's token: next[key] plus the lower lanes of that key
// (m: all of them); next[key] moves on by all of them
__device__ __forceinline__ int place_keys(uint32_t* next, int key, bool has, uint64_t m) {
  const int lane = threadIdx.x & 63;
  const int lead = has ? __builtin_ctzll(m) : lane;
  int old = 0;
  if (has && lead == lane) old = (int)atomicAdd(&next[key], (uint32_t)__popcll(m));
  return __shfl(old, lead) + __popcll(m & ((1ull << lane) - 1));
}

// Sorts tokens of bucket b, which begins at place base.  tokens(f) calls
// f(position, key) for this wave's tokens in order, a whole wave at a time; key:
// the row over kBuckets, -1 for a lane without a token.  They are the bucket's
// tokens, or part `part` of `parts` of them: then counts holds the tokens of
// every key in every part (kKeys each; only where the bucket has no more rows).
// The first part writes what is known of the rows.  Returns the bucket's end.
template <class T>
__device__ __forceinline__ int sort_bucket(int b, int V, int base, const Sorted& s, int part,
                                           int parts, const int32_t* __restrict__ counts,
                                           T tokens) {
  __shared__ uint32_t hist[kSortWaves * kKeys];
  __shared__ int nlong;
  const int rows = g2v::rows_of_bucket(V, b, kBuckets);
  const int first = base >> s.log2L, t = threadIdx.x;
  uint32_t* mine = hist + (t / 64) * kKeys;
  if (t == 0) nlong = 0;
  for (int w0 = 0; w0 < rows; w0 += kKeys) {
    const int rw = rows - w0 < kKeys ? rows - w0 : kKeys;
    const int bits = rw > 1 ? 32 - __builtin_clz(rw - 1) : 0;
    if (t < rw)
      for (int w = 0; w < kSortWaves; ++w) hist[w * kKeys + t] = 0;
    __syncthreads();
    tokens([&](int, int k) { count_keys(mine, k - w0, k >= w0 && k < w0 + rw); });
    __syncthreads();
    int c = 0, before = 0, all;
    if (t < rw) {
      if (parts > 1) {
#pragma unroll 8
        for (int q = 0; q < parts; ++q) {
          const int x = counts[q * kKeys + t];
          c += x;
          before += q < part ? x : 0;
        }
      } else {
        for (int w = 0; w < kSortWaves; ++w) c += (int)hist[w * kKeys + t];
      }
    }
    const int start = base + block_scan(c, all);
    if (t < rw) {
      if (part == 0) {
        const int v = (w0 + t) * kBuckets + b;
        s.rows[(int64_t)b * s.per_bucket + w0 + t] = make_int2(start, c);
        if (c > 1 << s.log2L) s.longs[first + atomicAdd(&nlong, 1)] = v;
      }
      int at = start + before;
      for (int w = 0; w < kSortWaves; ++w) {
        const int h = (int)hist[w * kKeys + t];
        hist[w * kKeys + t] = (uint32_t)at;
        at += h;
      }
    }
    __syncthreads();
    tokens([&](int i, int k) {
      const bool has = k >= w0 && k < w0 + rw;
      if (!__ballot(has)) return;
      const int p = place_keys(mine, k - w0, has, peers_skewed(k - w0, has, bits));
      if (!has) return;
      s.perm[p] = i;
      if ((p & ((1 << s.log2L) - 1)) == 0) s.at[p >> s.log2L] = k * kBuckets + b;
    });
    base += all;
    __syncthreads();
  }
  if (t == 0 && part == 0) {
    s.nlong[b] = rows ? nlong : 0;
    s.lfirst[b] = first;
    if (b == kBuckets - 1) *s.total = base;
  }
  return base;
}

// the row of a token, -1 if it names none or the padding
template <class I>
__device__ __forceinline__ int row_of(const I* __restrict__ ids, int64_t i, int V, int pad) {
  const int64_t id = (int64_t)ids[i];
  return id >= 0 && id < V && id != pad ? (int)id : -1;
}

template <class I>
__global__ __launch_bounds__(kSortThreads) void k_sort_scan(const I* __restrict__ ids, int n, int V,
                                                            int pad, Sorted s) {
  __shared__ uint32_t list[kSortWaves << kListBits];  // key << kListBits | position - i0
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  int64_t i0, i1;
  my_slice(n, i0, i1);
  uint32_t* mine = list + ((threadIdx.x / 64) << kListBits);
  int below = 0, mine_n = 0;
  for_slice(i0, i1, [&](int64_t i) { return row_of(ids, i, V, pad); },
            [&](int64_t i, int v) {
              const int d = v & (kBuckets - 1);
              const bool has = v >= 0 && d == b;
              below += v >= 0 && d < b;
              const uint64_t m = __ballot(has);
              if (!m) return;
              if (has)
                mine[mine_n + __popcll(m & ((1ull << lane) - 1))] =
                    (uint32_t)(v / kBuckets) << kListBits | (uint32_t)(i - i0);
              mine_n += __popcll(m);
            });
  int base;
  (void)block_scan(below, base);
  sort_bucket(b, V, base, s, 0, 1, nullptr, [&](auto f) {
    for (int j = lane; j - lane < mine_n; j += 64) {
      const bool in = j < mine_n;
      const uint32_t e = in ? mine[j] : 0;
      f((int)i0 + (int)(e & ((1 << kListBits) - 1)), in ? (int)(e >> kListBits) : -1);
    }
  });
}

// tokens of every bucket in every tile
template <class I>
__global__ __launch_bounds__(kSortThreads) void k_tile_count(const I* __restrict__ ids, int64_t n,
                                                             int64_t tile, int V, int pad,
                                                             int32_t* __restrict__ counts) {
  __shared__ uint32_t hist[kSortWaves * kBuckets];
  const int64_t t0 = (int64_t)blockIdx.x * tile, len = n - t0 < tile ? n - t0 : tile;
  for (int k = threadIdx.x; k < kSortWaves * kBuckets; k += kSortThreads) hist[k] = 0;
  __syncthreads();
  int64_t i0, i1;
  my_slice(len, i0, i1);
  uint32_t* mine = hist + (threadIdx.x / 64) * kBuckets;
  for_slice(i0, i1, [&](int64_t i) { return row_of(ids, t0 + i, V, pad); },
            [&](int64_t, int v) {
              if (v >= 0) atomicAdd(&mine[v & (kBuckets - 1)], 1u);
            });
  __syncthreads();
  if (threadIdx.x < kBuckets) {
    uint32_t c = 0;
    for (int w = 0; w < kSortWaves; ++w) c += hist[w * kBuckets + threadIdx.x];
    counts[blockIdx.x * kBuckets + threadIdx.x] = (int32_t)c;
  }
}

// the tokens as (row, position), bucket by bucket, in token order within one
template <class I>
__global__ __launch_bounds__(kSortThreads) void k_tile_scatter(
    const I* __restrict__ ids, int64_t n, int64_t tile, int V, int pad,
    const int32_t* __restrict__ counts, int32_t* __restrict__ bfirst, int2* __restrict__ pairs) {
  __shared__ uint32_t hist[kSortWaves * kBuckets];
  __shared__ int tsum[2][kSortThreads / kBuckets][kBuckets];
  const int64_t t0 = (int64_t)blockIdx.x * tile, len = n - t0 < tile ? n - t0 : tile;
  for (int k = threadIdx.x; k < kSortWaves * kBuckets; k += kSortThreads) hist[k] = 0;
  const int d = threadIdx.x % kBuckets, g = threadIdx.x / kBuckets;
  int before = 0, every = 0;
#pragma unroll 16
  for (int t = g; t < (int)gridDim.x; t += kSortThreads / kBuckets) {
    const int c = counts[t * kBuckets + d];
    every += c;
    before += t < (int)blockIdx.x ? c : 0;
  }
  tsum[0][g][d] = before;
  tsum[1][g][d] = every;
  __syncthreads();
  int64_t i0, i1;
  my_slice(len, i0, i1);
  uint32_t* mine = hist + (threadIdx.x / 64) * kBuckets;
  for_slice(i0, i1, [&](int64_t i) { return row_of(ids, t0 + i, V, pad); },
            [&](int64_t, int v) {
              if (v >= 0) atomicAdd(&mine[v & (kBuckets - 1)], 1u);
            });
  before = every = 0;
  if (threadIdx.x < kBuckets)
    for (int q = 0; q < kSortThreads / kBuckets; ++q) {
      before += tsum[0][q][d];
      every += tsum[1][q][d];
    }
  int all;
  const int b0 = block_scan(every, all);  // the bucket's first place (a barrier inside)
  if (threadIdx.x < kBuckets) {
    if (blockIdx.x == 0) {
      bfirst[d] = b0;
      if (d == 0) bfirst[kBuckets] = all;
    }
    uint32_t at = (uint32_t)(b0 + before);
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t h = hist[w * kBuckets + d];
      hist[w * kBuckets + d] = at;
      at += h;
    }
  }
  __syncthreads();
  for_slice(i0, i1, [&](int64_t i) { return row_of(ids, t0 + i, V, pad); },
            [&](int64_t i, int v) {
              if (!__ballot(v >= 0)) return;
              const int d = v & (kBuckets - 1);
              const int p = place_keys(mine, d, v >= 0, peers(d, v >= 0, 8));
              if (v >= 0) pairs[p] = make_int2(v, (int)(t0 + i));
            });
}

// The parts of the buckets of more than `hot` tokens, numbered through.
struct Part {
  int bucket, part, parts, first;  // first: the number of the bucket's part 0
};

__device__ __forceinline__ bool part_of(const int32_t* __restrict__ bfirst, int hot, int number,
                                        Part& p) {
  __shared__ Part found;
  int c = 0, all;
  if (threadIdx.x < kBuckets) {
    const int n = bfirst[threadIdx.x + 1] - bfirst[threadIdx.x];
    c = n > hot ? g2v::pieces(n, hot) : 0;
  }
  const int before = block_scan(c, all);
  if (number >= before && number < before + c)
    found = {(int)threadIdx.x, number - before, c, before};
  __syncthreads();
  if (number >= all) return false;
  p = found;
  return true;
}

__global__ __launch_bounds__(kSortThreads) void k_hot_count(const int2* __restrict__ pairs,
                                                            const int32_t* __restrict__ bfirst,
                                                            int hot, int32_t* __restrict__ counts) {
  __shared__ uint32_t hist[kKeys];
  Part p;
  if (!part_of(bfirst, hot, blockIdx.x, p)) return;
  hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t lo = bfirst[p.bucket] + (int64_t)p.part * hot, end = bfirst[p.bucket + 1];
  const int64_t len = end - lo < hot ? end - lo : hot;
  int64_t i0, i1;
  my_slice(len, i0, i1);
  for_slice(i0, i1, [&](int64_t i) { return pairs[lo + i].x / kBuckets; },
            [&](int64_t, int k) { count_keys(hist, k, k >= 0); });
  __syncthreads();
  counts[blockIdx.x * kKeys + threadIdx.x] = (int32_t)hist[threadIdx.x];
}

// the first workgroups: a part of a hot bucket each, as they take longest; the
// last kBuckets: a bucket that is not hot
__global__ __launch_bounds__(kSortThreads) void k_sort_bucket(const int2* __restrict__ pairs,
                                                              const int32_t* __restrict__ bfirst,
                                                              int V, int hot,
                                                              const int32_t* __restrict__ counts,
                                                              Sorted s) {
  const int cold = (int)blockIdx.x - ((int)gridDim.x - kBuckets);
  Part p{cold, 0, 1, 0};
  if (cold < 0 && !part_of(bfirst, hot, blockIdx.x, p)) return;
  const int base = bfirst[p.bucket], end = bfirst[p.bucket + 1];
  if (cold >= 0 && end - base > hot) return;
  const int64_t lo = base + (p.parts > 1 ? (int64_t)p.part * hot : 0);
  const int64_t len = end - lo < hot ? end - lo : hot;
  int64_t i0, i1;
  my_slice(len, i0, i1);
  sort_bucket(p.bucket, V, base, s, p.part, p.parts, counts + (int64_t)p.first * kKeys,
              [&](auto f) {
    const int lane = threadIdx.x & 63;
    for (int64_t i = i0; i < i1; i += 256) {
      int2 e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t j = i + u * 64 + lane;
        e[u] = j < i1 ? pairs[lo + j] : make_int2(-1, 0);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) f(e[u].y, e[u].x < 0 ? -1 : e[u].x / kBuckets);
    }
  });
}

// acc += the rows perm[p0 .. p1) of dy, in that order, eight loads in flight
template <class TY, int VEC>
__device__ __forceinline__ void sum_rows(const TY* __restrict__ dy, int64_t ld,
                                         const int32_t* __restrict__ perm, int p0, int p1,
                                         float (&acc)[VEC]) {
  auto some = [&](auto many) {
    constexpr int M = decltype(many)::value;
    int64_t r[M];
    float x[M][VEC];
#pragma unroll
    for (int m = 0; m < M; ++m) r[m] = perm[p0 + m];
#pragma unroll
    for (int m = 0; m < M; ++m) g2v::load_vec<TY, VEC>(dy + r[m] * ld, x[m]);
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += x[m][i];
    p0 += M;
  };
  while (p1 - p0 >= 8) some(std::integral_constant<int, 8>{});
  if ((p1 - p0) & 4) some(std::integral_constant<int, 4>{});
  if ((p1 - p0) & 2) some(std::integral_constant<int, 2>{});
  if ((p1 - p0) & 1) some(std::integral_constant<int, 1>{});
}

// G lanes per row; the sum of a row of at most L tokens goes to grad, of none
// zeros.  Memory bound by dy's rows and the whole of grad.  A group takes kPer
// times G vectors of a row, so that the many rows without a token are written by
// fewer groups that live long enough to pay for reading the count: the gradient
// of 16,384 tokens of 131,072 x 4,096 bf16 takes 272 us at 1, 247 at 2, 257 at 4;
// with ordinary stores, not past the caches, 268 at 2 (all with pieces of 64
// tokens; 237 with the 256 of today).  221 us are this kernel (1.2 GB, 5.4 TB/s;
// 160 where dy is still in the Infinity Cache, which is what filling a tensor of
// that size takes).
//
// A longer run is cut at every L-th of its tokens into pieces, first in the grid
// as they take longest and G vectors a group; their sums go to part.  Pieces are
// found by place: a run of more than L tokens that begins in [cL, cL + L) covers
// the place (c + 1) L, and one that begins before cL and has a piece there
// covers cL.  So slot 2c is the first piece of the run that begins there, slot
// 2c + 1 a later piece of one that began before; each exists at most once, as
// two such runs begin more than L places apart.
template <class TY, class TG, int VEC, int G>
__global__ __launch_bounds__(kThreads) void k_grad_rows(const TY* __restrict__ dy, int64_t ld,
                                                        Sorted s, float* __restrict__ part,
                                                        int64_t V, int D, int nv, int tiles,
                                                        int64_t slots, float scale,
                                                        TG* __restrict__ grad) {
  const int64_t it = block_number() * (kThreads / G) + threadIdx.x / G;
  const int lane = threadIdx.x % G, L = 1 << s.log2L;
  float acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  if (it < slots * tiles) {
    const int64_t slot = tiles == 1 ? it : it / tiles;
    const int unit = (int)(it - slot * tiles) * G + lane;
    if (unit >= nv) return;
    const int col = unit * VEC + VEC <= D ? unit * VEC : D - VEC;
    const int c = (int)(slot >> 1), later = (int)(slot & 1);
    const int64_t q = (int64_t)(c + 1 - later) << s.log2L;
    if (q >= *s.total) return;
    const int2 run = s.row(s.at[c + 1 - later]);
    const int p = run.x, n = run.y;
    if (n <= L) return;
    int p0 = p;
    if (later) {
      if (p >= q) return;
      const int64_t e = p + ((q - p + L - 1) >> s.log2L << s.log2L);
      if (e >= (int64_t)p + n) return;
      p0 = (int)e;
    } else if (p >> s.log2L != c) {
      return;
    }
    sum_rows<TY, VEC>(dy + col, ld, s.perm, p0, p + n - p0 > L ? p0 + L : p + n, acc);
    g2v::store_vec<float, VEC>(part + slot * D + col, acc);
    return;
  }
  const int64_t r = it - slots * tiles;
  const int parts = (tiles + kPer - 1) / kPer;
  const int64_t v = parts == 1 ? r : r / parts;
  if (v >= V) return;
  const int2 run = s.row((int)v);
  const int p = run.x, n = run.y;
  if (n > L) return;
  const int first = (int)(r - v * parts) * kPer * G;
  if (n == 0) {  // zeros, 16 bytes a lane side by side, whatever VEC is
    constexpr int Z = VEC * sizeof(TG) > 16 ? 16 / sizeof(TG) : VEC;
    const float zero[Z] = {};
    const int end = (first + kPer * G) * VEC < D ? (first + kPer * G) * VEC : D;
    for (int c = first * VEC + lane * Z; c < end; c += G * Z)
      g2v::store_vec_nt<TG, Z>(grad + v * D + (c + Z <= D ? c : D - Z), zero);
    return;
  }
  int unit = first + lane;
  for (int k = 0; k < kPer && unit < nv; ++k, unit += G) {
    const int col = unit * VEC + VEC <= D ? unit * VEC : D - VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    sum_rows<TY, VEC>(dy + col, ld, s.perm, p, p + n, acc);
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] *= scale;
    g2v::store_vec_nt<TG, VEC>(grad + v * D + col, acc);
  }
}

// The pieces of the long runs: kSortWaves waves add every kSortWaves-th piece of
// a run in order, the first wave those sums.  A workgroup takes 64 vectors of
// every gridDim.x-th long run; it numbers them itself, bucket by bucket.
template <class TG, int VEC>
__global__ __launch_bounds__(kSortThreads) void k_grad_join(Sorted s,
                                                            const float* __restrict__ part, int D,
                                                            int nv, float scale,
                                                            TG* __restrict__ grad) {
  __shared__ float sums[kSortWaves][64][VEC];
  __shared__ int before[kBuckets];
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  int all;
  const int mine = threadIdx.x < kBuckets ? s.nlong[threadIdx.x] : 0;
  const int sum = block_scan(mine, all);
  if (threadIdx.x < kBuckets) before[threadIdx.x] = sum;
  __syncthreads();
  const int unit = (int)blockIdx.y * 64 + lane;
  const bool in = unit < nv;
  const int col = !in ? 0 : unit * VEC + VEC <= D ? unit * VEC : D - VEC;
  for (int j = blockIdx.x; j < all; j += gridDim.x) {
    int b = 0;  // the last bucket with before[b] <= j: it holds run j
    for (int d = kBuckets / 2; d; d >>= 1)
      if (before[b + d] <= j) b += d;
    const int v = s.longs[s.lfirst[b] + j - before[b]];
    const int2 run = s.row(v);
    const int pieces = g2v::pieces_log2(run.y, s.log2L);
    const int64_t c0 = run.x >> s.log2L;
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    if (in) {
#pragma unroll 4
      for (int k = wave; k < pieces; k += kSortWaves) {
        float x[VEC];
        g2v::load_vec<float, VEC>(part + (2 * (c0 + k) + (k > 0)) * D + col, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += x[i];
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) sums[wave][lane][i] = acc[i];
    __syncthreads();
    if (wave == 0 && in) {
      for (int w = 1; w < kSortWaves; ++w)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += sums[w][lane][i];
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] *= scale;
      g2v::store_vec_nt<TG, VEC>(grad + (int64_t)v * D + col, acc);
    }
    __syncthreads();
  }
}

// where everything lies in the workspace
struct Plan {
  int log2L;
  int64_t chunks, slots;  // places of L tokens; pieces (none where no run can be long)
  int64_t tiles, tile;    // 0: every bucket reads all ids
  int64_t hot, parts;     // tokens of a part, and the most parts there can be
  int64_t per_bucket;
  int64_t perm, rows, at, longs, small, part, pairs, counts, bfirst, hcounts, bytes;
};

Plan plan(int64_t n, int64_t V, int64_t D) {
  Plan p{};
  // Short pieces spread a frequent row over more groups, long ones leave less to
  // join: the more elements, the more pieces there are to fill the card with, and
  // the longer they may be.  Microseconds of the gradient at L = 64 / 128 / 256,
  // rows by Zipf's law and (in brackets) two rows only:
  //   elements  64 columns bf16         200 fp32                512 bf16
  //   2^20      24 / 27 / 38            18 / 21 / 24            23 / 23 / 25
  //             (27 / 30 / 40)          (20 / 23 / 30)          (23 / 25 / 34)
  //   2^23      43 / 50 / 64            36 / 39 / 48            29 / 30 / 42
  //             (48 / 48 / 55)          (42 / 44 / 51)          (33 / 32 / 40)
  //   2^25.5    74 / 71 / 81            64 / 64 / 69            57 / 55 / 65
  //             (106 / 87 / 88)         (73 / 65 / 64)          (67 / 58 / 66)
  //   2^27      119 / 109 / 109         197 / 186 / 186         106 / 97 / 98
  //             (187 / 147 / 129)       (274 / 222 / 196)       (129 / 101 / 100)
  // Up to 256 tokens are not cut at all, which saves a launch of three (200
  // tokens: 11 us instead of 13; at 300 the longest run costs as much).
  const int64_t elements = n * D;
  p.log2L = n <= 256 ? 8 : elements < (int64_t)1 << 24 ? 6 : elements < (int64_t)1 << 26 ? 7 : 8;
  p.chunks = (n + ((int64_t)1 << p.log2L) - 1) >> p.log2L;
  p.slots = n > (int64_t)1 << p.log2L ? 2 * p.chunks : 0;
  if (n > kScanTokens || (n > 0 && V > kScanRows)) {
    p.tile = (n + kMaxTiles - 1) / kMaxTiles;
    p.tile = (p.tile + kTileTokens - 1) / kTileTokens * kTileTokens;
    p.tiles = (n + p.tile - 1) / p.tile;
    // a bucket is cut where its rows fit one window of counts
    p.hot = n / 1024 > kHotTokens ? n / 1024 : kHotTokens;
    if (V > (int64_t)kBuckets * kKeys) p.hot = n;
    // a hot bucket of m tokens has fewer than m / hot + 1 parts
    const int64_t most = n / p.hot;
    p.parts = p.hot < n ? most + (most < kBuckets ? most : kBuckets) : 0;
  }
  const auto take = [&](int64_t count, int64_t size) {
    const int64_t o = p.bytes;
    p.bytes += (count * size + 255) / 256 * 256;
    return o;
  };
  p.perm = take(n, 4);
  p.per_bucket = (V + kBuckets - 1) / kBuckets;
  p.rows = take(p.per_bucket * kBuckets, 8);
  p.at = take(p.chunks + 1, 4);
  p.longs = take(p.chunks + 1, 4);
  p.small = take(2 * kBuckets + 1, 4);
  p.part = take(p.slots, 4 * D);
  p.pairs = take(p.tiles ? n : 0, 8);
  p.counts = take(p.tiles * kBuckets, 4);
  p.bfirst = take(p.tiles ? kBuckets + 1 : 0, 4);
  p.hcounts = take(p.parts * kKeys, 4);
  return p;
}

template <class F>
int by_type(int type, F f) {
  switch (type) {
    case G2V_F32: return f(float{});
    case G2V_F16: return f(f16{});
    default: return f(bf16{});
  }
}

template <class F>
int by_id(int id_bytes, F f) {
  return id_bytes == 4 ? f(int32_t{}) : f(int64_t{});
}

int check_common(const char* what, int device, int64_t V, int64_t D, const void* ids,
                 int id_bytes, int64_t n) {
  OP_REQUIRE(device >= 0, G2V_EINVAL, "%s: device %d", what, device);
  OP_REQUIRE(V >= 1 && D >= 1 && n >= 0, G2V_EINVAL, "%s: V = %lld, D = %lld, n = %lld", what,
             (long long)V, (long long)D, (long long)n);
  OP_REQUIRE(V <= INT32_MAX && n <= INT32_MAX && D <= G2V_EMBED_MAX_DIM, G2V_ERANGE,
             "%s: V = %lld and n = %lld are at most 2^31 - 1, D = %lld at most %d", what,
             (long long)V, (long long)n, (long long)D, G2V_EMBED_MAX_DIM);
  OP_REQUIRE(id_bytes == 4 || id_bytes == 8, G2V_EINVAL, "%s: ids of %d bytes", what, id_bytes);
  OP_REQUIRE(n == 0 || (ids && (uintptr_t)ids % id_bytes == 0), G2V_EINVAL,
             "%s: ids are null or not aligned to their size", what);
  return G2V_OK;
}

int check_matrix(const char* what, const char* name, const void* p, int type, int64_t rows,
                 int64_t ld, int64_t D) {
  OP_REQUIRE(g2v::type_bytes(type) != 0, G2V_EINVAL, "%s: %s has the unknown type %d", what, name,
             type);
  OP_REQUIRE(rows == 0 || (p && (uintptr_t)p % g2v::type_bytes(type) == 0), G2V_EINVAL,
             "%s: %s is null or not aligned to its type", what, name);
  OP_REQUIRE(ld >= D, G2V_EINVAL, "%s: %s has rows of %lld elements every %lld", what, name,
             (long long)D, (long long)ld);
  OP_REQUIRE(ld <= (INT64_MAX / 4) / (rows > 1 ? rows : 1), G2V_ERANGE,
             "%s: %s spans more than 2^63 bytes", what, name);
  return G2V_OK;
}

// f(VEC, G) as constants, for rows of D elements: as few idle lanes as a power
// of two allows (a row of nv vectors on 64 lanes leaves all but nv without work)
template <int VEC, class F>
int by_width(int64_t D, F f) {
  const int64_t nv = (D + VEC - 1) / VEC;
  if (D < VEC) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
  const std::integral_constant<int, VEC> vec{};
  if (nv <= 8) return f(vec, std::integral_constant<int, 8>{});
  if (nv <= 16) return f(vec, std::integral_constant<int, 16>{});
  if (nv <= 32) return f(vec, std::integral_constant<int, 32>{});
  return f(vec, std::integral_constant<int, 64>{});
}

template <class TY, class TG>
int launch_rows(const TY* dy, int64_t ld, const Sorted& s, int64_t slots, float* part, int64_t V,
                int64_t D, float scale, TG* grad, hipStream_t st) {
  // 16 bytes of the narrower type: dy's rows are most of what is read
  constexpr int kVec = 16 / (sizeof(TY) < sizeof(TG) ? sizeof(TY) : sizeof(TG));
  return by_width<kVec>(D, [&](auto vec, auto g) {
    constexpr int VEC = decltype(vec)::value, G = decltype(g)::value;
    const int64_t nv = (D + VEC - 1) / VEC, tiles = (nv + G - 1) / G;
    const int64_t groups = slots * tiles + V * ((tiles + kPer - 1) / kPer);
    hipLaunchKernelGGL((k_grad_rows<TY, TG, VEC, G>),
                       grid_of((groups + kThreads / G - 1) / (kThreads / G)), dim3(kThreads), 0, st,
                       dy, ld, s, part, V, (int)D, (int)nv, (int)tiles, slots, scale, grad);
    OP_HIP(hipGetLastError(), "g2v_embed_grad");
    return (int)G2V_OK;
  });
}

template <class TG>
int launch_join(const Sorted& s, int64_t runs, const float* part, int64_t D, float scale,
                TG* grad, hipStream_t st) {
  const int vec = D >= 4 ? 4 : 1;
  const int64_t nv = (D + vec - 1) / vec, cols = (nv + 63) / 64;
  const int64_t blocks = kJoinBlocks > cols ? kJoinBlocks / cols : 1;
  hipLaunchKernelGGL((vec == 4 ? k_grad_join<TG, 4> : k_grad_join<TG, 1>),
                     dim3((unsigned)(runs < blocks ? runs : blocks), (unsigned)cols),
                     dim3(kSortThreads), 0, st, s, part, (int)D, (int)nv, scale, grad);
  OP_HIP(hipGetLastError(), "g2v_embed_grad");
  return G2V_OK;
}

template <class I>
int launch_sort(const I* ids, int64_t n, int64_t V, int pad, const Plan& p, const Sorted& s,
                char* ws, hipStream_t st) {
  if (!p.tiles) {
    hipLaunchKernelGGL(k_sort_scan<I>, dim3(kBuckets), dim3(kSortThreads), 0, st, ids, (int)n,
                       (int)V, pad, s);
  } else {
    int32_t* counts = reinterpret_cast<int32_t*>(ws + p.counts);
    int32_t* bfirst = reinterpret_cast<int32_t*>(ws + p.bfirst);
    int2* pairs = reinterpret_cast<int2*>(ws + p.pairs);
    hipLaunchKernelGGL(k_tile_count<I>, dim3((unsigned)p.tiles), dim3(kSortThreads), 0, st, ids, n,
                       p.tile, (int)V, pad, counts);
    OP_HIP(hipGetLastError(), "g2v_embed_grad");
    hipLaunchKernelGGL(k_tile_scatter<I>, dim3((unsigned)p.tiles), dim3(kSortThreads), 0, st, ids,
                       n, p.tile, (int)V, pad, counts, bfirst, pairs);
    OP_HIP(hipGetLastError(), "g2v_embed_grad");
    int32_t* hcounts = reinterpret_cast<int32_t*>(ws + p.hcounts);
    if (p.parts) {
      hipLaunchKernelGGL(k_hot_count, dim3((unsigned)p.parts), dim3(kSortThreads), 0, st, pairs,
                         bfirst, (int)p.hot, hcounts);
      OP_HIP(hipGetLastError(), "g2v_embed_grad");
    }
    hipLaunchKernelGGL(k_sort_bucket, dim3((unsigned)(kBuckets + p.parts)), dim3(kSortThreads), 0,
                       st, pairs, bfirst, (int)V, (int)p.hot, hcounts, s);
  }
  OP_HIP(hipGetLastError(), "g2v_embed_grad");
  return G2V_OK;
}

}  // namespace

extern "C" int g2v_embed_lookup(int device, const void* table, int table_type, int64_t V,
                                int64_t D, int64_t ld, const void* ids, int id_bytes, int64_t n,
                                float scale, void* out, int out_type, void* stream) {
  const char* what = "g2v_embed_lookup";
  int rc = check_common(what, device, V, D, ids, id_bytes, n);
  if (rc == G2V_OK) rc = check_matrix(what, "table", table, table_type, V, ld, D);
  if (rc == G2V_OK) rc = check_matrix(what, "out", out, out_type, n, D, D);
  if (rc != G2V_OK || n == 0) return rc;
  g2v::DeviceScope scope(device);
  OP_HIP(scope.error(), what);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(table_type, [&](auto w) {
    return by_type(out_type, [&](auto y) {
      return by_id(id_bytes, [&](auto i) {
        using TW = decltype(w);
        using TY = decltype(y);
        using I = decltype(i);
        // 16 bytes of the result: stores past the caches have to fill their
        // lines together (262,147 rows of 512, bf16 to fp32: 93 us, with
        // twice that a lane 227)
        constexpr int VEC = 16 / sizeof(TY);
        const int64_t nv = D >= VEC ? (D + VEC - 1) / VEC : D;
        const int64_t blocks = (n * nv + kThreads * kUnits - 1) / (kThreads * kUnits);
        const auto kernel =
            D >= VEC ? k_embed_lookup<TW, TY, I, VEC> : k_embed_lookup<TW, TY, I, 1>;
        hipLaunchKernelGGL(kernel, grid_of(blocks), dim3(kThreads), 0, st,
                           static_cast<const TW*>(table), V, (int)D, ld,
                           static_cast<const I*>(ids), n * nv, (int)nv, scale,
                           static_cast<TY*>(out));
        return 0;
      });
    });
  });
  OP_HIP(hipGetLastError(), what);
  return G2V_OK;
}

extern "C" int g2v_embed_grad_workspace(int64_t n, int64_t V, int64_t D, int64_t* bytes) {
  const char* what = "g2v_embed_grad_workspace";
  OP_REQUIRE(bytes, G2V_EINVAL, "%s: null output", what);
  *bytes = 0;
  const int rc = check_common(what, 0, V, D, nullptr, 4, 0);
  if (rc != G2V_OK) return rc;
  OP_REQUIRE(n >= 0 && n <= INT32_MAX, G2V_ERANGE, "%s: n = %lld", what, (long long)n);
  *bytes = plan(n, V, D).bytes;
  return G2V_OK;
}

extern "C" int g2v_embed_grad(int device, const void* dy, int dy_type, int64_t dy_ld,
                              const void* ids, int id_bytes, int64_t n, int64_t V, int64_t D,
                              float scale, int64_t padding_id, void* grad, int grad_type,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "g2v_embed_grad";
  int rc = check_common(what, device, V, D, ids, id_bytes, n);
  if (rc == G2V_OK) rc = check_matrix(what, "dy", dy, dy_type, n, dy_ld, D);
  if (rc == G2V_OK) rc = check_matrix(what, "grad", grad, grad_type, V, D, D);
  if (rc != G2V_OK) return rc;
  OP_REQUIRE(padding_id >= -1 && padding_id < V, G2V_EINVAL,
             "%s: padding id %lld outside [-1, %lld)", what, (long long)padding_id, (long long)V);
  int64_t need = 0;
  rc = g2v_embed_grad_workspace(n, V, D, &need);
  if (rc != G2V_OK) return rc;
  OP_REQUIRE(workspace_bytes >= need && workspace && (uintptr_t)workspace % 16 == 0, G2V_EINVAL,
             "%s: a 16-byte aligned workspace of %lld bytes is needed (got %lld)", what,
             (long long)need, (long long)workspace_bytes);
  g2v::DeviceScope scope(device);
  OP_HIP(scope.error(), what);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int pad = (int)padding_id;
  const auto by_types = [&](auto f) {
    return by_type(grad_type, [&](auto g) {
      return by_type(dy_type, [&](auto y) {
        return f(static_cast<const decltype(y)*>(dy), static_cast<decltype(g)*>(grad));
      });
    });
  };
  const Plan p = plan(n, V, D);
  char* ws = static_cast<char*>(workspace);
  const auto ints = [&](int64_t o) { return reinterpret_cast<int32_t*>(ws + o); };
  int32_t* small = ints(p.small);
  const Sorted s{ints(p.perm),  reinterpret_cast<int2*>(ws + p.rows),
                 ints(p.at),    ints(p.longs),
                 small,         small + kBuckets,
                 small + 2 * kBuckets, p.log2L,
                 (int)p.per_bucket};
  float* part = reinterpret_cast<float*>(ws + p.part);
  rc = by_id(id_bytes, [&](auto i) {
    using I = decltype(i);
    return launch_sort(static_cast<const I*>(ids), n, V, pad, p, s, ws, st);
  });
  if (rc != G2V_OK) return rc;
  return by_types([&](auto* y, auto* g) {
    const int r = launch_rows(y, dy_ld, s, p.slots, part, V, D, scale, g, st);
    return r != G2V_OK || p.slots == 0 ? r : launch_join(s, p.chunks, part, D, scale, g, st);
  });
}
