// A stable counting sort by bucket: what orders the assignments of tokens by expert, and, digit after digit, the
// entries of a batch by the row they name.
//
// position of entry i of bucket b = entries of smaller buckets + entries of b in earlier tiles + entries of b in earlier
// wavefronts of the tile + entries of b before i in its wavefront.  Each term comes out of counting alone, so the order is
// the same on every run.  A wavefront takes its entries 64 at a time in their order; the lanes whose buckets are equal find
// each other by one ballot per bit of the bucket, and the running count of a bucket is a word in LDS.
#pragma once

#include "ugk_internal.h"

namespace ugk {
namespace {

constexpr int kSortBlock = 512, kSortWaves = kSortBlock / kWave;
constexpr uint32_t kMaxBuckets = 2 * kSortBlock;  // a lane keeps the counts of two buckets
constexpr uint32_t kNoBucket = 0xffffffffu;

// kExperts: entries outside [0, buckets) have no bucket; kFirst: the lowest digit of an index, rows where it is outside [0,
// rows); kNext: a further digit of a key of an earlier pass
enum Pass { kExperts, kFirst, kNext };

struct Digits {
  uint64_t rows;     // kFirst
  uint32_t shift, mask;
  uint32_t buckets;  // of this pass
  uint32_t bits;     // ballots that tell buckets apart
};

template <Pass P, typename K>
__device__ __forceinline__ uint32_t sort_key(const K *keys, size_t i, const Digits &d) {
  if constexpr (P == kNext) return (uint32_t)keys[i];
  const long long id = (long long)keys[i];
  if constexpr (P == kExperts) return id >= 0 && id < (long long)d.buckets ? (uint32_t)id : kNoBucket;
  return id >= 0 && (uint64_t)id < d.rows ? (uint32_t)id : (uint32_t)d.rows;
}
template <Pass P>
__device__ __forceinline__ uint32_t sort_bucket(uint32_t key, const Digits &d) {
  return P == kExperts ? key : (key >> d.shift) & d.mask;
}

// the lanes of a wavefront with this lane's bucket; lanes without one are in nobody's set
__device__ __forceinline__ uint64_t same_bucket(uint32_t bucket, bool has, uint32_t bits) {
  uint64_t same = __ballot(has);
  for (uint32_t b = 0; b < bits; ++b) {
    const uint64_t ones = __ballot((bucket >> b) & 1u);
    same &= (bucket >> b) & 1u ? ones : ~ones;
  }
  return same;
}

// Where the counts of the other tiles come from.  kSingle: there is one tile.  kFew: counts[tile][bucket], which every
// workgroup adds up by itself.  kMany: a launch in between has added them up.
enum Reach { kSingle, kFew, kMany };

// the sum of a value over the lanes of the workgroup in front of this one, and over all of them
__device__ __forceinline__ uint32_t block_before(uint32_t v, uint32_t &total, uint32_t *wave_sum) {
  const unsigned lane = lane_id();
  uint32_t upto = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint32_t o = __shfl_up(upto, d);
    if ((int)lane >= d) upto += o;
  }
  if (lane == kWave - 1) wave_sum[threadIdx.x / kWave] = upto;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    if (w < (int)(threadIdx.x / kWave)) before += wave_sum[w];
    total += wave_sum[w];
  }
  return before + upto - v;
}

// counts[tile * buckets + bucket], for kMany counts[bucket * tiles + tile]
template <Pass P, typename K, int ITEMS, Reach R>
__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(const K *__restrict__ keys, size_t n, Digits d,
                                                                uint32_t *__restrict__ counts) {
  __shared__ uint32_t count[kMaxBuckets];
  const size_t base = (size_t)blockIdx.x * (kSortBlock * ITEMS) + threadIdx.x;
  uint32_t key[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const size_t i = base + (size_t)j * kSortBlock;
    key[j] = i < n ? sort_key<P>(keys, i, d) : kNoBucket;
  }
  for (uint32_t b = threadIdx.x; b < d.buckets; b += kSortBlock) count[b] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const size_t i = base + (size_t)j * kSortBlock;
    if (i < n && (P != kExperts || key[j] != kNoBucket)) atomicAdd(&count[sort_bucket<P>(key[j], d)], 1u);
  }
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < d.buckets; b += kSortBlock)
    counts[R == kMany ? (size_t)b * gridDim.x + blockIdx.x : (size_t)blockIdx.x * d.buckets + b] = count[b];
}

// workgroup b: before[tile * buckets + b] = entries of bucket b in earlier tiles; totals[b]
__global__ __launch_bounds__(kSortBlock) void sort_prefix_kernel(const uint32_t *__restrict__ counts, uint32_t tiles, uint32_t buckets,
                                                                 uint32_t *__restrict__ before, uint32_t *__restrict__ totals) {
  __shared__ uint32_t wave_sum[kSortWaves];
  const uint32_t b = blockIdx.x;
  uint32_t so_far = 0;
  for (uint32_t t0 = 0; t0 < tiles; t0 += kSortBlock) {
    const uint32_t t = t0 + threadIdx.x;
    uint32_t sum;
    const uint32_t at = block_before(t < tiles ? counts[(size_t)b * tiles + t] : 0u, sum, wave_sum);
    if (t < tiles) before[(size_t)t * buckets + b] = so_far + at;
    so_far += sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[b] = so_far;
}

// kExperts: slot[i], src[position], offsets[buckets + 1]; src is -1 behind the last position.  kFirst, kNext: key_out and
// entry_out at the position; entry is i in the first pass and entries[i] in the others.
template <Pass P, typename K, int ITEMS, Reach R>
__global__ __launch_bounds__(kSortBlock) void sort_place_kernel(const K *__restrict__ keys, const uint32_t *__restrict__ entries, size_t n,
                                                                Digits d, const uint32_t *__restrict__ counts,
                                                                const uint32_t *__restrict__ totals, uint32_t *__restrict__ out0,
                                                                uint32_t *__restrict__ out1, uint32_t *__restrict__ offsets) {
  __shared__ uint32_t seen[kSortWaves][kMaxBuckets];
  __shared__ uint32_t wave_sum[kSortWaves];
  const unsigned lane = lane_id(), wave = wave_in_block();
  const size_t first = (size_t)blockIdx.x * (kSortBlock * ITEMS) + (size_t)wave * (kWave * ITEMS) + lane;
  // everything that is read is on its way before the first of it is waited for
  uint32_t key[ITEMS], entry[ITEMS], rank[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const size_t i = first + (size_t)j * kWave;
    key[j] = i < n ? sort_key<P>(keys, i, d) : kNoBucket;
    entry[j] = P == kNext && i < n ? entries[i] : (uint32_t)i;
  }
  const uint32_t mine = 2 * threadIdx.x;  // this lane's two buckets
  uint32_t before[2] = {0, 0}, all[2] = {0, 0};
  const uint32_t at0 = min(mine, d.buckets - 1), at1 = min(mine + 1, d.buckets - 1);
  if constexpr (R == kMany) {
    before[0] = counts[(size_t)blockIdx.x * d.buckets + at0];
    before[1] = counts[(size_t)blockIdx.x * d.buckets + at1];
    all[0] = totals[at0];
    all[1] = totals[at1];
  } else if constexpr (R == kFew) {
    // sixteen tiles at a time and no branch in between: their counts come out of other XCDs' caches, a microsecond and a
    // half each if they are waited for one by one (16,384 entries in 16 tiles: 11.1 -> 5 us)
    constexpr uint32_t U = 16;
    for (uint32_t t0 = 0; t0 < gridDim.x; t0 += U) {
      uint32_t c[U][2];
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        const uint32_t *of = counts + min(t0 + u, gridDim.x - 1) * d.buckets;
        c[u][0] = of[at0];
        c[u][1] = of[at1];
      }
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          all[h] += t0 + u < gridDim.x ? c[u][h] : 0u;
          before[h] += t0 + u < blockIdx.x ? c[u][h] : 0u;
        }
    }
  }
  if constexpr (R != kSingle) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (mine + h >= d.buckets) all[h] = 0;
  }
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w)
    for (uint32_t b = threadIdx.x; b < d.buckets; b += kSortBlock) seen[w][b] = 0;
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1ull;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const size_t i = first + (size_t)j * kWave;
    const bool has = i < n && (P != kExperts || key[j] != kNoBucket);
    const uint32_t bucket = has ? sort_bucket<P>(key[j], d) : 0u;
    const uint64_t same = same_bucket(bucket, has, d.bits);
    rank[j] = 0;
    if (has) {
      const uint32_t so_far = seen[wave][bucket];
      rank[j] = so_far + (uint32_t)__popcll(same & below);
      __builtin_amdgcn_wave_barrier();  // the lanes of a set have read the count before one of them raises it
      if ((same & below) == 0) seen[wave][bucket] = so_far + (uint32_t)__popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  if constexpr (R == kSingle) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (mine + h < d.buckets)
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) all[h] += seen[w][mine + h];
  }
  uint32_t total;
  const uint32_t base = block_before(all[0] + all[1], total, wave_sum);
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (mine + h < d.buckets) {
      uint32_t at = base + (h ? all[0] : 0u);
      if (P == kExperts && blockIdx.x == 0) offsets[mine + h] = at;
      at += before[h];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t c = seen[w][mine + h];
        seen[w][mine + h] = at;
        at += c;
      }
    }
  if (P == kExperts && blockIdx.x == 0 && threadIdx.x == 0) offsets[d.buckets] = total;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const size_t i = first + (size_t)j * kWave;
    if (i >= n) continue;
    if constexpr (P == kExperts) {
      const bool has = key[j] != kNoBucket;
      const uint32_t at = has ? seen[wave][key[j]] + rank[j] : 0u;
      out0[i] = has ? at : 0xffffffffu;
      if (has) out1[at] = (uint32_t)i;
      if (i >= total) out1[i] = 0xffffffffu;
    } else {
      const uint32_t at = seen[wave][sort_bucket<P>(key[j], d)] + rank[j];
      out0[at] = key[j];
      out1[at] = entry[j];
    }
  }
}

static inline uint32_t bits_for(uint64_t values) {  // that tell `values` numbers from 0 on apart
  uint32_t bits = 0;
  while (((uint64_t)1 << bits) < values) ++bits;
  return bits;
}
// How a pass goes by its size.
struct SortShape {
  int items;
  Reach reach;
  uint32_t tiles;
};
static inline SortShape sort_shape(size_t n) {
  const auto tiles = [n](int items) { return (uint32_t)((n + kSortBlock * items - 1) / (kSortBlock * items)); };
  if (n <= 2 * kSortBlock) return SortShape{2, kSingle, 1};
  if (n <= 8 * kSortBlock) return SortShape{8, kSingle, 1};
  if (tiles(2) <= 16) return SortShape{2, kFew, tiles(2)};
  if (tiles(8) <= 32) return SortShape{8, kFew, tiles(8)};
  return SortShape{8, kMany, tiles(8)};
}
// words of the counts of a pass: of every tile, summed over the tiles before, and of all
static inline size_t sort_count_words(size_t n, uint32_t buckets) {
  const SortShape s = sort_shape(n);
  return s.reach == kSingle ? 0 : s.reach == kFew ? (size_t)s.tiles * buckets : (2 * (size_t)s.tiles + 1) * buckets;
}

template <Pass P, typename K, int ITEMS, Reach R>
static inline int sort_pass_as(const K *keys, const uint32_t *entries, size_t n, const Digits &d, uint32_t tiles, uint32_t *words,
                               uint32_t *out0, uint32_t *out1, uint32_t *offsets, hipStream_t stream) {
  uint32_t *counts = words, *before = counts + (size_t)tiles * d.buckets, *totals = before + (size_t)tiles * d.buckets;
  if constexpr (R != kSingle)
    hipLaunchKernelGGL((sort_count_kernel<P, K, ITEMS, R>), dim3(tiles), dim3(kSortBlock), 0, stream, keys, n, d, counts);
  if constexpr (R == kMany)
    hipLaunchKernelGGL(sort_prefix_kernel, dim3(d.buckets), dim3(kSortBlock), 0, stream, counts, tiles, d.buckets, before, totals);
  hipLaunchKernelGGL((sort_place_kernel<P, K, ITEMS, R>), dim3(tiles), dim3(kSortBlock), 0, stream, keys, entries, n, d,
                     R == kMany ? before : counts, totals, out0, out1, offsets);
  UGK_HIP(hipGetLastError());
  return 0;
}

template <Pass P, typename K>
static inline int sort_pass(const K *keys, const uint32_t *entries, size_t n, const Digits &d, uint32_t *words, uint32_t *out0,
                            uint32_t *out1, uint32_t *offsets, hipStream_t stream) {
  const SortShape s = sort_shape(n);
  if (s.reach == kMany) return sort_pass_as<P, K, 8, kMany>(keys, entries, n, d, s.tiles, words, out0, out1, offsets, stream);
  if (s.reach == kFew && s.items == 8) return sort_pass_as<P, K, 8, kFew>(keys, entries, n, d, s.tiles, words, out0, out1, offsets, stream);
  if (s.reach == kFew) return sort_pass_as<P, K, 2, kFew>(keys, entries, n, d, s.tiles, words, out0, out1, offsets, stream);
  if (s.items == 8) return sort_pass_as<P, K, 8, kSingle>(keys, entries, n, d, 1, words, out0, out1, offsets, stream);
  return sort_pass_as<P, K, 2, kSingle>(keys, entries, n, d, 1, words, out0, out1, offsets, stream);
}

}  // namespace
}  // namespace ugk
