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
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortBlock * kSortItems;
constexpr uint32_t kMaxBuckets = 1024;
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

// exclusive prefix sums of `count` words over a workgroup of kSortBlock lanes, in place; -> the total
__device__ __forceinline__ uint32_t block_prefix(uint32_t *v, uint32_t count, uint32_t *wave_sum) {
  const uint32_t per = (count + kSortBlock - 1) / kSortBlock;  // consecutive words of a lane
  const uint32_t first = threadIdx.x * per;
  uint32_t sum = 0;
  for (uint32_t i = 0; i < per; ++i) sum += first + i < count ? v[first + i] : 0u;
  uint32_t upto = sum;
  const unsigned lane = lane_id();
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint32_t o = __shfl_up(upto, d);
    if ((int)lane >= d) upto += o;
  }
  if (lane == kWave - 1) wave_sum[threadIdx.x / kWave] = upto;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    if (w < (int)(threadIdx.x / kWave)) before += wave_sum[w];
    total += wave_sum[w];
  }
  uint32_t at = before + upto - sum;
  for (uint32_t i = 0; i < per; ++i)
    if (first + i < count) {
      const uint32_t c = v[first + i];
      v[first + i] = at;
      at += c;
    }
  __syncthreads();
  return total;
}

// counts[bucket * tiles + tile]
template <Pass P, typename K>
__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(const K *__restrict__ keys, size_t n, Digits d,
                                                                uint32_t *__restrict__ counts) {
  __shared__ uint32_t count[kMaxBuckets];
  for (uint32_t b = threadIdx.x; b < d.buckets; b += kSortBlock) count[b] = 0;
  __syncthreads();
  const size_t base = (size_t)blockIdx.x * kSortTile;
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const size_t i = base + (size_t)j * kSortBlock + threadIdx.x;
    if (i < n) {
      const uint32_t key = sort_key<P>(keys, i, d);
      if (P != kExperts || key != kNoBucket) atomicAdd(&count[sort_bucket<P>(key, d)], 1u);
    }
  }
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < d.buckets; b += kSortBlock) counts[(size_t)b * gridDim.x + blockIdx.x] = count[b];
}

// workgroup b: before[tile * buckets + b] = entries of bucket b in earlier tiles; totals[b]
__global__ __launch_bounds__(kSortBlock) void sort_prefix_kernel(const uint32_t *__restrict__ counts, uint32_t tiles, uint32_t buckets,
                                                                 uint32_t *__restrict__ before, uint32_t *__restrict__ totals) {
  __shared__ uint32_t part[kSortBlock], wave_sum[kSortWaves];
  const uint32_t b = blockIdx.x;
  uint32_t so_far = 0;
  for (uint32_t t0 = 0; t0 < tiles; t0 += kSortBlock) {
    const uint32_t t = t0 + threadIdx.x;
    part[threadIdx.x] = t < tiles ? counts[(size_t)b * tiles + t] : 0u;
    __syncthreads();
    const uint32_t sum = block_prefix(part, kSortBlock, wave_sum);
    if (t < tiles) before[(size_t)t * buckets + b] = so_far + part[threadIdx.x];
    so_far += sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[b] = so_far;
}

// kExperts: slot[i], src[position], offsets[buckets + 1]; src is -1 behind the last position.  kFirst, kNext: key_out and
// entry_out at the position; entry is i in the first pass and entries[i] in the others.
template <Pass P, typename K>
__global__ __launch_bounds__(kSortBlock) void sort_place_kernel(const K *__restrict__ keys, const uint32_t *__restrict__ entries, size_t n,
                                                                Digits d, const uint32_t *__restrict__ before,
                                                                const uint32_t *__restrict__ totals, uint32_t *__restrict__ out0,
                                                                uint32_t *__restrict__ out1, uint32_t *__restrict__ offsets) {
  __shared__ uint32_t base[kMaxBuckets];
  __shared__ uint32_t seen[kSortWaves][kMaxBuckets];
  __shared__ uint32_t wave_sum[kSortWaves];
  for (uint32_t b = threadIdx.x; b < d.buckets; b += kSortBlock) {
    base[b] = totals[b];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) seen[w][b] = 0;
  }
  __syncthreads();
  const uint32_t total = block_prefix(base, d.buckets, wave_sum);
  const unsigned lane = lane_id(), wave = wave_in_block();
  const uint64_t below = (1ull << lane) - 1ull;
  const size_t tile0 = (size_t)blockIdx.x * kSortTile, first = tile0 + (size_t)wave * (kWave * kSortItems) + lane;
  uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const size_t i = first + (size_t)j * kWave;
    key[j] = i < n ? sort_key<P>(keys, i, d) : kNoBucket;
  }
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
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
  for (uint32_t b = threadIdx.x; b < d.buckets; b += kSortBlock) {
    if (P == kExperts && blockIdx.x == 0) offsets[b] = base[b];
    uint32_t at = base[b] + before[(size_t)blockIdx.x * d.buckets + b];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = seen[w][b];
      seen[w][b] = at;
      at += c;
    }
  }
  if (P == kExperts && blockIdx.x == 0 && threadIdx.x == 0) offsets[d.buckets] = total;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
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
      out1[at] = P == kFirst ? (uint32_t)i : entries[i];
    }
  }
}

static inline uint32_t bits_for(uint64_t values) {  // that tell `values` numbers from 0 on apart
  uint32_t bits = 0;
  while (((uint64_t)1 << bits) < values) ++bits;
  return bits;
}
static inline size_t sort_tiles(size_t n) { return (n + kSortTile - 1) / kSortTile; }
// words of the counts of a pass: of every tile, summed over the tiles before, and of all
static inline size_t sort_count_words(size_t n, uint32_t buckets) { return (2 * sort_tiles(n) + 1) * (size_t)buckets; }

template <Pass P, typename K>
static inline int sort_pass(const K *keys, const uint32_t *entries, size_t n, const Digits &d, uint32_t *words, uint32_t *out0,
                            uint32_t *out1, uint32_t *offsets, hipStream_t stream) {
  const size_t tiles = sort_tiles(n);
  uint32_t *counts = words, *before = counts + tiles * d.buckets, *totals = before + tiles * d.buckets;
  hipLaunchKernelGGL((sort_count_kernel<P, K>), dim3((unsigned)tiles), dim3(kSortBlock), 0, stream, keys, n, d, counts);
  hipLaunchKernelGGL(sort_prefix_kernel, dim3(d.buckets), dim3(kSortBlock), 0, stream, counts, (uint32_t)tiles, d.buckets, before, totals);
  hipLaunchKernelGGL((sort_place_kernel<P, K>), dim3((unsigned)tiles), dim3(kSortBlock), 0, stream, keys, entries, n, d, before, totals, out0,
                     out1, offsets);
  UGK_HIP(hipGetLastError());
  return 0;
}

}  // namespace
}  // namespace ugk
