// A stable counting sort by bucket: what orders the assignments of tokens by expert, and, digit after digit, the
// entries of a batch by the row they name.
//
// position of entry i of bucket b = entries of smaller buckets + entries of b in earlier tiles + entries of b in earlier
// wavefronts of the tile + entries of b before i in its wavefront.  Each term comes out of counting alone, so the order is
// the same on every run.  A wavefront takes its entries 64 at a time in their order; the lanes whose buckets are equal find
// each other by one ballot per bit of the bucket, and the running count of a bucket is a word in LDS.
#pragma once

#include <type_traits>

#include "ugk_internal.h"
#include "ugk_rows.cuh"

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

// the sum of a value over the lanes of the workgroup in front of this one, and over all of them (uint64_t: two sums of 32 bits)
template <typename V>
__device__ __forceinline__ V block_before(V v, V &total, V *wave_sum) {
  const unsigned lane = lane_id();
  V upto = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const V o = __shfl_up(upto, d);
    if ((int)lane >= d) upto += o;
  }
  if (lane == kWave - 1) wave_sum[threadIdx.x / kWave] = upto;
  __syncthreads();
  V before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    if (w < (int)(threadIdx.x / kWave)) before += wave_sum[w];
    total += wave_sum[w];
  }
  return before + upto - v;
}

// Memory that has to be zero before the launch behind the sort, cleared by workgroups that the sort's launches have beside
// those of the tiles: a sort of few entries leaves the memory and most of the chip alone.  Past
// the caches, which the sort and the sums behind it need (us, 16,384 entries over 50,000 rows of 2 KB: 56 -> 46).
struct Clear {
  char *to;        // at any element's address
  uint64_t bytes;  // a whole number of elements
  uint32_t first;  // the launch's first block of kClearBytes
};
constexpr uint32_t kClearBytes = kSortBlock * 32;
__device__ __forceinline__ void clear_block(const Clear &c, uint32_t block) {
  typedef typename ChunkOf<uint16_t, 8>::type chunk_t;
  const uint64_t base = ((uint64_t)c.first + block) * kClearBytes;
#pragma unroll
  for (uint32_t u = 0; u < kClearBytes / (16 * kSortBlock); ++u) {
    const uint64_t at = base + (u * kSortBlock + threadIdx.x) * 16;
    if (at + 16 <= c.bytes) put_chunk<uint16_t, 8, true>(reinterpret_cast<uint16_t *>(c.to + at), chunk_t{});
    else
      for (uint64_t i = at; i < c.bytes; i += 2) *reinterpret_cast<uint16_t *>(c.to + i) = 0;
  }
}

// counts[tile * buckets + bucket], for kMany counts[bucket * tiles + tile]
template <Pass P, typename K, int ITEMS, Reach R>
__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(const K *__restrict__ keys, size_t n, uint32_t tiles, Digits d, Clear clear,
                                                                uint32_t *__restrict__ counts) {
  __shared__ uint32_t count[kMaxBuckets];
  if (P != kExperts && blockIdx.x >= tiles) return clear_block(clear, blockIdx.x - tiles);
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
    counts[R == kMany ? (size_t)b * tiles + blockIdx.x : (size_t)blockIdx.x * d.buckets + b] = count[b];
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
    const uint32_t at = block_before<uint32_t>(t < tiles ? counts[(size_t)b * tiles + t] : 0u, sum, wave_sum);
    if (t < tiles) before[(size_t)t * buckets + b] = so_far + at;
    so_far += sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[b] = so_far;
}

// What the lanes of a workgroup need to put a tile in order.
template <int ITEMS>
struct TileSort {
  uint32_t seen[kSortWaves][kMaxBuckets];  // entries of a bucket that a wavefront has met, then where its first one goes
  uint32_t key[kSortBlock * ITEMS], entry[kSortBlock * ITEMS];  // in order
  uint64_t wave_sum[kSortWaves];
};

// The tile's entries, lane l of wavefront w holding entries w * 64 * ITEMS + j * 64 + l: rank[j] = entries of its bucket
// before it in its wavefront; here[h] = the tile's entries of the lane's two buckets; of_wave their shares.
template <int ITEMS>
__device__ __forceinline__ void rank_tile(TileSort<ITEMS> &t, const uint32_t (&bucket)[ITEMS], const Digits &d, uint32_t (&rank)[ITEMS],
                                          uint32_t (&of_wave)[2][kSortWaves], uint32_t (&here)[2]) {
  const unsigned lane = lane_id(), wave = wave_in_block();
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w)
    for (uint32_t b = threadIdx.x; b < d.buckets; b += kSortBlock) t.seen[w][b] = 0;
  const uint64_t below = (1ull << lane) - 1ull;
  uint32_t peers[ITEMS];  // lanes of this lane's bucket
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const uint64_t same = same_bucket(bucket[j], bucket[j] != kNoBucket, d.bits);
    rank[j] = (uint32_t)__popcll(same & below);
    peers[j] = (uint32_t)__popcll(same);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    if (bucket[j] != kNoBucket) {
      const uint32_t so_far = t.seen[wave][bucket[j]];
      __builtin_amdgcn_wave_barrier();  // the lanes of a bucket have read the count before the first of them raises it
      if (rank[j] == 0) t.seen[wave][bucket[j]] = so_far + peers[j];
      rank[j] += so_far;
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  const uint32_t mine = 2 * threadIdx.x;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    here[h] = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      of_wave[h][w] = mine + h < d.buckets ? t.seen[w][mine + h] : 0u;
      here[h] += of_wave[h][w];
    }
  }
}
// the entries of a lane's bucket `mine + h` begin at `at` in the tile
template <int ITEMS>
__device__ __forceinline__ void place_bucket(TileSort<ITEMS> &t, uint32_t bucket, uint32_t at, const uint32_t (&of_wave)[kSortWaves]) {
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    t.seen[w][bucket] = at;
    at += of_wave[w];
  }
}

// kExperts: slot[i], src[position], offsets[buckets + 1]; src is -1 behind the last position.  kFirst, kNext: key_out and
// entry_out at the position; entry is i in the first pass and entries[i] in the others.
//
// The tile is put in order in LDS first and leaves it in runs of a bucket's entries: stored from where they were read, 64
// lanes would touch 64 lines (262,144 entries in 256 buckets: 11.5 -> 9.9 us for this launch, 1 M in 128: 12.1 -> 11.5).
template <Pass P, typename K, int ITEMS, Reach R>
__global__ __launch_bounds__(kSortBlock) void sort_place_kernel(const K *__restrict__ keys, const uint32_t *__restrict__ entries, size_t n,
                                                                uint32_t tiles, Digits d, Clear clear, const uint32_t *__restrict__ counts,
                                                                const uint32_t *__restrict__ totals, uint32_t *__restrict__ out0,
                                                                uint32_t *__restrict__ out1, uint32_t *__restrict__ offsets) {
  __shared__ TileSort<ITEMS> tile;
  __shared__ uint32_t to_global[kMaxBuckets];  // what a position in the tile lacks to be one in the output
  if (P != kExperts && blockIdx.x >= tiles) return clear_block(clear, blockIdx.x - tiles);
  const unsigned lane = lane_id(), wave = wave_in_block();
  const size_t first = (size_t)blockIdx.x * (kSortBlock * ITEMS) + (size_t)wave * (kWave * ITEMS) + lane;
  // everything that is read is on its way before the first of it is waited for
  uint32_t key[ITEMS], entry[ITEMS], rank[ITEMS], bucket[ITEMS];
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
    // sixteen tiles at a time and no branch in between: their counts come out of other XCDs' caches, and waited for one by
    // one they cost half a microsecond each (16,384 entries in 16 tiles: 11.1 -> 6.5 us)
    constexpr uint32_t U = 16;
    for (uint32_t t0 = 0; t0 < tiles; t0 += U) {
      uint32_t c[U][2];
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        const uint32_t *of = counts + min(t0 + u, tiles - 1) * d.buckets;
        c[u][0] = of[at0];
        c[u][1] = of[at1];
      }
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          all[h] += t0 + u < tiles ? c[u][h] : 0u;
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
  for (int j = 0; j < ITEMS; ++j) {
    const size_t i = first + (size_t)j * kWave;
    bucket[j] = i < n && (P != kExperts || key[j] != kNoBucket) ? sort_bucket<P>(key[j], d) : kNoBucket;
  }
  uint32_t of_wave[2][kSortWaves], here[2];
  rank_tile<ITEMS>(tile, bucket, d, rank, of_wave, here);
  if constexpr (R == kSingle) all[0] = here[0], all[1] = here[1];
  uint64_t totals_of;
  const uint64_t starts = block_before<uint64_t>((uint64_t)(here[0] + here[1]) << 32 | (all[0] + all[1]), totals_of, tile.wave_sum);
  const uint32_t total = (uint32_t)totals_of, tile_total = (uint32_t)(totals_of >> 32);
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (mine + h < d.buckets) {
      const uint32_t at_global = (uint32_t)starts + (h ? all[0] : 0u), at = (uint32_t)(starts >> 32) + (h ? here[0] : 0u);
      if (P == kExperts && blockIdx.x == 0) offsets[mine + h] = at_global;
      to_global[mine + h] = at_global + before[h] - at;
      place_bucket<ITEMS>(tile, mine + h, at, of_wave[h]);
    }
  if (P == kExperts && blockIdx.x == 0 && threadIdx.x == 0) offsets[d.buckets] = total;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const size_t i = first + (size_t)j * kWave;
    const bool has = bucket[j] != kNoBucket;
    uint32_t at = 0;
    if (has) {
      at = tile.seen[wave][bucket[j]] + rank[j];
      tile.key[at] = key[j];
      tile.entry[at] = entry[j];
    }
    if constexpr (P == kExperts) {
      if (i < n) out0[i] = has ? at + to_global[bucket[j]] : 0xffffffffu;
      if (i < n && i >= total) out1[i] = 0xffffffffu;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const uint32_t at = (uint32_t)j * kSortBlock + threadIdx.x;
    if (at < tile_total) {
      const uint32_t to = at + to_global[sort_bucket<P>(tile.key[at], d)];
      if constexpr (P != kExperts) out0[to] = tile.key[at];
      out1[to] = tile.entry[at];
    }
  }
}

// all passes of a sort of at most kSortBlock * ITEMS entries by one workgroup, in LDS
template <typename K, int ITEMS>
__global__ __launch_bounds__(kSortBlock) void sort_one_tile_kernel(const K *__restrict__ keys, uint32_t n, uint32_t passes, Digits d,
                                                                   Clear clear, uint32_t *__restrict__ key_out,
                                                                   uint32_t *__restrict__ entry_out) {
  __shared__ TileSort<ITEMS> tile;
  if (blockIdx.x >= 1) return clear_block(clear, blockIdx.x - 1);
  const unsigned lane = lane_id(), wave = wave_in_block();
  const uint32_t first = wave * (kWave * ITEMS) + lane, mine = 2 * threadIdx.x;
  uint32_t key[ITEMS], entry[ITEMS], rank[ITEMS], bucket[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const uint32_t i = first + j * kWave;
    key[j] = i < n ? sort_key<kFirst>(keys, i, d) : kNoBucket;
    entry[j] = i;
  }
  for (uint32_t pass = 0; pass < passes; ++pass) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) bucket[j] = first + j * kWave < n ? (key[j] >> d.shift) & d.mask : kNoBucket;
    uint32_t of_wave[2][kSortWaves], here[2];
    rank_tile<ITEMS>(tile, bucket, d, rank, of_wave, here);
    uint64_t total;
    const uint32_t at = (uint32_t)block_before<uint64_t>(here[0] + here[1], total, tile.wave_sum);
    if (mine < d.buckets) place_bucket<ITEMS>(tile, mine, at, of_wave[0]);
    if (mine + 1 < d.buckets) place_bucket<ITEMS>(tile, mine + 1, at + here[0], of_wave[1]);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (bucket[j] != kNoBucket) {
        const uint32_t to = tile.seen[wave][bucket[j]] + rank[j];
        tile.key[to] = key[j];
        tile.entry[to] = entry[j];
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      key[j] = tile.key[first + j * kWave];
      entry[j] = tile.entry[first + j * kWave];
    }
    d.shift += d.bits;
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const uint32_t i = first + j * kWave;
    if (i < n) key_out[i] = key[j], entry_out[i] = entry[j];
  }
}

static inline uint32_t bits_for(uint64_t values) {  // that tell `values` numbers from 0 on apart
  uint32_t bits = 0;
  while (((uint64_t)1 << bits) < values) ++bits;
  return bits;
}
// How a pass goes by its size.  Small tiles spread a batch over the chip, large ones keep the counts of all tiles few.  us of a
// sort, entries per lane 2 / 4 / 8: 96,000 entries in 64 buckets 10.5 / 11.2 / 14.4, 480,000 11.6 / 11.9 / 15.1, 480,000 in 1,000
// 23.0 / 18.7 / 20.3, 1 M in 128 18.1 / 15.8 / 17.2, two passes of 1 M over 1,024 124 / 107 / 97; 32,000 in 64, counts of the
// tiles added up by every workgroup / by a launch of their own 8.5 / 10.5, 64,000 10.3 / 10.4.  Up to 4,096 entries are one tile: 1,200
// take 5.4 in one launch of four entries a lane and 7.6 in one of eight or in two launches; 4,000 take 9.5 in one and 8.6 in
// two, but a launch is 2.3 us of the host's time.
struct SortShape {
  int items;
  Reach reach;
  uint32_t tiles;
};
static inline SortShape sort_shape(size_t n, uint32_t buckets) {
  const auto tiles = [n](int items) { return (uint32_t)((n + kSortBlock * items - 1) / (kSortBlock * items)); };
  if (n <= 2 * kSortBlock) return SortShape{2, kSingle, 1};
  if (n <= 4 * kSortBlock) return SortShape{4, kSingle, 1};
  if (n <= 8 * kSortBlock) return SortShape{8, kSingle, 1};
  if (tiles(2) <= 32) return SortShape{2, kFew, tiles(2)};
  if ((uint64_t)tiles(2) * buckets <= 100'000) return SortShape{2, kMany, tiles(2)};
  if ((uint64_t)tiles(4) * buckets <= 250'000) return SortShape{4, kMany, tiles(4)};
  return SortShape{8, kMany, tiles(8)};
}
// words of the counts of a pass: of every tile, summed over the tiles before, and of all
static inline size_t sort_count_words(size_t n, uint32_t buckets) {
  const SortShape s = sort_shape(n, buckets);
  return s.reach == kSingle ? 0 : s.reach == kFew ? (size_t)s.tiles * buckets : (2 * (size_t)s.tiles + 1) * buckets;
}

// what is left to clear, and how much of it a launch takes
class Clearing {
 public:
  Clearing(void *to, size_t bytes) : _to(static_cast<char *>(to)), _bytes(bytes), _blocks((bytes + kClearBytes - 1) / kClearBytes) {}
  // `part` of `of` equal shares of what is left; -> the workgroups that takes
  uint32_t take(Clear &c, uint32_t part, uint32_t of) {
    const uint64_t blocks = ((_blocks - _done) * part + of - 1) / of;
    c = Clear{_to, _bytes, (uint32_t)_done};
    _done += blocks;
    return (uint32_t)blocks;
  }

 private:
  char *_to;
  uint64_t _bytes, _blocks, _done = 0;
};

template <Pass P, typename K, int ITEMS, Reach R>
static inline int sort_pass_as(const K *keys, const uint32_t *entries, size_t n, const Digits &d, uint32_t tiles, uint32_t *words,
                               uint32_t *out0, uint32_t *out1, uint32_t *offsets, Clearing *clearing, uint32_t passes_left, hipStream_t stream) {
  uint32_t *counts = words, *before = counts + (size_t)tiles * d.buckets, *totals = before + (size_t)tiles * d.buckets;
  Clear clear{};
  uint32_t blocks = 0;
  if constexpr (R != kSingle) {
    // a placement takes twice as long as the counting before it
    if (clearing) blocks = clearing->take(clear, 1, 3 * passes_left);
    hipLaunchKernelGGL((sort_count_kernel<P, K, ITEMS, R>), dim3(tiles + blocks), dim3(kSortBlock), 0, stream, keys, n, tiles, d, clear, counts);
  }
  if constexpr (R == kMany)
    hipLaunchKernelGGL(sort_prefix_kernel, dim3(d.buckets), dim3(kSortBlock), 0, stream, counts, tiles, d.buckets, before, totals);
  if (clearing) blocks = clearing->take(clear, 2, 3 * passes_left - 1);
  hipLaunchKernelGGL((sort_place_kernel<P, K, ITEMS, R>), dim3(tiles + blocks), dim3(kSortBlock), 0, stream, keys, entries, n, tiles, d, clear,
                     R == kMany ? before : counts, totals, out0, out1, offsets);
  UGK_HIP(hipGetLastError());
  return 0;
}

template <Pass P, typename K>
static inline int sort_pass(const K *keys, const uint32_t *entries, size_t n, const Digits &d, uint32_t *words, uint32_t *out0,
                            uint32_t *out1, uint32_t *offsets, Clearing *clearing, uint32_t passes_left, hipStream_t stream) {
  const SortShape s = sort_shape(n, d.buckets);
  const auto as = [&](auto items, auto reach) -> int {
    return sort_pass_as<P, K, decltype(items)::value, decltype(reach)::value>(keys, entries, n, d, s.tiles, words, out0, out1, offsets, clearing,
                                                                             passes_left, stream);
  };
  const std::integral_constant<int, 2> two;
  const std::integral_constant<int, 4> four;
  const std::integral_constant<int, 8> eight;
  const std::integral_constant<Reach, kMany> many;
  if (s.reach == kMany) return s.items == 2 ? as(two, many) : s.items == 4 ? as(four, many) : as(eight, many);
  if (s.reach == kFew) return as(two, std::integral_constant<Reach, kFew>());
  if constexpr (P == kExperts) {  // the others sort one tile by sort_one_tile_kernel
    const std::integral_constant<Reach, kSingle> single;
    return s.items == 2 ? as(two, single) : s.items == 4 ? as(four, single) : as(eight, single);
  }
  return ugk_set_error("ugk_bucket_sort: a single tile");
}

}  // namespace
}  // namespace ugk
