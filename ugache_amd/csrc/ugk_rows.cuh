// Rows of fp32, fp16 or bfloat16 elements of any length at any element boundary, as the kernels that add, weight and
// move them see them: 16-byte chunks held in registers as floats.
//
// A row of at least one chunk is covered by chunks at multiples of a chunk's length, the last one moved back so that it ends
// with the row: elements that two chunks share are computed twice, to the same bits, and no lane needs a loop over a
// tail.  gfx950 loads and stores 16 bytes at any element's address, so an odd number of two-byte elements costs no
// kernel of its own.  Rows shorter than a chunk go element by element (VEC 1).
#pragma once

#include <type_traits>

#include "ugk_internal.h"

namespace ugk {
namespace {

// the element types: how they are stored, and converted (to float exactly, back to the nearest, ties to even)
typedef _Float16 half_t;
typedef __bf16 bhalf_t;

template <typename T, int VEC>
struct ChunkOf {
  typedef T type __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
};
template <typename T>
struct ChunkOf<T, 1> {
  typedef T type;
};

// STREAM: past the caches (non-temporal), for what is read once or written to be read much later
template <typename T, int VEC, bool STREAM = false>
__device__ __forceinline__ typename ChunkOf<T, VEC>::type raw_chunk(const T *from) {
  const typename ChunkOf<T, VEC>::type *p = reinterpret_cast<const typename ChunkOf<T, VEC>::type *>(from);
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}
template <typename T, int VEC, bool STREAM = false>
__device__ __forceinline__ void put_chunk(T *to, const typename ChunkOf<T, VEC>::type &v) {
  typename ChunkOf<T, VEC>::type *p = reinterpret_cast<typename ChunkOf<T, VEC>::type *>(to);
  if constexpr (STREAM) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <typename T, int VEC>
__device__ __forceinline__ void to_floats(const typename ChunkOf<T, VEC>::type &v, float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    x[0] = (float)v;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = (float)v[i];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void load_chunk(const T *from, float (&x)[VEC]) {
  to_floats<T, VEC>(raw_chunk<T, VEC>(from), x);
}

template <typename T, int VEC, bool STREAM = false>
__device__ __forceinline__ void store_chunk(T *to, const float (&x)[VEC]) {
  typename ChunkOf<T, VEC>::type v;
  if constexpr (VEC == 1) {
    v = (T)x[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = (T)x[i];
  }
  put_chunk<T, VEC, STREAM>(to, v);
}

// a weight of any of the three types (a branch that the whole launch takes the same way)
__device__ __forceinline__ float load_weight(const void *w, int elem, size_t i) {
  if (elem == 4) return static_cast<const float *>(w)[i];
  if (elem == 2) return (float)static_cast<const half_t *>(w)[i];
  return (float)static_cast<const bhalf_t *>(w)[i];
}
__device__ __forceinline__ void store_weight(void *w, int elem, size_t i, float v) {
  if (elem == 4) static_cast<float *>(w)[i] = v;
  else if (elem == 2) static_cast<half_t *>(w)[i] = (half_t)v;
  else static_cast<bhalf_t *>(w)[i] = (bhalf_t)v;
}

// How the chunks of a batch of rows are dealt to lanes: numbered through, so that no lane idles whatever a row's length.
struct Split {
  uint32_t chunks;  // of a row
  uint32_t magic;   // floor(2^32 / chunks) + 1, where that has 32 bits
};
static inline Split split_of(size_t dim, int vec) {
  const uint32_t chunks = (uint32_t)((dim + vec - 1) / vec);
  return Split{chunks, (uint32_t)(((uint64_t)1 << 32) / chunks + 1)};
}
static inline size_t split_blocks(size_t rows, const Split &s) { return (rows * s.chunks + kBlock - 1) / kBlock; }

// The row and the chunk of a lane.  Every `chunks` workgroups take kBlock rows, so that 32 bits hold what is divided, and the
// divisions are scalar; what a lane adds to the second remainder stays below chunks + kBlock, where the product with the
// magic number is exact for up to kBlock chunks and a comparison does for more.
constexpr size_t kMaxDim = (size_t)1 << 25;
__device__ __forceinline__ void split_lane(const Split &s, uint32_t block, size_t &row, uint32_t &chunk) {
  const uint32_t group = block / s.chunks, first = (block - group * s.chunks) * kBlock, row0 = first / s.chunks;
  const uint32_t at = first - row0 * s.chunks + threadIdx.x;
  const uint32_t over = s.chunks == 1 ? at : s.chunks > (uint32_t)kBlock ? (at >= s.chunks ? 1u : 0u) : __umulhi(at, s.magic);
  row = (size_t)group * kBlock + (row0 + over);
  chunk = at - over * s.chunks;
}

// calls f with the element type and the elements per chunk that rows of `dim` elements of code `elem` take
template <typename F>
static inline int for_rows(int elem, size_t dim, F f) {
  if (elem == 4) return dim >= 4 ? f(float(), std::integral_constant<int, 4>()) : f(float(), std::integral_constant<int, 1>());
  if (elem == 2) return dim >= 8 ? f(half_t(), std::integral_constant<int, 8>()) : f(half_t(), std::integral_constant<int, 1>());
  return dim >= 8 ? f(bhalf_t(), std::integral_constant<int, 8>()) : f(bhalf_t(), std::integral_constant<int, 1>());
}
// ... and whether so many of them are more than the memory-side cache holds (us, past the caches / the ordinary way: the sums of
// 131,072 rows of 4 KB, 537 MB, 103 / 162; two passes over 12,297 rows of 4 KB, 49 MB, 37 / 32)
template <typename F>
static inline int for_rows_streamed(int elem, size_t dim, size_t rows, F f) {
  return for_rows(elem, dim, [&](auto type, auto vec) -> int {
    return rows * dim * sizeof(type) > kMemorySideCacheBytes ? f(type, vec, std::true_type()) : f(type, vec, std::false_type());
  });
}
// ... for kernels that move elements of two or four bytes without looking at them, and whether their output of so many rows is
// stored past the caches (49,152 rows of 4 KB, 201 MB, past the caches / the ordinary way 40 / 36 us; 131,072, and their gradient
// behind them, 224 / 259).  By size alone: what ugk_set_output_hint says is about the extractions of the thread.
template <typename F>
static inline int for_moved_rows(int elem, size_t dim, size_t out_rows, F f) {
  const auto stored = [&](auto type, auto vec) -> int {
    return out_rows * dim * sizeof(type) > kMemorySideCacheBytes ? f(type, vec, std::true_type()) : f(type, vec, std::false_type());
  };
  if (elem == 4) return dim >= 4 ? stored(uint32_t(), std::integral_constant<int, 4>()) : stored(uint32_t(), std::integral_constant<int, 1>());
  return dim >= 8 ? stored(uint16_t(), std::integral_constant<int, 8>()) : stored(uint16_t(), std::integral_constant<int, 1>());
}

// the work-items of a launch are counted in 32 bits
constexpr size_t kMaxBlocks = ((size_t)1 << 32) / kBlock - 1;

static inline size_t chunks_of(int elem, size_t dim) {  // of a row
  const size_t vec = elem == 4 ? 4 : 8;
  return dim >= vec ? (dim + vec - 1) / vec : dim;
}

static inline bool elem_ok(int elem) { return elem == 4 || elem == 2 || elem == UGK_ELEM_BF16; }
static inline size_t elem_size(int elem) { return elem == 4 ? 4 : 2; }

}  // namespace
}  // namespace ugk
