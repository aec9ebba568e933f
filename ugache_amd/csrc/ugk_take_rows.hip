// Rows taken by index, and the gradient of that: the rows of equal indices added up.
//
// The gradient sorts the entries by the row they name (digits of up to ten bits, ugk_bucket_sort.cuh), finds where every row's
// entries begin, and adds them in fp32 in the order of the batch, those of a row that many entries name in pieces that are
// then added in their order: no atomic touches a sum, so the same batch gives the same bits on every run.
#include <type_traits>

#include "ugk_bucket_sort.cuh"
#include "ugk_rows.cuh"

namespace ugk {
namespace {

// out[i] = table[index[i]], a zero row where the index is outside [0, rows)
template <typename T, int VEC, bool STREAM, typename I>
__global__ __launch_bounds__(kBlock) void take_rows_kernel(const T *__restrict__ table, uint64_t rows, size_t stride, const I *__restrict__ index,
                                                           size_t n, uint32_t dim, Split split, T *__restrict__ out) {
  size_t i;
  uint32_t c;
  split_lane(split, blockIdx.x, i, c);
  if (i >= n) return;
  const uint32_t at = min(c * VEC, dim - VEC);
  const long long r = (long long)index[i];
  typename ChunkOf<T, VEC>::type v = {};
  if (r >= 0 && (uint64_t)r < rows) v = raw_chunk<T, VEC>(table + (size_t)r * stride + at);
  put_chunk<T, VEC, STREAM>(out + i * dim + at, v);
}

// begin[r] = number of sorted keys below r, r = 0 .. rows.  A search per row, so that neither a run of rows nobody named nor a
// row everybody named is one lane's work; neighbouring rows walk the same way, a request for a wavefront.
__global__ __launch_bounds__(kBlock) void row_begin_kernel(const uint32_t *__restrict__ keys, uint32_t n, uint32_t rows,
                                                           uint32_t *__restrict__ begin) {
  const uint32_t r = blockIdx.x * kBlock + threadIdx.x;
  if (r > rows) return;
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (keys[mid] < r) lo = mid + 1;
    else hi = mid;
  }
  begin[r] = lo;
}

// sum += the rows grad[entries[j]], from <= j < to, in the order of j
template <typename T, int VEC>
__device__ __forceinline__ void add_entries(const T *grad, size_t stride, const uint32_t *entries, uint32_t from, uint32_t to, uint32_t at,
                                            float (&sum)[VEC]) {
  constexpr int U = 4;  // rows on their way
  uint32_t j = from;
  for (; j + U <= to; j += U) {
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) load_chunk<T, VEC>(grad + (size_t)entries[j + u] * stride + at, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] += v[u][e];
  }
  for (; j < to; ++j) {
    float v[VEC];
    load_chunk<T, VEC>(grad + (size_t)entries[j] * stride + at, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] += v[e];
  }
}

// A row of more than kPiece entries is summed in pieces: the positions are cut into pieces of kPiece, and a piece holds parts
// of at most two such rows, one that comes in from the piece before and one that begins in it and goes on behind it.
// parts[2 * piece] and parts[2 * piece + 1] are their sums.
constexpr uint32_t kPiece = 64;

// out[r] = sum of the rows grad[entries[j]], begin[r] <= j < begin[r + 1], in fp32 in the order of j.  The first row_blocks
// workgroups take the rows of at most kPiece entries, the others the pieces.
template <typename T, int VEC, bool STREAM>
__global__ __launch_bounds__(kBlock) void row_sum_kernel(const T *__restrict__ grad, size_t stride, const uint32_t *__restrict__ entries,
                                                         const uint32_t *__restrict__ keys, const uint32_t *__restrict__ begin,
                                                         uint32_t rows, uint32_t dim, Split split, uint32_t row_blocks, T *__restrict__ out,
                                                         float *__restrict__ parts) {
  size_t i;
  uint32_t c;
  const bool whole = blockIdx.x < row_blocks;
  split_lane(split, whole ? blockIdx.x : blockIdx.x - row_blocks, i, c);
  const uint32_t at = min(c * VEC, dim - VEC);
  float sum[VEC] = {};
  if (whole) {
    if (i >= rows) return;
    const uint32_t from = begin[i], to = begin[i + 1];
    if (to - from > kPiece) return;
    add_entries<T, VEC>(grad, stride, entries, from, to, at, sum);
    store_chunk<T, VEC, STREAM>(out + i * dim + at, sum);
    return;
  }
  const uint32_t live = begin[rows];
  const uint32_t from = (uint32_t)i * kPiece;  // below n + kPiece
  if (i * kPiece >= live) return;
  const uint32_t to = min(from + kPiece, live);
  const uint32_t r0 = keys[from], begin0 = begin[r0], end0 = begin[r0 + 1];
  if (begin0 < from && end0 - begin0 > kPiece) {
    add_entries<T, VEC>(grad, stride, entries, from, min(to, end0), at, sum);
    store_chunk<float, VEC>(parts + 2 * i * dim + at, sum);
  }
  const uint32_t r1 = keys[to - 1], begin1 = begin[r1];
  if (begin1 >= from && begin[r1 + 1] - begin1 > kPiece) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
    add_entries<T, VEC>(grad, stride, entries, begin1, to, at, sum);
    store_chunk<float, VEC>(parts + (2 * i + 1) * dim + at, sum);
  }
}

// The pieces of a row added up: a workgroup per piece in which such a row begins and per `lanes` chunks of it.  kBlock /
// lanes groups of lanes add a run of the pieces each, then the groups' sums are added in their order.
template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void row_join_kernel(const uint32_t *__restrict__ keys, const uint32_t *__restrict__ begin, uint32_t rows,
                                                          uint32_t dim, uint32_t chunks, uint32_t lanes, const float *__restrict__ parts,
                                                          T *__restrict__ out) {
  __shared__ float held[kBlock * VEC];
  const uint32_t live = begin[rows];
  const uint32_t first = blockIdx.x * kPiece;  // below n
  if (first >= live) return;
  const uint32_t r = keys[min(first + kPiece, live) - 1], from = begin[r], to = begin[r + 1];
  if (from < first || to - from <= kPiece) return;
  const uint32_t group = threadIdx.x / lanes, groups = kBlock / lanes;  // lanes: a power of two
  const uint32_t c = blockIdx.y * lanes + threadIdx.x % lanes;
  const uint32_t at = min(c * VEC, dim - VEC);
  const uint32_t p0 = blockIdx.x, pieces = (to - 1) / kPiece - p0 + 1;
  const uint32_t per = (pieces + groups - 1) / groups;
  float sum[VEC] = {};
  if (c < chunks) {
    constexpr uint32_t U = 8;  // parts on their way
    const uint32_t end = min((group + 1) * per, pieces);
    for (uint32_t p = group * per; p < end; p += U) {
      float v[U][VEC];
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        const uint32_t q = min(p + u, end - 1);
        load_chunk<float, VEC>(parts + (2 * (size_t)(p0 + q) + (q == 0 ? 1 : 0)) * dim + at, v[u]);
      }
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] += p + u < end ? v[u][e] : 0.f;
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) held[e * kBlock + threadIdx.x] = sum[e];
  __syncthreads();
  if (group != 0 || c >= chunks) return;
  for (uint32_t g = 1; g < groups; ++g)
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] += held[e * kBlock + g * lanes + threadIdx.x];
  store_chunk<T, VEC>(out + (size_t)r * dim + at, sum);
}

__global__ void preload_take_rows_kernel() {}

}  // namespace
void preload_take_rows(hipStream_t stream) { hipLaunchKernelGGL(preload_take_rows_kernel, dim3(1), dim3(1), 0, stream); }

namespace {

template <typename I>
int take_rows(const void *table, uint64_t num_rows, size_t stride, const I *index, size_t n, size_t dim, int elem, void *out, void *stream) {
  UGK_REQUIRE(elem_ok(elem), "ugk_take_rows: element code %d is none of fp32 (4), fp16 (2) and bfloat16 (UGK_ELEM_BF16)", elem);
  UGK_REQUIRE(dim >= 1 && dim < kMaxDim, "ugk_take_rows: rows of %zu elements", dim);
  UGK_REQUIRE(n < ((size_t)1 << 40) && num_rows < ((uint64_t)1 << 40), "ugk_take_rows: %zu of %zu rows", n, (size_t)num_rows);
  if (n == 0) return 0;
  UGK_REQUIRE((table || num_rows == 0) && index && out, "ugk_take_rows: null pointer");
  return for_moved_rows(elem, dim, n, [&](auto type, auto vec, auto stream_out) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    const Split s = split_of(dim, V);
    const size_t blocks = split_blocks(n, s);
    UGK_REQUIRE(blocks < ((size_t)1 << 31), "ugk_take_rows: %zu rows of %zu elements are more than one launch takes", n, dim);
    hipLaunchKernelGGL((take_rows_kernel<T, V, decltype(stream_out)::value, I>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream), (const T *)table, num_rows,
                       stride, index, n, (uint32_t)dim, s, (T *)out);
    UGK_HIP(hipGetLastError());
    return 0;
  });
}

// how a batch of n entries over `rows` rows is sorted: digits of equal length, the key `rows` (no row) among them
struct Plan {
  uint32_t passes, digit;
};
Plan plan_for(uint64_t rows) {
  const uint32_t bits = bits_for(rows + 1);
  const uint32_t passes = bits <= 10 ? 1u : bits <= 20 ? 2u : bits <= 30 ? 3u : 4u;
  return Plan{passes, (bits + passes - 1) / passes};
}

size_t pieces_of(size_t n) { return (n + kPiece - 1) / kPiece; }

template <typename I>
int take_rows_grad(const void *grad, size_t stride, const I *index, size_t n, uint64_t num_rows, size_t dim, int elem, void *out,
                   void *workspace, size_t workspace_bytes, void *stream) {
  UGK_REQUIRE(elem_ok(elem), "ugk_take_rows_grad: element code %d is none of fp32 (4), fp16 (2) and bfloat16 (UGK_ELEM_BF16)", elem);
  UGK_REQUIRE(dim >= 1 && dim < kMaxDim, "ugk_take_rows_grad: rows of %zu elements", dim);
  UGK_REQUIRE(n < ((size_t)1 << 31) && num_rows < ((uint64_t)1 << 31), "ugk_take_rows_grad: %zu entries of %zu rows, both have 31 bits", n,
              (size_t)num_rows);
  UGK_REQUIRE(stride >= dim || n <= 1, "ugk_take_rows_grad: rows of %zu elements overlap at a stride of %zu", dim, stride);
  if (num_rows == 0) return 0;
  UGK_REQUIRE(out && (n == 0 || (grad && index)), "ugk_take_rows_grad: null pointer");
  const size_t need = ugk_take_rows_grad_workspace_bytes(n, num_rows, dim);
  UGK_REQUIRE(workspace && workspace_bytes >= need, "ugk_take_rows_grad: a workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  uint32_t *begin = static_cast<uint32_t *>(workspace);
  uint32_t *key[2] = {begin + num_rows + 1, begin + num_rows + 1 + n}, *entry[2] = {key[1] + n, key[1] + 2 * n};
  float *parts = reinterpret_cast<float *>(entry[1] + n);
  uint32_t *words = reinterpret_cast<uint32_t *>(parts + 2 * pieces_of(n) * dim);
  const Plan p = plan_for(num_rows);
  int at = 0;
  if (n > 0) {
    Digits d{num_rows, 0, (1u << p.digit) - 1u, 1u << p.digit, p.digit};
    if (int rc = sort_pass<kFirst, I>(index, nullptr, n, d, words, key[0], entry[0], nullptr, as_stream(stream))) return rc;
    for (uint32_t pass = 1; pass < p.passes; ++pass, at ^= 1) {
      d.shift += p.digit;
      if (int rc = sort_pass<kNext, uint32_t>(key[at], entry[at], n, d, words, key[at ^ 1], entry[at ^ 1], nullptr, as_stream(stream)))
        return rc;
    }
  }
  hipLaunchKernelGGL(row_begin_kernel, dim3((unsigned)(num_rows / kBlock + 1)), dim3(kBlock), 0, as_stream(stream), key[at], (uint32_t)n,
                     (uint32_t)num_rows, begin);
  return for_rows_streamed(elem, dim, num_rows, [&](auto type, auto vec, auto stream_out) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    const Split s = split_of(dim, V);
    const size_t pieces = n > kPiece ? pieces_of(n) : 0;  // in fewer entries no row has more than a piece
    const size_t row_blocks = split_blocks(num_rows, s), blocks = row_blocks + split_blocks(pieces, s);
    uint32_t lanes = 1;
    while (lanes < s.chunks && lanes < 32) lanes *= 2;
    hipLaunchKernelGGL((row_sum_kernel<T, V, decltype(stream_out)::value>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream), (const T *)grad, stride, entry[at],
                       key[at], begin, (uint32_t)num_rows, (uint32_t)dim, s, (uint32_t)row_blocks, (T *)out, parts);
    if (pieces > 0)
      hipLaunchKernelGGL((row_join_kernel<T, V>), dim3((unsigned)pieces, (s.chunks + lanes - 1) / lanes), dim3(kBlock), 0, as_stream(stream),
                         key[at], begin, (uint32_t)num_rows, (uint32_t)dim, s.chunks, lanes, parts, (T *)out);
    UGK_HIP(hipGetLastError());
    return 0;
  });
}

}  // namespace
}  // namespace ugk

using namespace ugk;

extern "C" {

int ugk_take_rows_i32(const void *table_dev, uint64_t num_rows, size_t stride, const int32_t *index_dev, size_t n, size_t dim, int elem,
                      void *out_dev, void *stream) {
  return take_rows<int32_t>(table_dev, num_rows, stride, index_dev, n, dim, elem, out_dev, stream);
}
int ugk_take_rows_i64(const void *table_dev, uint64_t num_rows, size_t stride, const int64_t *index_dev, size_t n, size_t dim, int elem,
                      void *out_dev, void *stream) {
  return take_rows<int64_t>(table_dev, num_rows, stride, index_dev, n, dim, elem, out_dev, stream);
}

size_t ugk_take_rows_grad_workspace_bytes(size_t n, uint64_t num_rows, size_t dim) {
  return 4 * ((size_t)num_rows + 1 + 4 * n + 2 * pieces_of(n) * dim + sort_count_words(n, 1u << plan_for(num_rows).digit));
}
int ugk_take_rows_grad_i32(const void *grad_dev, size_t stride, const int32_t *index_dev, size_t n, uint64_t num_rows, size_t dim, int elem,
                           void *out_dev, void *workspace_dev, size_t workspace_bytes, void *stream) {
  return take_rows_grad<int32_t>(grad_dev, stride, index_dev, n, num_rows, dim, elem, out_dev, workspace_dev, workspace_bytes, stream);
}
int ugk_take_rows_grad_i64(const void *grad_dev, size_t stride, const int64_t *index_dev, size_t n, uint64_t num_rows, size_t dim, int elem,
                           void *out_dev, void *workspace_dev, size_t workspace_bytes, void *stream) {
  return take_rows_grad<int64_t>(grad_dev, stride, index_dev, n, num_rows, dim, elem, out_dev, workspace_dev, workspace_bytes, stream);
}

}  // extern "C"
