// Rows taken by index, and the gradient of that: the rows of equal indices added up.
//
// The gradient sorts the entries by the row they name (digits of up to ten bits, ugk_bucket_sort.cuh), finds where
// every row's entries begin, and adds them in fp32 in the order of the batch: no atomic touches a sum, so the same
// batch gives the same bits on every run.
#include <type_traits>

#include "ugk_bucket_sort.cuh"
#include "ugk_rows.cuh"

namespace ugk {
namespace {

// out[i] = table[index[i]], a zero row where the index is outside [0, rows)
template <typename T, int VEC, typename I>
__global__ __launch_bounds__(kBlock) void take_rows_kernel(const T *__restrict__ table, uint64_t rows, size_t stride, const I *__restrict__ index,
                                                           size_t n, uint32_t dim, Split split, T *__restrict__ out) {
  typedef typename ChunkOf<T, VEC>::type chunk_t;
  size_t i;
  uint32_t c;
  split_lane(split, i, c);
  if (i >= n) return;
  const uint32_t at = min(c * VEC, dim - VEC);
  const long long r = (long long)index[i];
  chunk_t v = {};
  if (r >= 0 && (uint64_t)r < rows) v = *reinterpret_cast<const chunk_t *>(table + (size_t)r * stride + at);
  *reinterpret_cast<chunk_t *>(out + i * dim + at) = v;
}

// begin[r] = number of sorted keys below r, r = 0 .. rows: lane i writes the rows that begin between entry i - 1 and entry i
__global__ __launch_bounds__(kBlock) void row_begin_kernel(const uint32_t *__restrict__ keys, size_t n, uint32_t rows,
                                                           uint32_t *__restrict__ begin) {
  const size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x;
  if (i > n) return;
  const uint32_t from = i == 0 ? 0u : keys[i - 1] + 1u, to = i == n ? rows : min(keys[i], rows);
  for (uint32_t r = from; r <= to; ++r) begin[r] = (uint32_t)i;
}

// out[r] = sum of the rows grad[entries[j]], begin[r] <= j < begin[r + 1], in fp32 in the order of j
template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void row_sum_kernel(const T *__restrict__ grad, size_t stride, const uint32_t *__restrict__ entries,
                                                         const uint32_t *__restrict__ begin, size_t rows, uint32_t dim, Split split,
                                                         T *__restrict__ out) {
  size_t r;
  uint32_t c;
  split_lane(split, r, c);
  if (r >= rows) return;
  const uint32_t at = min(c * VEC, dim - VEC);
  float sum[VEC] = {};
  const uint32_t end = begin[r + 1];
  for (uint32_t j = begin[r]; j < end; ++j) {
    float v[VEC];
    load_chunk<T, VEC>(grad + (size_t)entries[j] * stride + at, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] += v[e];
  }
  store_chunk<T, VEC>(out + r * dim + at, sum);
}

__global__ void preload_take_rows_kernel() {}

}  // namespace
void preload_take_rows(hipStream_t stream) { hipLaunchKernelGGL(preload_take_rows_kernel, dim3(1), dim3(1), 0, stream); }

namespace {

template <typename I>
int take_rows(const void *table, uint64_t num_rows, size_t stride, const I *index, size_t n, size_t dim, int elem, void *out, void *stream) {
  UGK_REQUIRE(elem_ok(elem), "ugk_take_rows: element code %d is none of fp32 (4), fp16 (2) and bfloat16 (UGK_ELEM_BF16)", elem);
  UGK_REQUIRE(dim >= 1 && dim < ((size_t)1 << 30), "ugk_take_rows: rows of %zu elements", dim);
  UGK_REQUIRE(n < ((size_t)1 << 40) && num_rows < ((uint64_t)1 << 40), "ugk_take_rows: %zu of %zu rows", n, (size_t)num_rows);
  if (n == 0) return 0;
  UGK_REQUIRE((table || num_rows == 0) && index && out, "ugk_take_rows: null pointer");
  return for_moved_rows(elem, dim, [&](auto type, auto vec) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    const Split s = split_of(dim, V);
    const size_t blocks = split_blocks(n, s);
    UGK_REQUIRE(blocks < ((size_t)1 << 31), "ugk_take_rows: %zu rows of %zu elements are more than one launch takes", n, dim);
    hipLaunchKernelGGL((take_rows_kernel<T, V, I>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream), (const T *)table, num_rows,
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

template <typename I>
int take_rows_grad(const void *grad, size_t stride, const I *index, size_t n, uint64_t num_rows, size_t dim, int elem, void *out,
                   void *workspace, size_t workspace_bytes, void *stream) {
  UGK_REQUIRE(elem_ok(elem), "ugk_take_rows_grad: element code %d is none of fp32 (4), fp16 (2) and bfloat16 (UGK_ELEM_BF16)", elem);
  UGK_REQUIRE(dim >= 1 && dim < ((size_t)1 << 30), "ugk_take_rows_grad: rows of %zu elements", dim);
  UGK_REQUIRE(n < ((size_t)1 << 31) && num_rows < ((uint64_t)1 << 31), "ugk_take_rows_grad: %zu entries of %zu rows, both have 31 bits", n,
              (size_t)num_rows);
  UGK_REQUIRE(stride >= dim || n <= 1, "ugk_take_rows_grad: rows of %zu elements overlap at a stride of %zu", dim, stride);
  if (num_rows == 0) return 0;
  UGK_REQUIRE(out && (n == 0 || (grad && index)), "ugk_take_rows_grad: null pointer");
  const size_t need = ugk_take_rows_grad_workspace_bytes(n, num_rows);
  UGK_REQUIRE(workspace && workspace_bytes >= need, "ugk_take_rows_grad: a workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  uint32_t *begin = static_cast<uint32_t *>(workspace);
  uint32_t *key[2] = {begin + num_rows + 1, begin + num_rows + 1 + n}, *entry[2] = {key[1] + n, key[1] + 2 * n};
  uint32_t *words = entry[1] + n;
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
  hipLaunchKernelGGL(row_begin_kernel, dim3((unsigned)(n / kBlock + 1)), dim3(kBlock), 0, as_stream(stream), key[at], n, (uint32_t)num_rows,
                     begin);
  return for_rows(elem, dim, [&](auto type, auto vec) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    const Split s = split_of(dim, V);
    const size_t blocks = split_blocks(num_rows, s);
    UGK_REQUIRE(blocks < ((size_t)1 << 31), "ugk_take_rows_grad: %zu rows of %zu elements are more than one launch takes", (size_t)num_rows, dim);
    hipLaunchKernelGGL((row_sum_kernel<T, V>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream), (const T *)grad, stride, entry[at],
                       begin, num_rows, (uint32_t)dim, s, (T *)out);
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

size_t ugk_take_rows_grad_workspace_bytes(size_t n, uint64_t num_rows) {
  return 4 * ((size_t)num_rows + 1 + 4 * n + sort_count_words(n, 1u << plan_for(num_rows).digit));
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
