// Rows sent to a router's experts and back: the order of the assignments by expert, the rows copied there, what comes
// back added up with the router's weights, and the gradients of both.
#include <type_traits>

#include "ugk_bucket_sort.cuh"
#include "ugk_rows.cuh"

namespace ugk {
namespace {

// rows[slot[t, k]] = x[t] for every assignment of token t; the positions behind the last live one are zero rows, so that
// what multiplies the whole buffer meets no stale bits.  The lane that holds a chunk of x[t] stores it `top` times; x is
// read once.
template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void dispatch_kernel(const T *__restrict__ x, size_t x_stride, const int32_t *__restrict__ slot,
                                                          const int32_t *__restrict__ live, size_t tokens, uint32_t top,
                                                          uint32_t dim, Split split, T *__restrict__ rows) {
  typedef typename ChunkOf<T, VEC>::type chunk_t;
  size_t t;
  uint32_t c;
  split_lane(split, blockIdx.x, t, c);
  if (t >= tokens) return;
  const uint32_t at = min(c * VEC, dim - VEC);
  const chunk_t v = *reinterpret_cast<const chunk_t *>(x + t * x_stride + at);
  const chunk_t zero = {};
  const uint32_t n = (uint32_t)(tokens * top), n_live = (uint32_t)*live;
  for (uint32_t k = 0; k < top; ++k) {
    const uint32_t i = (uint32_t)t * top + k;
    const uint32_t s = (uint32_t)slot[i];
    if (s < n) *reinterpret_cast<chunk_t *>(rows + (size_t)s * dim + at) = v;
    if (i >= n_live) *reinterpret_cast<chunk_t *>(rows + (size_t)i * dim + at) = zero;
  }
}

// out[t] = sum over k of w[t, k] * rows[slot[t, k]], added in fp32 in the order of k by fused multiply-adds and rounded once
template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void combine_kernel(const T *__restrict__ rows, size_t stride, uint32_t n_rows,
                                                         const int32_t *__restrict__ slot, size_t tokens, uint32_t top,
                                                         const void *__restrict__ weights, int weight_elem, uint32_t dim,
                                                         Split split, T *__restrict__ out) {
  size_t t;
  uint32_t c;
  split_lane(split, blockIdx.x, t, c);
  if (t >= tokens) return;
  const uint32_t at = min(c * VEC, dim - VEC);
  float sum[VEC] = {};
  constexpr uint32_t U = 8;  // rows on their way
  for (uint32_t k0 = 0; k0 < top; k0 += U) {
    const size_t i = t * top + k0;
    const uint32_t last = min(U, top - k0) - 1;
    uint32_t s[U];
    float w[U];
    typename ChunkOf<T, VEC>::type v[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      s[u] = (uint32_t)slot[i + min(u, last)];
      w[u] = weights ? load_weight(weights, weight_elem, i + min(u, last)) : 1.f;
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
      if (u <= last && s[u] < n_rows) v[u] = raw_chunk<T, VEC>(rows + s[u] * stride + at);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
      if (u <= last && s[u] < n_rows) {
        float x[VEC];
        to_floats<T, VEC>(v[u], x);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] = fmaf(w[u], x[e], sum[e]);
      }
  }
  store_chunk<T, VEC>(out + t * dim + at, sum);
}

// a wavefront per token: grad_rows[slot] = w * grad_out[t], grad_weights[t, k] = <rows[slot], grad_out[t]>, positions
// behind the last live one zero
template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void combine_grad_kernel(const T *__restrict__ grad_out, size_t grad_stride,
                                                              const T *__restrict__ rows, size_t stride,
                                                              const int32_t *__restrict__ slot, const int32_t *__restrict__ live,
                                                              size_t tokens, uint32_t top, const void *__restrict__ weights,
                                                              int weight_elem, uint32_t dim, uint32_t chunks,
                                                              T *__restrict__ grad_rows, void *__restrict__ grad_weights) {
  const size_t t = (size_t)blockIdx.x * (kBlock / kWave) + wave_in_block();
  if (t >= tokens) return;
  const uint32_t lane = lane_id(), n = (uint32_t)(tokens * top), n_live = (uint32_t)*live;
  for (uint32_t k = 0; k < top; ++k) {
    const uint32_t i = (uint32_t)t * top + k;
    const uint32_t s = (uint32_t)slot[i];
    const float w = weights ? load_weight(weights, weight_elem, i) : 1.f;
    float dot = 0.f;
    for (uint32_t c = lane; c < chunks; c += kWave) {
      const uint32_t at = min(c * VEC, dim - VEC);
      float g[VEC], v[VEC];
      if (i >= n_live) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = 0.f;
        store_chunk<T, VEC>(grad_rows + (size_t)i * dim + at, v);
      }
      if (s >= n) continue;
      load_chunk<T, VEC>(grad_out + t * grad_stride + at, g);
      if (grad_weights) {
        load_chunk<T, VEC>(rows + s * stride + at, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e)  // an element that the chunk before has too is counted there
          if (at + e >= c * VEC) dot = fmaf(v[e], g[e], dot);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = w * g[e];
      store_chunk<T, VEC>(grad_rows + (size_t)s * dim + at, v);
    }
    if (grad_weights) {
#pragma unroll
      for (int d = kWave / 2; d > 0; d /= 2) dot += __shfl_xor(dot, d);
      if (lane == 0) store_weight(grad_weights, weight_elem, i, dot);
    }
  }
}

__global__ void preload_expert_kernel() {}

}  // namespace
void preload_expert(hipStream_t stream) { hipLaunchKernelGGL(preload_expert_kernel, dim3(1), dim3(1), 0, stream); }

namespace {

template <typename K>
int expert_sort(const K *ids, size_t n, uint32_t num_experts, int32_t *slot, int32_t *src, int32_t *offsets, void *workspace,
                size_t workspace_bytes, void *stream) {
  UGK_REQUIRE(num_experts >= 1 && num_experts <= kMaxBuckets, "ugk_expert_sort: %u experts, 1 to %u are sorted", num_experts, kMaxBuckets);
  UGK_REQUIRE(n < ((size_t)1 << 31), "ugk_expert_sort: %zu assignments, positions have 31 bits", n);
  UGK_REQUIRE(offsets && (n == 0 || (ids && slot && src)), "ugk_expert_sort: null pointer");
  if (n == 0) return ugk_fill_u32(reinterpret_cast<uint32_t *>(offsets), 0, (size_t)num_experts + 1, stream);
  const size_t need = ugk_expert_sort_workspace_bytes(n, num_experts);
  UGK_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "ugk_expert_sort: a workspace of %zu bytes, %zu are needed", workspace_bytes,
              need);
  const Digits d{0, 0, 0, num_experts, bits_for(num_experts)};
  return sort_pass<kExperts, K>(ids, nullptr, n, d, static_cast<uint32_t *>(workspace), reinterpret_cast<uint32_t *>(slot),
                                reinterpret_cast<uint32_t *>(src), reinterpret_cast<uint32_t *>(offsets), as_stream(stream));
}

// what the entry points that move rows ask of their sizes
int check_rows(const char *what, size_t tokens, uint32_t top, size_t dim, int elem, size_t stride) {
  UGK_REQUIRE(elem_ok(elem), "%s: element code %d is none of fp32 (4), fp16 (2) and bfloat16 (UGK_ELEM_BF16)", what, elem);
  UGK_REQUIRE(top >= 1 && tokens < ((size_t)1 << 31) && tokens * top < ((size_t)1 << 31),
              "%s: %zu tokens of %u assignments, positions have 31 bits", what, tokens, top);
  UGK_REQUIRE(dim >= 1 && dim < kMaxDim, "%s: rows of %zu elements", what, dim);
  UGK_REQUIRE(stride >= dim || tokens <= 1, "%s: rows of %zu elements overlap at a stride of %zu", what, dim, stride);
  return 0;
}

}  // namespace
}  // namespace ugk

using namespace ugk;

extern "C" {

size_t ugk_expert_sort_workspace_bytes(size_t n, uint32_t num_experts) { return 4 * sort_count_words(n, num_experts); }

int ugk_expert_sort_i32(const int32_t *ids_dev, size_t n, uint32_t num_experts, int32_t *slot_dev, int32_t *src_dev, int32_t *offsets_dev,
                        void *workspace_dev, size_t workspace_bytes, void *stream) {
  return expert_sort<int32_t>(ids_dev, n, num_experts, slot_dev, src_dev, offsets_dev, workspace_dev, workspace_bytes, stream);
}
int ugk_expert_sort_i64(const int64_t *ids_dev, size_t n, uint32_t num_experts, int32_t *slot_dev, int32_t *src_dev, int32_t *offsets_dev,
                        void *workspace_dev, size_t workspace_bytes, void *stream) {
  return expert_sort<int64_t>(ids_dev, n, num_experts, slot_dev, src_dev, offsets_dev, workspace_dev, workspace_bytes, stream);
}

int ugk_expert_dispatch(const void *x_dev, size_t x_stride, const int32_t *slot_dev, const int32_t *live_dev, size_t tokens, uint32_t top,
                        size_t dim, int elem, void *rows_dev, void *stream) {
  if (int rc = check_rows("ugk_expert_dispatch", tokens, top, dim, elem, x_stride)) return rc;
  if (tokens == 0) return 0;
  UGK_REQUIRE(x_dev && slot_dev && live_dev && rows_dev, "ugk_expert_dispatch: null pointer");
  return for_moved_rows(elem, dim, [&](auto type, auto vec) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    const Split s = split_of(dim, V);
    const size_t blocks = split_blocks(tokens, s);
    UGK_REQUIRE(blocks < ((size_t)1 << 31), "ugk_expert_dispatch: %zu tokens of %zu elements are more than one launch takes", tokens, dim);
    hipLaunchKernelGGL((dispatch_kernel<T, V>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream), (const T *)x_dev, x_stride,
                       slot_dev, live_dev, tokens, top, (uint32_t)dim, s, (T *)rows_dev);
    UGK_HIP(hipGetLastError());
    return 0;
  });
}

int ugk_expert_combine(const void *rows_dev, size_t n_rows, size_t row_stride, const int32_t *slot_dev, size_t tokens, uint32_t top,
                       const void *weights_dev, int weight_elem, size_t dim, int elem, void *out_dev, void *stream) {
  if (int rc = check_rows("ugk_expert_combine", tokens, top, dim, elem, row_stride)) return rc;
  UGK_REQUIRE(n_rows < ((size_t)1 << 31), "ugk_expert_combine: %zu rows, positions have 31 bits", n_rows);
  UGK_REQUIRE(!weights_dev || elem_ok(weight_elem), "ugk_expert_combine: element code %d of the weights", weight_elem);
  if (tokens == 0) return 0;
  UGK_REQUIRE((rows_dev || n_rows == 0) && slot_dev && out_dev, "ugk_expert_combine: null pointer");
  return for_rows(elem, dim, [&](auto type, auto vec) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    const Split s = split_of(dim, V);
    const size_t blocks = split_blocks(tokens, s);
    UGK_REQUIRE(blocks < ((size_t)1 << 31), "ugk_expert_combine: %zu tokens of %zu elements are more than one launch takes", tokens, dim);
    hipLaunchKernelGGL((combine_kernel<T, V>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream), (const T *)rows_dev, row_stride,
                       (uint32_t)n_rows, slot_dev, tokens, top, weights_dev, weight_elem, (uint32_t)dim, s, (T *)out_dev);
    UGK_HIP(hipGetLastError());
    return 0;
  });
}

int ugk_expert_combine_grad(const void *grad_out_dev, size_t grad_stride, const void *rows_dev, size_t row_stride, const int32_t *slot_dev,
                            const int32_t *live_dev, size_t tokens, uint32_t top, const void *weights_dev, int weight_elem, size_t dim,
                            int elem, void *grad_rows_dev, void *grad_weights_dev, void *stream) {
  if (int rc = check_rows("ugk_expert_combine_grad", tokens, top, dim, elem, grad_stride)) return rc;
  UGK_REQUIRE(row_stride >= dim || tokens * top <= 1 || !grad_weights_dev, "ugk_expert_combine_grad: rows of %zu elements overlap at a stride of %zu",
              dim, row_stride);
  UGK_REQUIRE((!weights_dev && !grad_weights_dev) || elem_ok(weight_elem), "ugk_expert_combine_grad: element code %d of the weights", weight_elem);
  if (tokens == 0) return 0;
  UGK_REQUIRE(grad_out_dev && slot_dev && live_dev && grad_rows_dev && (rows_dev || !grad_weights_dev), "ugk_expert_combine_grad: null pointer");
  return for_rows(elem, dim, [&](auto type, auto vec) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    constexpr int kPer = kBlock / kWave;
    hipLaunchKernelGGL((combine_grad_kernel<T, V>), dim3((unsigned)((tokens + kPer - 1) / kPer)), dim3(kBlock), 0, as_stream(stream),
                       (const T *)grad_out_dev, grad_stride, (const T *)rows_dev, row_stride, slot_dev, live_dev, tokens, top, weights_dev,
                       weight_elem, (uint32_t)dim, split_of(dim, V).chunks, (T *)grad_rows_dev, grad_weights_dev);
    UGK_HIP(hipGetLastError());
    return 0;
  });
}

}  // extern "C"
