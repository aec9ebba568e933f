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
template <typename T, int VEC, bool STREAM>
__global__ __launch_bounds__(kBlock) void dispatch_kernel(const T *__restrict__ x, size_t x_stride, const int32_t *__restrict__ slot,
                                                          const int32_t *__restrict__ live, size_t tokens, uint32_t top,
                                                          uint32_t dim, Split split, T *__restrict__ rows) {
  typedef typename ChunkOf<T, VEC>::type chunk_t;
  size_t t;
  uint32_t c;
  split_lane(split, blockIdx.x, t, c);
  if (t >= tokens) return;
  const uint32_t at = min(c * VEC, dim - VEC);
  const chunk_t v = raw_chunk<T, VEC>(x + t * x_stride + at), zero = {};
  const uint32_t n = (uint32_t)(tokens * top), n_live = (uint32_t)*live;
  for (uint32_t k = 0; k < top; ++k) {
    const uint32_t i = (uint32_t)t * top + k;
    const uint32_t s = (uint32_t)slot[i];
    if (s < n) put_chunk<T, VEC, STREAM>(rows + (size_t)s * dim + at, v);
    if (i >= n_live) put_chunk<T, VEC, STREAM>(rows + (size_t)i * dim + at, zero);
  }
}

// out[t] = sum over k of w[t, k] * rows[slot[t, k]], added in fp32 in the order of k by fused multiply-adds and rounded once.
// STREAM: the rows are more than the memory-side cache holds and are read past the caches.
template <typename T, int VEC, bool STREAM>
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
  constexpr uint32_t U = 4;  // rows on their way (8: the same for eight experts a token, 65 us against 58 for two)
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
      if (u <= last && s[u] < n_rows) v[u] = raw_chunk<T, VEC, STREAM>(rows + s[u] * stride + at);
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

// grad_rows[slot] = w * grad_out[t], grad_weights[t, k] = <rows[slot], grad_out[t]>, positions behind the last live one zero.
// A group of `lanes` lanes, up to a wavefront, per token, or the whole workgroup (WIDE): it has U of the token's rows on
// their way, CH chunks of each to a lane, and the chunks of grad_out that go with them.
template <typename T, int VEC, bool STREAM, bool WIDE>
__global__ __launch_bounds__(kBlock) void combine_grad_kernel(const T *__restrict__ grad_out, size_t grad_stride,
                                                              const T *__restrict__ rows, size_t stride,
                                                              const int32_t *__restrict__ slot, const int32_t *__restrict__ live,
                                                              size_t tokens, uint32_t top, const void *__restrict__ weights,
                                                              int weight_elem, uint32_t dim, uint32_t chunks, uint32_t lanes,
                                                              T *__restrict__ grad_rows, void *__restrict__ grad_weights) {
  typedef typename ChunkOf<T, VEC>::type chunk_t;
  constexpr uint32_t U = 4, CH = 2;
  __shared__ float wave_dot[WIDE ? kBlock / kWave : 1][U];
  const uint32_t lane = threadIdx.x & (lanes - 1);
  const size_t t = WIDE ? blockIdx.x : (size_t)blockIdx.x * (kBlock / lanes) + threadIdx.x / lanes;
  if (t >= tokens) return;
  const uint32_t n = (uint32_t)(tokens * top), n_live = (uint32_t)*live;
  const T *from = grad_out + t * grad_stride;
  for (uint32_t k0 = 0; k0 < top; k0 += U) {
    const uint32_t i = (uint32_t)t * top + k0, last = min(U, top - k0) - 1;
    uint32_t s[U];
    float w[U], dot[U] = {};
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      s[u] = u <= last ? (uint32_t)slot[i + u] : n;
      w[u] = weights ? load_weight(weights, weight_elem, i + min(u, last)) : 1.f;
    }
    for (uint32_t c0 = lane; c0 < chunks; c0 += lanes * CH) {
      uint32_t at[CH];
      chunk_t g[CH], v[U][CH];
#pragma unroll
      for (uint32_t h = 0; h < CH; ++h) {
        at[h] = min((c0 + h * lanes) * VEC, dim - VEC);
        g[h] = raw_chunk<T, VEC>(from + at[h]);
      }
      if (grad_weights) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
          if (s[u] < n)
#pragma unroll
            for (uint32_t h = 0; h < CH; ++h) v[u][h] = raw_chunk<T, VEC, STREAM>(rows + s[u] * stride + at[h]);
      }
#pragma unroll
      for (uint32_t h = 0; h < CH; ++h) {
        const uint32_t c = c0 + h * lanes;
        if (c >= chunks) break;
        float x[VEC];
        to_floats<T, VEC>(g[h], x);
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          if (i + u >= n_live && u <= last) put_chunk<T, VEC, STREAM>(grad_rows + (size_t)(i + u) * dim + at[h], chunk_t{});
          if (s[u] >= n) continue;
          float y[VEC];
          if (grad_weights) {
            to_floats<T, VEC>(v[u][h], y);
#pragma unroll
            for (int e = 0; e < VEC; ++e)  // an element that the chunk before has too is counted there
              if (at[h] + e >= c * VEC) dot[u] = fmaf(y[e], x[e], dot[u]);
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) y[e] = w[u] * x[e];
          store_chunk<T, VEC, STREAM>(grad_rows + (size_t)s[u] * dim + at[h], y);
        }
      }
    }
    if (!grad_weights) continue;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
      for (uint32_t d = min(lanes, (uint32_t)kWave) / 2; d > 0; d /= 2) dot[u] += __shfl_xor(dot[u], d);
    if constexpr (WIDE) {
      __syncthreads();  // the sums of the rows before have been read
      if (lane_id() == 0)
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) wave_dot[wave_in_block()][u] = dot[u];
      __syncthreads();
      if (threadIdx.x <= last) {
        float sum = 0.f;
#pragma unroll
        for (int q = 0; q < kBlock / kWave; ++q) sum += wave_dot[q][threadIdx.x];
        store_weight(grad_weights, weight_elem, i + threadIdx.x, sum);
      }
    } else if (lane == 0) {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
        if (u <= last) store_weight(grad_weights, weight_elem, i + u, dot[u]);
    }
  }
}


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
                                reinterpret_cast<uint32_t *>(src), reinterpret_cast<uint32_t *>(offsets), nullptr, 1, as_stream(stream));
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
  return for_moved_rows(elem, dim, tokens * top, [&](auto type, auto vec, auto stream_out) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    const Split s = split_of(dim, V);
    const size_t blocks = split_blocks(tokens, s);
    UGK_REQUIRE(blocks <= kMaxBlocks, "ugk_expert_dispatch: %zu tokens of %zu elements are more than one launch takes", tokens, dim);
    hipLaunchKernelGGL((dispatch_kernel<T, V, decltype(stream_out)::value>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream),
                       (const T *)x_dev, x_stride, slot_dev, live_dev, tokens, top, (uint32_t)dim, s, (T *)rows_dev);
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
  return for_rows_streamed(elem, dim, n_rows, [&](auto type, auto vec, auto stream_rows) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    const Split s = split_of(dim, V);
    const size_t blocks = split_blocks(tokens, s);
    UGK_REQUIRE(blocks <= kMaxBlocks, "ugk_expert_combine: %zu tokens of %zu elements are more than one launch takes", tokens, dim);
    hipLaunchKernelGGL((combine_kernel<T, V, decltype(stream_rows)::value>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream),
                       (const T *)rows_dev, row_stride, (uint32_t)n_rows, slot_dev, tokens, top, weights_dev, weight_elem, (uint32_t)dim, s, (T *)out_dev);
    UGK_HIP(hipGetLastError());
    return 0;
  });
}

int ugk_expert_combine_grad(const void *grad_out_dev, size_t grad_stride, const void *rows_dev, size_t row_stride, const int32_t *slot_dev,
                            const int32_t *live_dev, size_t tokens, uint32_t top, const void *weights_dev, int weight_elem, size_t dim,
                            int elem, void *grad_rows_dev, void *grad_weights_dev, void *stream) {
  if (int rc = check_rows("ugk_expert_combine_grad", tokens, top, dim, elem, grad_stride)) return rc;
  UGK_REQUIRE(row_stride >= dim || tokens * top <= 1 || !grad_weights_dev,
              "ugk_expert_combine_grad: rows of %zu elements overlap at a stride of %zu",
              dim, row_stride);
  UGK_REQUIRE((!weights_dev && !grad_weights_dev) || elem_ok(weight_elem),
              "ugk_expert_combine_grad: element code %d of the weights", weight_elem);
  if (tokens == 0) return 0;
  UGK_REQUIRE(grad_out_dev && slot_dev && live_dev && grad_rows_dev && (rows_dev || !grad_weights_dev), "ugk_expert_combine_grad: null pointer");
  return for_rows_streamed(elem, dim, tokens * top, [&](auto type, auto vec, auto stream_rows) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    constexpr bool S = decltype(stream_rows)::value;
    const uint32_t chunks = split_of(dim, V).chunks;
    uint32_t lanes = 4;
    while (lanes < chunks && lanes < (uint32_t)kWave) lanes *= 2;
    // a workgroup per token from 256 chunks on (us, a wavefront / a workgroup per token, bfloat16 rows: 1 GB of them, eight a token, of
    // 128 chunks 396 / 492, 192 408 / 399, 256 410 / 391, 512 459 / 411, 1,024 453 / 422; 16 MB, eight a token, 256 16.5 / 12.1; two a
    // token, where fewer rows are on their way in a workgroup, change over later: 1 GB, 256 477 / 541, 320 485 / 495, 512 535 / 465;
    // 16 MB, 256 10.1 / 12.7, 512 11.7 / 10.1)
    const bool wide = chunks >= (uint32_t)kBlock;
    const auto launch = [&](auto is_wide, size_t blocks, uint32_t of) -> int {
      hipLaunchKernelGGL((combine_grad_kernel<T, V, S, decltype(is_wide)::value>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream),
                         (const T *)grad_out_dev, grad_stride, (const T *)rows_dev, row_stride, slot_dev, live_dev, tokens, top, weights_dev,
                         weight_elem, (uint32_t)dim, chunks, of, (T *)grad_rows_dev, grad_weights_dev);
      UGK_HIP(hipGetLastError());
      return 0;
    };
    const size_t per = kBlock / lanes, blocks = wide ? tokens : (tokens + per - 1) / per;
    UGK_REQUIRE(blocks <= kMaxBlocks, "ugk_expert_combine_grad: %zu tokens are more than one launch takes", tokens);
    return wide ? launch(std::true_type(), blocks, kBlock) : launch(std::false_type(), blocks, lanes);
  });
}

}  // extern "C"
