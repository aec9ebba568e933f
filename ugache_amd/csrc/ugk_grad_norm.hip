// The l2 norm over all gradients of a training step, and the gradients scaled down to a limit.
//
// norm = sqrt(sum over tensors and elements of x^2).  Squares and sums are held in 64 bits: a float's square needs twice
// its exponent, and a thousand million terms need more than 24 bits.  Every workgroup sums one piece of one tensor, the
// pieces' sums are added in their order, so the same gradients give the same bits on every run.
#include "ugk_rows.cuh"

namespace ugk {
namespace {

// What a launch is told of its tensors travels in its arguments (the list of a training step changes with every step):
// up to kListed tensors at a time, each a run of consecutive pieces.
constexpr int kListed = 120;
constexpr uint32_t kPieceBytes = 32768;
struct TensorList {
  const void *data[kListed];
  void *out[kListed];
  uint64_t count[kListed];
  uint32_t first[kListed];  // the tensor's first piece in this launch
  int32_t elem[kListed];
  uint32_t n;
};

static inline uint64_t pieces_of(const ugk_tensor_t &t) { return (t.count * elem_size(t.elem) + kPieceBytes - 1) / kPieceBytes; }

__device__ __forceinline__ uint32_t tensor_of(const TensorList &list, uint32_t piece) {
  uint32_t at = 0;
  for (uint32_t i = 1; i < list.n; ++i) at += list.first[i] <= piece ? 1u : 0u;
  return at;
}

template <typename T, typename F>
__device__ __forceinline__ void for_elements(const T *data, uint64_t count, uint32_t piece, F f) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr uint32_t kElems = kPieceBytes / sizeof(T);
  const uint64_t begin = (uint64_t)piece * kElems;
  const uint32_t n = (uint32_t)min((uint64_t)kElems, count - begin);
  for (uint32_t i = threadIdx.x * VEC; i + VEC <= n; i += kBlock * VEC) {
    float x[VEC];
    load_chunk<T, VEC>(data + begin + i, x);
    f(begin + i, x, std::integral_constant<int, VEC>());
  }
  const uint32_t tail = n / VEC * VEC + threadIdx.x;
  if (tail < n) {
    float x[1];
    load_chunk<T, 1>(data + begin + tail, x);
    f(begin + tail, x, std::integral_constant<int, 1>());
  }
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double wave_sum[kBlock / kWave];
#pragma unroll
  for (int d = kWave / 2; d > 0; d /= 2) v += __shfl_xor(v, d);
  if (lane_id() == 0) wave_sum[wave_in_block()] = v;
  __syncthreads();
  double sum = 0;
#pragma unroll
  for (int w = 0; w < kBlock / kWave; ++w) sum += wave_sum[w];
  return sum;
}

template <typename T>
__device__ __forceinline__ double squares(const void *data, uint64_t count, uint32_t piece) {
  double sum = 0;
  for_elements<T>(static_cast<const T *>(data), count, piece, [&](uint64_t, const auto &x, auto vec) {
#pragma unroll
    for (int e = 0; e < decltype(vec)::value; ++e) sum = fma((double)x[e], (double)x[e], sum);
  });
  return sum;
}

__global__ __launch_bounds__(kBlock) void grad_squares_kernel(TensorList list, double *__restrict__ sums) {
  const uint32_t t = tensor_of(list, blockIdx.x), piece = blockIdx.x - list.first[t];
  const double mine = list.elem[t] == 4   ? squares<float>(list.data[t], list.count[t], piece)
                      : list.elem[t] == 2 ? squares<half_t>(list.data[t], list.count[t], piece)
                                          : squares<bhalf_t>(list.data[t], list.count[t], piece);
  const double sum = block_sum(mine);
  if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// one workgroup: the pieces' sums added up; total[0] = their sum
__global__ __launch_bounds__(kBlock) void grad_norm_kernel(const double *__restrict__ sums, size_t pieces, double *__restrict__ total,
                                                           float *__restrict__ norm) {
  double mine = 0;
  for (size_t i = threadIdx.x; i < pieces; i += kBlock) mine += sums[i];
  const double sum = block_sum(mine);
  if (threadIdx.x == 0) {
    *total = sum;
    *norm = (float)sqrt(sum);
  }
}

template <typename T>
__device__ __forceinline__ void scaled(const void *data, void *out, uint64_t count, uint32_t piece, float factor, float after) {
  for_elements<T>(static_cast<const T *>(data), count, piece, [&](uint64_t at, const auto &x, auto vec) {
    constexpr int VEC = decltype(vec)::value;
    float y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] = x[e] * factor * after;
    store_chunk<T, VEC>(static_cast<T *>(out) + at, y);
  });
}

// out = data * min(1, max_norm / (norm + 1e-6)), rounded once; nothing to do in place where the factor is 1.  A norm that is
// no number makes every element none.
__global__ __launch_bounds__(kBlock) void grad_scale_kernel(TensorList list, const double *__restrict__ total, double max_norm) {
  const double ratio = max_norm / (sqrt(*total) + 1e-6);
  // a factor near the end of float's range, which a norm beyond it brings, would lose its digits: it is multiplied in two steps
  const bool small = ratio < 0x1p-100;
  const float factor = ratio >= 1.0 ? 1.f : (float)(small ? ratio * 0x1p100 : ratio), after = small ? 0x1p-100f : 1.f;
  const uint32_t t = tensor_of(list, blockIdx.x), piece = blockIdx.x - list.first[t];
  if (factor == 1.f && list.out[t] == list.data[t]) return;
  if (list.elem[t] == 4) scaled<float>(list.data[t], list.out[t], list.count[t], piece, factor, after);
  else if (list.elem[t] == 2) scaled<half_t>(list.data[t], list.out[t], list.count[t], piece, factor, after);
  else scaled<bhalf_t>(list.data[t], list.out[t], list.count[t], piece, factor, after);
}

__global__ void preload_grad_norm_kernel() {}

}  // namespace
void preload_grad_norm(hipStream_t stream) { hipLaunchKernelGGL(preload_grad_norm_kernel, dim3(1), dim3(1), 0, stream); }

namespace {

// calls launch(list, pieces of it, pieces before it) for the tensors in lists that fit a launch's arguments
template <typename F>
int for_lists(const ugk_tensor_t *tensors, size_t n, F launch) {
  TensorList list;
  uint64_t pieces = 0, before = 0;
  list.n = 0;
  for (size_t i = 0; i <= n; ++i) {
    const uint64_t more = i < n ? pieces_of(tensors[i]) : 0;
    if (i < n && more == 0) continue;
    if (list.n > 0 && (i == n || list.n == (uint32_t)kListed || pieces + more >= ((uint64_t)1 << 31))) {
      if (int rc = launch(list, pieces, before)) return rc;
      before += pieces, pieces = 0, list.n = 0;
    }
    if (i == n) break;
    const uint32_t at = list.n++;
    list.data[at] = tensors[i].data;
    list.out[at] = tensors[i].out ? tensors[i].out : const_cast<void *>(tensors[i].data);
    list.count[at] = tensors[i].count;
    list.first[at] = (uint32_t)pieces;
    list.elem[at] = tensors[i].elem;
    pieces += more;
  }
  return 0;
}

int grad_norm(const char *what, const ugk_tensor_t *tensors, size_t n, void *workspace, size_t workspace_bytes, float *norm, hipStream_t stream) {
  UGK_REQUIRE(tensors || n == 0, "%s: null list of tensors", what);
  uint64_t pieces = 0;
  for (size_t i = 0; i < n; ++i) {
    UGK_REQUIRE(elem_ok(tensors[i].elem), "%s: element code %d of tensor %zu is none of fp32 (4), fp16 (2) and bfloat16 (UGK_ELEM_BF16)", what,
                tensors[i].elem, i);
    UGK_REQUIRE(tensors[i].data || tensors[i].count == 0, "%s: null data of tensor %zu", what, i);
    UGK_REQUIRE(tensors[i].count < ((uint64_t)1 << 44), "%s: %zu elements in tensor %zu", what, (size_t)tensors[i].count, i);
    pieces += pieces_of(tensors[i]);
  }
  UGK_REQUIRE(norm, "%s: null output", what);
  UGK_REQUIRE(workspace && workspace_bytes >= (pieces + 1) * sizeof(double), "%s: a workspace of %zu bytes, %zu are needed", what, workspace_bytes,
              (size_t)(pieces + 1) * sizeof(double));
  double *total = static_cast<double *>(workspace), *sums = total + 1;
  const int rc = for_lists(tensors, n, [&](const TensorList &list, uint64_t count, uint64_t before) -> int {
    hipLaunchKernelGGL(grad_squares_kernel, dim3((unsigned)count), dim3(kBlock), 0, stream, list, sums + before);
    UGK_HIP(hipGetLastError());
    return 0;
  });
  if (rc) return rc;
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kBlock), 0, stream, sums, (size_t)pieces, total, norm);
  UGK_HIP(hipGetLastError());
  return 0;
}

}  // namespace
}  // namespace ugk

using namespace ugk;

extern "C" {

size_t ugk_grad_norm_workspace_bytes(const ugk_tensor_t *tensors, size_t n) {
  uint64_t pieces = 0;
  for (size_t i = 0; tensors && i < n; ++i) pieces += pieces_of(tensors[i]);
  return (size_t)(pieces + 1) * sizeof(double);
}

int ugk_grad_norm(const ugk_tensor_t *tensors, size_t n, void *workspace_dev, size_t workspace_bytes, float *norm_dev, void *stream) {
  return grad_norm("ugk_grad_norm", tensors, n, workspace_dev, workspace_bytes, norm_dev, as_stream(stream));
}

int ugk_grad_clip(const ugk_tensor_t *tensors, size_t n, double max_norm, void *workspace_dev, size_t workspace_bytes, float *norm_dev,
                  void *stream) {
  UGK_REQUIRE(max_norm >= 0, "ugk_grad_clip: a limit of %g", max_norm);
  if (int rc = grad_norm("ugk_grad_clip", tensors, n, workspace_dev, workspace_bytes, norm_dev, as_stream(stream))) return rc;
  return for_lists(tensors, n, [&](const TensorList &list, uint64_t count, uint64_t) -> int {
    hipLaunchKernelGGL(grad_scale_kernel, dim3((unsigned)count), dim3(kBlock), 0, as_stream(stream), list,
                       static_cast<const double *>(workspace_dev), max_norm);
    UGK_HIP(hipGetLastError());
    return 0;
  });
}

}  // extern "C"
