// The l2 norm over all gradients of a training step, and the gradients scaled down to a limit.
//
// norm = sqrt(sum over tensors and elements of x^2).  Squares and sums are held in 64 bits: a float's square needs twice
// its exponent, and a thousand million terms need more than 24 bits.  Every workgroup sums one piece of one tensor, the
// pieces' sums are added in their order, so the same gradients give the same bits on every run.
#include <algorithm>

#include "ugk_rows.cuh"

namespace ugk {
namespace {

// What a launch is told of its tensors travels in its arguments (the list of a training step changes with every step):
// up to kListed parts of tensors at a time, each a run of consecutive pieces (with the hidden ones the arguments stay in 4 KB).
constexpr int kListed = 144;
constexpr uint32_t kPieceBytes = 32768;
constexpr uint64_t kPartElems = (uint64_t)1 << 31;  // of a tensor that has more; a multiple of a piece
struct TensorList {
  const void *data[kListed];
  void *out[kListed];
  uint32_t count[kListed];
  uint32_t first[kListed];  // a part's first piece in this launch
  uint8_t elem[kListed];    // 4, 2 or 1 for bfloat16
  uint32_t n, pieces;
};
struct Listed {
  const void *data;
  void *out;
  uint32_t count;
  int elem;
};

__host__ __device__ static inline uint32_t pieces_in(uint64_t count, int elem) {
  return (uint32_t)((count * (elem == 4 ? 4 : 2) + kPieceBytes - 1) / kPieceBytes);
}
static inline uint64_t pieces_of(const ugk_tensor_t &t) { return pieces_in(t.count, t.elem); }

__device__ __forceinline__ Listed listed(const TensorList &list, uint32_t at) {
  return Listed{list.data[at], list.out[at], list.count[at], list.elem[at]};
}

// the tensor of a piece: how many of the first pieces are not behind it
__device__ __forceinline__ uint32_t tensor_of(const TensorList &list, uint32_t piece) {
  uint32_t found = 0;
#pragma unroll
  for (uint32_t i = 0; i < kListed; i += kWave) {
    const uint32_t at = i + lane_id();
    found += (uint32_t)__popcll(__ballot(at < list.n && list.first[min(at, (uint32_t)kListed - 1)] <= piece));
  }
  return __builtin_amdgcn_readfirstlane(found - 1);
}

// f for the 16-byte chunks of a piece, all of a lane's on their way at once where the piece is a whole one, and for the
// elements behind the last chunk
template <typename T, bool STREAM, typename F>
__device__ __forceinline__ void for_elements(const T *data, uint64_t count, uint32_t piece, F f) {
  constexpr int VEC = 16 / sizeof(T), U = kPieceBytes / (16 * kBlock);
  constexpr uint32_t kElems = kPieceBytes / sizeof(T);
  const uint64_t begin = (uint64_t)piece * kElems;
  // (a shift and not min(): of a 64-bit minimum in scalar registers that a branch depends on as well, this compiler makes a
  // select without its condition)
  const uint64_t left = count - begin;
  const bool whole = left / kElems != 0;
  const uint32_t n = whole ? kElems : (uint32_t)left;
  const T *from = data + begin;
  if (whole) {
    typename ChunkOf<T, VEC>::type v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = raw_chunk<T, VEC, STREAM>(from + (u * kBlock + threadIdx.x) * VEC);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[VEC];
      to_floats<T, VEC>(v[u], x);
      f(begin + (u * kBlock + threadIdx.x) * VEC, x, std::integral_constant<int, VEC>());
    }
    return;
  }
  for (uint32_t i = threadIdx.x * VEC; i + VEC <= n; i += kBlock * VEC) {
    float x[VEC];
    load_chunk<T, VEC>(from + i, x);
    f(begin + i, x, std::integral_constant<int, VEC>());
  }
  const uint32_t tail = n / VEC * VEC + threadIdx.x;
  if (tail < n) {
    float x[1];
    load_chunk<T, 1>(from + tail, x);
    f(begin + tail, x, std::integral_constant<int, 1>());
  }
}

template <int BLOCK>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double wave_sum[BLOCK / kWave];
#pragma unroll
  for (int d = kWave / 2; d > 0; d /= 2) v += __shfl_xor(v, d);
  if (lane_id() == 0) wave_sum[wave_in_block()] = v;
  __syncthreads();
  double sum = 0;
#pragma unroll
  for (int w = 0; w < BLOCK / kWave; ++w) sum += wave_sum[w];
  return sum;
}

template <typename T, bool STREAM>
__device__ __forceinline__ double squares(const void *data, uint64_t count, uint32_t piece) {
  double sum = 0;
  for_elements<T, STREAM>(static_cast<const T *>(data), count, piece, [&](uint64_t, const auto &x, auto vec) {
#pragma unroll
    for (int e = 0; e < decltype(vec)::value; ++e) sum = fma((double)x[e], (double)x[e], sum);
  });
  return sum;
}

template <bool STREAM>
__device__ __forceinline__ double squares_of(const Listed &t, uint32_t piece) {
  return t.elem == 4   ? squares<float, STREAM>(t.data, t.count, piece)
         : t.elem == 2 ? squares<half_t, STREAM>(t.data, t.count, piece)
                       : squares<bhalf_t, STREAM>(t.data, t.count, piece);
}

// What the memory-side cache keeps between the two passes over the gradients: the last kKept pieces (224 MiB) are read for
// the norm the ordinary way, the ones before them past the caches, and the second pass goes from the last piece to the first;
// its stores go past the caches too where gradients and outputs are more than the cache holds.  us, norm and scaling into
// other tensors, all ordinary / these rules: 1.4 GB of bfloat16 766 / 702, 302 MB 173 / 138, 151 MB 76 / 72.
constexpr uint64_t kKept = ((uint64_t)224 << 20) / kPieceBytes;

// the first `streamed` pieces past the caches
__global__ __launch_bounds__(kBlock) void grad_squares_kernel(TensorList list, uint32_t streamed, double *__restrict__ sums) {
  const uint32_t at = tensor_of(list, blockIdx.x), piece = blockIdx.x - list.first[at];
  const Listed t = listed(list, at);
  const double mine = blockIdx.x < streamed ? squares_of<true>(t, piece) : squares_of<false>(t, piece);
  const double sum = block_sum<kBlock>(mine);
  if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// the pieces' sums added up by a workgroup, the same way on every call of a block size
template <int BLOCK>
__device__ __forceinline__ double sum_of_pieces(const double *sums, uint64_t pieces) {
  constexpr int U = 8;  // sums on their way
  double mine = 0;
  for (uint64_t i = threadIdx.x; i < pieces; i += U * BLOCK) {
    double v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = sums[i + u * BLOCK < pieces ? i + u * BLOCK : i];
#pragma unroll
    for (int u = 0; u < U; ++u) mine += i + u * BLOCK < pieces ? v[u] : 0.0;
  }
  return block_sum<BLOCK>(mine);
}

// one workgroup: total[0] = the sum of all squares
constexpr int kNormBlock = 1024;
__global__ __launch_bounds__(kNormBlock) void grad_norm_kernel(const double *__restrict__ sums, uint64_t pieces, double *__restrict__ total,
                                                               float *__restrict__ norm) {
  const double sum = sum_of_pieces<kNormBlock>(sums, pieces);
  if (threadIdx.x == 0) {
    *total = sum;
    *norm = (float)sqrt(sum);
  }
}

template <typename T, bool STREAM, bool STREAM_OUT>
__device__ __forceinline__ void scaled(const void *data, void *out, uint64_t count, uint32_t piece, float factor, float after) {
  for_elements<T, STREAM>(static_cast<const T *>(data), count, piece, [&](uint64_t at, const auto &x, auto vec) {
    constexpr int VEC = decltype(vec)::value;
    float y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] = x[e] * factor * after;
    store_chunk<T, VEC, STREAM_OUT>(static_cast<T *>(out) + at, y);
  });
}
template <bool STREAM, bool STREAM_OUT>
__device__ __forceinline__ void scale_one(const Listed &t, uint32_t piece, float factor, float after) {
  if (t.elem == 4) scaled<float, STREAM, STREAM_OUT>(t.data, t.out, t.count, piece, factor, after);
  else if (t.elem == 2) scaled<half_t, STREAM, STREAM_OUT>(t.data, t.out, t.count, piece, factor, after);
  else scaled<bhalf_t, STREAM, STREAM_OUT>(t.data, t.out, t.count, piece, factor, after);
}

// out = data * min(1, max_norm / (norm + 1e-6)), rounded once; nothing to do in place where the factor is 1.  A norm that is
// no number makes every element none.  An infinite max_norm scales nothing, whatever the norm is.
// The first `kept` pieces are read the ordinary way.  Few pieces are added up by every workgroup, and the norm is left by the
// first, without a launch in between (`norm` set; 98,816 gradients in twelve tensors: 9.0 -> 7.3 us); the sum of more is in
// total[0], in front of the pieces'.  The launch saved is worth the same at any number (us of the kernels, added up by a launch / by
// every workgroup: one tensor of 100 pieces 8.3 / 7.0, 1,024 pieces 21.8 / 20.2, 2,048 36.0 / 34.3, 4,096 64.7 / 63.4; 1,000 pieces in
// 100 tensors 22.1 / 20.3, 4,000 64.8 / 63.0), while what every workgroup reads grows with it; the line keeps that to 8 KB.
constexpr uint64_t kFewPieces = 1024;
template <bool STREAM_OUT>
__global__ __launch_bounds__(kBlock) void grad_scale_kernel(TensorList list, uint32_t kept, const double *__restrict__ total, uint32_t pieces,
                                                            float *__restrict__ norm, double max_norm) {
  const double length = sqrt(norm ? sum_of_pieces<kBlock>(total + 1, pieces) : *total);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)length;  // the same in every list
  const double ratio = isinf(max_norm) ? 1.0 : max_norm / (length + 1e-6);
  // a factor near the end of float's range, which a norm beyond it brings, would lose its digits: it is multiplied in two steps
  const bool small = ratio < 0x1p-100;
  const float factor = ratio >= 1.0 ? 1.f : (float)(small ? ratio * 0x1p100 : ratio), after = small ? 0x1p-100f : 1.f;
  // from the last piece to the first: the last ones read for the norm are the ones the memory-side cache still holds
  // (the tensors are listed from the last to the first)
  const uint32_t at = tensor_of(list, blockIdx.x);
  const Listed t = listed(list, at);
  const uint32_t piece = pieces_in(t.count, t.elem) - 1 - (blockIdx.x - list.first[at]);
  if (factor == 1.f && t.out == t.data) return;
  if (blockIdx.x < kept) scale_one<false, STREAM_OUT>(t, piece, factor, after);
  else scale_one<true, STREAM_OUT>(t, piece, factor, after);
}


// calls launch(list, pieces before it) for the parts of the tensors in lists that fit a launch's arguments, from the last part
// to the first where `backwards`
template <typename F>
int for_lists(const ugk_tensor_t *tensors, size_t n, bool backwards, F launch) {
  TensorList list;
  uint64_t before = 0;
  list.n = list.pieces = 0;
  for (size_t k = 0; k < n; ++k) {
    const ugk_tensor_t &t = tensors[backwards ? n - 1 - k : k];
    const uint64_t parts = (t.count + kPartElems - 1) / kPartElems;
    for (uint64_t j = 0; j < parts; ++j) {
      const uint64_t from = (backwards ? parts - 1 - j : j) * kPartElems, count = std::min(kPartElems, t.count - from);
      const uint32_t more = pieces_in(count, t.elem);
      if (list.n > 0 && (list.n == (uint32_t)kListed || (uint64_t)list.pieces + more > kMaxBlocks)) {
        if (int rc = launch(list, before)) return rc;
        before += list.pieces;
        list.n = list.pieces = 0;
      }
      const uint32_t at = list.n++;
      const size_t bytes = from * elem_size(t.elem);
      list.data[at] = static_cast<const char *>(t.data) + bytes;
      list.out[at] = (t.out ? static_cast<char *>(t.out) : const_cast<char *>(static_cast<const char *>(t.data))) + bytes;
      list.count[at] = (uint32_t)count;
      list.elem[at] = t.elem == UGK_ELEM_BF16 ? 1 : (uint8_t)t.elem;
      list.first[at] = list.pieces;
      list.pieces += more;
    }
  }
  return list.n > 0 ? launch(list, before) : 0;
}

// the sums of squares of all pieces, behind the first word of the workspace
int grad_squares(const char *what, const ugk_tensor_t *tensors, size_t n, void *workspace, size_t workspace_bytes, const float *norm,
                 uint64_t &pieces, hipStream_t stream) {
  UGK_REQUIRE(tensors || n == 0, "%s: null list of tensors", what);
  pieces = 0;
  for (size_t i = 0; i < n; ++i) {
    UGK_REQUIRE(elem_ok(tensors[i].elem), "%s: element code %d of tensor %zu is none of fp32 (4), fp16 (2) and bfloat16 (UGK_ELEM_BF16)", what,
                tensors[i].elem, i);
    UGK_REQUIRE(tensors[i].data || tensors[i].count == 0, "%s: null data of tensor %zu", what, i);
    UGK_REQUIRE(tensors[i].count < ((uint64_t)1 << 42), "%s: %zu elements in tensor %zu", what, (size_t)tensors[i].count, i);
    pieces += pieces_of(tensors[i]);
  }
  UGK_REQUIRE(norm, "%s: null output", what);
  UGK_REQUIRE(workspace && workspace_bytes >= (pieces + 1) * sizeof(double), "%s: a workspace of %zu bytes, %zu are needed", what, workspace_bytes,
              (size_t)(pieces + 1) * sizeof(double));
  double *sums = static_cast<double *>(workspace) + 1;
  return for_lists(tensors, n, false, [&](const TensorList &list, uint64_t before) -> int {
    // pieces in front of the last kKept of all
    const uint64_t streamed = pieces > kKept + before ? pieces - kKept - before : 0;
    hipLaunchKernelGGL(grad_squares_kernel, dim3(list.pieces), dim3(kBlock), 0, stream, list, (uint32_t)std::min<uint64_t>(streamed, list.pieces),
                       sums + before);
    UGK_HIP(hipGetLastError());
    return 0;
  });
}

int grad_norm(void *workspace, uint64_t pieces, float *norm, hipStream_t stream) {
  double *total = static_cast<double *>(workspace);
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kNormBlock), 0, stream, total + 1, pieces, total, norm);
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
  uint64_t pieces;
  if (int rc = grad_squares("ugk_grad_norm", tensors, n, workspace_dev, workspace_bytes, norm_dev, pieces, as_stream(stream))) return rc;
  return grad_norm(workspace_dev, pieces, norm_dev, as_stream(stream));
}

int ugk_grad_clip(const ugk_tensor_t *tensors, size_t n, double max_norm, void *workspace_dev, size_t workspace_bytes, float *norm_dev,
                  void *stream) {
  UGK_REQUIRE(max_norm >= 0, "ugk_grad_clip: a limit of %g", max_norm);
  uint64_t pieces;
  if (int rc = grad_squares("ugk_grad_clip", tensors, n, workspace_dev, workspace_bytes, norm_dev, pieces, as_stream(stream))) return rc;
  const bool few = pieces > 0 && pieces <= kFewPieces;
  if (!few)
    if (int rc = grad_norm(workspace_dev, pieces, norm_dev, as_stream(stream))) return rc;
  uint64_t read = 0, written = 0;  // bytes
  for (size_t i = 0; i < n; ++i) {
    read += tensors[i].count * elem_size(tensors[i].elem);
    if (tensors[i].out && tensors[i].out != tensors[i].data) written += tensors[i].count * elem_size(tensors[i].elem);
  }
  const bool stream_out = read + written > kMemorySideCacheBytes;
  return for_lists(tensors, n, true, [&](const TensorList &list, uint64_t before) -> int {
    const uint32_t kept = before < kKept ? (uint32_t)(kKept - before) : 0;
    if (stream_out)
      hipLaunchKernelGGL(grad_scale_kernel<true>, dim3(list.pieces), dim3(kBlock), 0, as_stream(stream), list, kept,
                         static_cast<const double *>(workspace_dev), (uint32_t)pieces, few ? norm_dev : nullptr, max_norm);
    else
      hipLaunchKernelGGL(grad_scale_kernel<false>, dim3(list.pieces), dim3(kBlock), 0, as_stream(stream), list, kept,
                         static_cast<const double *>(workspace_dev), (uint32_t)pieces, few ? norm_dev : nullptr, max_norm);
    UGK_HIP(hipGetLastError());
    return 0;
  });
}

}  // extern "C"
