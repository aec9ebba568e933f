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

// the first position in [lo, hi) whose key is not below r; hi if there is none
__device__ __forceinline__ uint32_t first_of(const uint32_t *keys, uint32_t lo, uint32_t hi, uint32_t r) {
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (keys[mid] < r) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}
// the first position behind `at` where another row's keys begin; `at` is row r's or the one behind its last
__device__ __forceinline__ uint32_t end_of(const uint32_t *keys, uint32_t at, uint32_t n, uint32_t r, uint32_t step) {
  while (step < n - at && keys[at + step] == r) at += step, step *= 2;
  return first_of(keys, at, min(at + min(step, n - at) + 1, n), r + 1);
}
// the same as first_of for a wavefront that searches for one row: 64 keys a step
__device__ __forceinline__ uint32_t wave_first_of(const uint32_t *keys, uint32_t lo, uint32_t hi, uint32_t r) {
  while (hi > lo) {
    const uint32_t step = (hi - lo + kWave - 1) / kWave, at = lo + lane_id() * step;
    const uint32_t less = (uint32_t)__popcll(__ballot(at < hi && keys[min(at, hi - 1)] < r));  // they come first
    if (step == 1) return lo + less;
    hi = min(lo + less * step, hi);
    lo = less ? lo + (less - 1) * step + 1 : lo;
  }
  return lo;
}

// begin[r] = number of sorted keys below r, r = 0 .. rows.  A search per row, so that neither a run of rows nobody named nor a
// row everybody named is one lane's work: wavefronts find the workgroup's first and last row among all keys, its lanes
// theirs between the two.
__global__ __launch_bounds__(kBlock) void row_begin_kernel(const uint32_t *__restrict__ keys, uint32_t n, uint32_t rows,
                                                           uint32_t *__restrict__ begin) {
  __shared__ uint32_t ends[2];
  const uint32_t r0 = blockIdx.x * kBlock, r = r0 + threadIdx.x, wave = wave_in_block();
  if (wave < 2) {
    const uint32_t found = wave_first_of(keys, 0, n, wave == 0 ? r0 : min(r0 + kBlock, rows));
    if (lane_id() == 0) ends[wave] = found;
  }
  __syncthreads();
  if (r <= rows) begin[r] = first_of(keys, ends[0], ends[1], r);
}

// sum += the rows grad[entries[j]], from <= j < to, in the order of j
template <typename T, int VEC>
__device__ __forceinline__ void add_entries(const T *grad, size_t stride, const uint32_t *entries, uint32_t from, uint32_t to, uint32_t at,
                                            float (&sum)[VEC]) {
  constexpr uint32_t U = 4;  // rows on their way
  uint32_t j = from;
  for (; j + U <= to; j += U) {
    typename ChunkOf<T, VEC>::type v[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) v[u] = raw_chunk<T, VEC>(grad + (size_t)entries[j + u] * stride + at);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      float x[VEC];
      to_floats<T, VEC>(v[u], x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] += x[e];
    }
  }
  for (; j < to; ++j) {
    float x[VEC];
    load_chunk<T, VEC>(grad + (size_t)entries[j] * stride + at, x);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] += x[e];
  }
}

// A row of more than `piece` entries is summed in pieces: the positions are cut into runs of `piece`, and a run holds parts of
// at most two such rows, one that comes in from the run before and one that begins in it and goes on behind it.
// parts[2 * run] and parts[2 * run + 1] are their sums.
//
// Where a row's entries are is in begin[] (BY_ROW), or is searched for among the keys.
struct Sorted {
  const uint32_t *keys, *begin;
  uint32_t n, rows, piece;
};

// (Keys that a decision needs are loaded together, whether or not the first of them settles it: they were written by another
// XCD and are a microsecond away each.)

// whether a row that is summed in pieces begins in a run; the row, its first position, and where the run's entries end
template <bool BY_ROW>
__device__ __forceinline__ bool long_row_from(const Sorted &s, uint32_t run, uint32_t &row, uint32_t &first, uint32_t &to) {
  const uint32_t from = run * s.piece;
  to = min(from + s.piece, s.n);
  row = s.keys[to - 1];
  if constexpr (BY_ROW) {
    const uint32_t live = s.begin[s.rows];
    if (row >= s.rows) {  // entries without a row come last
      if (from >= live) return false;
      to = live;
      row = s.keys[to - 1];
    }
    first = s.begin[row];
    return first >= from && s.begin[row + 1] - first > s.piece;
  } else {
    const uint32_t behind = s.keys[min(to, s.n - 1)], head = s.keys[from], before = s.keys[max(from, 1u) - 1];
    // it goes on behind the run, and did not begin before it
    if (row >= s.rows || to == s.n || behind != row || (from > 0 && before == row)) return false;
    first = head == row ? from : first_of(s.keys, from + 1, to, row);
    return first + s.piece < s.n && s.keys[first + s.piece] == row;
  }
}
// whether a row that is summed in pieces comes into a run from the one before, and where its entries end there
template <bool BY_ROW>
__device__ __forceinline__ bool long_row_into(const Sorted &s, uint32_t run, uint32_t &end) {
  const uint32_t from = run * s.piece, to = min(from + s.piece, s.n);
  if (from >= s.n || from == 0) return false;
  const uint32_t row = s.keys[from];
  if constexpr (BY_ROW) {
    if (row >= s.rows) return false;
    const uint32_t first = s.begin[row], last = s.begin[row + 1];
    end = min(to, last);
    return first < from && last - first > s.piece;
  } else {
    const uint32_t before = s.keys[from - 1], back = s.keys[from - s.piece], tail = s.keys[to - 1];
    if (row >= s.rows || before != row) return false;
    const uint32_t first = back == row ? from - s.piece : first_of(s.keys, from - s.piece + 1, from, row);
    if (first + s.piece >= s.n || s.keys[first + s.piece] != row) return false;
    end = tail == row ? to : first_of(s.keys, from + 1, to, row + 1);
    return true;
  }
}

// The parts of the runs, and the rows of at most `piece` entries.  BY_ROW: a lane's row is i (the first row_blocks workgroups),
// and one without entries is zero.  Otherwise i is a position, the lane's row the one that begins there, and out holds zeros.
template <typename T, int VEC, bool BY_ROW, bool STREAM>
__global__ __launch_bounds__(kBlock) void row_sum_kernel(const T *__restrict__ grad, size_t stride, const uint32_t *__restrict__ entries,
                                                         Sorted s, uint32_t dim, Split split, uint32_t row_blocks, T *__restrict__ out,
                                                         float *__restrict__ parts) {
  size_t i;
  uint32_t c;
  const bool whole = blockIdx.x < row_blocks;
  split_lane(split, whole ? blockIdx.x : blockIdx.x - row_blocks, i, c);
  const uint32_t at = min(c * VEC, dim - VEC);
  float sum[VEC] = {};
  uint32_t from, to;
  if (whole) {
    if constexpr (BY_ROW) {
      if (i >= s.rows) return;
      from = s.begin[i], to = s.begin[i + 1];
      if (to - from > s.piece) return;
    } else {
      if (i >= s.n) return;
      from = (uint32_t)i;
      to = min(from + s.piece, s.n);
      const uint32_t r = s.keys[from], before = s.keys[max(from, 1u) - 1], next = s.keys[min(from + 1, s.n - 1)],
                     behind = s.keys[min(to, s.n - 1)];
      if (r >= s.rows || (from > 0 && before == r) || (to < s.n && behind == r)) return;
      to = from + 1 < s.n && next == r ? first_of(s.keys, from + 2, to, r + 1) : from + 1;
      i = r;
    }
    add_entries<T, VEC>(grad, stride, entries, from, to, at, sum);
    store_chunk<T, VEC, STREAM>(out + i * dim + at, sum);
    return;
  }
  if (i * s.piece >= s.n) return;
  if (long_row_into<BY_ROW>(s, (uint32_t)i, to)) {
    add_entries<T, VEC>(grad, stride, entries, (uint32_t)i * s.piece, to, at, sum);
    store_chunk<float, VEC>(parts + 2 * i * dim + at, sum);
  }
  uint32_t row;
  if (long_row_from<BY_ROW>(s, (uint32_t)i, row, from, to)) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
    add_entries<T, VEC>(grad, stride, entries, from, to, at, sum);
    store_chunk<float, VEC>(parts + (2 * i + 1) * dim + at, sum);
  }
}

// sum += the parts from .. to of a row whose first is in run p0
template <int VEC>
__device__ __forceinline__ void add_parts(const float *parts, uint32_t dim, uint32_t p0, uint32_t from, uint32_t to, uint32_t at,
                                          float (&sum)[VEC]) {
  constexpr uint32_t U = 8;  // parts on their way
  for (uint32_t p = from; p < to; p += U) {
    float v[U][VEC];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t q = min(p + u, to - 1);
      load_chunk<float, VEC>(parts + (2 * (size_t)(p0 + q) + (q == 0 ? 1 : 0)) * dim + at, v[u]);
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] += p + u < to ? v[u][e] : 0.f;
  }
}

// The parts of a row added up, for `lanes` chunks of it.  A group of `lanes` lanes looks after a run: if a row that is summed
// in pieces begins there it adds the row's parts; those of a row of many parts the workgroup's kBlock / lanes groups add
// together, consecutive ones each, and the groups' sums are added in their order.  (us of the gradient, many from 8 / 16 / 32 /
// 64 on: 16,384 entries over 50,000 rows, 8 groups 46.0 / 46.0 / 47.2 / 51.9; 202,156 over 3,277 rows of 16 bytes, 256 groups
// 150 / 105 / 80 / 72.)
template <typename T, int VEC, bool BY_ROW>
__global__ __launch_bounds__(kBlock) void row_join_kernel(Sorted s, uint32_t runs, uint32_t dim, uint32_t chunks, uint32_t lanes, uint32_t columns,
                                                          const float *__restrict__ parts, T *__restrict__ out) {
  __shared__ float held[kBlock * VEC];
  __shared__ uint32_t many[kBlock][3], n_many;  // rows of many parts: the row, its first run, its parts
  if (threadIdx.x == 0) n_many = 0;
  __syncthreads();
  const uint32_t group = threadIdx.x / lanes, groups = kBlock / lanes;  // lanes: a power of two
  const uint32_t run0 = blockIdx.x / columns * groups, column = blockIdx.x % columns;
  const uint32_t c = column * lanes + threadIdx.x % lanes;
  const uint32_t at = min(c * VEC, dim - VEC);
  const uint32_t run = run0 + group, few = max(16u, groups / 4);
  uint32_t r = 0, from = 0, to = 0, pieces = 0;
  if (run < runs && long_row_from<BY_ROW>(s, run, r, from, to)) {
    if constexpr (BY_ROW) to = s.begin[r + 1];
    else to = end_of(s.keys, to, s.n, r, s.piece);
    pieces = (to - 1) / s.piece - run + 1;
  }
  if (threadIdx.x % lanes == 0 && pieces > few) {
    const uint32_t g = atomicAdd(&n_many, 1u);  // rows are added up one by one: in whatever order
    many[g][0] = r, many[g][1] = run, many[g][2] = pieces;
  }
  if (pieces > 0 && pieces <= few && c < chunks) {
    float sum[VEC] = {};
    add_parts<VEC>(parts, dim, run, 0, pieces, at, sum);
    store_chunk<T, VEC>(out + (size_t)r * dim + at, sum);
  }
  __syncthreads();
  for (uint32_t g = 0; g < n_many; ++g) {
    pieces = many[g][2];
    const uint32_t per = (pieces + groups - 1) / groups;
    float sum[VEC] = {};
    if (c < chunks) add_parts<VEC>(parts, dim, many[g][1], min(group * per, pieces), min((group + 1) * per, pieces), at, sum);
#pragma unroll
    for (int e = 0; e < VEC; ++e) held[e * kBlock + threadIdx.x] = sum[e];
    __syncthreads();
    if (group == 0 && c < chunks) {
      for (uint32_t h = 1; h < groups; ++h)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] += held[e * kBlock + h * lanes + threadIdx.x];
      store_chunk<T, VEC>(out + (size_t)many[g][0] * dim + at, sum);
    }
    __syncthreads();
  }
}

// more of the output than the sort's launches clear on their side
__global__ __launch_bounds__(kSortBlock) void clear_kernel(Clear clear) { clear_block(clear, blockIdx.x); }


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
    UGK_REQUIRE(blocks <= kMaxBlocks, "ugk_take_rows: %zu rows of %zu elements are more than one launch takes", n, dim);
    hipLaunchKernelGGL((take_rows_kernel<T, V, decltype(stream_out)::value, I>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream),
                       (const T *)table, num_rows, stride, index, n, (uint32_t)dim, s, (T *)out);
    UGK_HIP(hipGetLastError());
    return 0;
  });
}

// how a batch of n entries over `rows` rows is sorted: digits of equal length, the key `rows` (no row) among them
// (as few digits as ten bits allow; us of the gradient of rows of 32 bytes by position over 2^20 - 1 rows, two digits of ten bits,
// and over 2^20 + 1, three of seven: 250,000 entries 52.5 and 50.4, 500,000 67.3 and 63.0, 1,000,000 91.2 and 84.5)
struct Plan {
  uint32_t passes, digit;
};
Plan plan_for(uint64_t rows) {
  const uint32_t bits = bits_for(rows + 1);
  const uint32_t passes = bits <= 10 ? 1u : bits <= 20 ? 2u : bits <= 30 ? 3u : 4u;
  return Plan{passes, (bits + passes - 1) / passes};
}

// Where some rows are named by nobody for certain the output is cleared on the side of the sort, which leaves the memory idle,
// and only rows with entries are visited after it; where most may be named that would store them twice, but for small outputs,
// and a row's entries are found by a launch of its own instead of searches by whoever adds them.  us, by position / by row:
// 16,384 entries over 50,000 bfloat16 rows of 2 KB 46 / 62, 40,000 over 50,000 76 / 98, 100,000 over 200,000 of 256 bytes 70 / 69;
// 3,000 over 3,000 of 128 bytes 18.6 / 21.0, 10,000 over 5,000 of 256 bytes 30 / 31, 213,119 over as many of 16 bytes 37 / 42;
// 40,000 over 40,000 of 4 KB 145 / 111, 262,144 over 60,000 of 512 bytes 133 / 105, 100,000 over 2,000 of 1 KB 59 / 48, 928,382 over
// 42,603 of 8 bytes 84 / 70.  The line of 4,000,000 elements is between the types' own, which lie near 12 MB of output (fp32
// rows of 400 bytes 2.8 M elements 34.6 / 32.5, 3.8 M 39.4 / 35.4; bfloat16 rows of 1,000 bytes 4.2 M 25.7 / 26.5, 5.6 M 28.1 / 29.4,
// 8.4 M 37.1 / 34.4).  Rows that outnumber the entries a little are visited by position too, which costs where they are many MB:
// 285,714 bfloat16 rows of 2 KB and 200,000 entries 392 / 281, of 16 bytes 42.6 / 47.3.
bool sums_by_row(size_t n, uint64_t rows, size_t dim) { return rows <= n && (rows * dim > 4'000'000 || (n > 32768 && n > 2 * rows)); }

// Entries a lane adds one after the other: few where the batch is small and their latency is what it costs, more where the
// parts are traffic.  us, of 16 / 32 / 64: 16,384 bfloat16 rows of 1,024 elements 56 / 59 / 63, 30,000 95 / 95 / 104, 100,000 fp32
// rows of 128 120 / 124 / 137, 262,144 of them 115 / 105 / 107, 30,000 bfloat16 rows of 2,048 132 / 126 / 132.
uint32_t piece_for(size_t n, size_t dim) { return n * dim <= 20'000'000 ? 16u : 32u; }
size_t pieces_of(size_t n, size_t dim) { return (n + piece_for(n, dim) - 1) / piece_for(n, dim); }

size_t begin_words(size_t n, uint64_t rows, size_t dim) { return sums_by_row(n, rows, dim) ? (size_t)rows + 1 : 0; }

template <typename I>
int take_rows_grad(const void *grad, size_t stride, const I *index, size_t n, uint64_t num_rows, size_t dim, int elem, void *out,
                   void *workspace, size_t workspace_bytes, void *stream) {
  UGK_REQUIRE(elem_ok(elem), "ugk_take_rows_grad: element code %d is none of fp32 (4), fp16 (2) and bfloat16 (UGK_ELEM_BF16)", elem);
  UGK_REQUIRE(dim >= 1 && dim < kMaxDim, "ugk_take_rows_grad: rows of %zu elements", dim);
  UGK_REQUIRE(n < ((size_t)1 << 31) && num_rows < ((uint64_t)1 << 31), "ugk_take_rows_grad: %zu entries of %zu rows, both have 31 bits", n,
              (size_t)num_rows);
  UGK_REQUIRE(stride >= dim || n <= 1, "ugk_take_rows_grad: rows of %zu elements overlap at a stride of %zu", dim, stride);
  // a workgroup's 256 chunks, of the rows, of the entries and of the parts
  UGK_REQUIRE((num_rows + 2 * n) * chunks_of(elem, dim) / kBlock + 2 < kMaxBlocks,
              "ugk_take_rows_grad: %zu rows and %zu entries of %zu elements are more than one launch takes", (size_t)num_rows, n, dim);
  if (num_rows == 0) return 0;
  UGK_REQUIRE(out && (n == 0 || (grad && index)), "ugk_take_rows_grad: null pointer");
  const size_t need = ugk_take_rows_grad_workspace_bytes(n, num_rows, dim);
  UGK_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "ugk_take_rows_grad: a workspace of %zu bytes, %zu are needed",
              workspace_bytes, need);
  uint32_t *begin = static_cast<uint32_t *>(workspace);
  uint32_t *key[2] = {begin + begin_words(n, num_rows, dim), begin + begin_words(n, num_rows, dim) + n}, *entry[2] = {key[1] + n, key[1] + 2 * n};
  float *parts = reinterpret_cast<float *>(entry[1] + n);
  uint32_t *words = reinterpret_cast<uint32_t *>(parts + 2 * pieces_of(n, dim) * dim);
  if (n == 0) {
    Clearing all(out, num_rows * dim * elem_size(elem));
    Clear clear;
    const uint32_t blocks = all.take(clear, 1, 1);
    hipLaunchKernelGGL(clear_kernel, dim3(blocks), dim3(kSortBlock), 0, as_stream(stream), clear);
    UGK_HIP(hipGetLastError());
    return 0;
  }
  const Plan p = plan_for(num_rows);
  const bool by_row = sums_by_row(n, num_rows, dim);
  Clearing clearing(out, by_row ? 0 : num_rows * dim * elem_size(elem));
  Digits d{num_rows, 0, (1u << p.digit) - 1u, 1u << p.digit, p.digit};
  int at = 0;
  const SortShape shape = sort_shape(n, d.buckets);
  if (shape.reach == kSingle) {
    Clear clear;
    const uint32_t blocks = clearing.take(clear, 1, 1);
    const auto one = [&](auto items) {
      hipLaunchKernelGGL((sort_one_tile_kernel<I, decltype(items)::value>), dim3(1 + blocks), dim3(kSortBlock), 0, as_stream(stream), index,
                         (uint32_t)n, p.passes, d, clear, key[0], entry[0]);
    };
    if (shape.items == 2) one(std::integral_constant<int, 2>());
    else if (shape.items == 4) one(std::integral_constant<int, 4>());
    else one(std::integral_constant<int, 8>());
    UGK_HIP(hipGetLastError());
  } else {
    if (int rc = sort_pass<kFirst, I>(index, nullptr, n, d, words, key[0], entry[0], nullptr, &clearing, p.passes, as_stream(stream))) return rc;
    for (uint32_t pass = 1; pass < p.passes; ++pass, at ^= 1) {
      d.shift += p.digit;
      if (int rc = sort_pass<kNext, uint32_t>(key[at], entry[at], n, d, words, key[at ^ 1], entry[at ^ 1], nullptr, &clearing, p.passes - pass,
                                              as_stream(stream)))
        return rc;
    }
  }
  if (by_row)
    hipLaunchKernelGGL(row_begin_kernel, dim3((unsigned)(num_rows / kBlock + 1)), dim3(kBlock), 0, as_stream(stream), key[at], (uint32_t)n,
                       (uint32_t)num_rows, begin);
  return for_rows_streamed(elem, dim, num_rows, [&](auto type, auto vec, auto stream_out) -> int {
    typedef decltype(type) T;
    constexpr int V = decltype(vec)::value;
    const Split s = split_of(dim, V);
    const uint32_t piece = piece_for(n, dim);
    const Sorted sorted{key[at], begin, (uint32_t)n, (uint32_t)num_rows, piece};
    const size_t pieces = n > piece ? pieces_of(n, dim) : 0;  // in fewer entries no row has more than a piece
    const size_t row_blocks = split_blocks(by_row ? num_rows : n, s), blocks = row_blocks + split_blocks(pieces, s);
    uint32_t lanes = 1;
    while (lanes < s.chunks && lanes < 32) lanes *= 2;
    const uint32_t columns = (s.chunks + lanes - 1) / lanes;
    const auto launch = [&](auto rowwise, auto stored) {
      constexpr bool R = decltype(rowwise)::value;
      hipLaunchKernelGGL((row_sum_kernel<T, V, R, decltype(stored)::value>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream),
                         (const T *)grad, stride, entry[at], sorted, (uint32_t)dim, s, (uint32_t)row_blocks, (T *)out, parts);
      if (pieces > 0)
        hipLaunchKernelGGL((row_join_kernel<T, V, R>), dim3((unsigned)((pieces + kBlock / lanes - 1) / (kBlock / lanes)) * columns),
                           dim3(kBlock), 0, as_stream(stream), sorted, (uint32_t)pieces, (uint32_t)dim, s.chunks, lanes, columns, parts, (T *)out);
    };
    if (by_row) launch(std::true_type(), stream_out);
    else launch(std::false_type(), std::false_type());
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
  return 4 * (begin_words(n, num_rows, dim) + 4 * n + 2 * pieces_of(n, dim) * dim + sort_count_words(n, 1u << plan_for(num_rows).digit));
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
