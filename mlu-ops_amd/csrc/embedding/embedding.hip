// mluOpExtEmbeddingForward / Backward (no counterpart in the reference): rows of a table by their numbers, scaled, and the
// gradient of the table.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "core/core.h"
#include "core/device_sort.h"
#include "core/elements.h"
#include "mlu_op_ext.h"

namespace {

using namespace mluop;
typedef unsigned long long u64;

constexpr int kThreads = 256;
template <int V>
using Lanes = RowLanes<V, kThreads>;

// Tokens of either type.
struct Tokens {
  const void *at;
  bool wide;
  uint32_t rows;
  // The row that token i names; `rows` where it names none.
  __device__ __forceinline__ uint32_t row(int64_t i) const {
    const int64_t t = wide ? static_cast<const int64_t *>(at)[i] : (int64_t) static_cast<const int32_t *>(at)[i];
    return (u64)t < rows ? (uint32_t)t : rows;
  }
};

// ---- forward -------------------------------------------------------------------------------

constexpr int kRowsAThread = 4;  // whose loads are in flight together

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void embeddingRows(const T *__restrict__ table, int64_t row_stride, int channels,
                                                          Tokens tokens, int64_t n, float scale, T *__restrict__ out) {
  const Lanes<V> l(channels);
  if (l.row < 0) return;
  const int64_t first = (int64_t)blockIdx.x * l.rows_at_once * kRowsAThread + l.row;
  uint32_t row[kRowsAThread];
#pragma unroll
  for (int j = 0; j < kRowsAThread; ++j) {
    const int64_t t = first + j * l.rows_at_once;
    row[j] = t < n ? tokens.row(t) : tokens.rows;
  }
  float v[kRowsAThread][V];
#pragma unroll
  for (int j = 0; j < kRowsAThread; ++j) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[j][i] = 0.f;
    if (row[j] < tokens.rows) loadFloats<T, V>(table + (int64_t)row[j] * row_stride + l.channel, v[j]);
  }
#pragma unroll
  for (int j = 0; j < kRowsAThread; ++j) {
    const int64_t t = first + j * l.rows_at_once;
    // (not zero times the scale, which may be infinite)
    if (row[j] < tokens.rows) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] *= scale;
    }
    if (t < n) storeFloats<T, V>(out + t * channels + l.channel, v[j]);
  }
}

// ---- backward ------------------------------------------------------------------------------
//
// The places of the tokens are sorted by the row they name (equal rows in ascending place): each row of the table then has
// its gradients' places side by side, and adds them up in a fixed order, without atomics.  Rows named at most kPiece times
// are summed by the threads that own them.  Longer ones are cut into pieces at multiples of kPiece of the sorted places;
// each piece is summed by a workgroup of its own, and a last launch adds the pieces.

constexpr int kPiece = 64;

// Sorted words: the row above, the place below.
struct FirstPass {
  typedef u64 Item;
  Tokens tokens;
  u64 *out;
  uint32_t mask;
  __device__ Item load(int64_t i) const { return (u64)tokens.row(i) << 32 | (u64)i; }
  __device__ uint32_t digit(const Item &t) const { return (uint32_t)(t >> 32) & mask; }
  __device__ void store(size_t to, const Item &t, int64_t) const { out[to] = t; }
};

// The place of the first sorted word of every row, and of `rows`, where the words end that name a row.
__global__ __launch_bounds__(kThreads) void embeddingRowStarts(const u64 *__restrict__ sorted, uint32_t n, uint32_t rows,
                                                               uint32_t *__restrict__ starts) {
  const uint32_t row = blockIdx.x * kThreads + threadIdx.x;
  if (row > rows) return;
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if ((uint32_t)(sorted[mid] >> 32) < row)
      lo = mid + 1;
    else
      hi = mid;
  }
  starts[row] = lo;
}

// Adds the gradients of sorted words [begin, end) to sum, one after the other, a few loads in flight.
template <typename T, int V>
__device__ __forceinline__ void addRows(const T *__restrict__ grad, int64_t row_stride, const u64 *__restrict__ sorted,
                                        uint32_t begin, uint32_t end, int channel, float (&sum)[V]) {
  constexpr int kAhead = 4;
  for (uint32_t i = begin; i < end; i += kAhead) {
    float v[kAhead][V];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      // (behind the end the last one again, which is not added)
      const uint32_t place = (uint32_t)sorted[i + j < end ? i + j : end - 1];
      loadFloats<T, V>(grad + (int64_t)place * row_stride + channel, v[j]);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j < end) {
#pragma unroll
        for (int c = 0; c < V; ++c) sum[c] += v[j][c];
      }
  }
}

struct Sorted {
  const u64 *words;
  const uint32_t *starts;
  uint32_t n, rows, pieces;
};

// The first row_blocks workgroups own rows of the table.  The others take a piece each: of the rows that are longer than
// one, at most two reach into it, that of its first word and that of its last.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void embeddingGradRows(const T *__restrict__ grad, int64_t row_stride,
                                                              int channels, Sorted s, float scale, int row_blocks,
                                                              float *__restrict__ partial, T *__restrict__ out) {
  const Lanes<V> l(channels);
  if ((int)blockIdx.x < row_blocks) {
    const uint32_t row = blockIdx.x * l.rows_at_once + l.row;
    if (l.row < 0 || row >= s.rows) return;
    const uint32_t begin = s.starts[row], end = s.starts[row + 1];
    if (end - begin > (uint32_t)kPiece) return;
    float sum[V] = {};
    addRows<T, V>(grad, row_stride, s.words, begin, end, l.channel, sum);
    if (begin < end) {
#pragma unroll
      for (int c = 0; c < V; ++c) sum[c] *= scale;
    }
    storeFloats<T, V>(out + (int64_t)row * channels + l.channel, sum);
    return;
  }
  const uint32_t piece = blockIdx.x - row_blocks;
  const uint32_t lo = piece * kPiece, hi = min(lo + kPiece, s.n);
  if (l.row < 0 || l.row > 1) return;
  // (one row of threads where a row has all of them)
  for (int side = l.row; side < 2; side += min(l.rows_at_once, 2)) {
    const uint32_t row = (uint32_t)(s.words[side == 0 ? lo : hi - 1] >> 32);
    if (row >= s.rows) continue;
    const uint32_t begin = s.starts[row], end = s.starts[row + 1];
    if (end - begin <= (uint32_t)kPiece || (side == 1 && begin <= lo)) continue;
    float sum[V] = {};
    addRows<T, V>(grad, row_stride, s.words, max(begin, lo), min(end, hi), l.channel, sum);
    storeFloats<float, V>(partial + ((int64_t)piece * 2 + side) * channels + l.channel, sum);
  }
}

// Adds up the pieces of the long row that begins in piece blockIdx.x, if one does (only one can reach beyond its end).
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void embeddingGradJoin(int channels, Sorted s, float scale,
                                                              const float *__restrict__ partial, T *__restrict__ out) {
  const uint32_t lo = blockIdx.x * kPiece, hi = min(lo + kPiece, s.n);
  const uint32_t row = (uint32_t)(s.words[hi - 1] >> 32);
  if (row >= s.rows) return;
  const uint32_t begin = s.starts[row], end = s.starts[row + 1];
  if (end - begin <= (uint32_t)kPiece || begin < lo) return;
  const Lanes<V> l(channels);
  if (l.row != 0) return;
  float sum[V] = {};
  const uint32_t last = (end - 1) / kPiece;
  for (uint32_t p = blockIdx.x; p <= last; ++p) {
    // (a row that begins with a piece's first word is that piece's first)
    const int side = p == blockIdx.x && begin > lo ? 1 : 0;
    float v[V];
    loadFloats<float, V>(partial + ((int64_t)p * 2 + side) * channels + l.channel, v);
#pragma unroll
    for (int c = 0; c < V; ++c) sum[c] += v[c];
  }
#pragma unroll
  for (int c = 0; c < V; ++c) sum[c] *= scale;
  storeFloats<T, V>(out + (int64_t)row * channels + l.channel, sum);
}

// ---- host side -----------------------------------------------------------------------------

struct Plan {
  int bits, pass_bits;
  uint32_t pieces;
  size_t words, counters, starts, partial;  // bytes of each part
  size_t all() const { return 256 + 2 * words + counters + starts + partial; }
};

size_t rounded(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

Plan planOf(int64_t n, int64_t rows, int64_t channels) {
  Plan p;
  p.bits = 1;
  while ((rows >> p.bits) != 0) ++p.bits;  // (up to `rows` itself, of tokens that name no row)
  p.pass_bits = device_sort::sortPassBits(p.bits);
  p.pieces = (uint32_t)((n + kPiece - 1) / kPiece);
  p.words = rounded((size_t)n * sizeof(u64));
  p.counters = rounded(device_sort::sortCounterWords(n) * sizeof(uint32_t));
  p.starts = rounded((size_t)(rows + 1) * sizeof(uint32_t));
  p.partial = rounded((size_t)p.pieces * 2 * channels * sizeof(float));
  return p;
}

mluOpStatus_t checkTable(const char *api, int64_t n, int64_t rows, int64_t channels) {
  PARAM_CHECK(api, n >= 0);
  PARAM_CHECK(api, rows > 0);
  PARAM_CHECK(api, channels > 0);
  if (n > INT32_MAX - 4096 || rows > INT32_MAX - 4096 || channels > (1 << 20) || n * channels > ((int64_t)1 << 46) ||
      rows * channels > ((int64_t)1 << 46)) {
    MLUOP_LOG(ERROR) << api << " At most 2^31 - 4097 tokens and rows, 2^20 channels and 2^46 values are supported.";
    return MLUOP_STATUS_NOT_SUPPORTED;
  }
  return MLUOP_STATUS_SUCCESS;
}

// Calls f(element type, V): 16 bytes a thread where rows and addresses allow, else pairs or single elements.
template <typename F>
void byType(mluOpDataType_t type, int64_t channels, int64_t row_stride, uintptr_t addresses, F f) {
  auto fits = [&](int v) {
    return channels % v == 0 && row_stride % v == 0 && addresses % (v * (size_t)elementBytes(type)) == 0;
  };
  auto sixteen = [&](auto zero) {
    if (fits(8))
      f(zero, std::integral_constant<int, 8>());
    else if (fits(2))
      f(zero, std::integral_constant<int, 2>());
    else
      f(zero, std::integral_constant<int, 1>());
  };
  if (type == MLUOP_DTYPE_HALF) {
    sixteen((_Float16)0);
  } else if (type == MLUOP_DTYPE_BFLOAT16) {
    sixteen((__bf16)0.f);
  } else if (fits(4)) {
    f(0.f, std::integral_constant<int, 4>());
  } else {
    f(0.f, std::integral_constant<int, 1>());
  }
}

int rowsAtOnce(int64_t vectors) { return vectors >= kThreads ? 1 : (int)(kThreads / vectors); }
unsigned slabsOf(int64_t vectors) { return (unsigned)((vectors + kThreads - 1) / kThreads); }

}  // namespace

mluOpStatus_t MLUOP_WIN_API mluOpExtEmbeddingForward(mluOpHandle_t handle, mluOpDataType_t type, const void *table,
                                                     int64_t rows, int64_t channels, int64_t row_stride,
                                                     mluOpDataType_t token_type, const void *tokens, int64_t num_tokens,
                                                     float scale, void *out) {
  const char *api = "[mluOpExtEmbeddingForward]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  PARAM_CHECK(api, token_type == MLUOP_DTYPE_INT32 || token_type == MLUOP_DTYPE_INT64);
  const mluOpStatus_t status = checkTable(api, num_tokens, rows, channels);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, row_stride >= channels);
  PARAM_CHECK(api, row_stride <= ((int64_t)1 << 46) / rows);
  PARAM_CHECK(api, table != NULL);
  PARAM_CHECK(api, num_tokens == 0 || (tokens != NULL && out != NULL));
  DEVICE_HANDLE_CHECK(api, handle);
  if (num_tokens == 0) return MLUOP_STATUS_SUCCESS;
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  handle->forgetNotesIn(out, (size_t)num_tokens * channels * elementBytes(type));
  const Tokens t = {tokens, token_type == MLUOP_DTYPE_INT64, (uint32_t)rows};
  const mluop::LaunchCtx lc = handle->launchCtx();
  byType(type, channels, row_stride, reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out), [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    // (the last slab has fewer channels and more rows at once: its surplus workgroups find nothing)
    const int64_t per_block = (int64_t)rowsAtOnce(channels / V) * kRowsAThread;
    lc.begin("embeddingRows");
    embeddingRows<T, V><<<dim3((unsigned)((num_tokens + per_block - 1) / per_block), slabsOf(channels / V)), kThreads, 0, lc.stream>>>(
        static_cast<const T *>(table), row_stride, (int)channels, t, num_tokens, scale, static_cast<T *>(out));
    lc.end();
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtGetEmbeddingBackwardWorkspaceSize(int64_t num_tokens, int64_t rows,
                                                                      int64_t channels, size_t *size) {
  const char *api = "[mluOpExtGetEmbeddingBackwardWorkspaceSize]";
  PARAM_CHECK(api, size != NULL);
  const mluOpStatus_t status = checkTable(api, num_tokens, rows, channels);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  *size = planOf(num_tokens, rows, channels).all();
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtEmbeddingBackward(mluOpHandle_t handle, mluOpDataType_t type,
                                                      const void *output_grad, int64_t row_stride,
                                                      mluOpDataType_t token_type, const void *tokens, int64_t num_tokens,
                                                      int64_t rows, int64_t channels, float scale, void *workspace,
                                                      size_t workspace_size, void *grad_table) {
  const char *api = "[mluOpExtEmbeddingBackward]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  PARAM_CHECK(api, token_type == MLUOP_DTYPE_INT32 || token_type == MLUOP_DTYPE_INT64);
  const mluOpStatus_t status = checkTable(api, num_tokens, rows, channels);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, num_tokens == 0 || row_stride >= channels);
  PARAM_CHECK(api, num_tokens == 0 || row_stride <= ((int64_t)1 << 46) / num_tokens);
  PARAM_CHECK(api, num_tokens == 0 || (output_grad != NULL && tokens != NULL));
  PARAM_CHECK(api, grad_table != NULL);
  PARAM_CHECK(api, workspace != NULL);
  const Plan p = planOf(num_tokens, rows, channels);
  PARAM_CHECK(api, workspace_size >= p.all());
  DEVICE_HANDLE_CHECK(api, handle);
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  if (handle->hasNotes()) {
    handle->forgetNotesIn(grad_table, (size_t)rows * channels * elementBytes(type));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  // (the caller's memory need not be aligned)
  char *at = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~(uintptr_t)255);
  u64 *words[2] = {reinterpret_cast<u64 *>(at), reinterpret_cast<u64 *>(at + p.words)};
  uint32_t *counters = reinterpret_cast<uint32_t *>(at + 2 * p.words);
  uint32_t *starts = reinterpret_cast<uint32_t *>(at + 2 * p.words + p.counters);
  float *partial = reinterpret_cast<float *>(at + 2 * p.words + p.counters + p.starts);

  const mluop::LaunchCtx lc = handle->launchCtx();
  bool in_second = false;
  if (num_tokens > 0) {
    const FirstPass first = {{tokens, token_type == MLUOP_DTYPE_INT64, (uint32_t)rows}, words[0], (1u << p.pass_bits) - 1u};
    lc.begin("embeddingSort");
    HIP_CHECK_RETURN(api, device_sort::partition(lc.stream, first, num_tokens, device_sort::sortDigits(p.pass_bits),
                                                 p.pass_bits, counters));
    HIP_CHECK_RETURN(api, (device_sort::sortPairs<u64, false>(lc.stream, counters, words[0], words[1], nullptr, nullptr,
                                                              num_tokens, 32 + p.pass_bits, 32 + p.bits, p.pass_bits,
                                                              &in_second)));
    lc.end();
  }
  const Sorted s = {words[in_second ? 1 : 0], starts, (uint32_t)num_tokens, (uint32_t)rows, p.pieces};
  lc.begin("embeddingRowStarts");
  embeddingRowStarts<<<(unsigned)(rows / kThreads + 1), kThreads, 0, lc.stream>>>(s.words, s.n, s.rows, starts);
  lc.end();
  byType(type, channels, row_stride, reinterpret_cast<uintptr_t>(output_grad) | reinterpret_cast<uintptr_t>(grad_table),
         [&](auto zero, auto v) {
           typedef decltype(zero) T;
           constexpr int V = decltype(v)::value;
           const int64_t at_once = rowsAtOnce(channels / V);
           const int row_blocks = (int)((rows + at_once - 1) / at_once);
           lc.begin("embeddingGradRows");
           embeddingGradRows<T, V><<<dim3((unsigned)row_blocks + p.pieces, slabsOf(channels / V)), kThreads, 0, lc.stream>>>(
               static_cast<const T *>(output_grad), row_stride, (int)channels, s, scale, row_blocks, partial,
               static_cast<T *>(grad_table));
           lc.end();
           if (num_tokens <= kPiece) return;  // (no row can be longer)
           lc.begin("embeddingGradJoin");
           embeddingGradJoin<T, V><<<dim3(p.pieces, slabsOf(channels / V)), kThreads, 0, lc.stream>>>(
               (int)channels, s, scale, partial, static_cast<T *>(grad_table));
           lc.end();
         });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
