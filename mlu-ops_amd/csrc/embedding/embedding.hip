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

// Tokens of either type, read without a branch: one between loads would make each wait for the one before.
struct Tokens {
  const uint32_t *at;
  uint32_t rows;
  int step, high;  // words of a token, and where its upper half is (32 bits: the token again, of which nothing counts)
  uint32_t upper;
  Tokens(const void *tokens, mluOpDataType_t type, int64_t table_rows)
      : at(static_cast<const uint32_t *>(tokens)), rows((uint32_t)table_rows), step(type == MLUOP_DTYPE_INT64 ? 2 : 1),
        high(step - 1), upper(high != 0 ? ~0u : 0u) {}
  // The row that token i names; `rows` where it names none.
  __device__ __forceinline__ uint32_t row(int64_t i) const {
    const uint32_t *word = at + i * step;
    const uint32_t lo = word[0], hi = word[high];
    const uint32_t none = (hi & upper) | (lo < rows ? 0u : 1u);
    return none == 0 ? lo : rows;
  }
};

// ---- forward -------------------------------------------------------------------------------

// out[t] = scale * table[token t], in one pass; bound by memory, or by the launch where there is little: 240 612 rows of 512
// fp16 (247 MB) 36 us, 64 rows of 1024 bf16 5.6.
constexpr int kRowsAThread = 4;  // whose loads are in flight together

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void embeddingRows(const T *__restrict__ table, int64_t row_stride, int channels,
                                                          Tokens tokens, int64_t n, float scale, int64_t first_block,
                                                          T *__restrict__ out) {
  const Lanes<V> l(channels);
  if (l.row < 0) return;
  const int64_t first = (first_block + blockIdx.x) * l.rows_at_once * kRowsAThread + l.row;
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
// its gradients' places side by side, and adds them up in a fixed order, without atomics.  Rows named no more often
// than a piece is long are summed by the threads that own them.  Longer ones are cut at multiples of it in the sorted places;
// each piece is summed by a workgroup of its own, and a last launch adds the pieces.

// Whether all rows of threads of a workgroup share a row of the table: one that is named often, as all are in a small table.
// us of the gradient of 5000 x 64 bf16 without / with this: named 8 times on average 38 / 42, 16 times 41 / 44, 32 times 55 / 47,
// 64 times 75 / 52; 517 x 64 fp32, 232 times, 47 / 31.
bool rowsShared(int64_t n, int64_t rows, int64_t channels) { return n >= 24 * rows && channels < 1024; }

// Words of a piece: as many as the rows of threads of a workgroup (which V = 4 has) read at once, eight each, where they
// share rows of the table.  Where one of them sums a row alone, fewer; but where a row has many channels there are no
// threads to share a piece either, and sums to keep.  us of the whole gradient at pieces of 32 / 64 words, 65 536 tokens,
// 131 072 x 2048 bf16: 222 / 216.
int pieceOf(int64_t n, int64_t rows, int64_t channels) {
  if (rowsShared(n, rows, channels)) return (int)std::max<int64_t>(8 * (kThreads * 4 / std::max<int64_t>(channels, 4)), 64);
  return channels >= 1024 ? 64 : 32;
}

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

// Few tokens (rankedTokens): the place of a word is the number of words below it, counted for kRanked words by a workgroup whose
// waves share the others.  One launch, whose work grows with the square of the tokens.  us of a whole gradient of 64 bf16
// channels with this / with the sort: one pass of it (500 rows) 1024 tokens 13.2 / 15.9, 4096 18.4 / 19.4, 6000 22.0 / 19.4; two
// (91 000 rows) 1024 15.3 / 30.0, 8192 25.7 / 35.5, 12 288 34.9 / 36.4, 16 384 46.0 / 37.7.
constexpr int kRanked = 16;
int rankedTokens(int passes) { return passes == 1 ? 4096 : 12288; }
__global__ __launch_bounds__(kThreads) void embeddingRankWords(Tokens tokens, uint32_t n, u64 *__restrict__ sorted) {
  constexpr int kAhead = 4;
  __shared__ uint32_t s_below[kRanked][kThreads];
  const uint32_t first = blockIdx.x * kRanked, wave = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63u), lane = threadIdx.x & 63;
  uint32_t row[kRanked], below[kRanked] = {};
#pragma unroll
  for (int j = 0; j < kRanked; ++j) row[j] = __builtin_amdgcn_readfirstlane(tokens.row(min(first + j, n - 1))) + 1;
  uint32_t next[kAhead];
  auto request = [&](uint32_t i0) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const uint32_t i = i0 + a * kThreads + lane;
      const uint32_t row = tokens.row(min(i, n - 1));
      next[a] = i < n ? row + 1 : 0x80000000u;  // (below nothing)
    }
  };
  request(wave);
  for (uint32_t i0 = wave; i0 < n; i0 += kThreads * kAhead) {
    uint32_t other[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) other[a] = next[a];
    request(i0 + kThreads * kAhead);
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const uint32_t from = i0 + a * kThreads;
      // (of equal rows those of the places in front are below: all of these 64 or none, mostly)
      if (from + 63 < first || from >= first + kRanked) {
        const uint32_t as = other[a] - (from < first ? 1 : 0);
#pragma unroll
        for (int j = 0; j < kRanked; ++j) below[j] += as < row[j] ? 1u : 0u;
      } else {
#pragma unroll
        for (int j = 0; j < kRanked; ++j)
          below[j] += other[a] < row[j] + (from + lane < first + j ? 1u : 0u) ? 1u : 0u;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kRanked; ++j) s_below[j][threadIdx.x] = below[j];
  __syncthreads();
  // sixteen threads a word, lines of them
  constexpr int kShare = kThreads / kRanked;
  const uint32_t word = threadIdx.x / kShare, share = threadIdx.x % kShare;
  uint32_t sum = 0;
#pragma unroll
  for (int k = 0; k < kThreads / kShare; ++k) sum += s_below[word][k * kShare + share];
#pragma unroll
  for (int d = kShare / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
  if (share == 0 && first + word < n) sorted[sum] = (u64)tokens.row(first + word) << 32 | (first + word);
}

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

// Adds the gradients of the sorted words begin, begin + step, ... below end to sum, a few loads in flight.
template <typename T, int V>
__device__ __forceinline__ void addRows(const T *__restrict__ grad, int64_t row_stride, const u64 *__restrict__ sorted,
                                        uint32_t begin, uint32_t end, uint32_t step, int channel, float (&sum)[V]) {
  constexpr int kAhead = 8;
  for (uint32_t i = begin; i < end; i += kAhead * step) {
    Vector<T, V> v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      // (behind the end the first one again, which is not added)
      const uint32_t place = (uint32_t)sorted[i + j * step < end ? i + j * step : i];
      v[j] = *reinterpret_cast<const Vector<T, V> *>(grad + (int64_t)place * row_stride + channel);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j * step < end) {
#pragma unroll
        for (int c = 0; c < V; ++c) sum[c] += (float)v[j].v[c];
      }
  }
}

// Sums of V values over the `rows` rows of threads of a workgroup (in `scratch`, THREADS * V floats), in the threads of row 0.
// By the whole workgroup.
template <int V>
__device__ __forceinline__ void sumOverThreadRows(int row, int rows, int across, float *scratch, float (&sum)[V]) {
  for (int left = rows; left > 1;) {
    const int half = (left + 1) / 2;
    if (row >= half && row < left) {
#pragma unroll
      for (int v = 0; v < V; ++v) scratch[threadIdx.x * V + v] = sum[v];
    }
    __syncthreads();
    if (row >= 0 && row + half < left) {
#pragma unroll
      for (int v = 0; v < V; ++v) sum[v] += scratch[(threadIdx.x + half * across) * V + v];
    }
    left = half;
  }
}

struct Sorted {
  const u64 *words;
  const uint32_t *starts;
  uint32_t n, rows, piece;
  uint32_t first_block;  // of the launch, of all that its kernel has
  bool streamed;
};

// out[row] = scale * (the gradients of the row's words, added up in fp32 in an order that the words decide).  Bound by memory:
// 131 072 x 2048 bf16 from 65 536 tokens (805 MB) 140 us, 5.7 TB/s.
// The first row_blocks workgroups own rows of the table.  The others take a piece each: of the rows that are longer than
// one, at most two reach into it, that of its first word and that of its last.
// SHARED: a row of the table a workgroup, whose rows of threads share the words.
template <typename T, int V, int kTableRows, bool SHARED>
__global__ __launch_bounds__(kThreads) void embeddingGradRows(const T *__restrict__ grad, int64_t row_stride,
                                                              int channels, Sorted s, float scale, uint32_t row_blocks,
                                                              float *__restrict__ partial, T *__restrict__ out) {
  __shared__ float s_sum[kThreads * V];
  const uint32_t block = s.first_block + blockIdx.x;
  const Lanes<V> l(channels);
  if (SHARED && block < row_blocks) {
    const uint32_t row = block, begin = s.starts[row], end = s.starts[row + 1];
    if (end - begin > s.piece) return;
    float sum[V] = {};
    if (l.row >= 0) addRows<T, V>(grad, row_stride, s.words, begin + l.row, end, l.rows_at_once, l.channel, sum);
    sumOverThreadRows<V>(l.row, l.rows_at_once, l.across, s_sum, sum);
    if (l.row != 0) return;
    if (begin < end) {
#pragma unroll
      for (int c = 0; c < V; ++c) sum[c] *= scale;
    }
    storeFloats<T, V>(out + (int64_t)row * channels + l.channel, sum, s.streamed);
    return;
  }
  if (block < row_blocks) {
    if (l.row < 0) return;
    const uint32_t first = block * l.rows_at_once * kTableRows + l.row;
    uint32_t begin[kTableRows], end[kTableRows];
#pragma unroll
    for (int j = 0; j < kTableRows; ++j) {
      const uint32_t row = min(first + j * l.rows_at_once, s.rows - 1);
      begin[j] = s.starts[row];
      end[j] = s.starts[row + 1];
    }
#pragma unroll
    for (int j = 0; j < kTableRows; ++j) {
      const uint32_t row = first + j * l.rows_at_once;
      if (row >= s.rows) return;
      if (end[j] - begin[j] > s.piece) continue;
      float sum[V] = {};
      if (begin[j] < end[j]) {
        addRows<T, V>(grad, row_stride, s.words, begin[j], end[j], 1, l.channel, sum);
#pragma unroll
        for (int c = 0; c < V; ++c) sum[c] *= scale;
      }
      storeFloats<T, V>(out + (int64_t)row * channels + l.channel, sum, s.streamed);
    }
    return;
  }
  const uint32_t piece = block - row_blocks;
  const uint32_t lo = piece * s.piece, hi = min(lo + s.piece, s.n);
  for (int side = 0; side < 2; ++side) {
    const uint32_t row = (uint32_t)(s.words[side == 0 ? lo : hi - 1] >> 32);
    if (row >= s.rows) continue;
    const uint32_t begin = s.starts[row], end = s.starts[row + 1];
    if (end - begin <= s.piece || (side == 1 && begin <= lo)) continue;
    float sum[V] = {};
    if (l.row >= 0)
      addRows<T, V>(grad, row_stride, s.words, max(begin, lo) + l.row, min(end, hi), l.rows_at_once, l.channel, sum);
    __syncthreads();
    sumOverThreadRows<V>(l.row, l.rows_at_once, l.across, s_sum, sum);
    if (l.row == 0) storeFloats<float, V>(partial + ((int64_t)piece * 2 + side) * channels + l.channel, sum);
  }
}

// Adds up the pieces of the long row that begins in a workgroup's own piece, if one does (only one can reach beyond its end).  A
// wave's width of threads across the channels, so that the workgroup's rows of threads share the pieces.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void embeddingGradJoin(int channels, Sorted s, float scale,
                                                              const float *__restrict__ partial, T *__restrict__ out) {
  constexpr int kAhead = 4;
  __shared__ float s_sum[kThreads * V];
  const uint32_t own = s.first_block + blockIdx.x, lo = own * s.piece, hi = min(lo + s.piece, s.n);
  const uint32_t row = (uint32_t)(s.words[hi - 1] >> 32);
  if (row >= s.rows) return;
  const uint32_t begin = s.starts[row], end = s.starts[row + 1];
  if (end - begin <= s.piece || begin < lo) return;
  const int across = min(channels / V - (int)blockIdx.y * 64, 64), rows = kThreads / across;
  const int my_row = (int)threadIdx.x / across < rows ? (int)threadIdx.x / across : -1;
  const int channel = ((int)blockIdx.y * 64 + (int)threadIdx.x % across) * V;
  float sum[V] = {};
  if (my_row >= 0) {
    const uint32_t last = (end - 1) / s.piece;
    for (uint32_t p0 = own + my_row; p0 <= last; p0 += kAhead * rows) {
      Vector<float, V> v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const uint32_t p = min(p0 + j * rows, last);
        // (a row that begins with a piece's first word is that piece's first)
        const int side = p == own && begin > lo ? 1 : 0;
        v[j] = *reinterpret_cast<const Vector<float, V> *>(partial + ((int64_t)p * 2 + side) * channels + channel);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (p0 + j * rows > last) break;
#pragma unroll
        for (int c = 0; c < V; ++c) sum[c] += v[j].v[c];
      }
    }
  }
  sumOverThreadRows<V>(my_row, rows, across, s_sum, sum);
  if (my_row != 0) return;
#pragma unroll
  for (int c = 0; c < V; ++c) sum[c] *= scale;
  storeFloats<T, V>(out + (int64_t)row * channels + channel, sum);
}

// ---- host side -----------------------------------------------------------------------------

struct Plan {
  int bits, pass_bits, piece;
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
  p.piece = pieceOf(n, rows, channels);
  p.pieces = (uint32_t)((n + p.piece - 1) / p.piece);
  p.words = rounded((size_t)n * sizeof(u64));
  p.counters = rounded(device_sort::sortCounterWords(n) * sizeof(uint32_t));
  p.starts = rounded((size_t)std::max<int64_t>(rows + 1, device_sort::kMaxDigits) * sizeof(uint32_t));
  p.partial = rounded((size_t)p.pieces * 2 * channels * sizeof(float));
  return p;
}

mluOpStatus_t checkTable(const char *api, int64_t n, int64_t rows, int64_t channels) {
  PARAM_CHECK(api, n >= 0);
  PARAM_CHECK(api, rows > 0 || (rows == 0 && n == 0));
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

// Rows of the table that a row of threads owns, of `turns` it would own one at a time: several of a large table, most of
// whose rows nobody names, and a workgroup for each would mostly start and end; one of a small table.  us of a gradient with
// one / with four: 131 072 x 2048 bf16 from 65 536 tokens 202 / 186, 600 000 x 64 from 30 000 55 / 52; 500 x 512 from 4000 18 /
// 23.
int tableRows(int64_t turns) { return turns >= 16384 ? 4 : 1; }

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
  PARAM_CHECK(api, rows == 0 || row_stride <= ((int64_t)1 << 46) / rows);
  PARAM_CHECK(api, rows == 0 || table != NULL);
  PARAM_CHECK(api, num_tokens == 0 || (tokens != NULL && out != NULL));
  DEVICE_HANDLE_CHECK(api, handle);
  if (num_tokens == 0) return MLUOP_STATUS_SUCCESS;
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  handle->forgetNotesIn(out, (size_t)num_tokens * channels * elementBytes(type));
  const Tokens t(tokens, token_type, rows);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out);
  byType(type, channels, row_stride, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    // (the last slab has fewer channels and more rows at once: its surplus workgroups find nothing)
    const int64_t per_block = (int64_t)rowsAtOnce(channels / V) * kRowsAThread;
    inLaunches((num_tokens + per_block - 1) / per_block, kThreads, [&](int64_t first, unsigned blocks) {
      lc.begin("embeddingRows");
      embeddingRows<T, V><<<dim3(blocks, slabsOf(channels / V)), kThreads, 0, lc.stream>>>(
          static_cast<const T *>(table), row_stride, (int)channels, t, num_tokens, scale, first, static_cast<T *>(out));
      lc.end();
    });
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
  PARAM_CHECK(api, rows == 0 || grad_table != NULL);
  PARAM_CHECK(api, workspace != NULL);
  const Plan p = planOf(num_tokens, rows, channels);
  PARAM_CHECK(api, workspace_size >= p.all());
  DEVICE_HANDLE_CHECK(api, handle);
  if (rows == 0) return MLUOP_STATUS_SUCCESS;
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
  const Tokens names(tokens, token_type, rows);
  bool in_second = false, started = false;
  if (num_tokens > rankedTokens((p.bits + p.pass_bits - 1) / p.pass_bits)) {
    lc.begin("embeddingSort");
    const bool few = device_sort::tilesFor(num_tokens) <= device_sort::kFewTiles;
    const int digits = device_sort::sortDigits(p.pass_bits);
    const uint32_t mask = (1u << p.pass_bits) - 1u;
    // (where one pass sorts, its digits are the rows)
    started = p.pass_bits >= p.bits;
    uint32_t *firsts = started ? starts : nullptr;
    auto pass = [&](const auto &items) {
      return few ? device_sort::partitionFew(lc.stream, items, num_tokens, digits, p.pass_bits, counters, firsts)
                 : device_sort::partition(lc.stream, items, num_tokens, digits, p.pass_bits, counters, firsts);
    };
    HIP_CHECK_RETURN(api, pass(FirstPass{names, words[0], mask}));
    for (int shift = 32 + p.pass_bits; shift < 32 + p.bits; shift += p.pass_bits) {
      const device_sort::KeysAndValues<u64, false> items = {words[in_second ? 1 : 0], nullptr, words[in_second ? 0 : 1],
                                                            nullptr, shift, mask};
      HIP_CHECK_RETURN(api, pass(items));
      in_second = !in_second;
    }
    lc.end();
  } else if (num_tokens > 0) {
    lc.begin("embeddingRankWords");
    embeddingRankWords<<<(unsigned)((num_tokens + kRanked - 1) / kRanked), kThreads, 0, lc.stream>>>(names, (uint32_t)num_tokens,
                                                                                                     words[0]);
    lc.end();
  }
  Sorted s = {words[in_second ? 1 : 0], starts, (uint32_t)num_tokens, (uint32_t)rows, (uint32_t)p.piece, 0,
              (size_t)rows * channels * elementBytes(type) >= kStreamedBytes};
  if (!started) {
    lc.begin("embeddingRowStarts");
    embeddingRowStarts<<<(unsigned)(rows / kThreads + 1), kThreads, 0, lc.stream>>>(s.words, s.n, s.rows, starts);
    lc.end();
  }
  byType(type, channels, row_stride, reinterpret_cast<uintptr_t>(output_grad) | reinterpret_cast<uintptr_t>(grad_table),
         [&](auto zero, auto v) {
           typedef decltype(zero) T;
           constexpr int V = decltype(v)::value;
           const int64_t at_once = rowsAtOnce(channels / V);
           const bool shared = rowsShared(num_tokens, rows, channels);
           const int each = tableRows(rows / at_once);
           const int64_t row_blocks = shared ? rows : (rows + at_once * each - 1) / (at_once * each);
           auto kernel = shared      ? embeddingGradRows<T, V, 1, true>
                         : each == 1 ? embeddingGradRows<T, V, 1, false>
                                     : embeddingGradRows<T, V, 4, false>;
           inLaunches(row_blocks + p.pieces, kThreads, [&](int64_t first, unsigned blocks) {
             s.first_block = (uint32_t)first;
             lc.begin("embeddingGradRows");
             kernel<<<dim3(blocks, slabsOf(channels / V)), kThreads, 0, lc.stream>>>(
                 static_cast<const T *>(output_grad), row_stride, (int)channels, s, scale, (uint32_t)row_blocks, partial,
                 static_cast<T *>(grad_table));
             lc.end();
           });
           if (num_tokens <= p.piece) return;  // (no row can be longer)
           inLaunches(p.pieces, kThreads, [&](int64_t first, unsigned blocks) {
             constexpr int W = V < 4 ? V : 4;
             s.first_block = (uint32_t)first;
             lc.begin("embeddingGradJoin");
             embeddingGradJoin<T, W><<<dim3(blocks, (unsigned)((channels / W + 63) / 64)), kThreads, 0, lc.stream>>>(
                 (int)channels, s, scale, partial, static_cast<T *>(grad_table));
             lc.end();
           });
         });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
