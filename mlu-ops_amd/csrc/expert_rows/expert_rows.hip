// mluOpExtExpertOrder, mluOpExtExpertDispatch, mluOpExtExpertCombine and its gradients (no counterpart in the reference): rows
// brought into the order of the experts they are sent to, and the experts' results back, weighted and added up.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "core/core.h"
#include "core/device_sort.h"
#include "core/elements.h"
#include "core/lane_sum.h"
#include "mlu_op_ext.h"

namespace {

using namespace mluop;

constexpr int kThreads = 256;

// ---- the order -----------------------------------------------------------------------------

// Choices [rows * choices] to be partitioned by their expert, stably: those of no expert behind the last.
struct Choices {
  const uint32_t *at;
  int step, high;  // words of a number, and where its upper half is (32 bits: the number again, of which nothing counts)
  uint32_t upper, experts, choices;
  int32_t *ordered_rows, *places;
  struct Item {
    uint32_t expert;
  };
  __device__ __forceinline__ Item load(int64_t i) const {
    const uint32_t *word = at + i * step;
    const uint32_t lo = word[0], hi = word[high];
    return {((hi & upper) == 0 && lo < experts) ? lo : experts};
  }
  __device__ __forceinline__ uint32_t digit(const Item &item) const { return item.expert; }
  __device__ __forceinline__ void store(size_t to, const Item &item, int64_t i) const {
    const bool sent = item.expert < experts;
    ordered_rows[to] = sent ? (int32_t)((uint32_t)i / choices) : -1;
    places[i] = sent ? (int32_t)to : -1;
  }
};

// Tiles of kOrderTile choices, a workgroup each: one launch where one holds them all, else one that counts and one that places.
// A wave has 64 * kTurns consecutive choices, 64 at a time in order; choices of one expert find each other with a ballot for each
// bit of its number.  A choice's place is behind those of lower experts, of its expert in earlier tiles, in earlier waves, in
// earlier turns of its wave, and in lower lanes.  us of the general partition / of these: 24 choices of 32 experts 7.8 / 3.6,
// 65 536 of 64 15 / 10, 240 000 of 8 26 / 9.
constexpr int kOrderThreads = 512, kOrderWaves = kOrderThreads / 64, kTurns = 4, kOrderTile = kOrderThreads * kTurns;
constexpr int kMostDigits = device_sort::kMaxDigits;

__global__ __launch_bounds__(kOrderThreads) void expertCounts(Choices items, int64_t n, int digits,
                                                              uint32_t *__restrict__ hist) {
  __shared__ uint32_t s_count[kMostDigits];
  const int64_t base = (int64_t)blockIdx.x * kOrderTile + threadIdx.x;
  Choices::Item item[kTurns];
#pragma unroll
  for (int j = 0; j < kTurns; ++j) item[j] = items.load(min(base + j * kOrderThreads, n - 1));
  for (int d = threadIdx.x; d < digits; d += kOrderThreads) s_count[d] = 0;
  __syncthreads();
  // (integer adds in LDS: the order they land in does not matter for a count)
#pragma unroll
  for (int j = 0; j < kTurns; ++j)
    if (base + j * kOrderThreads < n) atomicAdd(&s_count[item[j].expert], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kOrderThreads) hist[(size_t)blockIdx.x * digits + d] = s_count[d];
}

// Choices of every digit in all tiles, and in those in front of this workgroup's, to s_total and s_before: as many threads a
// digit as there are, `across` (a power of two) digits side by side.
__device__ __forceinline__ void countsOfTiles(const uint32_t *__restrict__ hist, int tiles, int digits, int across,
                                              uint32_t *s_total, uint32_t *s_before) {
  constexpr int kAtOnce = 8;
  for (int d = threadIdx.x; d < digits; d += kOrderThreads) s_total[d] = s_before[d] = 0;
  __syncthreads();
  const int shares = kOrderThreads / across, share = (int)threadIdx.x / across;
  for (int d = (int)threadIdx.x % across; d < digits; d += across) {
    uint32_t total = 0, before = 0;
    for (int t0 = share; t0 < tiles; t0 += kAtOnce * shares) {
      uint32_t v[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) v[j] = hist[(size_t)min(t0 + j * shares, tiles - 1) * digits + d];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int t = t0 + j * shares;
        total += t < tiles ? v[j] : 0u;
        before += t < tiles && t < (int)blockIdx.x ? v[j] : 0u;
      }
    }
    atomicAdd(&s_total[d], total);
    atomicAdd(&s_before[d], before);
  }
  __syncthreads();
}

// ALONE: one workgroup has all choices.
template <bool ALONE>
__global__ __launch_bounds__(kOrderThreads) void expertPlaces(Choices items, int64_t n, int digits, int digit_bits, int across,
                                                              const uint32_t *__restrict__ hist,
                                                              int32_t *__restrict__ starts) {
  __shared__ uint16_t s_count[kOrderWaves][kMostDigits];
  __shared__ uint32_t s_first[kMostDigits], s_before[ALONE ? 1 : kMostDigits], s_wave[kOrderWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned long long below = (1ull << lane) - 1ull;
  const int64_t base = (int64_t)blockIdx.x * kOrderTile + wave * 64 * kTurns + lane;
  Choices::Item item[kTurns];
#pragma unroll
  for (int j = 0; j < kTurns; ++j) item[j] = items.load(min(base + j * 64, n - 1));
  for (int d = threadIdx.x; d < digits; d += kOrderThreads)
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) s_count[w][d] = 0;
  __syncthreads();
  volatile uint16_t *mine = s_count[wave];
  uint32_t place[kTurns];
#pragma unroll
  for (int j = 0; j < kTurns; ++j) {
    const bool valid = base + j * 64 < n;
    const uint32_t digit = item[j].expert;
    unsigned long long peers = __ballot(valid);
    for (int b = 0; b < digit_bits; ++b) {
      const bool bit = (digit >> b) & 1u;
      const unsigned long long with = __ballot(bit);
      peers &= bit ? with : ~with;
    }
    const int leader = valid ? __ffsll((long long)peers) - 1 : lane;
    uint32_t before = 0;
    if (valid && lane == leader) {
      before = mine[digit];
      mine[digit] = (uint16_t)(before + (uint32_t)__popcll(peers));
    }
    before = __shfl(before, leader, 64);
    place[j] = before + (uint32_t)__popcll(peers & below);
  }
  __syncthreads();
  // counts of a digit become those of the waves in front, and its total; a run of digits for each thread
  const int per = (digits + kOrderThreads - 1) / kOrderThreads, d0 = (int)threadIdx.x * per;
  for (int d = d0; d < min(d0 + per, digits); ++d) {
    uint32_t run = 0;
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) {
      const uint32_t c = s_count[w][d];
      s_count[w][d] = (uint16_t)run;
      run += c;
    }
    if (ALONE) s_first[d] = run;
  }
  if (!ALONE) countsOfTiles(hist, (int)gridDim.x, digits, across, s_first, s_before);
  // totals become starts
  uint32_t sum = 0;
  for (int d = d0; d < min(d0 + per, digits); ++d) sum += s_first[d];
  const uint32_t upto = device_sort::waveInclusiveSum(sum);
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  uint32_t run = upto - sum;
  for (int w = 0; w < wave; ++w) run += s_wave[w];
  for (int d = d0; d < min(d0 + per, digits); ++d) {
    const uint32_t total = s_first[d];
    if (blockIdx.x == 0) starts[d] = (int32_t)run;
    s_first[d] = ALONE ? run : run + s_before[d];
    run += total;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kTurns; ++j)
    if (base + j * 64 < n)
      items.store((size_t)s_first[item[j].expert] + s_count[wave][item[j].expert] + place[j], item[j], base + j * 64);
}

__global__ __launch_bounds__(kThreads) void expertStarts(const uint32_t *__restrict__ from, int count,
                                                         int32_t *__restrict__ to) {
  const int i = (int)blockIdx.x * kThreads + (int)threadIdx.x;
  if (i < count) to[i] = from == nullptr ? 0 : (int32_t)from[i];
}

// ---- rows to their places and back ---------------------------------------------------------

// LANES threads have a row, 16 bytes each whatever the vectors' width, as often as the row needs.  (A vector each: 60 000 rows of
// 250 bf16 from two places 60 us, 16 bytes 30.  Eight threads or more, where two hold a row: 1 875 000 rows of 16 bf16 back 92
// us, two 47.)
template <typename T, int V>
constexpr int kVectors = 16 / (int)sizeof(T) / V;

// Rows that are not whole lines of 128 bytes share lines with their neighbours.  Workgroups go to the eight XCDs in turn: with
// runs of rows for each, what shares a line in front and behind mostly meets in one L2, and results stay in the caches, where a
// line is filled before it goes to memory (sent past them 1 875 000 rows of 16 bf16 take 54 us, else 37, in runs 30; 227 272 x 4
// x 33 bf16 49 and in runs 39, their gradients 81 and 66).  Whole lines are better off in turn (32 768 x 2 x 2048 bf16 76 and in
// runs 80).
__device__ __forceinline__ int64_t inRuns(int64_t block, int64_t blocks) {
  const int64_t run = blocks / 8;
  return block < run * 8 ? block % 8 * run + block / 8 : block;
}
inline bool wholeLines(int64_t channels, mluOpDataType_t type) { return channels * elementBytes(type) % 128 == 0; }

// The places behind the last expert's are zero: there is one for every choice without an expert, and the threads of row r have
// every one that is r further on, and as many rows again.  (By 64 workgroups of their own: 157 us, where 30 % of 16 384 x 4 x
// 1024 fp16 are sent nowhere, and their gradients 162; so 34 and 56.)
template <typename T, int V, int LANES>
__device__ __forceinline__ void zeroTail(int tail, int64_t r, int64_t rows, int64_t n, int channels, bool streamed, T *out) {
  const float zero[V] = {};
  for (int64_t p = (tail < 0 ? 0 : tail) + r; p < n; p += rows)
    for (int c = (int)threadIdx.x % LANES * V; c < channels; c += LANES * V)
      storeFloats<T, V>(out + p * channels + c, zero, streamed);
}

// out[place of (r, k)] = x[r] for every choice k: a row is read once and written as often as it is sent.  Bound by memory: 32 768
// x 2 x 2048 bf16 (403 MB) 70 us, 5.7 TB/s.
template <typename T, int V, int LANES>
__global__ __launch_bounds__(kThreads) void expertDispatch(const T *__restrict__ x, int64_t x_stride, int64_t rows,
                                                           int channels, int choices, const int32_t *__restrict__ places,
                                                           const int32_t *__restrict__ starts, int experts,
                                                           int64_t first_block, int64_t row_blocks, bool lines,
                                                           bool streamed, T *__restrict__ out) {
  constexpr int N = kVectors<T, V>;
  const int64_t n = rows * choices, block = first_block + blockIdx.x;
  const int tail = starts[experts];
  const int64_t r = (lines ? block : inRuns(block, row_blocks)) * (kThreads / LANES) + (int)threadIdx.x / LANES;
  if (r >= rows) return;
  for (int c = (int)threadIdx.x % LANES * V; c < channels; c += LANES * V * N) {
    float v[N][V];
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (c + j * LANES * V < channels) loadFloats<T, V>(x + r * x_stride + c + j * LANES * V, v[j]);
    for (int k = 0; k < choices; ++k) {
      const int64_t p = places[r * choices + k];
      if (p < 0 || p >= n) continue;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c + j * LANES * V < channels) storeFloats<T, V>(out + p * channels + c + j * LANES * V, v[j], streamed);
    }
  }
  zeroTail<T, V, LANES>(tail, r, rows, n, channels, streamed, out);
}

// Weights of either type, or none (one each).
struct Weights {
  const void *at;
  mluOpDataType_t type;
  __device__ __forceinline__ float load(int64_t i) const {
    if (at == nullptr) return 1.f;
    if (type == MLUOP_DTYPE_FLOAT) return static_cast<const float *>(at)[i];
    if (type == MLUOP_DTYPE_HALF) return (float)static_cast<const _Float16 *>(at)[i];
    return (float)static_cast<const __bf16 *>(at)[i];
  }
  __device__ __forceinline__ void store(void *to, int64_t i, float v) const {
    if (type == MLUOP_DTYPE_FLOAT)
      static_cast<float *>(to)[i] = v;
    else if (type == MLUOP_DTYPE_HALF)
      static_cast<_Float16 *>(to)[i] = (_Float16)v;
    else
      static_cast<__bf16 *>(to)[i] = (__bf16)v;
  }
};

constexpr int kAhead = 4;  // choices whose rows are on their way together

// out[r] = sum over k of weight (r, k) * y[place of (r, k)], in the choices' order; a choice without a place adds nothing.
// Bound by memory, which it reads in places all over: 32 768 x 2 x 2048 bf16 (403 MB) 70 us, 5.7 TB/s.  (Choices that a row has
// not read as its first: 79.)
template <typename T, int V, int LANES>
__global__ __launch_bounds__(kThreads) void expertCombine(const T *__restrict__ y, int64_t y_stride, int64_t rows,
                                                          int channels, int choices, const int32_t *__restrict__ places,
                                                          Weights weights, int64_t first_block, int64_t row_blocks,
                                                          bool lines, bool streamed, T *__restrict__ out) {
  constexpr int N = kVectors<T, V>;
  const int64_t n = rows * choices, block = first_block + blockIdx.x;
  const int64_t r = (lines ? block : inRuns(block, row_blocks)) * (kThreads / LANES) + (int)threadIdx.x / LANES;
  if (r >= rows) return;
  for (int c = (int)threadIdx.x % LANES * V; c < channels; c += LANES * V * N) {
    float sum[N][V] = {};
    for (int k0 = 0; k0 < choices; k0 += kAhead) {
      Vector<T, V> v[kAhead][N];
      float w[kAhead];
      bool there[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        there[j] = false;
        if (k0 + j >= choices) continue;
        const int64_t at = r * choices + k0 + j, p = places[at];
        there[j] = p >= 0 && p < n;
        w[j] = weights.load(at);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int at_c = c + i * LANES * V;
          v[j][i] = *reinterpret_cast<const Vector<T, V> *>(y + (there[j] ? p : 0) * y_stride + (at_c < channels ? at_c : c));
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (!there[j]) continue;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) sum[i][e] = fmaf(w[j], (float)v[j][i].v[e], sum[i][e]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i * LANES * V < channels) storeFloats<T, V>(out + r * channels + c + i * LANES * V, sum[i], streamed);
  }
}

// The gradients of the weighted sum: dout_r goes to the places times its weights, and the weights' gradients are products with
// what lies there.  Up to 64 lanes, one wave's, a row.  Bound by memory: 16 384 x 4 x 1024 fp16 (302 MB) 54 us, 5.6 TB/s.
// (Stores past the caches, which serve the others: 32 768 x 2 x 2048 bf16 144 us in place of 126.)
template <typename T, int V, int LANES>
__global__ __launch_bounds__(kThreads) void expertCombineGrad(const T *__restrict__ dout, int64_t dout_stride,
                                                              const T *__restrict__ y, int64_t y_stride, int64_t rows,
                                                              int channels, int choices,
                                                              const int32_t *__restrict__ places,
                                                              const int32_t *__restrict__ starts, int experts,
                                                              Weights weights, int64_t first_block, int64_t row_blocks,
                                                              bool lines, T *__restrict__ dy,
                                                              void *__restrict__ dweights) {
  constexpr int N = kVectors<T, V>;
  const int lane = (int)threadIdx.x % LANES;
  const int64_t n = rows * choices, block = first_block + blockIdx.x;
  const int tail = starts[experts];
  const int64_t r = (lines ? block : inRuns(block, row_blocks)) * (kThreads / LANES) + (int)threadIdx.x / LANES;
  const bool row = r < rows;
  if (row) zeroTail<T, V, LANES>(tail, r, rows, n, channels, false, dy);
  for (int k0 = 0; k0 < choices; k0 += kAhead) {
    int64_t p[kAhead];
    float w[kAhead], along[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      p[j] = -1;
      w[j] = along[j] = 0.f;
      if (row && k0 + j < choices) {
        p[j] = places[r * choices + k0 + j];
        if (p[j] >= n) p[j] = -1;
        w[j] = weights.load(r * choices + k0 + j);
      }
    }
    if (row) {
      for (int c = lane * V; c < channels; c += LANES * V * N) {
        float g[N][V] = {};
        Vector<T, V> v[kAhead][N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int at = c + i * LANES * V;
          if (at < channels) loadFloats<T, V>(dout + r * dout_stride + at, g[i]);
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            v[j][i] = {};
            if (p[j] >= 0 && dweights != nullptr && at < channels)
              v[j][i] = *reinterpret_cast<const Vector<T, V> *>(y + p[j] * y_stride + at);
          }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (p[j] < 0) continue;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            float d[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
              d[e] = w[j] * g[i][e];
              along[j] = fmaf(g[i][e], (float)v[j][i].v[e], along[j]);
            }
            if (c + i * LANES * V < channels) storeFloats<T, V>(dy + p[j] * channels + c + i * LANES * V, d);
          }
        }
      }
    }
    if (dweights == nullptr) continue;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float sum = sumOverLanes<LANES>(along[j]);
      if (row && lane == 0 && k0 + j < choices) weights.store(dweights, r * choices + k0 + j, sum);
    }
  }
}

// ---- host side -----------------------------------------------------------------------------

constexpr int kMostExperts = device_sort::kMaxDigits - 1;
constexpr int kCounterWords = 16 * device_sort::kMaxDigits;  // that every workgroup of the second launch adds up by itself

struct Plan {
  int tiles, digits, digit_bits;
  bool few;  // two launches: the tiles' counters are few enough for every workgroup to add them up
  size_t counters, starts;
  size_t all() const { return 256 + counters + starts; }
};

Plan planOf(int64_t n, int64_t experts) {
  Plan p;
  const int64_t tiles = (n + kOrderTile - 1) / kOrderTile;
  p.few = tiles * (experts + 1) <= kCounterWords;
  p.tiles = (int)tiles;
  p.digits = (int)(p.few ? experts + 1
                         : (experts + device_sort::kColumns) / device_sort::kColumns * device_sort::kColumns);
  p.digit_bits = 1;
  while (((int64_t)1 << p.digit_bits) < experts + 1) ++p.digit_bits;
  const size_t words = p.few ? (size_t)tiles * p.digits : device_sort::counterWords(n, p.digits);
  p.counters = (words * sizeof(uint32_t) + 255) & ~(size_t)255;
  p.starts = (size_t)p.digits * sizeof(uint32_t);
  return p;
}

mluOpStatus_t checkOrder(const char *api, int64_t rows, int64_t choices, int64_t experts) {
  PARAM_CHECK(api, rows >= 0);
  PARAM_CHECK(api, choices > 0);
  PARAM_CHECK(api, experts > 0);
  if (experts > kMostExperts || choices > INT32_MAX || rows > (INT32_MAX - 4096) / choices) {
    MLUOP_LOG(ERROR) << api << " At most 2047 experts and 2^31 - 4097 choices of all rows are supported.";
    return MLUOP_STATUS_NOT_SUPPORTED;
  }
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t checkRows(const char *api, int64_t rows, int64_t channels, int64_t choices) {
  PARAM_CHECK(api, rows >= 0);
  PARAM_CHECK(api, channels > 0);
  PARAM_CHECK(api, choices > 0);
  if (channels > (1 << 20) || choices > INT32_MAX || rows > (INT32_MAX - 4096) / choices ||
      rows * choices * channels > ((int64_t)1 << 46)) {
    MLUOP_LOG(ERROR) << api << " At most 2^20 channels, 2^31 - 4097 choices of all rows and 2^46 values are supported.";
    return MLUOP_STATUS_NOT_SUPPORTED;
  }
  return MLUOP_STATUS_SUCCESS;
}

bool strideFits(int64_t rows, int64_t channels, int64_t stride) {
  return stride >= channels && (rows == 0 || stride <= ((int64_t)1 << 46) / rows);
}

// Calls f(element type, V): vectors that divide a row and lie at multiples of their length.
template <typename F>
void byType(mluOpDataType_t type, int64_t channels, int64_t strides, uintptr_t addresses, F f) {
  auto fits = [&](int v) {
    return channels % v == 0 && strides % v == 0 && addresses % (v * (size_t)elementBytes(type)) == 0;
  };
  auto sixteen = [&](auto zero) {
    if (fits(8))
      f(zero, std::integral_constant<int, 8>());
    else if (fits(4))
      f(zero, std::integral_constant<int, 4>());
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

// Calls f(LANES): threads for a row of so many pieces of 16 bytes, at most MOST.
template <int MOST, typename F>
void byLanes(int64_t pieces, F f) {
  if (pieces <= 2)
    f(std::integral_constant<int, 2>());
  else if (pieces <= 4)
    f(std::integral_constant<int, 4>());
  else if (pieces <= 8)
    f(std::integral_constant<int, 8>());
  else if (pieces <= 16)
    f(std::integral_constant<int, 16>());
  else if (pieces <= 32)
    f(std::integral_constant<int, 32>());
  else if (pieces <= 64 || MOST <= 64)
    f(std::integral_constant<int, 64>());
  else if (pieces <= 128)
    f(std::integral_constant<int, (MOST < 128 ? MOST : 128)>());
  else
    f(std::integral_constant<int, MOST>());
}
template <typename T>
int64_t piecesOf(int64_t channels) { return (channels * (int64_t)sizeof(T) + 15) / 16; }

}  // namespace

mluOpStatus_t MLUOP_WIN_API mluOpExtGetExpertOrderWorkspaceSize(int64_t rows, int64_t choices, int64_t experts,
                                                                size_t *size) {
  const char *api = "[mluOpExtGetExpertOrderWorkspaceSize]";
  PARAM_CHECK(api, size != NULL);
  const mluOpStatus_t status = checkOrder(api, rows, choices, experts);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  *size = planOf(std::max<int64_t>(rows * choices, 1), experts).all();
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtExpertOrder(mluOpHandle_t handle, mluOpDataType_t index_type,
                                                const void *experts_of_rows, int64_t rows, int64_t choices,
                                                int64_t experts, void *workspace, size_t workspace_size,
                                                int32_t *ordered_rows, int32_t *group_starts, int32_t *places) {
  const char *api = "[mluOpExtExpertOrder]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, index_type == MLUOP_DTYPE_INT32 || index_type == MLUOP_DTYPE_INT64);
  const mluOpStatus_t status = checkOrder(api, rows, choices, experts);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, rows == 0 || (experts_of_rows != NULL && ordered_rows != NULL && places != NULL));
  PARAM_CHECK(api, group_starts != NULL);
  PARAM_CHECK(api, workspace != NULL);
  const int64_t n = rows * choices;
  const Plan p = planOf(std::max<int64_t>(n, 1), experts);
  PARAM_CHECK(api, workspace_size >= p.all());
  DEVICE_HANDLE_CHECK(api, handle);
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  if (handle->hasNotes()) {
    handle->forgetNotesIn(ordered_rows, (size_t)n * sizeof(int32_t));
    handle->forgetNotesIn(places, (size_t)n * sizeof(int32_t));
    handle->forgetNotesIn(group_starts, (size_t)(experts + 1) * sizeof(int32_t));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  // (the caller's memory need not be aligned)
  char *at = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~(uintptr_t)255);
  uint32_t *counters = reinterpret_cast<uint32_t *>(at), *starts = reinterpret_cast<uint32_t *>(at + p.counters);
  const bool wide = index_type == MLUOP_DTYPE_INT64;
  const Choices items = {static_cast<const uint32_t *>(experts_of_rows), wide ? 2 : 1, wide ? 1 : 0, wide ? ~0u : 0u,
                         (uint32_t)experts, (uint32_t)choices, ordered_rows, places};
  const mluop::LaunchCtx lc = handle->launchCtx();
  lc.begin("expertOrder");
  if (n == 0) {
    expertStarts<<<(unsigned)(experts / kThreads + 1), kThreads, 0, lc.stream>>>(nullptr, (int)experts + 1, group_starts);
  } else if (n <= kOrderTile) {
    expertPlaces<true><<<1, kOrderThreads, 0, lc.stream>>>(items, n, (int)experts + 1, p.digit_bits, 0, nullptr, group_starts);
  } else if (p.few) {
    int across = 1;
    while (across < experts + 1 && across < kOrderThreads) across <<= 1;
    expertCounts<<<p.tiles, kOrderThreads, 0, lc.stream>>>(items, n, p.digits, counters);
    expertPlaces<false><<<p.tiles, kOrderThreads, 0, lc.stream>>>(items, n, p.digits, p.digit_bits, across, counters,
                                                                  group_starts);
  } else {
    HIP_CHECK_RETURN(api, device_sort::partition(lc.stream, items, n, p.digits, p.digit_bits, counters, starts));
    expertStarts<<<(unsigned)(experts / kThreads + 1), kThreads, 0, lc.stream>>>(starts, (int)experts + 1, group_starts);
  }
  lc.end();
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtExpertDispatch(mluOpHandle_t handle, mluOpDataType_t type, const void *features,
                                                   int64_t features_stride, int64_t rows, int64_t channels,
                                                   int64_t choices, const int32_t *places, const int32_t *group_starts,
                                                   int64_t experts, void *out) {
  const char *api = "[mluOpExtExpertDispatch]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  const mluOpStatus_t status = checkRows(api, rows, channels, choices);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, experts > 0 && experts <= INT32_MAX);
  PARAM_CHECK(api, strideFits(rows, channels, features_stride));
  PARAM_CHECK(api, rows == 0 || (features != NULL && places != NULL && out != NULL));
  PARAM_CHECK(api, group_starts != NULL);
  DEVICE_HANDLE_CHECK(api, handle);
  if (rows == 0) return MLUOP_STATUS_SUCCESS;
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  const size_t bytes = (size_t)rows * choices * channels * elementBytes(type);
  handle->forgetNotesIn(out, bytes);
  const bool lines = wholeLines(channels, type);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(out);
  byType(type, channels, features_stride, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    byLanes<256>(piecesOf<T>(channels), [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value;
      const int64_t blocks = (rows + kThreads / LANES - 1) / (kThreads / LANES);
      inLaunches(blocks, kThreads, [&](int64_t first, unsigned count) {
        lc.begin("expertDispatch");
        expertDispatch<T, V, LANES><<<count, kThreads, 0, lc.stream>>>(
            static_cast<const T *>(features), features_stride, rows, (int)channels, (int)choices, places, group_starts,
            (int)experts, first, blocks, lines, lines && bytes >= kStreamedBytes, static_cast<T *>(out));
        lc.end();
      });
    });
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtExpertCombine(mluOpHandle_t handle, mluOpDataType_t type, const void *results,
                                                  int64_t results_stride, int64_t rows, int64_t channels, int64_t choices,
                                                  const int32_t *places, mluOpDataType_t weight_type, const void *weights,
                                                  void *out) {
  const char *api = "[mluOpExtExpertCombine]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  PARAM_CHECK(api, weight_type == type || weight_type == MLUOP_DTYPE_FLOAT);
  const mluOpStatus_t status = checkRows(api, rows, channels, choices);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, strideFits(rows * choices, channels, results_stride));
  PARAM_CHECK(api, rows == 0 || (results != NULL && places != NULL && out != NULL));
  DEVICE_HANDLE_CHECK(api, handle);
  if (rows == 0) return MLUOP_STATUS_SUCCESS;
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  const size_t bytes = (size_t)rows * channels * elementBytes(type);
  handle->forgetNotesIn(out, bytes);
  const bool lines = wholeLines(channels, type);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(results) | reinterpret_cast<uintptr_t>(out);
  byType(type, channels, results_stride, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    byLanes<256>(piecesOf<T>(channels), [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value;
      const int64_t blocks = (rows + kThreads / LANES - 1) / (kThreads / LANES);
      inLaunches(blocks, kThreads, [&](int64_t first, unsigned count) {
        lc.begin("expertCombine");
        expertCombine<T, V, LANES><<<count, kThreads, 0, lc.stream>>>(
            static_cast<const T *>(results), results_stride, rows, (int)channels, (int)choices, places,
            Weights{weights, weight_type}, first, blocks, lines, bytes >= kStreamedBytes, static_cast<T *>(out));
        lc.end();
      });
    });
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtExpertCombineBackward(mluOpHandle_t handle, mluOpDataType_t type,
                                                          const void *output_grad, int64_t output_grad_stride,
                                                          const void *results, int64_t results_stride, int64_t rows,
                                                          int64_t channels, int64_t choices, const int32_t *places,
                                                          const int32_t *group_starts, int64_t experts,
                                                          mluOpDataType_t weight_type, const void *weights,
                                                          void *results_grad, void *weights_grad) {
  const char *api = "[mluOpExtExpertCombineBackward]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  PARAM_CHECK(api, weight_type == type || weight_type == MLUOP_DTYPE_FLOAT);
  const mluOpStatus_t status = checkRows(api, rows, channels, choices);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, experts > 0 && experts <= INT32_MAX);
  PARAM_CHECK(api, strideFits(rows, channels, output_grad_stride) && strideFits(rows * choices, channels, results_stride));
  PARAM_CHECK(api, rows == 0 || (output_grad != NULL && places != NULL && results_grad != NULL));
  PARAM_CHECK(api, rows == 0 || weights_grad == NULL || results != NULL);
  PARAM_CHECK(api, group_starts != NULL);
  DEVICE_HANDLE_CHECK(api, handle);
  if (rows == 0) return MLUOP_STATUS_SUCCESS;
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  const size_t bytes = (size_t)rows * choices * channels * elementBytes(type);
  if (handle->hasNotes()) {
    handle->forgetNotesIn(results_grad, bytes);
    if (weights_grad) handle->forgetNotesIn(weights_grad, (size_t)rows * choices * elementBytes(weight_type));
  }
  const bool lines = wholeLines(channels, type);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(output_grad) | reinterpret_cast<uintptr_t>(results) |
                              reinterpret_cast<uintptr_t>(results_grad);
  byType(type, channels, output_grad_stride | results_stride, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    T *dy = static_cast<T *>(results_grad);
    auto launch = [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value;
      const int64_t blocks = (rows + kThreads / LANES - 1) / (kThreads / LANES);
      inLaunches(blocks, kThreads, [&](int64_t first, unsigned count) {
        lc.begin("expertCombineGrad");
        expertCombineGrad<T, V, LANES><<<count, kThreads, 0, lc.stream>>>(
            static_cast<const T *>(output_grad), output_grad_stride, static_cast<const T *>(results), results_stride, rows,
            (int)channels, (int)choices, places, group_starts, (int)experts, Weights{weights, weight_type}, first, blocks,
            lines, dy, weights_grad);
        lc.end();
      });
    };
    byLanes<64>(piecesOf<T>(channels), launch);
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
