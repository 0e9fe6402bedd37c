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

__global__ __launch_bounds__(kThreads) void expertStarts(const uint32_t *__restrict__ from, int count,
                                                         int32_t *__restrict__ to) {
  const int i = (int)blockIdx.x * kThreads + (int)threadIdx.x;
  if (i < count) to[i] = from == nullptr ? 0 : (int32_t)from[i];
}

// ---- rows to their places and back ---------------------------------------------------------

// What a row's choices have in common: threads of V channels each over rows, as many rows at once as fit.
template <int V>
using Lanes = RowLanes<V, kThreads>;

constexpr int kTailBlocks = 64;  // workgroups for the places behind the last expert's, which are zero

template <typename T, int V>
__device__ void zeroTail(const Lanes<V> &l, const int32_t *starts, int experts, int64_t n, int channels, int block, T *out) {
  const int64_t first = starts[experts];
  const float zero[V] = {};
  for (int64_t p = (first < 0 ? 0 : first) + (int64_t)block * l.rows_at_once + l.row; p < n;
       p += (int64_t)kTailBlocks * l.rows_at_once)
    storeFloats<T, V>(out + p * channels + l.channel, zero);
}

// out[place of (r, k)] = x[r] for every choice k: a row is read once and written as often as it is sent.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void expertDispatch(const T *__restrict__ x, int64_t x_stride, int64_t rows,
                                                           int channels, int choices, const int32_t *__restrict__ places,
                                                           const int32_t *__restrict__ starts, int experts,
                                                           int64_t first_block, int64_t row_blocks, bool streamed,
                                                           T *__restrict__ out) {
  const Lanes<V> l(channels);
  if (l.row < 0) return;
  const int64_t n = rows * choices, block = first_block + blockIdx.x;
  if (block >= row_blocks) {
    zeroTail<T, V>(l, starts, experts, n, channels, (int)(block - row_blocks), out);
    return;
  }
  const int64_t r = block * l.rows_at_once + l.row;
  if (r >= rows) return;
  const Vector<T, V> v = *reinterpret_cast<const Vector<T, V> *>(x + r * x_stride + l.channel);
  float f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = (float)v.v[i];
  for (int k = 0; k < choices; ++k) {
    const int64_t p = places[r * choices + k];
    if (p >= 0 && p < n) storeFloats<T, V>(out + p * channels + l.channel, f, streamed);
  }
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
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void expertCombine(const T *__restrict__ y, int64_t y_stride, int64_t rows,
                                                          int channels, int choices, const int32_t *__restrict__ places,
                                                          Weights weights, int64_t first_block, bool streamed,
                                                          T *__restrict__ out) {
  const Lanes<V> l(channels);
  if (l.row < 0) return;
  const int64_t n = rows * choices, r = (first_block + blockIdx.x) * l.rows_at_once + l.row;
  if (r >= rows) return;
  float sum[V] = {};
  for (int k0 = 0; k0 < choices; k0 += kAhead) {
    Vector<T, V> v[kAhead];
    float w[kAhead];
    bool there[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t at = r * choices + (k0 + j < choices ? k0 + j : k0);
      const int64_t p = places[at];
      there[j] = k0 + j < choices && p >= 0 && p < n;
      w[j] = weights.load(at);
      v[j] = *reinterpret_cast<const Vector<T, V> *>(y + (there[j] ? p : 0) * y_stride + l.channel);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (!there[j]) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] = fmaf(w[j], (float)v[j].v[i], sum[i]);
    }
  }
  storeFloats<T, V>(out + r * channels + l.channel, sum, streamed);
}

// The gradients of the weighted sum: dy_r goes to the places times its weights, and the weights' gradients are products with what
// lies there.  LANES lanes of a wave a row.
template <typename T, int V, int LANES>
__global__ __launch_bounds__(kThreads) void expertCombineGrad(const T *__restrict__ dout, int64_t dout_stride,
                                                              const T *__restrict__ y, int64_t y_stride, int64_t rows,
                                                              int channels, int choices,
                                                              const int32_t *__restrict__ places, Weights weights,
                                                              int64_t first_block, bool streamed, T *__restrict__ dy,
                                                              void *__restrict__ dweights) {
  constexpr int kRows = kThreads / LANES;
  const int lane = (int)threadIdx.x % LANES;
  const int64_t n = rows * choices, r = (first_block + blockIdx.x) * kRows + (int)threadIdx.x / LANES;
  const bool row = r < rows;
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
      for (int c = lane * V; c < channels; c += LANES * V) {
        float g[V];
        loadFloats<T, V>(dout + r * dout_stride + c, g);
        Vector<T, V> v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          v[j] = {};
          if (p[j] >= 0 && dweights != nullptr) v[j] = *reinterpret_cast<const Vector<T, V> *>(y + p[j] * y_stride + c);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (p[j] < 0) continue;
          float d[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            d[i] = w[j] * g[i];
            along[j] = fmaf(g[i], (float)v[j].v[i], along[j]);
          }
          storeFloats<T, V>(dy + p[j] * channels + c, d, streamed);
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

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void expertZeroTail(const int32_t *__restrict__ starts, int experts, int64_t n,
                                                           int channels, T *__restrict__ out) {
  const Lanes<V> l(channels);
  if (l.row >= 0) zeroTail<T, V>(l, starts, experts, n, channels, (int)blockIdx.x, out);
}

// ---- host side -----------------------------------------------------------------------------

constexpr int kMostExperts = device_sort::kMaxDigits - 1;
constexpr int kCounterWords = 16 * device_sort::kMaxDigits;  // that a workgroup of the order's second launch reads by itself

struct Plan {
  int tiles, digits, digit_bits;
  bool few;  // two launches: the tiles' counters are few enough for every workgroup to add them up
  size_t counters, starts;
  size_t all() const { return 256 + counters + starts; }
};

Plan planOf(int64_t n, int64_t experts) {
  Plan p;
  p.tiles = device_sort::tilesFor(n);
  p.few = device_sort::roundsFor(n) == 1 && p.tiles * (experts + 1) <= kCounterWords;
  p.digits = (int)(p.few ? experts + 1
                         : (experts + device_sort::kColumns) / device_sort::kColumns * device_sort::kColumns);
  p.digit_bits = 1;
  while (((int64_t)1 << p.digit_bits) < experts + 1) ++p.digit_bits;
  p.counters = (device_sort::counterWords(n, p.digits) * sizeof(uint32_t) + 255) & ~(size_t)255;
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
  } else if (p.few) {
    uint32_t *hist = counters + device_sort::kMaxDigits;
    device_sort::countTiles<Choices><<<p.tiles, device_sort::kTileThreads, 0, lc.stream>>>(items, n, p.digits, 1, hist);
    device_sort::partitionTiles<Choices, false><<<p.tiles, device_sort::kTileThreads, 0, lc.stream>>>(
        items, n, p.digits, p.digit_bits, 1, hist, nullptr, reinterpret_cast<uint32_t *>(group_starts));
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
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(out);
  byType(type, channels, features_stride, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    const int64_t at_once = rowsAtOnce(channels / V), blocks = (rows + at_once - 1) / at_once;
    inLaunches(blocks + kTailBlocks, kThreads, [&](int64_t first, unsigned count) {
      lc.begin("expertDispatch");
      expertDispatch<T, V><<<dim3(count, slabsOf(channels / V)), kThreads, 0, lc.stream>>>(
          static_cast<const T *>(features), features_stride, rows, (int)channels, (int)choices, places, group_starts,
          (int)experts, first, blocks, bytes >= kStreamedBytes, static_cast<T *>(out));
      lc.end();
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
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(results) | reinterpret_cast<uintptr_t>(out);
  byType(type, channels, results_stride, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    const int64_t at_once = rowsAtOnce(channels / V);
    inLaunches((rows + at_once - 1) / at_once, kThreads, [&](int64_t first, unsigned count) {
      lc.begin("expertCombine");
      expertCombine<T, V><<<dim3(count, slabsOf(channels / V)), kThreads, 0, lc.stream>>>(
          static_cast<const T *>(results), results_stride, rows, (int)channels, (int)choices, places,
          Weights{weights, weight_type}, first, bytes >= kStreamedBytes, static_cast<T *>(out));
      lc.end();
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
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(output_grad) | reinterpret_cast<uintptr_t>(results) |
                              reinterpret_cast<uintptr_t>(results_grad);
  byType(type, channels, output_grad_stride | results_stride, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    T *dy = static_cast<T *>(results_grad);
    auto launch = [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value;
      inLaunches((rows + kThreads / LANES - 1) / (kThreads / LANES), kThreads, [&](int64_t first, unsigned count) {
        lc.begin("expertCombineGrad");
        expertCombineGrad<T, V, LANES><<<count, kThreads, 0, lc.stream>>>(
            static_cast<const T *>(output_grad), output_grad_stride, static_cast<const T *>(results), results_stride, rows,
            (int)channels, (int)choices, places, Weights{weights, weight_type}, first, bytes >= kStreamedBytes, dy,
            weights_grad);
        lc.end();
      });
    };
    if (channels / V <= 8)
      launch(std::integral_constant<int, 8>());
    else if (channels / V <= 16)
      launch(std::integral_constant<int, 16>());
    else
      launch(std::integral_constant<int, 64>());
    lc.begin("expertZeroTail");
    expertZeroTail<T, V><<<dim3(kTailBlocks, slabsOf(channels / V)), kThreads, 0, lc.stream>>>(
        group_starts, (int)experts, rows * choices, (int)channels, dy);
    lc.end();
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
