// mluOpExtGroupNormForward / Backward (no counterpart in the reference): group norm with an activation over ragged samples
// of rows whose channels lie side by side.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "core/core.h"
#include "core/elements.h"
#include "core/ragged.h"
#include "mlu_op_ext.h"

namespace {

using namespace mluop;

constexpr int kThreads = 256;

// The problem as its kernels see it.
struct Shape {
  int rows, channels, groups, samples;
  int tile_rows, most_tiles;
  const int32_t *starts;
};

// Rows of a tile: enough tiles to fill the GPU, enough values in each for what a workgroup does once.
int tileRows(int64_t rows, int64_t channels) {
  const int64_t fill = (rows + 2047) / 2048, least = (8192 + channels - 1) / channels;
  const int64_t r = std::min<int64_t>(std::max(fill, least), 1024);
  return (int)((r + 15) / 16 * 16);
}

struct Params {
  const void *weight, *bias;
  mluOpDataType_t type;
  __device__ __forceinline__ float at(const void *p, int c, float none) const {
    if (p == nullptr) return none;
    if (type == MLUOP_DTYPE_FLOAT) return static_cast<const float *>(p)[c];
    if (type == MLUOP_DTYPE_HALF) return (float)static_cast<const _Float16 *>(p)[c];
    return (float)static_cast<const __bf16 *>(p)[c];
  }
  __device__ __forceinline__ float weightAt(int c) const { return at(weight, c, 1.f); }
  __device__ __forceinline__ float biasAt(int c) const { return at(bias, c, 0.f); }
};

template <int V>
using Lanes = RowLanes<V, kThreads>;

__device__ __forceinline__ float sigmoid(float z) {
  // (an exponential beyond the range is infinite, and its reciprocal zero)
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}

template <int ACT>
__device__ __forceinline__ float activated(float z) {
  if (ACT == MLUOP_EXT_ACTIVATION_RELU) return z < 0.f ? 0.f : z;  // (a NaN stays one)
  if (ACT == MLUOP_EXT_ACTIVATION_SILU) return z * sigmoid(z);
  return z;
}

template <int ACT>
__device__ __forceinline__ float slope(float z) {
  if (ACT == MLUOP_EXT_ACTIVATION_RELU) return z > 0.f ? 1.f : 0.f;
  if (ACT == MLUOP_EXT_ACTIVATION_SILU) {
    const float t = sigmoid(z);
    return t * (1.f + z * (1.f - t));
  }
  return 1.f;
}

// Sums a[V] and b[V] of a channel over the rows a workgroup holds at once; valid in its first row of threads.
template <int V>
__device__ __forceinline__ void sumOverRows(const Lanes<V> &l, float (&a)[V], float (&b)[V]) {
  __shared__ float s_a[kThreads * V], s_b[kThreads * V];
  const int at = threadIdx.x * V;
  int left = l.rows_at_once;
  while (left > 1) {
    const int half = (left + 1) / 2;
    if (l.row >= half && l.row < left) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        s_a[at + v] = a[v];
        s_b[at + v] = b[v];
      }
    }
    __syncthreads();
    if (l.row >= 0 && l.row + half < left) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        a[v] += s_a[at + half * l.across * V + v];
        b[v] += s_b[at + half * l.across * V + v];
      }
    }
    left = half;
  }
}

// A tile's mean and sum of squared deviations of every channel, to partial[tile][channel].  The sums are taken of
// differences from the tile's first row, so that channels far off zero lose nothing.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void groupNormMoments(const T *__restrict__ x, Shape s,
                                                             float2 *__restrict__ partial) {
  const RaggedTile t = findRaggedTile<false>(s.starts, s.rows, s.samples, s.tile_rows, blockIdx.x);
  if (t.segment < 0) return;
  const Lanes<V> l(s.channels);
  float base[V], sum[V] = {}, squares[V] = {};
  if (l.row >= 0) {
    const T *from = x + (int64_t)t.first * s.channels + l.channel;
    loadFloats<T, V>(from, base);
    for (int r = l.row; r < t.rows; r += l.rows_at_once) {
      float v[V];
      loadFloats<T, V>(from + (int64_t)r * s.channels, v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = v[i] - base[i];
        sum[i] += d;
        squares[i] = fmaf(d, d, squares[i]);
      }
    }
  }
  sumOverRows<V>(l, sum, squares);
  if (l.row == 0) {
    const float by = 1.f / (float)t.rows;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float off = sum[i] * by;
      partial[(int64_t)blockIdx.x * s.channels + l.channel + i] =
          make_float2(base[i] + off, fmaxf(squares[i] - sum[i] * off, 0.f));
    }
  }
}

// Sum of v over a workgroup, in all threads.
__device__ __forceinline__ float sumOfWorkgroup(float v) {
  __shared__ float s_wave[kThreads / 64];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = v;
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) sum += s_wave[w];
  return sum;
}

// Mean and rstd of a (sample, group) from its tiles' moments: the mean first, then the deviations from it.
__global__ __launch_bounds__(kThreads) void groupNormJoinMoments(const float2 *__restrict__ partial, Shape s, float eps,
                                                                 float *__restrict__ mean, float *__restrict__ rstd) {
  const int sample = blockIdx.x / s.groups, group = blockIdx.x - sample * s.groups;
  const int per_group = s.channels / s.groups;
  int first, rows;
  const int tiles = raggedTilesOf(s.starts, s.rows, sample, s.tile_rows, s.most_tiles, &first, &rows);
  const float2 *from = partial + (int64_t)first * s.channels + group * per_group;
  const int entries = tiles * per_group;
  auto rowsOf = [&](int tile) { return (float)min(s.tile_rows, rows - tile * s.tile_rows); };
  float sum = 0.f;
  for (int e = threadIdx.x; e < entries; e += kThreads) {
    const int tile = e / per_group;
    sum += from[(int64_t)tile * s.channels + (e - tile * per_group)].x * rowsOf(tile);
  }
  const float by = rows > 0 ? 1.f / ((float)rows * (float)per_group) : 0.f;
  const float m = sumOfWorkgroup(sum) * by;
  float squares = 0.f;
  for (int e = threadIdx.x; e < entries; e += kThreads) {
    const int tile = e / per_group;
    const float2 p = from[(int64_t)tile * s.channels + (e - tile * per_group)];
    squares += fmaf((p.x - m) * (p.x - m), rowsOf(tile), p.y);
  }
  squares = sumOfWorkgroup(squares);
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = m;
    rstd[blockIdx.x] = 1.f / sqrtf(squares * by + eps);
  }
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void groupNormApply(const T *__restrict__ x, Shape s, Params p,
                                                           const float *__restrict__ mean,
                                                           const float *__restrict__ rstd, T *__restrict__ out) {
  const RaggedTile t = findRaggedTile<true>(s.starts, s.rows, s.samples, s.tile_rows, blockIdx.x);
  if (t.segment < 0) return;
  const Lanes<V> l(s.channels);
  if (l.row < 0) return;
  const bool inside = t.segment > 0 && t.segment <= s.samples;
  float m[V] = {}, a[V] = {}, b[V] = {};
  if (inside) {
    const int per_group = s.channels / s.groups;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int g = (t.segment - 1) * s.groups + (l.channel + i) / per_group;
      m[i] = mean[g];
      a[i] = rstd[g] * p.weightAt(l.channel + i);
      b[i] = p.biasAt(l.channel + i);
    }
  }
  const int64_t at = (int64_t)t.first * s.channels + l.channel;
  for (int r = l.row; r < t.rows; r += l.rows_at_once) {
    float v[V] = {};
    if (inside) {
      loadFloats<T, V>(x + at + (int64_t)r * s.channels, v);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = activated<ACT>(fmaf(v[i] - m[i], a[i], b[i]));
    }
    storeFloats<T, V>(out + at + (int64_t)r * s.channels, v);
  }
}

// dz = dy * activation'(z) of V channels, and the normed values.
template <typename T, int V, int ACT>
__device__ __forceinline__ void gradOfNormed(const T *dy, const T *x, const float (&m)[V], const float (&r)[V],
                                             const float (&w)[V], const float (&b)[V], float (&dz)[V],
                                             float (&normed)[V]) {
  loadFloats<T, V>(dy, dz);
  loadFloats<T, V>(x, normed);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    normed[i] = (normed[i] - m[i]) * r[i];
    if (ACT != MLUOP_EXT_ACTIVATION_NONE) dz[i] *= slope<ACT>(fmaf(normed[i], w[i], b[i]));
  }
}

// A tile's sums of dz and dz * normed of every channel, to partial[tile][channel].
template <typename T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void groupNormGradSums(const T *__restrict__ dy, const T *__restrict__ x, Shape s,
                                                              Params p, const float *__restrict__ mean,
                                                              const float *__restrict__ rstd,
                                                              float2 *__restrict__ partial) {
  const RaggedTile t = findRaggedTile<false>(s.starts, s.rows, s.samples, s.tile_rows, blockIdx.x);
  if (t.segment < 0) return;
  const Lanes<V> l(s.channels);
  float sum[V] = {}, with_normed[V] = {};
  if (l.row >= 0) {
    const int per_group = s.channels / s.groups;
    float m[V], r[V], w[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int g = t.segment * s.groups + (l.channel + i) / per_group;
      m[i] = mean[g];
      r[i] = rstd[g];
      w[i] = p.weightAt(l.channel + i);
      b[i] = p.biasAt(l.channel + i);
    }
    const int64_t at = (int64_t)t.first * s.channels + l.channel;
    for (int row = l.row; row < t.rows; row += l.rows_at_once) {
      float dz[V], normed[V];
      const int64_t from = at + (int64_t)row * s.channels;
      gradOfNormed<T, V, ACT>(dy + from, x + from, m, r, w, b, dz, normed);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        sum[i] += dz[i];
        with_normed[i] = fmaf(dz[i], normed[i], with_normed[i]);
      }
    }
  }
  sumOverRows<V>(l, sum, with_normed);
  if (l.row == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      partial[(int64_t)blockIdx.x * s.channels + l.channel + i] = make_float2(sum[i], with_normed[i]);
  }
}

template <typename T>
__device__ __forceinline__ void storeParam(void *to, int c, float v) {
  static_cast<T *>(to)[c] = (T)v;
}

// The first samples * groups workgroups: the means of w dz and w dz * normed of a (sample, group).  The others: the
// gradients of the parameters of kChannels channels each, over all tiles.
constexpr int kChannels = 16;
__global__ __launch_bounds__(kThreads) void groupNormJoinGradSums(const float2 *__restrict__ partial, Shape s, Params p,
                                                                  float2 *__restrict__ means, void *weight_grad,
                                                                  void *bias_grad) {
  const int pairs = s.samples * s.groups;
  if ((int)blockIdx.x < pairs) {
    const int sample = blockIdx.x / s.groups, group = blockIdx.x - sample * s.groups;
    const int per_group = s.channels / s.groups;
    int first, rows;
    const int entries = raggedTilesOf(s.starts, s.rows, sample, s.tile_rows, s.most_tiles, &first, &rows) * per_group;
    const float2 *from = partial + (int64_t)first * s.channels + group * per_group;
    float a = 0.f, b = 0.f;
    for (int e = threadIdx.x; e < entries; e += kThreads) {
      const int tile = e / per_group, c = e - tile * per_group;
      const float2 v = from[(int64_t)tile * s.channels + c];
      const float w = p.weightAt(group * per_group + c);
      a = fmaf(v.x, w, a);
      b = fmaf(v.y, w, b);
    }
    a = sumOfWorkgroup(a);
    b = sumOfWorkgroup(b);
    const float by = rows > 0 ? 1.f / ((float)rows * (float)per_group) : 0.f;
    if (threadIdx.x == 0) means[blockIdx.x] = make_float2(a * by, b * by);
    return;
  }
  int last, rows;
  const int of_last = raggedTilesOf(s.starts, s.rows, s.samples - 1, s.tile_rows, s.most_tiles, &last, &rows);
  const int tiles = last + of_last;
  const int lane = threadIdx.x % kChannels, share = threadIdx.x / kChannels;
  const int c = ((int)blockIdx.x - pairs) * kChannels + lane;
  __shared__ float2 s_sum[kThreads / kChannels][kChannels];
  float a = 0.f, b = 0.f;
  if (c < s.channels) {
    for (int t = share; t < tiles; t += kThreads / kChannels) {
      const float2 v = partial[(int64_t)t * s.channels + c];
      a += v.x;
      b += v.y;
    }
  }
  s_sum[share][lane] = make_float2(a, b);
  __syncthreads();
  if (share != 0 || c >= s.channels) return;
  for (int i = 1; i < kThreads / kChannels; ++i) {
    a += s_sum[i][lane].x;
    b += s_sum[i][lane].y;
  }
  auto store = [&](void *to, float v) {
    if (to == nullptr) return;
    if (p.type == MLUOP_DTYPE_FLOAT)
      storeParam<float>(to, c, v);
    else if (p.type == MLUOP_DTYPE_HALF)
      storeParam<_Float16>(to, c, v);
    else
      storeParam<__bf16>(to, c, v);
  };
  store(bias_grad, a);
  store(weight_grad, b);
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void groupNormGradApply(const T *__restrict__ dy, const T *__restrict__ x, Shape s,
                                                               Params p, const float *__restrict__ mean,
                                                               const float *__restrict__ rstd,
                                                               const float2 *__restrict__ means, T *__restrict__ dx) {
  const RaggedTile t = findRaggedTile<true>(s.starts, s.rows, s.samples, s.tile_rows, blockIdx.x);
  if (t.segment < 0) return;
  const Lanes<V> l(s.channels);
  if (l.row < 0) return;
  const bool inside = t.segment > 0 && t.segment <= s.samples;
  float m[V] = {}, r[V] = {}, w[V] = {}, b[V] = {};
  float2 c[V] = {};
  if (inside) {
    const int per_group = s.channels / s.groups;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int g = (t.segment - 1) * s.groups + (l.channel + i) / per_group;
      m[i] = mean[g];
      r[i] = rstd[g];
      c[i] = means[g];
      w[i] = p.weightAt(l.channel + i);
      b[i] = p.biasAt(l.channel + i);
    }
  }
  const int64_t at = (int64_t)t.first * s.channels + l.channel;
  for (int row = l.row; row < t.rows; row += l.rows_at_once) {
    const int64_t from = at + (int64_t)row * s.channels;
    float d[V] = {};
    if (inside) {
      float dz[V], normed[V];
      gradOfNormed<T, V, ACT>(dy + from, x + from, m, r, w, b, dz, normed);
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = r[i] * (fmaf(dz[i], w[i], -c[i].x) - normed[i] * c[i].y);
    }
    storeFloats<T, V>(dx + from, d);
  }
}

// ---- host side -----------------------------------------------------------------------------

size_t partialBytes(int64_t rows, int64_t channels, int64_t samples) {
  return (size_t)mostRaggedTiles(rows, samples, tileRows(rows, channels)) * channels * sizeof(float2);
}

mluOpStatus_t checkShape(const char *api, int64_t rows, int64_t channels, int64_t groups, int64_t samples) {
  PARAM_CHECK(api, rows >= 0);
  PARAM_CHECK(api, channels > 0);
  PARAM_CHECK(api, groups > 0);
  PARAM_CHECK(api, channels % groups == 0);
  PARAM_CHECK(api, samples > 0);
  if (rows > INT32_MAX - 4096 || channels > (1 << 20) || samples > (1 << 20) || samples * groups > (1 << 28) ||
      rows * channels > ((int64_t)1 << 46)) {
    MLUOP_LOG(ERROR) << api << " At most 2^31 - 4097 rows, 2^20 channels, 2^20 samples, 2^28 pairs of a sample and a "
                     << "group and 2^46 values are supported.";
    return MLUOP_STATUS_NOT_SUPPORTED;
  }
  return MLUOP_STATUS_SUCCESS;
}

struct Workspace {
  float2 *partial, *means;
};

// (the caller's memory need not be aligned)
size_t workspaceBytes(int64_t rows, int64_t channels, int64_t groups, int64_t samples) {
  return 16 + partialBytes(rows, channels, samples) + (size_t)samples * groups * sizeof(float2);
}
Workspace carve(void *workspace, int64_t rows, int64_t channels, int64_t samples) {
  char *at = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~(uintptr_t)15);
  return {reinterpret_cast<float2 *>(at), reinterpret_cast<float2 *>(at + partialBytes(rows, channels, samples))};
}

// Calls f(element type, V, activation) as constants.
template <typename F>
void byActivation(int activation, F f) {
  if (activation == MLUOP_EXT_ACTIVATION_RELU)
    f(std::integral_constant<int, MLUOP_EXT_ACTIVATION_RELU>());
  else if (activation == MLUOP_EXT_ACTIVATION_SILU)
    f(std::integral_constant<int, MLUOP_EXT_ACTIVATION_SILU>());
  else
    f(std::integral_constant<int, MLUOP_EXT_ACTIVATION_NONE>());
}

// (vectors that divide a row and lie at multiples of their length: 16 bytes, 8 of a 2-byte type, single elements)
template <typename F>
void byType(mluOpDataType_t type, int channels, uintptr_t addresses, F f) {
  auto fits = [&](int v) { return channels % v == 0 && addresses % (v * (size_t)elementBytes(type)) == 0; };
  auto sixteen = [&](auto zero) {
    if (fits(8))
      f(zero, std::integral_constant<int, 8>());
    else if (fits(4))
      f(zero, std::integral_constant<int, 4>());
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

}  // namespace

mluOpStatus_t MLUOP_WIN_API mluOpExtGetGroupNormWorkspaceSize(int64_t rows, int64_t channels, int64_t groups,
                                                              int64_t samples, size_t *size) {
  const char *api = "[mluOpExtGetGroupNormWorkspaceSize]";
  PARAM_CHECK(api, size != NULL);
  const mluOpStatus_t status = checkShape(api, rows, channels, groups, samples);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  *size = workspaceBytes(rows, channels, groups, samples);
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtGroupNormForward(mluOpHandle_t handle, mluOpDataType_t type, const void *features,
                                                     int64_t rows, int64_t channels, int64_t groups,
                                                     const int32_t *row_starts, int64_t samples,
                                                     mluOpDataType_t param_type, const void *weight, const void *bias,
                                                     float eps, mluOpExtActivation_t activation, void *workspace,
                                                     size_t workspace_size, void *out, float *mean, float *rstd) {
  const char *api = "[mluOpExtGroupNormForward]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  PARAM_CHECK(api, param_type == type || param_type == MLUOP_DTYPE_FLOAT);
  const mluOpStatus_t status = checkShape(api, rows, channels, groups, samples);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, row_starts != NULL || samples == 1);
  PARAM_CHECK(api, activation >= MLUOP_EXT_ACTIVATION_NONE && activation <= MLUOP_EXT_ACTIVATION_SILU);
  PARAM_CHECK(api, eps >= 0.f && std::isfinite(eps));
  PARAM_CHECK(api, rows == 0 || (features != NULL && out != NULL));
  PARAM_CHECK(api, mean != NULL && rstd != NULL);
  PARAM_CHECK(api, workspace != NULL);
  PARAM_CHECK(api, workspace_size >= workspaceBytes(rows, channels, groups, samples));
  DEVICE_HANDLE_CHECK(api, handle);
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  if (handle->hasNotes()) {
    handle->forgetNotesIn(out, (size_t)rows * channels * elementBytes(type));
    handle->forgetNotesIn(mean, (size_t)samples * groups * sizeof(float));
    handle->forgetNotesIn(rstd, (size_t)samples * groups * sizeof(float));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  const Shape s = {(int)rows, (int)channels, (int)groups, (int)samples, tileRows(rows, channels),
                   (int)mostRaggedTiles(rows, samples, tileRows(rows, channels)), row_starts};
  const Params p = {weight, bias, param_type};
  const Workspace w = carve(workspace, rows, channels, samples);
  const mluop::LaunchCtx lc = handle->launchCtx();
  byType(type, s.channels, reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(out), [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    const unsigned slabs = (unsigned)((s.channels / V + kThreads - 1) / kThreads);
    const unsigned tiles = (unsigned)mostRaggedTiles(rows, samples, s.tile_rows);
    if (tiles > 0) {
      lc.begin("groupNormMoments");
      groupNormMoments<T, V><<<dim3(tiles, slabs), kThreads, 0, lc.stream>>>(static_cast<const T *>(features), s, w.partial);
      lc.end();
    }
    lc.begin("groupNormJoinMoments");
    groupNormJoinMoments<<<(unsigned)(samples * groups), kThreads, 0, lc.stream>>>(w.partial, s, eps, mean, rstd);
    lc.end();
    const unsigned all = (unsigned)mostRaggedTiles(rows, samples + 2, s.tile_rows);
    if (all == 0) return;
    byActivation(activation, [&](auto act) {
      lc.begin("groupNormApply");
      groupNormApply<T, V, decltype(act)::value><<<dim3(all, slabs), kThreads, 0, lc.stream>>>(
          static_cast<const T *>(features), s, p, mean, rstd, static_cast<T *>(out));
      lc.end();
    });
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtGroupNormBackward(mluOpHandle_t handle, mluOpDataType_t type,
                                                      const void *output_grad, const void *features, int64_t rows,
                                                      int64_t channels, int64_t groups, const int32_t *row_starts,
                                                      int64_t samples, mluOpDataType_t param_type, const void *weight,
                                                      const void *bias, const float *mean, const float *rstd,
                                                      mluOpExtActivation_t activation, void *workspace,
                                                      size_t workspace_size, void *input_grad, void *weight_grad,
                                                      void *bias_grad) {
  const char *api = "[mluOpExtGroupNormBackward]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  PARAM_CHECK(api, param_type == type || param_type == MLUOP_DTYPE_FLOAT);
  const mluOpStatus_t status = checkShape(api, rows, channels, groups, samples);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, row_starts != NULL || samples == 1);
  PARAM_CHECK(api, activation >= MLUOP_EXT_ACTIVATION_NONE && activation <= MLUOP_EXT_ACTIVATION_SILU);
  PARAM_CHECK(api, rows == 0 || (output_grad != NULL && features != NULL && input_grad != NULL));
  PARAM_CHECK(api, mean != NULL && rstd != NULL);
  PARAM_CHECK(api, workspace != NULL);
  PARAM_CHECK(api, workspace_size >= workspaceBytes(rows, channels, groups, samples));
  DEVICE_HANDLE_CHECK(api, handle);
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  if (handle->hasNotes()) {
    handle->forgetNotesIn(input_grad, (size_t)rows * channels * elementBytes(type));
    if (weight_grad) handle->forgetNotesIn(weight_grad, (size_t)channels * elementBytes(param_type));
    if (bias_grad) handle->forgetNotesIn(bias_grad, (size_t)channels * elementBytes(param_type));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  const Shape s = {(int)rows, (int)channels, (int)groups, (int)samples, tileRows(rows, channels),
                   (int)mostRaggedTiles(rows, samples, tileRows(rows, channels)), row_starts};
  const Params p = {weight, bias, param_type};
  const Workspace w = carve(workspace, rows, channels, samples);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(output_grad) |
                              reinterpret_cast<uintptr_t>(input_grad);
  byType(type, s.channels, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    const unsigned slabs = (unsigned)((s.channels / V + kThreads - 1) / kThreads);
    const T *dy = static_cast<const T *>(output_grad), *x = static_cast<const T *>(features);
    byActivation(activation, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      const unsigned tiles = (unsigned)mostRaggedTiles(rows, samples, s.tile_rows);
      if (tiles > 0) {
        lc.begin("groupNormGradSums");
        groupNormGradSums<T, V, ACT><<<dim3(tiles, slabs), kThreads, 0, lc.stream>>>(dy, x, s, p, mean, rstd, w.partial);
        lc.end();
      }
      lc.begin("groupNormJoinGradSums");
      groupNormJoinGradSums<<<(unsigned)(samples * groups + (channels + kChannels - 1) / kChannels), kThreads, 0,
                              lc.stream>>>(w.partial, s, p, w.means, weight_grad, bias_grad);
      lc.end();
      const unsigned all = (unsigned)mostRaggedTiles(rows, samples + 2, s.tile_rows);
      if (all == 0) return;
      lc.begin("groupNormGradApply");
      groupNormGradApply<T, V, ACT><<<dim3(all, slabs), kThreads, 0, lc.stream>>>(dy, x, s, p, mean, rstd, w.means,
                                                                                  static_cast<T *>(input_grad));
      lc.end();
    });
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
