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
constexpr int kAhead = 4;      // rows of a thread whose loads are in flight together
constexpr int kGradAhead = 2;  // the same of two tensors

// The problem as its kernels see it.
struct Shape {
  int rows, channels, groups, samples;
  int tile_rows, most_tiles;  // tiles that are summed
  int apply_rows;             // rows of a tile of the pass that applies them
  const int32_t *starts;
  bool streamed;              // results go past the caches
};

// Rows of a tile: tiles for four workgroups a CU, and values enough in each for what a workgroup does once.  248 636 x 128
// fp16 with SiLU, us of the pass that applies, and gradient sums of 400 000 x 128 bf16, at 512 / 1024 / 2048 tiles: 24 / 23 /
// 23 and 58 / 41 / 45.
constexpr int64_t kTiles = 1024;
int tileRows(int64_t rows, int64_t channels) {
  const int64_t fill = (rows + kTiles - 1) / kTiles, least = (8192 + channels - 1) / channels;
  const int64_t r = std::min<int64_t>(std::max(fill, least), 1024);
  return (int)((r + 15) / 16 * 16);
}

// Rows of a tile of the pass that applies: nothing is added up there, so that smaller tiles cost little.
int applyRows(int64_t rows, int64_t channels) {
  const int64_t fill = (rows + kTiles - 1) / kTiles, least = (2048 + channels - 1) / channels;
  const int64_t r = std::min<int64_t>(std::max(fill, least), 1024);
  return (int)((r + 15) / 16 * 16);
}

struct Params {
  const void *weight, *bias;
  mluOpDataType_t type;
  bool wide;  // 16-byte loads of both

  template <typename T, int V>
  __device__ __forceinline__ void loadAs(const void *p, int c, float (&to)[V]) const {
    if (wide) {
      loadFloats<T, V>(static_cast<const T *>(p) + c, to);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) to[i] = (float)static_cast<const T *>(p)[c + i];
    }
  }
  template <int V>
  __device__ __forceinline__ void load(const void *p, int c, float none, float (&to)[V]) const {
    if (p == nullptr) {
#pragma unroll
      for (int i = 0; i < V; ++i) to[i] = none;
    } else if (type == MLUOP_DTYPE_FLOAT) {
      loadAs<float, V>(p, c, to);
    } else if (type == MLUOP_DTYPE_HALF) {
      loadAs<_Float16, V>(p, c, to);
    } else {
      loadAs<__bf16, V>(p, c, to);
    }
  }
  // A gradient of the parameters (nowhere where it is not wanted).
  __device__ __forceinline__ void store(void *to, int c, float v) const {
    if (to == nullptr) return;
    if (type == MLUOP_DTYPE_FLOAT)
      static_cast<float *>(to)[c] = v;
    else if (type == MLUOP_DTYPE_HALF)
      static_cast<_Float16 *>(to)[c] = (_Float16)v;
    else
      static_cast<__bf16 *>(to)[c] = (__bf16)v;
  }
  template <int V>
  __device__ __forceinline__ void weights(int c, float (&to)[V]) const {
    load<V>(weight, c, 1.f, to);
  }
  template <int V>
  __device__ __forceinline__ void biases(int c, float (&to)[V]) const {
    load<V>(bias, c, 0.f, to);
  }
};

// The groups of the channels c to c + V - 1 (one division: V of them are a third of what a small workgroup does).
template <int V>
__device__ __forceinline__ void groupsOf(int c, int per_group, int (&group)[V]) {
  int g = c / per_group, in_group = c - g * per_group;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    group[i] = g;
    const bool next = ++in_group == per_group;
    g += next ? 1 : 0;
    in_group = next ? 0 : in_group;
  }
}

template <int V>
using Lanes = RowLanes<V, kThreads>;

__device__ __forceinline__ float sigmoid(float z) {
  // (An exponential beyond the range is infinite, and its reciprocal zero.  The exponential's argument is rounded once more: SiLU is
  // off by up to 1.3 (1 + |z|) units of 2^-24 of itself below -5, where z's own rounding moves it by |z| / 2, and by 6 units
  // around zero; expf and a division have 3.)
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
// differences from the tile's first row, so that channels far off zero lose nothing.  Bound by memory: 248 636 x 128 fp16
// (64 MB) 12.6 us, 5.1 TB/s.
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
    for (int r0 = l.row; r0 < t.rows; r0 += kAhead * l.rows_at_once) {
      Vector<T, V> v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        // (behind the tile the first row again, which adds nothing)
        const int r = r0 + j * l.rows_at_once;
        v[j] = *reinterpret_cast<const Vector<T, V> *>(from + (int64_t)(r < t.rows ? r : 0) * s.channels);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = (float)v[j].v[i] - base[i];
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

// Mean and squared deviations of a group from its tiles' moments at `from`: the mean first, then the deviations from it.  By
// LANES lanes, number `lane` of them this; `all` adds up over them.
template <int LANES, typename ALL>
__device__ __forceinline__ void joinMoments(const float2 *from, const Shape &s, int tiles, int rows, int lane, ALL all,
                                            float *mean, float *squares, float *by, int lanes = LANES) {
  const int per_group = s.channels / s.groups, entries = tiles * per_group;
  auto rowsOf = [&](int tile) { return (float)min(s.tile_rows, rows - tile * s.tile_rows); };
  float sum = 0.f;
  for (int e0 = lane; e0 < entries; e0 += kAhead * lanes) {
    float v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int e = min(e0 + j * lanes, entries - 1), tile = e / per_group;
      v[j] = from[(int64_t)tile * s.channels + (e - tile * per_group)].x * rowsOf(tile);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) sum += e0 + j * lanes < entries ? v[j] : 0.f;
  }
  *by = rows > 0 ? 1.f / ((float)rows * (float)per_group) : 0.f;
  const float m = all(sum) * *by;
  sum = 0.f;
  for (int e0 = lane; e0 < entries; e0 += kAhead * lanes) {
    float v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int e = min(e0 + j * lanes, entries - 1), tile = e / per_group;
      const float2 p = from[(int64_t)tile * s.channels + (e - tile * per_group)];
      v[j] = fmaf((p.x - m) * (p.x - m), rowsOf(tile), p.y);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) sum += e0 + j * lanes < entries ? v[j] : 0.f;
  }
  *squares = all(sum);
  *mean = m;
}

// Mean and rstd of a (sample, group).
__global__ __launch_bounds__(kThreads) void groupNormJoinMoments(const float2 *__restrict__ partial, Shape s, float eps,
                                                                 float *__restrict__ mean, float *__restrict__ rstd) {
  const int sample = blockIdx.x / s.groups, group = blockIdx.x - sample * s.groups;
  int first, rows;
  const int tiles = raggedTilesOf(s.starts, s.rows, sample, s.tile_rows, s.most_tiles, &first, &rows);
  const float2 *from = partial + (int64_t)first * s.channels + group * (s.channels / s.groups);
  float m, squares, by;
  joinMoments<kThreads>(from, s, tiles, rows, threadIdx.x, [](float v) { return sumOfWorkgroup(v); }, &m, &squares, &by);
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = m;
    rstd[blockIdx.x] = 1.f / sqrtf(squares * by + eps);
  }
}

// JOINED: the moments are there.  Otherwise every workgroup joins those of its sample's tiles itself, a few lanes a group, and
// the first of a sample writes them down: few tiles, for which that costs less than a launch of its own.
// Bound by memory: 248 636 x 128 fp16 with SiLU, read and written (127 MB) 23.3 us, 5.5 TB/s.
template <typename T, int V, int ACT, bool JOINED>
__global__ __launch_bounds__(kThreads) void groupNormApply(const T *__restrict__ x, Shape s, Params p, float eps,
                                                           const float2 *__restrict__ partial, float *__restrict__ mean,
                                                           float *__restrict__ rstd, T *__restrict__ out) {
  const RaggedTile t = findRaggedTile<true>(s.starts, s.rows, s.samples, s.apply_rows, blockIdx.x);
  if (t.segment < 0) return;
  const bool inside = t.segment > 0 && t.segment <= s.samples;
  __shared__ float s_mean[JOINED ? 1 : kThreads], s_rstd[JOINED ? 1 : kThreads];
  if constexpr (!JOINED) {
    if (blockIdx.x == 0 && blockIdx.y == 0) {
      // (samples without rows have no workgroup of their own)
      for (int i = threadIdx.x; i < s.samples * s.groups; i += kThreads) {
        int first, rows;
        segmentRows(s.starts, s.rows, i / s.groups, &first, &rows);
        if (rows == 0) {
          mean[i] = 0.f;
          rstd[i] = 1.f / sqrtf(eps);
        }
      }
    }
    if (inside) {
      const int sample = t.segment - 1;
      int lanes = 64;
      while (lanes * s.groups > kThreads) lanes >>= 1;
      const int group = (int)threadIdx.x / lanes, lane = (int)threadIdx.x % lanes;
      int first, rows;
      const int tiles = raggedTilesOf(s.starts, s.rows, sample, s.tile_rows, s.most_tiles, &first, &rows);
      if (group < s.groups) {
        auto all = [&](float v) {
          for (int d = lanes >> 1; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
          return v;
        };
        float m, squares, by;
        joinMoments<64>(partial + (int64_t)first * s.channels + group * (s.channels / s.groups), s, tiles, rows, lane, all,
                        &m, &squares, &by, lanes);
        if (lane == 0) {
          s_mean[group] = m;
          s_rstd[group] = 1.f / sqrtf(squares * by + eps);
          if (t.in_segment == 0 && blockIdx.y == 0) {
            mean[sample * s.groups + group] = m;
            rstd[sample * s.groups + group] = s_rstd[group];
          }
        }
      }
    }
    __syncthreads();
  }
  const Lanes<V> l(s.channels);
  if (l.row < 0) return;
  float m[V] = {}, a[V] = {}, b[V] = {};
  if (inside) {
    int in_sample[V];
    groupsOf<V>(l.channel, s.channels / s.groups, in_sample);
    p.weights<V>(l.channel, a);
    p.biases<V>(l.channel, b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int g = (t.segment - 1) * s.groups + in_sample[i];
      m[i] = JOINED ? mean[g] : s_mean[in_sample[i]];
      a[i] *= JOINED ? rstd[g] : s_rstd[in_sample[i]];
    }
  }
  const int64_t at = (int64_t)t.first * s.channels + l.channel;
  for (int r0 = l.row; r0 < t.rows; r0 += kAhead * l.rows_at_once) {
    float v[kAhead][V] = {};
    if (inside) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int r = r0 + j * l.rows_at_once;
        loadFloats<T, V>(x + at + (int64_t)(r < t.rows ? r : r0) * s.channels, v[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int r = r0 + j * l.rows_at_once;
      if (r >= t.rows) break;
      if (inside) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = activated<ACT>(fmaf(v[j][i] - m[i], a[i], b[i]));
      }
      storeFloats<T, V>(out + at + (int64_t)r * s.channels, v[j], s.streamed);
    }
  }
}

// dz = dy * activation'(z) of V channels, and the normed values.
template <typename T, int V, int ACT>
__device__ __forceinline__ void gradOfNormed(const Vector<T, V> &dy, const Vector<T, V> &x, const float (&m)[V],
                                             const float (&r)[V], const float (&w)[V], const float (&b)[V],
                                             float (&dz)[V], float (&normed)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    dz[i] = (float)dy.v[i];
    normed[i] = ((float)x.v[i] - m[i]) * r[i];
    if (ACT != MLUOP_EXT_ACTIVATION_NONE) dz[i] *= slope<ACT>(fmaf(normed[i], w[i], b[i]));
  }
}

// A tile's sums of dz and dz * normed of every channel, to partial[tile][channel].  Bound by memory: two tensors of
// 400 000 x 128 bf16 (205 MB) 37 us, 5.5 TB/s.
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
    float m[V], r[V], w[V], b[V];
    int in_sample[V];
    groupsOf<V>(l.channel, s.channels / s.groups, in_sample);
    p.weights<V>(l.channel, w);
    p.biases<V>(l.channel, b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      m[i] = mean[t.segment * s.groups + in_sample[i]];
      r[i] = rstd[t.segment * s.groups + in_sample[i]];
    }
    const int64_t at = (int64_t)t.first * s.channels + l.channel;
    for (int r0 = l.row; r0 < t.rows; r0 += kGradAhead * l.rows_at_once) {
      Vector<T, V> dys[kGradAhead], xs[kGradAhead];
#pragma unroll
      for (int j = 0; j < kGradAhead; ++j) {
        const int row = r0 + j * l.rows_at_once;
        const int64_t from = at + (int64_t)(row < t.rows ? row : r0) * s.channels;
        dys[j] = *reinterpret_cast<const Vector<T, V> *>(dy + from);
        xs[j] = *reinterpret_cast<const Vector<T, V> *>(x + from);
      }
#pragma unroll
      for (int j = 0; j < kGradAhead; ++j) {
        if (r0 + j * l.rows_at_once >= t.rows) break;
        float dz[V], normed[V];
        gradOfNormed<T, V, ACT>(dys[j], xs[j], m, r, w, b, dz, normed);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          sum[i] += dz[i];
          with_normed[i] = fmaf(dz[i], normed[i], with_normed[i]);
        }
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

// The first samples * groups workgroups: the means of w dz and w dz * normed of a (sample, group).  The others: the
// gradients of the parameters of kChannels channels each, over all tiles.
constexpr int kChannels = 4;
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
    for (int e0 = threadIdx.x; e0 < entries; e0 += kAhead * kThreads) {
      float2 v[kAhead];
      float w[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int e = min(e0 + j * kThreads, entries - 1), tile = e / per_group, c = e - tile * per_group;
        v[j] = from[(int64_t)tile * s.channels + c];
        float one[1];
        p.weights<1>(group * per_group + c, one);
        w[j] = one[0];
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (e0 + j * kThreads >= entries) break;
        a = fmaf(v[j].x, w[j], a);
        b = fmaf(v[j].y, w[j], b);
      }
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
    constexpr int kShares = kThreads / kChannels;
    for (int t0 = share; t0 < tiles; t0 += kAhead * kShares) {
      float2 v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = partial[(int64_t)min(t0 + j * kShares, tiles - 1) * s.channels + c];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (t0 + j * kShares >= tiles) break;
        a += v[j].x;
        b += v[j].y;
      }
    }
  }
  s_sum[share][lane] = make_float2(a, b);
  __syncthreads();
  if (share != 0 || c >= s.channels) return;
  for (int i = 1; i < kThreads / kChannels; ++i) {
    a += s_sum[i][lane].x;
    b += s_sum[i][lane].y;
  }
  p.store(bias_grad, c, a);
  p.store(weight_grad, c, b);
}

// dx = rstd (w dz - mean of w dz - normed * mean of w dz normed).  Tiles from the last to the first: what the sums read last is
// still in the caches.  Bound by memory: 400 000 x 128 bf16 (307 MB) 49 us, 6.3 TB/s.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void groupNormGradApply(const T *__restrict__ dy, const T *__restrict__ x, Shape s,
                                                               Params p, const float *__restrict__ mean,
                                                               const float *__restrict__ rstd,
                                                               const float2 *__restrict__ means, T *__restrict__ dx) {
  const RaggedTile t = findRaggedTile<true>(s.starts, s.rows, s.samples, s.apply_rows, gridDim.x - 1 - blockIdx.x);
  if (t.segment < 0) return;
  const Lanes<V> l(s.channels);
  if (l.row < 0) return;
  const bool inside = t.segment > 0 && t.segment <= s.samples;
  float m[V] = {}, r[V] = {}, w[V] = {}, b[V] = {};
  float2 c[V] = {};
  if (inside) {
    int in_sample[V];
    groupsOf<V>(l.channel, s.channels / s.groups, in_sample);
    p.weights<V>(l.channel, w);
    p.biases<V>(l.channel, b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int g = (t.segment - 1) * s.groups + in_sample[i];
      m[i] = mean[g];
      r[i] = rstd[g];
      c[i] = means[g];
    }
  }
  const int64_t at = (int64_t)t.first * s.channels + l.channel;
  for (int r0 = l.row; r0 < t.rows; r0 += kGradAhead * l.rows_at_once) {
    Vector<T, V> dys[kGradAhead], xs[kGradAhead];
    if (inside) {
#pragma unroll
      for (int j = 0; j < kGradAhead; ++j) {
        const int row = r0 + j * l.rows_at_once;
        const int64_t from = at + (int64_t)(row < t.rows ? row : r0) * s.channels;
        dys[j] = *reinterpret_cast<const Vector<T, V> *>(dy + from);
        xs[j] = *reinterpret_cast<const Vector<T, V> *>(x + from);
      }
    }
#pragma unroll
    for (int j = 0; j < kGradAhead; ++j) {
      const int row = r0 + j * l.rows_at_once;
      if (row >= t.rows) break;
      float d[V] = {};
      if (inside) {
        float dz[V], normed[V];
        gradOfNormed<T, V, ACT>(dys[j], xs[j], m, r, w, b, dz, normed);
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = r[i] * (fmaf(dz[i], w[i], -c[i].x) - normed[i] * c[i].y);
      }
      storeFloats<T, V>(dx + at + (int64_t)row * s.channels, d, s.streamed);
    }
  }
}

// ---- few rows ------------------------------------------------------------------------------
//
// One launch, in which a workgroup keeps a sample's rows of `columns` * V channels, whole groups, in registers: it reads them
// once, takes the mean, then the squares of the differences from it, and writes the results.  All lanes of a wave have
// the same V channels of rows of their own.  Bound by what a launch and a few barriers take.  us in two or three launches /
// in one, forward and gradients: 1000 x 64 fp16 in 16 groups 11.1 / 6.6 and 12.8 / 7.9, 4096 rows 11.2 / 9.5 and 13.1 / 12.7,
// 1000 x 16 fp32 in one group 11.2 / 6.5 and 12.2 / 11.0.  From the rows on that no longer fit there is nothing to choose.

constexpr int kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64;
constexpr int kSmallRows = 4;         // of a thread
constexpr int kSmallGradSamples = 4;  // taken one after the other
constexpr int64_t kMostAlongY = 65535;  // workgroups of a grid

// Sum over the lanes, in lane 63.
__device__ __forceinline__ float waveSumAtLast(float v) {
#define MLUOP_ADD_MOVED(ctrl, rows) \
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, rows, 0xf, false));
  MLUOP_ADD_MOVED(0x111, 0xf)  // within rows of 16 lanes: from 1, 2, 4 and 8 lanes below
  MLUOP_ADD_MOVED(0x112, 0xf)
  MLUOP_ADD_MOVED(0x114, 0xf)
  MLUOP_ADD_MOVED(0x118, 0xf)
  MLUOP_ADD_MOVED(0x142, 0xa)  // and from row to row
  MLUOP_ADD_MOVED(0x143, 0xc)
#undef MLUOP_ADD_MOVED
  return v;
}

template <int V>
struct SmallLanes {
  int columns, column, wave, lane;
  int channel;       // first of this thread's
  int in_slab;       // the same, within the workgroup's
  int row, at_once;  // the thread's first row, rows of the workgroup at once
  __device__ explicit SmallLanes(int c) : columns(c) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    column = wave % columns;
    in_slab = column * V;
    channel = ((int)blockIdx.x * columns + column) * V;
    at_once = kSmallWaves / columns * 64;
    row = wave / columns * 64 + lane;
  }
  // Sums of every channel of the slab over the workgroup's rows, to `sums`.  By the whole workgroup.
  __device__ __forceinline__ void sumRows(const float (&v)[V], float *sums) const {
    __shared__ float s_wave[kSmallWaves][V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float sum = waveSumAtLast(v[i]);
      if (lane == 63) s_wave[wave][i] = sum;
    }
    __syncthreads();
    const int c = threadIdx.x;
    if (c < columns * V) {
      float sum = 0.f;
      for (int w = c / V; w < kSmallWaves; w += columns) sum += s_wave[w][c % V];
      sums[c] = sum;
    }
    __syncthreads();
  }
};

// Zeros in the rows that belong to no sample, by the workgroups of the first and the last.
template <typename T, int V>
__device__ __forceinline__ void smallOutside(const SmallLanes<V> &l, const Shape &s, int sample, T *out) {
  const float zero[V] = {};
  for (int side = 0; side < 2; ++side) {
    if (sample != (side == 0 ? 0 : s.samples - 1)) continue;
    int first, rows;
    segmentOrOutside(s.starts, s.rows, s.samples, side == 0 ? 0 : s.samples + 1, &first, &rows);
    for (int r = l.row; r < rows; r += l.at_once) storeFloats<T, V>(out + (int64_t)(first + r) * s.channels + l.channel, zero);
  }
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(kSmallThreads) void groupNormSmall(const T *__restrict__ x, Shape s, Params p, float eps,
                                                                int columns, int first_sample, float *__restrict__ mean,
                                                                float *__restrict__ rstd, T *__restrict__ out) {
  __shared__ float s_sum[kSmallWaves * V], s_mean[kSmallWaves * V], s_rstd[kSmallWaves * V];
  const SmallLanes<V> l(columns);
  const int sample = first_sample + blockIdx.y, per_group = s.channels / s.groups, slab = columns * V;
  int first, rows;
  segmentRows(s.starts, s.rows, sample, &first, &rows);
  const int64_t at = (int64_t)first * s.channels + l.channel;
  Vector<T, V> v[kSmallRows];
  float sum[V] = {};
#pragma unroll
  for (int j = 0; j < kSmallRows; ++j) {
    const int r = l.row + j * l.at_once;
    v[j] = {};
    if (r < rows) v[j] = *reinterpret_cast<const Vector<T, V> *>(x + at + (int64_t)r * s.channels);
  }
  float w[V], b[V];
  int group[V];
  p.weights<V>(l.channel, w);
  p.biases<V>(l.channel, b);
  groupsOf<V>(l.in_slab, per_group, group);
#pragma unroll
  for (int j = 0; j < kSmallRows; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] += (float)v[j].v[i];
  const float by = rows > 0 ? 1.f / ((float)rows * (float)per_group) : 0.f;
  // a group's sum, from those of its channels
  auto join = [&](int g) {
    float all = 0.f;
    for (int c = g * per_group; c < (g + 1) * per_group; ++c) all += s_sum[c];
    return all;
  };
  const int groups = slab / per_group;
  l.sumRows(sum, s_sum);
  if ((int)threadIdx.x < groups) s_mean[threadIdx.x] = join(threadIdx.x) * by;
  __syncthreads();
  float m[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    m[i] = s_mean[group[i]];
    sum[i] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < kSmallRows; ++j) {
    const bool there = l.row + j * l.at_once < rows;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = there ? (float)v[j].v[i] - m[i] : 0.f;
      sum[i] = fmaf(d, d, sum[i]);
    }
  }
  l.sumRows(sum, s_sum);
  if ((int)threadIdx.x < groups) {
    const float r = 1.f / sqrtf(join(threadIdx.x) * by + eps);
    s_rstd[threadIdx.x] = r;
    const int g = sample * s.groups + (int)blockIdx.x * groups + (int)threadIdx.x;
    mean[g] = s_mean[threadIdx.x];
    rstd[g] = r;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] *= s_rstd[group[i]];
#pragma unroll
  for (int j = 0; j < kSmallRows; ++j) {
    const int r = l.row + j * l.at_once;
    if (r >= rows) continue;
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = activated<ACT>(fmaf((float)v[j].v[i] - m[i], w[i], b[i]));
    storeFloats<T, V>(out + at + (int64_t)r * s.channels, z);
  }
  smallOutside<T, V>(l, s, sample, out);
}

// The gradients in one launch, sample after sample: a workgroup has all rows of its channels, and so the gradients of their
// parameters.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(kSmallThreads) void groupNormSmallGrad(const T *__restrict__ dy, const T *__restrict__ x, Shape s,
                                                                    Params p, int columns, const float *__restrict__ mean,
                                                                    const float *__restrict__ rstd, T *__restrict__ dx,
                                                                    void *weight_grad, void *bias_grad) {
  __shared__ float s_dz[kSmallWaves * V], s_with[kSmallWaves * V], s_weight[kSmallWaves * V];
  __shared__ float2 s_means[kSmallWaves * V];
  const SmallLanes<V> l(columns);
  const int per_group = s.channels / s.groups, slab = columns * V, groups = slab / per_group;
  float w[V], b[V];
  int group[V];
  p.weights<V>(l.channel, w);
  p.biases<V>(l.channel, b);
  groupsOf<V>(l.in_slab, per_group, group);
  if (l.lane == 0 && l.wave < columns) {
#pragma unroll
    for (int i = 0; i < V; ++i) s_weight[l.in_slab + i] = w[i];
  }
  float dw = 0.f, db = 0.f;  // of channel threadIdx.x of the slab
  for (int sample = 0; sample < s.samples; ++sample) {
    int first, rows;
    segmentRows(s.starts, s.rows, sample, &first, &rows);
    const int64_t at = (int64_t)first * s.channels + l.channel;
    Vector<T, V> dys[kSmallRows], xs[kSmallRows];
#pragma unroll
    for (int j = 0; j < kSmallRows; ++j) {
      const int r = l.row + j * l.at_once;
      dys[j] = xs[j] = {};
      if (r < rows) {
        dys[j] = *reinterpret_cast<const Vector<T, V> *>(dy + at + (int64_t)r * s.channels);
        xs[j] = *reinterpret_cast<const Vector<T, V> *>(x + at + (int64_t)r * s.channels);
      }
    }
    float m[V], rs[V], sum[V] = {}, with[V] = {};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int g = sample * s.groups + (int)blockIdx.x * groups + group[i];
      m[i] = mean[g];
      rs[i] = rstd[g];
    }
#pragma unroll
    for (int j = 0; j < kSmallRows; ++j) {
      if (l.row + j * l.at_once >= rows) continue;
      float dz[V], normed[V];
      gradOfNormed<T, V, ACT>(dys[j], xs[j], m, rs, w, b, dz, normed);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        sum[i] += dz[i];
        with[i] = fmaf(dz[i], normed[i], with[i]);
      }
    }
    l.sumRows(sum, s_dz);
    l.sumRows(with, s_with);
    const float by = rows > 0 ? 1.f / ((float)rows * (float)per_group) : 0.f;
    if ((int)threadIdx.x < slab) {
      db += s_dz[threadIdx.x];
      dw += s_with[threadIdx.x];
    }
    if ((int)threadIdx.x < groups) {
      float a = 0.f, c = 0.f;
      for (int i = threadIdx.x * per_group; i < ((int)threadIdx.x + 1) * per_group; ++i) {
        a = fmaf(s_dz[i], s_weight[i], a);
        c = fmaf(s_with[i], s_weight[i], c);
      }
      s_means[threadIdx.x] = make_float2(a * by, c * by);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSmallRows; ++j) {
      const int r = l.row + j * l.at_once;
      if (r >= rows) continue;
      float dz[V], normed[V];
      gradOfNormed<T, V, ACT>(dys[j], xs[j], m, rs, w, b, dz, normed);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 c = s_means[group[i]];
        dz[i] = rs[i] * (fmaf(dz[i], w[i], -c.x) - normed[i] * c.y);
      }
      storeFloats<T, V>(dx + at + (int64_t)r * s.channels, dz);
    }
    __syncthreads();
  }
  smallOutside<T, V>(l, s, 0, dx);
  if (s.samples > 1) smallOutside<T, V>(l, s, s.samples - 1, dx);
  const int c = (int)blockIdx.x * slab + (int)threadIdx.x;
  if ((int)threadIdx.x < slab) {
    p.store(bias_grad, c, db);
    p.store(weight_grad, c, dw);
  }
}

// ---- host side -----------------------------------------------------------------------------

size_t partialBytes(int64_t rows, int64_t channels, int64_t samples) {
  return (size_t)mostRaggedTiles(rows, samples, tileRows(rows, channels)) * channels * sizeof(float2);
}

// Whether the pass that applies joins the moments itself: each of its workgroups then reads those of a sample's tiles, of
// no more than a few KB.  us in three launches / in two: 20 000 x 16 fp32 in two samples 11.2 / 10.0, 20 000 x 32 bf16 in 16
// 12.5 / 10.7.
bool joinedByApply(const Shape &s) {
  return s.rows > 0 && s.samples <= 64 && s.groups <= kThreads && (int64_t)s.most_tiles * s.channels <= 4096;
}

// Threads' columns of the kernels of few rows, 0: they do not take this.  Their workgroups hold whole groups: V channels of
// several, or one of up to 16 V.
int smallColumns(const Shape &s, int v) {
  const int per_group = s.channels / s.groups;
  const int columns = v % per_group == 0 ? 1 : (per_group % v == 0 ? per_group / v : 0);
  if (columns == 0 || columns > kSmallWaves || kSmallWaves % columns != 0) return 0;
  return s.rows <= kSmallRows * (kSmallThreads / columns) ? columns : 0;
}

constexpr int64_t kMostPairs = 15 << 20;

mluOpStatus_t checkShape(const char *api, int64_t rows, int64_t channels, int64_t groups, int64_t samples) {
  PARAM_CHECK(api, rows >= 0);
  PARAM_CHECK(api, channels > 0);
  PARAM_CHECK(api, groups > 0);
  PARAM_CHECK(api, channels % groups == 0);
  PARAM_CHECK(api, samples > 0);
  // (a pair, and four channels, have a workgroup each, in one launch)
  static_assert(kMostPairs + (1 << 20) / kChannels <= mostBlocks(kThreads), "a grid's threads");
  if (rows > INT32_MAX - 4096 || channels > (1 << 20) || samples > (1 << 20) || samples * groups > kMostPairs ||
      rows * channels > ((int64_t)1 << 46)) {
    MLUOP_LOG(ERROR) << api << " At most 2^31 - 4097 rows, 2^20 channels, 2^20 samples, 15 * 2^20 pairs of a sample and a "
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
                   (int)mostRaggedTiles(rows, samples, tileRows(rows, channels)), applyRows(rows, channels), row_starts,
                   (size_t)rows * channels * elementBytes(type) >= kStreamedBytes};
  const Params p = {weight, bias, param_type, alignedTo(weight, 16) && alignedTo(bias, 16)};
  const Workspace w = carve(workspace, rows, channels, samples);
  const mluop::LaunchCtx lc = handle->launchCtx();
  byType(type, s.channels, reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(out), [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    const unsigned slabs = (unsigned)((s.channels / V + kThreads - 1) / kThreads);
    constexpr int W = V < 4 ? V : 4;  // (eight channels a lane: twice the sums over its waves in half as many workgroups)
    const int columns = smallColumns(s, W);
    if (columns > 0) {
      byActivation(activation, [&](auto act) {
        for (int64_t first = 0; first < samples; first += kMostAlongY) {
          const unsigned count = (unsigned)std::min(samples - first, kMostAlongY);
          lc.begin("groupNormSmall");
          groupNormSmall<T, W, decltype(act)::value><<<dim3(s.channels / (columns * W), count), kSmallThreads, 0, lc.stream>>>(
              static_cast<const T *>(features), s, p, eps, columns, (int)first, mean, rstd, static_cast<T *>(out));
          lc.end();
        }
      });
      return;
    }
    const unsigned tiles = (unsigned)mostRaggedTiles(rows, samples, s.tile_rows);
    if (tiles > 0) {
      lc.begin("groupNormMoments");
      groupNormMoments<T, V><<<dim3(tiles, slabs), kThreads, 0, lc.stream>>>(static_cast<const T *>(features), s, w.partial);
      lc.end();
    }
    const bool joined = !joinedByApply(s);
    if (joined) {
      lc.begin("groupNormJoinMoments");
      groupNormJoinMoments<<<(unsigned)(samples * groups), kThreads, 0, lc.stream>>>(w.partial, s, eps, mean, rstd);
      lc.end();
    }
    const unsigned all = (unsigned)mostRaggedTiles(rows, samples + 2, s.apply_rows);
    if (all == 0) return;
    byActivation(activation, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      auto kernel = joined ? groupNormApply<T, V, ACT, true> : groupNormApply<T, V, ACT, false>;
      lc.begin("groupNormApply");
      kernel<<<dim3(all, slabs), kThreads, 0, lc.stream>>>(static_cast<const T *>(features), s, p, eps, w.partial, mean,
                                                           rstd, static_cast<T *>(out));
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
                   (int)mostRaggedTiles(rows, samples, tileRows(rows, channels)), applyRows(rows, channels), row_starts,
                   (size_t)rows * channels * elementBytes(type) >= kStreamedBytes};
  const Params p = {weight, bias, param_type, alignedTo(weight, 16) && alignedTo(bias, 16)};
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
      constexpr int W = V < 4 ? V : 4;
      const int columns = samples <= kSmallGradSamples ? smallColumns(s, W) : 0;
      if (columns > 0) {
        lc.begin("groupNormSmallGrad");
        groupNormSmallGrad<T, W, ACT><<<s.channels / (columns * W), kSmallThreads, 0, lc.stream>>>(
            dy, x, s, p, columns, mean, rstd, static_cast<T *>(input_grad), weight_grad, bias_grad);
        lc.end();
        return;
      }
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
      const unsigned all = (unsigned)mostRaggedTiles(rows, samples + 2, s.apply_rows);
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
