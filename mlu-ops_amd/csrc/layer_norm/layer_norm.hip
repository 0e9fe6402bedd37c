// mluOpExtLayerNormForward / Backward (no counterpart in the reference): every row normed over its channels.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "core/channel_params.h"
#include "core/core.h"
#include "core/elements.h"
#include "core/lane_sum.h"
#include "mlu_op_ext.h"

namespace {

using namespace mluop;

constexpr int kThreads = 256;
constexpr int kMostChannels = 1 << 15;

// The problem as its kernels see it.
struct Shape {
  int64_t rows;
  int channels;
  int64_t x_stride, dy_stride;  // elements from row to row; results lie row by row
  bool streamed;                // results go past the caches
};

// A row is read once and kept in the registers of its team: LANES lanes of a wave, or a workgroup of LANES threads, N vectors of
// V channels each, lane after lane.
template <int V, int LANES, int N>
struct Team {
  static constexpr int kWorkgroup = LANES > kThreads ? LANES : kThreads;
  static constexpr int kTeams = kWorkgroup / LANES;  // of a workgroup
  int lane, team;
  __device__ Team() : lane((int)threadIdx.x % LANES), team((int)threadIdx.x / LANES) {}
  __device__ __forceinline__ int channel(int n) const { return (lane + n * LANES) * V; }

  // Sums over the team, in all its threads.  By whole workgroups.
  template <int COUNT>
  __device__ __forceinline__ void sum(float (&v)[COUNT]) const {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = sumOverLanes<(LANES < 64 ? LANES : 64)>(v[i]);
    if constexpr (LANES > 64) {
      constexpr int kWaves = LANES / 64;
      __shared__ float s_wave[kWaves][COUNT];
      __syncthreads();
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) s_wave[threadIdx.x >> 6][i] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < COUNT; ++i) {
        v[i] = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v[i] += s_wave[w][i];
      }
    }
  }
};

// ---- forward -------------------------------------------------------------------------------

// y = (x - mean) * rstd * weight + bias.  The mean is the sum's, put right by the mean of the differences from it, so that rows far
// off zero lose nothing; the variance is that of the differences.  R rows of a team are on their way together.
template <typename T, int V, int LANES, int N, int R>
__global__ __launch_bounds__((Team<V, LANES, N>::kWorkgroup)) void layerNormRows(const T *__restrict__ x, Shape s,
                                                                                ChannelParams p, float eps,
                                                                                T *__restrict__ out,
                                                                                float *__restrict__ mean,
                                                                                float *__restrict__ rstd) {
  typedef Team<V, LANES, N> Lanes;
  const Lanes l;
  float w[N][V] = {}, b[N][V] = {};
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = l.channel(n);
    if (c < s.channels) {
      p.weights<V>(c, w[n]);
      p.biases<V>(c, b[n]);
    }
  }
  const float by = 1.f / (float)s.channels;
  const int64_t step = (int64_t)gridDim.x * Lanes::kTeams;
  // (all teams of a workgroup take as many turns: sums are taken by whole waves)
  for (int64_t first = (int64_t)blockIdx.x * Lanes::kTeams; first < s.rows; first += R * step) {
    Vector<T, V> v[R][N];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int64_t r = first + l.team + j * step;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        v[j][n] = {};
        if (r < s.rows && l.channel(n) < s.channels)
          v[j][n] = *reinterpret_cast<const Vector<T, V> *>(x + r * s.x_stride + l.channel(n));
      }
    }
    float m[R], moments[2 * R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      m[j] = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < V; ++i) m[j] += (float)v[j][n].v[i];
    }
    l.sum(m);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      m[j] *= by;
      float sum = 0.f, squares = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const bool there = l.channel(n) < s.channels;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = there ? (float)v[j][n].v[i] - m[j] : 0.f;
          sum += d;
          squares = fmaf(d, d, squares);
        }
      }
      moments[2 * j] = sum;
      moments[2 * j + 1] = squares;
    }
    l.sum(moments);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int64_t r = first + l.team + j * step;
      const float off = moments[2 * j] * by;
      const float variance = fmaf(-off, off, moments[2 * j + 1] * by);
      const float inv = 1.f / sqrtf((variance < 0.f ? 0.f : variance) + eps);  // (NaN stays NaN)
      if (r >= s.rows) continue;
      if (l.lane == 0) {
        mean[r] = m[j] + off;
        rstd[r] = inv;
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (l.channel(n) >= s.channels) continue;
        float y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = fmaf(((float)v[j][n].v[i] - m[j] - off) * inv, w[n][i], b[n][i]);
        storeFloats<T, V>(out + r * s.channels + l.channel(n), y, s.streamed);
      }
    }
  }
}

// ---- backward ------------------------------------------------------------------------------

// dx = rstd (d - mean of d - normed * mean of d normed) with d = dy * weight, and with SUMS a workgroup's sums of dy * normed
// and dy of every channel over its rows, to partial[workgroup][2][channels].  A team's lanes have the same channels in
// every row, so that these stay in registers until the last row.
template <typename T, int V, int LANES, int N, int R, bool SUMS>
__global__ __launch_bounds__((Team<V, LANES, N>::kWorkgroup)) void layerNormGrad(const T *__restrict__ dy,
                                                                                const T *__restrict__ x, Shape s,
                                                                                ChannelParams p,
                                                                                const float *__restrict__ mean,
                                                                                const float *__restrict__ rstd,
                                                                                T *__restrict__ dx,
                                                                                float *__restrict__ partial) {
  typedef Team<V, LANES, N> Lanes;
  const Lanes l;
  float w[N][V] = {}, dw[SUMS ? N : 1][V] = {}, db[SUMS ? N : 1][V] = {};
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (l.channel(n) < s.channels) p.weights<V>(l.channel(n), w[n]);
  const float by = 1.f / (float)s.channels;
  const int64_t step = (int64_t)gridDim.x * Lanes::kTeams;
  for (int64_t first = (int64_t)blockIdx.x * Lanes::kTeams; first < s.rows; first += R * step) {
    Vector<T, V> dys[R][N], xs[R][N];
    float m[R], inv[R], sums[2 * R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int64_t r = first + l.team + j * step;
      m[j] = inv[j] = 0.f;
      if (r < s.rows) {
        m[j] = mean[r];
        inv[j] = rstd[r];
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        dys[j][n] = xs[j][n] = {};
        if (r < s.rows && l.channel(n) < s.channels) {
          dys[j][n] = *reinterpret_cast<const Vector<T, V> *>(dy + r * s.dy_stride + l.channel(n));
          xs[j][n] = *reinterpret_cast<const Vector<T, V> *>(x + r * s.x_stride + l.channel(n));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool row = first + l.team + j * step < s.rows;
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (!row || l.channel(n) >= s.channels) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float g = (float)dys[j][n].v[i], normed = ((float)xs[j][n].v[i] - m[j]) * inv[j], d = g * w[n][i];
          a += d;
          b = fmaf(d, normed, b);
          if constexpr (SUMS) {
            dw[n][i] = fmaf(g, normed, dw[n][i]);
            db[n][i] += g;
          }
        }
      }
      sums[2 * j] = a;
      sums[2 * j + 1] = b;
    }
    l.sum(sums);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int64_t r = first + l.team + j * step;
      const float a = sums[2 * j] * by, b = sums[2 * j + 1] * by;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (r >= s.rows || l.channel(n) >= s.channels) continue;
        float d[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float normed = ((float)xs[j][n].v[i] - m[j]) * inv[j];
          d[i] = inv[j] * (fmaf((float)dys[j][n].v[i], w[n][i], -a) - normed * b);
        }
        storeFloats<T, V>(dx + r * s.channels + l.channel(n), d, s.streamed);
      }
    }
  }
  if constexpr (SUMS) {
    // teams' sums of a vector of channels after the other's
    __shared__ float s_sum[Lanes::kWorkgroup * V];
    float *to = partial + (int64_t)blockIdx.x * 2 * s.channels;
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        if constexpr (Lanes::kTeams > 1) {
          __syncthreads();
#pragma unroll
          for (int i = 0; i < V; ++i) s_sum[threadIdx.x * V + i] = which == 0 ? dw[n][i] : db[n][i];
          __syncthreads();
          for (int e = threadIdx.x; e < LANES * V; e += Lanes::kWorkgroup) {
            float sum = 0.f;
#pragma unroll 8
            for (int t = 0; t < Lanes::kTeams; ++t) sum += s_sum[t * LANES * V + e];
            const int c = n * LANES * V + e;
            if (c < s.channels) to[which * s.channels + c] = sum;
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (l.channel(n) < s.channels) to[which * s.channels + l.channel(n) + i] = which == 0 ? dw[n][i] : db[n][i];
        }
      }
    }
  }
}

// The same sums of rows too wide for registers: a thread has one channel of every slice of rows.
template <typename T>
__global__ __launch_bounds__(kThreads) void layerNormColumnSums(const T *__restrict__ dy, const T *__restrict__ x, Shape s,
                                                                const float *__restrict__ mean,
                                                                const float *__restrict__ rstd,
                                                                float *__restrict__ partial) {
  const int c = (int)blockIdx.y * kThreads + (int)threadIdx.x;
  if (c >= s.channels) return;
  float dw = 0.f, db = 0.f;
#pragma unroll 4
  for (int64_t r = blockIdx.x; r < s.rows; r += gridDim.x) {
    const float g = (float)dy[r * s.dy_stride + c];
    dw = fmaf(g, ((float)x[r * s.x_stride + c] - mean[r]) * rstd[r], dw);
    db += g;
  }
  float *to = partial + (int64_t)blockIdx.x * 2 * s.channels;
  to[c] = dw;
  to[s.channels + c] = db;
}

// partial[parts][2][channels] added up: kChannels sums a workgroup, each by kThreads / kChannels threads.
constexpr int kChannels = 16, kAhead = 4;
__global__ __launch_bounds__(kThreads) void layerNormJoinSums(const float *__restrict__ partial, int parts, int channels,
                                                              ChannelParams p, void *weight_grad, void *bias_grad) {
  constexpr int kShares = kThreads / kChannels;
  __shared__ float s_sum[kShares][kChannels];
  const int lane = threadIdx.x % kChannels, share = threadIdx.x / kChannels;
  const int at = (int)blockIdx.x * kChannels + lane;
  float sum = 0.f;
  if (at < 2 * channels) {
    for (int t0 = share; t0 < parts; t0 += kAhead * kShares) {
      float v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = partial[(int64_t)min(t0 + j * kShares, parts - 1) * 2 * channels + at];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) sum += t0 + j * kShares < parts ? v[j] : 0.f;
    }
  }
  s_sum[share][lane] = sum;
  __syncthreads();
  if (share != 0 || at >= 2 * channels) return;
#pragma unroll
  for (int i = 1; i < kShares; ++i) sum += s_sum[i][lane];
  if (at < channels)
    p.store(weight_grad, at, sum);
  else
    p.store(bias_grad, at - channels, sum);
}

// ---- host side -----------------------------------------------------------------------------

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

// Calls f(LANES, N): the smallest team that holds a row of `vectors` vectors.
template <typename F>
void byTeam(int64_t vectors, F f) {
  auto one = std::integral_constant<int, 1>();
  if (vectors <= 8)
    f(std::integral_constant<int, 8>(), one);
  else if (vectors <= 16)
    f(std::integral_constant<int, 16>(), one);
  else if (vectors <= 32)
    f(std::integral_constant<int, 32>(), one);
  else if (vectors <= 64)
    f(std::integral_constant<int, 64>(), one);
  else if (vectors <= 128)
    f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
  else if (vectors <= 256)
    f(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
  else
    f(std::integral_constant<int, 256>(), std::integral_constant<int, 4>());
}
constexpr int kTeamVectors = 1024;  // that byTeam's largest holds
constexpr int kWideThreads = 1024;  // of a workgroup that holds a row of up to kMostChannels

constexpr int kSumParts = 512;      // most rows of partial sums

mluOpStatus_t checkShape(const char *api, int64_t rows, int64_t channels) {
  PARAM_CHECK(api, rows >= 0);
  PARAM_CHECK(api, channels > 0);
  if (channels > kMostChannels || rows > ((int64_t)1 << 46) / channels) {
    MLUOP_LOG(ERROR) << api << " At most 2^15 channels and 2^46 values are supported.";
    return MLUOP_STATUS_NOT_SUPPORTED;
  }
  return MLUOP_STATUS_SUCCESS;
}

bool strideFits(int64_t rows, int64_t channels, int64_t stride) {
  return stride >= channels && (rows == 0 || stride <= ((int64_t)1 << 46) / rows);
}

size_t workspaceBytes(int64_t channels) { return 16 + (size_t)kSumParts * 2 * channels * sizeof(float); }

}  // namespace

mluOpStatus_t MLUOP_WIN_API mluOpExtLayerNormForward(mluOpHandle_t handle, mluOpDataType_t type, const void *features,
                                                     int64_t features_stride, int64_t rows, int64_t channels,
                                                     mluOpDataType_t param_type, const void *weight, const void *bias,
                                                     float eps, void *out, float *mean, float *rstd) {
  const char *api = "[mluOpExtLayerNormForward]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  PARAM_CHECK(api, param_type == type || param_type == MLUOP_DTYPE_FLOAT);
  const mluOpStatus_t status = checkShape(api, rows, channels);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, strideFits(rows, channels, features_stride));
  PARAM_CHECK(api, eps >= 0.f && std::isfinite(eps));
  PARAM_CHECK(api, rows == 0 || (features != NULL && out != NULL && mean != NULL && rstd != NULL));
  DEVICE_HANDLE_CHECK(api, handle);
  if (rows == 0) return MLUOP_STATUS_SUCCESS;
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  const size_t bytes = (size_t)rows * channels * elementBytes(type);
  if (handle->hasNotes()) {
    handle->forgetNotesIn(out, bytes);
    handle->forgetNotesIn(mean, (size_t)rows * sizeof(float));
    handle->forgetNotesIn(rstd, (size_t)rows * sizeof(float));
  }
  const Shape s = {rows, (int)channels, features_stride, 0, bytes >= kStreamedBytes};
  const ChannelParams p = {weight, bias, param_type, alignedTo(weight, 16) && alignedTo(bias, 16)};
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(out);
  byType(type, channels, features_stride, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    auto launch = [&](auto lanes, auto vectors) {
      constexpr int LANES = decltype(lanes)::value, N = decltype(vectors)::value;
      typedef Team<V, LANES, N> L;
      constexpr int R = LANES > 64 ? 1 : 4 / N;
      // (weight and bias stay in registers: workgroups for all CUs to hold, and rows for each)
      const int64_t blocks = (rows + L::kTeams * R - 1) / (L::kTeams * R);
      const unsigned grid = (unsigned)std::min<int64_t>(blocks, LANES > kThreads ? 512 : 2048);
      lc.begin("layerNormRows");
      layerNormRows<T, V, LANES, N, R><<<grid, L::kWorkgroup, 0, lc.stream>>>(
          static_cast<const T *>(features), s, p, eps, static_cast<T *>(out), mean, rstd);
      lc.end();
    };
    if (channels / V <= kTeamVectors)
      byTeam(channels / V, launch);
    else
      launch(std::integral_constant<int, kWideThreads>(), std::integral_constant<int, kMostChannels / kWideThreads / V>());
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtGetLayerNormBackwardWorkspaceSize(int64_t rows, int64_t channels, size_t *size) {
  const char *api = "[mluOpExtGetLayerNormBackwardWorkspaceSize]";
  PARAM_CHECK(api, size != NULL);
  const mluOpStatus_t status = checkShape(api, rows, channels);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  *size = workspaceBytes(channels);
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtLayerNormBackward(mluOpHandle_t handle, mluOpDataType_t type, const void *output_grad,
                                                      int64_t output_grad_stride, const void *features,
                                                      int64_t features_stride, int64_t rows, int64_t channels,
                                                      mluOpDataType_t param_type, const void *weight, const float *mean,
                                                      const float *rstd, void *workspace, size_t workspace_size,
                                                      void *input_grad, void *weight_grad, void *bias_grad) {
  const char *api = "[mluOpExtLayerNormBackward]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  PARAM_CHECK(api, param_type == type || param_type == MLUOP_DTYPE_FLOAT);
  const mluOpStatus_t status = checkShape(api, rows, channels);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, strideFits(rows, channels, output_grad_stride) && strideFits(rows, channels, features_stride));
  PARAM_CHECK(api, rows == 0 || (output_grad != NULL && features != NULL && input_grad != NULL));
  PARAM_CHECK(api, rows == 0 || (mean != NULL && rstd != NULL));
  PARAM_CHECK(api, workspace != NULL);
  PARAM_CHECK(api, workspace_size >= workspaceBytes(channels));
  DEVICE_HANDLE_CHECK(api, handle);
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  const size_t bytes = (size_t)rows * channels * elementBytes(type);
  if (handle->hasNotes()) {
    handle->forgetNotesIn(input_grad, bytes);
    if (weight_grad) handle->forgetNotesIn(weight_grad, (size_t)channels * elementBytes(param_type));
    if (bias_grad) handle->forgetNotesIn(bias_grad, (size_t)channels * elementBytes(param_type));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  const bool sums = weight_grad != nullptr || bias_grad != nullptr;
  const Shape s = {rows, (int)channels, features_stride, output_grad_stride, bytes >= kStreamedBytes};
  const ChannelParams p = {weight, nullptr, param_type, alignedTo(weight, 16)};
  // (the caller's memory need not be aligned)
  float *partial = reinterpret_cast<float *>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~(uintptr_t)15);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(output_grad) |
                              reinterpret_cast<uintptr_t>(input_grad);
  int parts = 0;
  if (rows > 0) {
    byType(type, channels, features_stride | output_grad_stride, addresses, [&](auto zero, auto v) {
      typedef decltype(zero) T;
      constexpr int V = decltype(v)::value;
      const T *dy = static_cast<const T *>(output_grad), *x = static_cast<const T *>(features);
      T *dx = static_cast<T *>(input_grad);
      if (channels / V <= kTeamVectors) {
        byTeam(channels / V, [&](auto lanes, auto vectors) {
          constexpr int LANES = decltype(lanes)::value, N = decltype(vectors)::value;
          typedef Team<V, LANES, N> L;
          constexpr int R = LANES > 64 || N > 1 ? 1 : 2;
          const int64_t blocks = (rows + L::kTeams * R - 1) / (L::kTeams * R);
          parts = (int)std::min<int64_t>(blocks, kSumParts);
          lc.begin("layerNormGrad");
          if (sums)
            layerNormGrad<T, V, LANES, N, R, true><<<(unsigned)parts, L::kWorkgroup, 0, lc.stream>>>(dy, x, s, p, mean, rstd,
                                                                                                     dx, partial);
          else
            layerNormGrad<T, V, LANES, N, R, false><<<(unsigned)std::min<int64_t>(blocks, 2048), L::kWorkgroup, 0, lc.stream>>>(
                dy, x, s, p, mean, rstd, dx, nullptr);
          lc.end();
        });
      } else {
        constexpr int N = kMostChannels / kWideThreads / V;
        lc.begin("layerNormGrad");
        layerNormGrad<T, V, kWideThreads, N, 1, false><<<(unsigned)std::min<int64_t>(rows, 512), kWideThreads, 0, lc.stream>>>(
            dy, x, s, p, mean, rstd, dx, nullptr);
        lc.end();
        if (sums) {
          parts = (int)std::min<int64_t>((rows + 15) / 16, 128);
          lc.begin("layerNormColumnSums");
          layerNormColumnSums<T><<<dim3((unsigned)parts, (unsigned)((channels + kThreads - 1) / kThreads)), kThreads, 0,
                                   lc.stream>>>(dy, x, s, mean, rstd, partial);
          lc.end();
        }
      }
    });
  }
  if (sums) {
    lc.begin("layerNormJoinSums");
    layerNormJoinSums<<<(unsigned)((2 * channels + kChannels - 1) / kChannels), kThreads, 0, lc.stream>>>(
        partial, parts, (int)channels, p, weight_grad, bias_grad);
    lc.end();
  }
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
