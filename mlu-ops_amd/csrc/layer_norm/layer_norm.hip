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
      __shared__ float s_wave[kTeams][kWaves][COUNT];
      __syncthreads();
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) s_wave[team][lane >> 6][i] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < COUNT; ++i) {
        v[i] = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v[i] += s_wave[team][w][i];
      }
    }
  }
};

// ---- forward -------------------------------------------------------------------------------

// y = (x - mean) * rstd * weight + bias.  The mean is the sum's, put right by the mean of the differences from it, so that rows
// far off zero lose nothing; the variance is that of the differences.  Weight and bias stay in registers.  Bound by memory:
// 248 636 x 128 fp16 (127 MB) 23.7 us, 5.4 TB/s; 32 768 x 2048 bf16 (268 MB) 52 us, 5.2 TB/s.
template <typename T, int V, int LANES, int N>
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
  // (all teams of a workgroup take as many turns: sums are taken by whole waves)
  for (int64_t first = (int64_t)blockIdx.x * Lanes::kTeams; first < s.rows; first += (int64_t)gridDim.x * Lanes::kTeams) {
    const int64_t r = first + l.team;
    const bool row = r < s.rows;
    Vector<T, V> v[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = {};
      if (row && l.channel(n) < s.channels) v[n] = *reinterpret_cast<const Vector<T, V> *>(x + r * s.x_stride + l.channel(n));
    }
    float m[1] = {0.f}, moments[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i) m[0] += (float)v[n].v[i];
    l.sum(m);
    m[0] *= by;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const bool there = l.channel(n) < s.channels;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = there ? (float)v[n].v[i] - m[0] : 0.f;
        moments[0] += d;
        moments[1] = fmaf(d, d, moments[1]);
      }
    }
    l.sum(moments);
    const float off = moments[0] * by, variance = fmaf(-off, off, moments[1] * by);
    const float inv = 1.f / sqrtf((variance < 0.f ? 0.f : variance) + eps);  // (NaN stays NaN)
    if (!row) continue;
    if (l.lane == 0) {
      mean[r] = m[0] + off;
      rstd[r] = inv;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (l.channel(n) >= s.channels) continue;
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = fmaf(((float)v[n].v[i] - m[0] - off) * inv, w[n][i], b[n][i]);
      storeFloats<T, V>(out + r * s.channels + l.channel(n), y, s.streamed);
    }
  }
}

// ---- backward ------------------------------------------------------------------------------

// dx = rstd (d - mean of d - normed * mean of d normed) with d = dy * weight, and with SUMS a workgroup's sums of dy * normed
// and dy of every channel over its rows, to partial[workgroup][2][channels].  A team's lanes have the same channels in
// every row, so that these stay in registers until the last row.  Bound by memory: 32 768 x 2048 bf16 (403 MB) 77 us, 5.2 TB/s.
template <typename T, int V, int LANES, int N, bool SUMS>
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
  for (int64_t first = (int64_t)blockIdx.x * Lanes::kTeams; first < s.rows; first += (int64_t)gridDim.x * Lanes::kTeams) {
    const int64_t r = first + l.team;
    const bool row = r < s.rows;
    Vector<T, V> dys[N], xs[N];
    const float m = row ? mean[r] : 0.f, inv = row ? rstd[r] : 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      dys[n] = xs[n] = {};
      if (row && l.channel(n) < s.channels) {
        dys[n] = *reinterpret_cast<const Vector<T, V> *>(dy + r * s.dy_stride + l.channel(n));
        xs[n] = *reinterpret_cast<const Vector<T, V> *>(x + r * s.x_stride + l.channel(n));
      }
    }
    float sums[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!row || l.channel(n) >= s.channels) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float g = (float)dys[n].v[i], normed = ((float)xs[n].v[i] - m) * inv, d = g * w[n][i];
        sums[0] += d;
        sums[1] = fmaf(d, normed, sums[1]);
        if constexpr (SUMS) {
          dw[n][i] = fmaf(g, normed, dw[n][i]);
          db[n][i] += g;
        }
      }
    }
    l.sum(sums);
    const float a = sums[0] * by, b = sums[1] * by;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!row || l.channel(n) >= s.channels) continue;
      float d[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float normed = ((float)xs[n].v[i] - m) * inv;
        d[i] = inv * (fmaf((float)dys[n].v[i], w[n][i], -a) - normed * b);
      }
      storeFloats<T, V>(dx + r * s.channels + l.channel(n), d, s.streamed);
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

// The same sums of rows too wide for registers, more than 16 KB: a thread has one channel of every slice of rows, and dy and x
// are read a second time (2000 x 8192 fp32, 197 MB: gradients 48 us, these 23, and 7 to add them up).
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

// partial[parts][2][channels] added up: kChannels sums a workgroup, each by kShares threads.
constexpr int kJoinThreads = 1024, kChannels = 16, kShares = kJoinThreads / kChannels, kAhead = 8;
__global__ __launch_bounds__(kJoinThreads) void layerNormJoinSums(const float *__restrict__ partial, int parts, int channels,
                                                                  ChannelParams p, void *weight_grad, void *bias_grad) {
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

// Vectors of a thread: 16 bytes, whatever their width.  (More, and no barrier between the waves of a wide row, leaves few waves a
// SIMD: 32 768 x 2048 bf16, 64 bytes a thread 106 us forward and 117 backward, 16 bytes 53 and 77.  Less has a wave add up few
// values: 200 000 x 33 bf16, 2 bytes a thread 35 us forward, 16 bytes 17.)
template <typename T, int V>
constexpr int kVectors = 16 / (int)sizeof(T) / V;

// Calls f(LANES): the smallest team that holds a row whose threads' 16 bytes are `pieces`.  (Teams of eight for 1 875 000 rows of
// 16 bf16: 57 us forward and 61 backward, of two 24 and 40.)
template <typename F>
void byTeam(int64_t pieces, F f) {
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
  else if (pieces <= 64)
    f(std::integral_constant<int, 64>());
  else if (pieces <= 128)
    f(std::integral_constant<int, 128>());
  else if (pieces <= 256)
    f(std::integral_constant<int, 256>());
  else if (pieces <= 512)
    f(std::integral_constant<int, 512>());
  else
    f(std::integral_constant<int, 1024>());
}
constexpr int kTeamPieces = 1024;   // that byTeam's largest holds
constexpr int kWideThreads = 1024;  // of a workgroup that holds a row of up to kMostChannels

constexpr int kBlocks = 4096;       // most workgroups of 256 threads

// Most rows of partial sums: as many workgroups as the CUs hold together, and fewer where a row of sums is long (32 768 x 2048
// bf16: 512 workgroups 95 us and 5 to add up, 1024 77 and 7; 16 384 x 8192: 149 and 12, 154 and 22; 60 000 x 250: 31 and 5, 2048
// 22 and 6).  How many rows there are is not looked at: of 2048 x 2048 bf16 every workgroup has two, and 16.8 MB of sums are
// written and read beside 25 MB of tensors (14 us and 9).
int64_t sumParts(int64_t channels) { return channels <= 512 ? 2048 : channels <= 2048 ? 1024 : 512; }

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

size_t workspaceBytes(int64_t channels) { return 16 + (size_t)sumParts(channels) * 2 * channels * sizeof(float); }

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
      const unsigned grid = (unsigned)std::min<int64_t>((rows + L::kTeams - 1) / L::kTeams, kBlocks * kThreads / L::kWorkgroup);
      lc.begin("layerNormRows");
      layerNormRows<T, V, LANES, N><<<grid, L::kWorkgroup, 0, lc.stream>>>(
          static_cast<const T *>(features), s, p, eps, static_cast<T *>(out), mean, rstd);
      lc.end();
    };
    constexpr int kN = kVectors<T, V>;
    const int64_t pieces = (channels + V * kN - 1) / (V * kN);
    if (pieces <= kTeamPieces)
      byTeam(pieces, [&](auto lanes) { launch(lanes, std::integral_constant<int, kN>()); });
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
      constexpr int kN = kVectors<T, V>;
      const int64_t pieces = (channels + V * kN - 1) / (V * kN);
      if (pieces <= kTeamPieces) {
        byTeam(pieces, [&](auto lanes) {
          constexpr int LANES = decltype(lanes)::value, N = kN;
          typedef Team<V, LANES, N> L;
          const int64_t blocks = (rows + L::kTeams - 1) / L::kTeams;
          parts = (int)std::min<int64_t>(blocks, sumParts(channels));
          lc.begin("layerNormGrad");
          if (sums) {
            layerNormGrad<T, V, LANES, N, true><<<(unsigned)parts, L::kWorkgroup, 0, lc.stream>>>(dy, x, s, p, mean, rstd, dx,
                                                                                                  partial);
          } else {
            const unsigned grid = (unsigned)std::min<int64_t>(blocks, kBlocks * kThreads / L::kWorkgroup);
            layerNormGrad<T, V, LANES, N, false><<<grid, L::kWorkgroup, 0, lc.stream>>>(dy, x, s, p, mean, rstd, dx, nullptr);
          }
          lc.end();
        });
      } else {
        constexpr int N = kMostChannels / kWideThreads / V;
        lc.begin("layerNormGrad");
        layerNormGrad<T, V, kWideThreads, N, false><<<(unsigned)std::min<int64_t>(rows, 512), kWideThreads, 0, lc.stream>>>(
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
    layerNormJoinSums<<<(unsigned)((2 * channels + kChannels - 1) / kChannels), kJoinThreads, 0, lc.stream>>>(
        partial, parts, (int)channels, p, weight_grad, bias_grad);
    lc.end();
  }
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
