// Kernels of the products grouped by expert.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "core/elements.h"
#include "core/ragged.h"
#include "grouped_matmul/grouped_matmul.h"

namespace mluop {
namespace grouped_matmul {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr int kForward = MLUOP_EXT_GROUPED_FORWARD;
constexpr int kBackwardData = MLUOP_EXT_GROUPED_BACKWARD_DATA;
constexpr int kBackwardFilter = MLUOP_EXT_GROUPED_BACKWARD_FILTER;

// Operand fragments of a multiply are 16 bytes a lane: eight 2-byte elements of the reduction, or four fp32 ones, which take
// four multiplies, number s of which pairs element s of both sides.
template <typename T>
struct Fragment;
template <>
struct Fragment<_Float16> {
  typedef half8 type;
  static constexpr int kDepth = 32;  // reduction of a fragment over the wave
  static __device__ __forceinline__ float4v mma(type a, type b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Fragment<__bf16> {
  typedef bf16x8 type;
  static constexpr int kDepth = 32;
  static __device__ __forceinline__ float4v mma(type a, type b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Fragment<float> {
  typedef float4v type;
  static constexpr int kDepth = 16;
  static __device__ __forceinline__ float4v mma(type a, type b, float4v c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    return c;
  }
};

// What the kernels take.
struct Args {
  int rows, groups, ci, co;
  const int32_t *starts;
  int64_t left_stride, right_stride;
  int slice_rows;   // backward filter: rows of a slice; 0: a group's rows are one slice, and its sums the result
  int most_slices;
  float *partial;   // backward filter in slices: sums [slice, ci, co]
};

// ---- any shape, stride and alignment -------------------------------------------------------
//
// A workgroup of four waves has 64 x 64 results, 2 x 2 blocks of 16 x 16 a wave.  Both operands go through registers to LDS as
// [result row or column][reduction], transposed on the way where memory has them the other way round.

constexpr int kAnyTile = 64, kAnyDepth = 32, kAnyThreads = 256;

template <typename T>
constexpr int kAnyPitch = kAnyDepth + 16 / (int)sizeof(T);  // elements: rows 16 bytes past a multiple of the banks

// Eight elements of an operand tile a thread: along the reduction where memory has that side by side (TOGETHER), else along
// the results.  Elements outside [0, extent) x [0, depth) are zero.
template <typename T, bool TOGETHER>
struct AnyLoader {
  const T *base;
  int64_t stride;     // of the other index
  int extent, depth;  // results and reduction that there are
  bool aligned;       // 16-byte loads of whole pieces
  float value[8];
  int at, from;       // first result and first step of the reduction, in the tile

  __device__ AnyLoader(const T *b, int64_t s, int e, int d) : base(b), stride(s), extent(e), depth(d) {
    at = TOGETHER ? (int)threadIdx.x / 4 : (int)threadIdx.x % 8 * 8;
    from = TOGETHER ? (int)threadIdx.x % 4 * 8 : (int)threadIdx.x / 8;
    aligned = (reinterpret_cast<uintptr_t>(b) & 15) == 0 && (s * (int64_t)sizeof(T)) % 16 == 0;
  }
  __device__ __forceinline__ void load(int k0) {
    const int k = k0 + from;
    const int64_t place = TOGETHER ? (int64_t)at * stride + k : (int64_t)k * stride + at;
    const bool line = TOGETHER ? at < extent : k < depth;
    const int left = TOGETHER ? depth - k : extent - at;
    if (line && left >= 8 && aligned) {
      loadFloats<T, 8>(base + place, value);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) value[i] = line && i < left ? (float)base[place + i] : 0.f;
    }
  }
  __device__ __forceinline__ void store(T *tile) const {
    if (TOGETHER) {
      storeFloats<T, 8>(tile + at * kAnyPitch<T> + from, value);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) tile[(at + i) * kAnyPitch<T> + from] = (T)value[i];
    }
  }
};

template <typename T, int MODE>
__global__ __launch_bounds__(kAnyThreads) void groupedAny(const T *__restrict__ left, const T *__restrict__ right, Args a,
                                                          T *__restrict__ out) {
  constexpr bool kFilter = MODE == kBackwardFilter;
  typedef Fragment<T> F;
  const int columns = MODE == kBackwardData ? a.ci : a.co;
  const int n0 = blockIdx.y * kAnyTile;
  int group, m0 = 0, extent, depth;
  const T *l, *r;
  int64_t out_row;     // of result row 0
  bool result = true;  // sums are the result, and not a slice's
  if (kFilter) {
    int first, count;
    m0 = blockIdx.z * kAnyTile;
    extent = a.ci - m0;
    if (a.slice_rows > 0) {
      const RaggedTile t = findRaggedTile<false>(a.starts, a.rows, a.groups, a.slice_rows, blockIdx.x);
      if (t.segment < 0) return;
      group = t.segment;
      first = t.first;
      count = t.rows;
      out_row = (int64_t)blockIdx.x * a.ci + m0;
      result = false;
    } else {
      group = blockIdx.x;
      segmentRows(a.starts, a.rows, group, &first, &count);
      out_row = (int64_t)group * a.ci + m0;
    }
    depth = count;
    l = left + first * a.left_stride + m0;
    r = right + first * a.right_stride + n0;
  } else {
    const RaggedTile t = findRaggedTile<true>(a.starts, a.rows, a.groups, kAnyTile, blockIdx.x);
    if (t.segment < 0) return;
    group = t.segment - 1;
    extent = t.rows;
    out_row = t.first;
    // (rows of no group: nothing to add up)
    depth = group >= 0 && group < a.groups ? (MODE == kForward ? a.ci : a.co) : 0;
    l = left + t.first * a.left_stride;
    r = right + (int64_t)(depth > 0 ? group : 0) * a.ci * a.co + (MODE == kForward ? (int64_t)n0 : (int64_t)n0 * a.co);
  }
  const int width = columns - n0;

  __shared__ __attribute__((aligned(16))) T s_left[kAnyTile * kAnyPitch<T>];
  __shared__ __attribute__((aligned(16))) T s_right[kAnyTile * kAnyPitch<T>];
  AnyLoader<T, !kFilter> from_left(l, a.left_stride, extent, depth);
  AnyLoader<T, MODE == kBackwardData> from_right(r, a.right_stride, width, depth);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sub = lane & 15, quarter = lane >> 4;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  float4v acc[2][2] = {};
  for (int k0 = 0; k0 < depth; k0 += kAnyDepth) {
    from_left.load(k0);
    from_right.load(k0);
    __syncthreads();
    from_left.store(s_left);
    from_right.store(s_right);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kAnyDepth; k += F::kDepth) {
      constexpr int kPiece = 16 / (int)sizeof(T);
      typename F::type x[2], y[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[i] = *reinterpret_cast<const typename F::type *>(s_left + (wm + i * 16 + sub) * kAnyPitch<T> + k + quarter * kPiece);
        y[i] = *reinterpret_cast<const typename F::type *>(s_right + (wn + i * 16 + sub) * kAnyPitch<T> + k + quarter * kPiece);
      }
      // (the right side first: a lane then has four results side by side in a row)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = F::mma(y[j], x[i], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = wm + i * 16 + sub;
    if (m >= extent) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = wn + j * 16 + quarter * 4 + e;
        if (n >= width) continue;
        const int64_t at = (out_row + m) * columns + n0 + n;
        if (result)
          out[at] = (T)acc[i][j][e];
        else
          a.partial[at] = acc[i][j][e];
      }
  }
}

// Adds up the slices of every group, in order.
template <typename T>
__global__ __launch_bounds__(256) void groupedSumSlices(Args a, T *__restrict__ out) {
  const int64_t filter = (int64_t)a.ci * a.co;
  const int group = blockIdx.y;
  int first, count;
  const int slices = raggedTilesOf(a.starts, a.rows, group, a.slice_rows, a.most_slices, &first, &count);
  const float *from = a.partial + first * filter;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < filter; i += (int64_t)gridDim.x * 256) {
    float sum = 0.f;
    for (int s = 0; s < slices; ++s) sum += from[s * filter + i];
    out[group * filter + i] = (T)sum;
  }
}

// ---- host side -----------------------------------------------------------------------------

int tilesOf(int64_t n, int tile) { return (int)((n + tile - 1) / tile); }

// Rows of a slice of the backward filter; 0: one slice a group.  Slices where tiles alone leave most of the GPU idle.
int sliceRows(const Problem &p, int cu_count) {
  const int64_t tiles = (int64_t)tilesOf(p.ci, kAnyTile) * tilesOf(p.co, kAnyTile);
  const int64_t wanted = 4 * (int64_t)cu_count;
  if (tiles * p.groups >= wanted || p.rows <= 512) return 0;
  const int64_t slices = (wanted + tiles - 1) / tiles;
  const int64_t r = std::max<int64_t>((p.rows + slices - 1) / slices, 256);
  if (r >= p.rows) return 0;
  return (int)((r + 63) / 64 * 64);
}

template <typename T, int MODE>
hipError_t launchAny(const LaunchCtx &lc, const Problem &p, const Args &a) {
  const T *l = static_cast<const T *>(p.left), *r = static_cast<const T *>(p.right);
  T *out = static_cast<T *>(p.out);
  const int columns = MODE == kBackwardData ? p.ci : p.co;
  dim3 grid;
  if (MODE == kBackwardFilter) {
    const int64_t slices = a.slice_rows > 0 ? mostRaggedTiles(p.rows, p.groups, a.slice_rows) : p.groups;
    grid = dim3((unsigned)slices, tilesOf(columns, kAnyTile), tilesOf(p.ci, kAnyTile));
  } else {
    grid = dim3((unsigned)mostRaggedTiles(p.rows, p.groups + 2, kAnyTile), tilesOf(columns, kAnyTile), 1);
  }
  lc.begin("groupedAny");
  groupedAny<T, MODE><<<grid, kAnyThreads, 0, lc.stream>>>(l, r, a, out);
  lc.end();
  if (MODE == kBackwardFilter && a.slice_rows > 0) {
    const int64_t blocks = ((int64_t)p.ci * p.co + 255) / 256;
    lc.begin("groupedSumSlices");
    groupedSumSlices<T><<<dim3((unsigned)std::min<int64_t>(blocks, 4096), p.groups), 256, 0, lc.stream>>>(a, out);
    lc.end();
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launchOf(const LaunchCtx &lc, const Problem &p, const Args &a) {
  switch (p.which) {
    case MLUOP_EXT_GROUPED_FORWARD: return launchAny<T, kForward>(lc, p, a);
    case MLUOP_EXT_GROUPED_BACKWARD_DATA: return launchAny<T, kBackwardData>(lc, p, a);
    default: return launchAny<T, kBackwardFilter>(lc, p, a);
  }
}

}  // namespace

size_t workspaceBytes(const Problem &p, int cu_count) {
  if (p.which != MLUOP_EXT_GROUPED_BACKWARD_FILTER) return 0;
  const int slice = sliceRows(p, cu_count);
  if (slice == 0) return 0;
  return (size_t)mostRaggedTiles(p.rows, p.groups, slice) * p.ci * p.co * sizeof(float);
}

hipError_t launch(const LaunchCtx &lc, const Problem &p, int cu_count, void *workspace) {
  Args a = {p.rows, p.groups, p.ci, p.co, p.starts, p.left_stride, p.right_stride, 0, 0, nullptr};
  if (p.which == MLUOP_EXT_GROUPED_BACKWARD_FILTER) {
    a.slice_rows = sliceRows(p, cu_count);
    a.most_slices = a.slice_rows > 0 ? (int)mostRaggedTiles(p.rows, p.groups, a.slice_rows) : 0;
    a.partial = static_cast<float *>(workspace);
  }
  if (p.type == MLUOP_DTYPE_HALF) return launchOf<_Float16>(lc, p, a);
  if (p.type == MLUOP_DTYPE_BFLOAT16) return launchOf<__bf16>(lc, p, a);
  return launchOf<float>(lc, p, a);
}

}  // namespace grouped_matmul
}  // namespace mluop
