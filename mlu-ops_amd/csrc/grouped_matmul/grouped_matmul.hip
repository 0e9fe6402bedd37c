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
  int blocks;       // backward filter: slices there can be, or groups
  int works;        // numbers of works (some of which may not be there)
  float *partial;   // backward filter in slices: sums [slice, ci, co]
};

// ---- any shape, stride and alignment -------------------------------------------------------
//
// A workgroup of four waves has 64 x 64 results, a quarter a wave.  Both operands go through registers to LDS as
// [result row or column][reduction], transposed on the way where memory has them the other way round; the registers of a step
// are filled while the one before is multiplied.

constexpr int kAnyTile = 64, kAnyThreads = 256;
template <typename T>
constexpr int kAnyDepth = 128 / (int)sizeof(T);  // of a step: 128 bytes
template <typename T>
constexpr int kAnyPitch = kAnyDepth<T> + 16 / (int)sizeof(T);  // elements: rows 16 bytes past a multiple of the banks

// A thread's part of an operand tile: eight elements kParts times, along the reduction where memory has that side by side
// (TOGETHER), else along the results.  Elements outside [0, extent) x [0, depth) are zero.
template <typename T, bool TOGETHER>
struct AnyLoader {
  static constexpr int kParts = kAnyTile * kAnyDepth<T> / 8 / kAnyThreads;  // (two of 2-byte types, one of fp32)
  static constexpr int kAcross = TOGETHER ? kAnyDepth<T> / 8 : kAnyTile / 8;
  const T *base;
  int64_t stride;     // of the other index
  int extent, depth;  // results and reduction that there are
  int whole;          // how eight elements that are all there are read: 2: as 16 bytes, 1: as 8, 0: one by one
  Vector<T, 8> value[kParts];

  __device__ AnyLoader(const T *b, int64_t s, int e, int d) : base(b), stride(s), extent(e), depth(d) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(b) | (uintptr_t)(s * (int64_t)sizeof(T));
    whole = (all & 15) == 0 ? 2 : ((all & 7) == 0 ? 1 : 0);
  }
  static __device__ __forceinline__ int at(int part) {  // first result
    const int eight = (int)threadIdx.x + kAnyThreads * part;
    return TOGETHER ? eight / kAcross : eight % kAcross * 8;
  }
  static __device__ __forceinline__ int from(int part) {  // first of the reduction
    const int eight = (int)threadIdx.x + kAnyThreads * part;
    return TOGETHER ? eight % kAcross * 8 : eight / kAcross;
  }
  __device__ __forceinline__ void load(int k0) {
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const int r = at(part), k = k0 + from(part);
      const T *place = base + (TOGETHER ? (int64_t)r * stride + k : (int64_t)k * stride + r);
      const bool line = TOGETHER ? r < extent : k < depth;
      const int left = TOGETHER ? depth - k : extent - r;
      Vector<T, 8> &v = value[part];
      if (line && left >= 8 && whole == 2) {
        v = *reinterpret_cast<const Vector<T, 8> *>(place);
      } else if (line && left >= 8 && whole == 1) {
        struct alignas(8) Pieces {
          uint2 piece[sizeof(T)];
        } pieces;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) pieces.piece[i] = reinterpret_cast<const uint2 *>(place)[i];
        v = __builtin_bit_cast(Vector<T, 8>, pieces);
      } else {
        // (loads of a place that is there, whether wanted or not: under a condition each would wait for the one before)
#pragma unroll
        for (int i = 0; i < 8; ++i) v.v[i] = *(line && i < left ? place + i : base);
#pragma unroll
        for (int i = 0; i < 8; ++i) v.v[i] = line && i < left ? v.v[i] : (T)0.f;
      }
    }
  }
  __device__ __forceinline__ void store(T *tile) const {
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      if (TOGETHER) {
        *reinterpret_cast<Vector<T, 8> *>(tile + at(part) * kAnyPitch<T> + from(part)) = value[part];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) tile[(at(part) + i) * kAnyPitch<T> + from(part)] = value[part].v[i];
      }
    }
  }
};

template <typename T, int MODE>
__global__ __launch_bounds__(kAnyThreads) void groupedAny(const T *__restrict__ left, const T *__restrict__ right, Args a,
                                                          T *__restrict__ out) {
  constexpr bool kFilter = MODE == kBackwardFilter;
  constexpr int kBlocks = kAnyTile / 32;  // of 16 results, of a wave
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
  const int wm = (wave >> 1) * (kAnyTile / 2), wn = (wave & 1) * (kAnyTile / 2);
  float4v acc[kBlocks][kBlocks] = {};
  if (depth > 0) {
    from_left.load(0);
    from_right.load(0);
  }
  for (int k0 = 0; k0 < depth; k0 += kAnyDepth<T>) {
    __syncthreads();
    from_left.store(s_left);
    from_right.store(s_right);
    __syncthreads();
    if (k0 + kAnyDepth<T> < depth) {
      from_left.load(k0 + kAnyDepth<T>);
      from_right.load(k0 + kAnyDepth<T>);
    }
#pragma unroll
    for (int k = 0; k < kAnyDepth<T>; k += F::kDepth) {
      constexpr int kPiece = 16 / (int)sizeof(T);
      typename F::type x[kBlocks], y[kBlocks];
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        x[i] = *reinterpret_cast<const typename F::type *>(s_left + (wm + i * 16 + sub) * kAnyPitch<T> + k + quarter * kPiece);
        y[i] = *reinterpret_cast<const typename F::type *>(s_right + (wn + i * 16 + sub) * kAnyPitch<T> + k + quarter * kPiece);
      }
      // (the right side first: a lane then has four results side by side in a row)
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) acc[i][j] = F::mma(y[j], x[i], acc[i][j]);
    }
  }
  const bool fours = (columns & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) {
    const int m = wm + i * 16 + sub;
    if (m >= extent) continue;
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) {
      const int n = wn + j * 16 + quarter * 4;
      const int64_t at = (out_row + m) * columns + n0 + n;
      const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      if (fours && n < width) {
        if (result)
          storeFloats<T, 4>(out + at, v);
        else
          storeFloats<float, 4>(a.partial + at, v);
        continue;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (n + e >= width) continue;
        if (result)
          out[at + e] = (T)v[e];
        else
          a.partial[at + e] = v[e];
      }
    }
  }
}

// ---- rows in whole 16-byte pieces ----------------------------------------------------------
//
// A workgroup has BM x BN results; the reduction goes through two LDS buffers in steps of 128 bytes (64 elements of 2 bytes, 32
// of fp32), which loads fill directly, 16 bytes a lane.  An operand that memory has along the reduction lies in LDS as
// [result][step], and a fragment is one 16-byte read.  One that memory has along the results lies as [step][results]:
// 2-byte elements are transposed by `ds_read_b64_tr_b16` (within 16 lanes, lane i gives the address of four results of the
// reduction's part i / 4, and lane j receives result j of the four parts), fp32 ones are read one by one.  Either way rows are a multiple of the banks apart,
// and their 16-byte pieces are permuted by row so that the lanes of a read meet all banks; the loads permute, since a
// lane's place in LDS is fixed.

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef short v8i16 __attribute__((ext_vector_type(8)));

template <typename T>
constexpr int kDepth = 128 / (int)sizeof(T);  // of a step
constexpr uint32_t kNowhere = 0x80000000u;  // behind the end of every buffer

// 16 bytes per lane from byte `offset` of a buffer straight into LDS: lane l writes bytes [16 l, 16 l + 16) behind
// `lds_address`; zeros for offsets behind the buffer's end.  The caller waits (vmcnt).
__device__ __forceinline__ void requestToLds(u32x4 buffer, uint32_t offset, uint32_t lds_address) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds_address), "v"(offset), "s"(buffer) : "memory", "m0");
}
// Everybody's requests and reads are done.
__device__ __forceinline__ void stepBarrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// One operand of a tile: RESULTS results by the reduction.  TOGETHER: memory has the reduction side by side.
template <typename T, bool TOGETHER, int RESULTS, int WAVES>
struct Operand {
  static constexpr int kSize = (int)sizeof(T), kStep = kDepth<T>;
  static constexpr int kRowBytes = TOGETHER ? 128 : RESULTS * kSize;
  static constexpr int kBytes = RESULTS * 128;
  static constexpr int kAll = kBytes / 1024;                      // wave-loads of a step
  static constexpr int kLoads = kAll < WAVES ? 1 : kAll / WAVES;  // of a wave
  static constexpr int kPieces = kRowBytes / 16;
  static_assert(kAll < WAVES ? WAVES % kAll == 0 : kBytes % (1024 * WAVES) == 0, "whole wave-loads");
  // (fewer than there are waves: several waves make the same one, so that all wait for the same number)
  static __device__ __forceinline__ int ownWave() {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    return kAll < WAVES ? wave % kAll : wave;
  }

  // By which a row's pieces are permuted (LDS row: a result or a step).
  static __device__ __forceinline__ int moved(int row) {
    if (TOGETHER) return (row >> 1) & 7;
    if (kSize == 4) return kPieces >= 16 ? row & 12 : (row >> 1) & 4;
    return kPieces >= 16 ? ((row & 1) << 1) | ((row & 2) << 1) | (row & 8) : (row & 2) | ((row & 8) >> 1);
  }

  const char *base;       // of the step to be requested
  int64_t step_bytes;     // from step to step
  uint32_t stride;        // bytes from row to row
  int extent;             // results that there are
  uint32_t offset[kLoads];
  uint32_t lds;           // of the first buffer, this wave's first load
  int part;               // of the reduction: the first of this lane's pieces (TOGETHER: the same in all its loads)
  u32x4 words;            // the step's buffer,
  uint32_t behind;        // what a lane's offsets are ored with in this step

  __device__ Operand(const T *from, int64_t stride_elements, int results, const char *lds_base) {
    base = reinterpret_cast<const char *>(from);
    stride = (uint32_t)stride_elements * kSize;
    extent = results < RESULTS ? results : RESULTS;
    step_bytes = TOGETHER ? 128 : (int64_t)kStep * stride;
    const int lane = threadIdx.x & 63, wave = ownWave();
    lds = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)lds_base + wave * 1024;
    static_assert(!TOGETHER || WAVES % 2 == 0, "every load of a lane has the same parts of its rows");
    part = ((lane % kPieces) ^ moved((wave * 64 + lane) / kPieces)) * (16 / kSize);
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int piece = (u * WAVES + wave) * 64 + lane;
      const int row = piece / kPieces;
      offset[u] = (uint32_t)row * stride + (uint32_t)((piece % kPieces) ^ moved(row)) * 16u;
    }
  }
  // Goes on to the next step, of which `left` parts of the reduction are there (none or less: its loads give zeros).
  __device__ __forceinline__ void next(int left) {
    const int there = left < kStep ? left : kStep;
    // (past the last row's own bytes nothing is read: what lies there is another's)
    const uint32_t end = TOGETHER ? (uint32_t)(extent - 1) * stride + (uint32_t)(there * kSize)
                                  : (uint32_t)(there - 1) * stride + (uint32_t)(extent * kSize);
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    words = u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                  (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32)),
                  (uint32_t)__builtin_amdgcn_readfirstlane(left > 0 ? (int)end : 0), 0x00020000u};
    // (pieces behind the reduction's end are those of the next row)
    behind = TOGETHER && part >= left ? kNowhere : 0u;
    base += step_bytes;
  }
  __device__ __forceinline__ void request(int u, int buffer) const {
    requestToLds(words, TOGETHER ? offset[u] | behind : offset[u], lds + buffer * kBytes + u * WAVES * 1024);
  }

  // Where in a buffer a lane's fragment of the results from `first` on (a multiple of 16) and of one half of the step lies.
  static __device__ __forceinline__ int place(int first, int half) {
    const int lane = threadIdx.x & 63, sub = lane & 15, quarter = lane >> 4;
    if (TOGETHER) {
      const int row = first + sub;
      return row * kRowBytes + ((half * 4 + quarter) ^ moved(row)) * 16;
    }
    if (kSize == 4) {
      const int row = half * 16 + quarter * 4, result = first + sub;
      return row * kRowBytes + ((result / 4) ^ moved(row)) * 16 + result % 4 * 4;
    }
    const int row = half * 32 + quarter * 8 + (sub >> 2);
    return row * kRowBytes + (((first / 8) + ((sub & 3) >> 1)) ^ moved(row)) * 16 + (sub & 1) * 8;
  }
  static __device__ __forceinline__ typename Fragment<T>::type fragment(const char *at) {
    if constexpr (TOGETHER) {
      return *reinterpret_cast<const typename Fragment<T>::type *>(at);
    } else if constexpr (kSize == 4) {
      // (four rows whose pieces are permuted alike)
      float4v v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const float *>(at + i * kRowBytes);
      return v;
    } else {
      typedef __attribute__((address_space(3))) v4i16 *Place;
      const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Place)(at));
      const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Place)(at + 4 * kRowBytes));
      return __builtin_bit_cast(typename Fragment<T>::type, (v8i16)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// What a workgroup multiplies next.
template <typename T>
struct Work {
  bool there;
  int extent, width, depth;  // results of the tile that there are, and the reduction
  const T *left, *right;
  int64_t out;               // element of the result's (or the partial sums') first
};

// Tile of rows number `number`, and which of the tiles_n tiles of columns.  Workgroups go to the eight XCDs in turn, and so
// do the numbers; an XCD has a run of tiles that share operands in its L2: four tiles of rows by all columns, then the
// next four.
template <int BM>
__device__ __forceinline__ RaggedTile tileOfRows(int number, const int32_t *starts, const Args &a, int tiles_n, int *column) {
  constexpr int kBand = 4;
  const int total_m = raggedTiles<true>(starts, a.rows, a.groups, BM), total = total_m * tiles_n, each = (total + 7) / 8;
  const int in_xcd = number >> 3, tile = (number & 7) * each + in_xcd;
  if (in_xcd >= each || tile >= total) {
    RaggedTile none = {};
    none.segment = -1;
    return none;
  }
  const int band = tile / (kBand * tiles_n), in_band = tile - band * (kBand * tiles_n);
  const int height = min(total_m - band * kBand, kBand);
  *column = in_band / height;
  return findRaggedTile<true>(starts, a.rows, a.groups, BM, band * kBand + in_band % height);
}

// Work number `number` of args.works, from the starts in LDS.  Workgroups go to the eight XCDs in turn, and so do the
// numbers; those of an XCD take tiles that share operands in its L2.
template <typename T, int MODE, int BM, int BN>
__device__ __forceinline__ Work<T> workOf(int number, const int32_t *starts, const uint16_t *longest, const Args &a,
                                          const T *left, const T *right) {
  Work<T> w;
  w.there = false;
  w.extent = w.width = w.depth = 0;
  w.left = left;
  w.right = right;
  w.out = 0;
  if (number >= a.works) return w;
  const int columns = MODE == kBackwardData ? a.ci : a.co;
  const int tiles_n = (columns + BN - 1) / BN;
  const int xcd = number & 7;
  int in_xcd = number >> 3, n0;
  if (MODE == kBackwardFilter) {
    // an eighth of every block's tiles (a group, or a slice of its rows) for each XCD: groups have very different lengths
    const int per_block = (a.ci + BM - 1) / BM * tiles_n;
    int block, tile;
    if (per_block >= 8) {
      // (every second round of the workgroups backwards: who had a long one has a short one next)
      const int wide = gridDim.x >> 3, round = in_xcd / wide;
      if (longest != nullptr && (round & 1) != 0)
        in_xcd = 2 * round * wide + min(wide, (a.works >> 3) - round * wide) - 1 - in_xcd;
      const int each = (per_block + 7) / 8;
      block = in_xcd / each;
      tile = xcd * each + in_xcd - block * each;
      if (tile >= min(per_block, (xcd + 1) * each)) return w;
    } else {
      block = number / per_block;
      tile = number - block * per_block;
    }
    if (block >= a.blocks) return w;
    const int m0 = tile / tiles_n * BM;
    n0 = tile % tiles_n * BN;
    int first;
    if (a.slice_rows > 0) {
      const RaggedTile t = findRaggedTile<false>(starts, a.rows, a.groups, a.slice_rows, block);
      if (t.segment < 0) return w;
      first = t.first;
      w.depth = t.rows;
    } else {
      if (longest != nullptr) block = __builtin_amdgcn_readfirstlane(longest[block]);
      segmentRows(starts, a.rows, block, &first, &w.depth);
      first = __builtin_amdgcn_readfirstlane(first);
      w.depth = __builtin_amdgcn_readfirstlane(w.depth);
    }
    w.extent = a.ci - m0;
    w.left += first * a.left_stride + m0;
    w.right += first * a.right_stride + n0;
    w.out = ((int64_t)block * a.ci + m0) * columns + n0;
  } else {
    const RaggedTile t = tileOfRows<BM>(number, starts, a, tiles_n, &n0);
    if (t.segment < 0) return w;
    n0 *= BN;
    const int group = t.segment - 1;
    const bool inside = group >= 0 && group < a.groups;
    w.depth = inside ? (MODE == kForward ? a.ci : a.co) : 0;
    w.extent = t.rows;
    w.left += t.first * a.left_stride;
    w.right += (int64_t)(inside ? group : 0) * a.ci * a.co + (MODE == kForward ? (int64_t)n0 : (int64_t)n0 * a.co);
    w.out = (int64_t)t.first * columns + n0;
  }
  w.width = columns - n0;
  w.there = true;
  return w;
}

constexpr int kStartsInLds = 2048, kRankedGroups = 256;

// Workgroups stay: each takes the works blockIdx.x, blockIdx.x + gridDim.x, ...  The first loads of the next are under way
// while the results of this one are stored.
template <typename T, int MODE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64) void groupedTiles(const T *__restrict__ left, const T *__restrict__ right,
                                                            Args a, T *__restrict__ out) {
  constexpr bool kFilter = MODE == kBackwardFilter;
  constexpr int kWaves = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  typedef Operand<T, !kFilter, BM, kWaves> Left;
  typedef Operand<T, MODE == kBackwardData, BN, kWaves> Right;
  typedef typename Fragment<T>::type fragment;
  extern __shared__ __attribute__((aligned(1024))) char s_tiles[];  // two buffers of the left side, two of the right
  __shared__ int32_t s_starts[kStartsInLds];

  for (int i = threadIdx.x; i <= a.groups; i += kWaves * 64) s_starts[i] = a.starts[i];
  __syncthreads();
  // groups by falling length (few enough for everybody to rank them): static rounds of works of very different lengths
  // would wait for whoever has most of the long ones
  const uint16_t *longest = nullptr;
  if (kFilter && a.slice_rows == 0 && a.groups <= kRankedGroups) {
    __shared__ uint16_t s_longest[kRankedGroups];
    for (int g = threadIdx.x; g < a.groups; g += kWaves * 64) {
      int first, rows, place = 0;
      segmentRows(s_starts, a.rows, g, &first, &rows);
      for (int o = 0; o < a.groups; ++o) {
        int others;
        segmentRows(s_starts, a.rows, o, &first, &others);
        place += others > rows || (others == rows && o < g) ? 1 : 0;
      }
      s_longest[place] = (uint16_t)g;
    }
    __syncthreads();
    longest = s_longest;
  }
  const int columns = MODE == kBackwardData ? a.ci : a.co;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const char *x_tile = s_tiles, *y_tile = s_tiles + 2 * Left::kBytes;

  // A step has kSlots slots of TN multiplies each.  In slot n the left fragment of slot n + 2 is read, and in the first half
  // the right ones of the second.  In the last two slots they are those of the next step: in front of them everybody's
  // loads are waited for and everybody has read this step's buffer, which the loads of the step after next then
  // fill, kAtOnce a slot.
  constexpr int kSlots = 2 * TM, kLoads = Left::kLoads + Right::kLoads, kAtOnce = (2 * kLoads + kSlots - 1) / kSlots;
  static_assert(TM >= 2 && kAtOnce * (kSlots - 2) >= kLoads, "all loads are requested in front of the slots that wait for them");
  static_assert(TN % 2 == 0, "columns are stored two blocks at once");
  constexpr int kStores = sizeof(T) == 2 ? TM * TN / 2 : TM * TN;  // (partial sums of 2-byte types take twice as many: the wait is for some of them too)
  Left x(left, 0, 1, s_tiles);
  Right y(right, 0, 1, s_tiles + 2 * Left::kBytes);
  auto request = [&](int slot, int buffer) {  // slot: since the wait
#pragma unroll
    for (int u = slot * kAtOnce; u < (slot + 1) * kAtOnce; ++u) {
      if (u < Left::kLoads)
        x.request(u, buffer);
      else if (u < kLoads)
        y.request(u - Left::kLoads, buffer);
    }
  };
  auto begin = [&](const Work<T> &w) {
    x = Left(w.left, a.left_stride, w.extent, s_tiles);
    y = Right(w.right, a.right_stride, w.width, s_tiles + 2 * Left::kBytes);
    x.next(w.depth);
    y.next(w.depth);
#pragma unroll
    for (int n = 0; n < kSlots; ++n) request(n, 0);
  };
  auto left_fragment = [&](int slot, int buffer) {
    return Left::fragment(x_tile + buffer * Left::kBytes + Left::place(wm + slot % TM * 16, slot / TM));
  };
  auto right_fragment = [&](int j, int half, int buffer) {
    return Right::fragment(y_tile + buffer * Right::kBytes + Right::place(wn + j * 16, half));
  };

  int number = blockIdx.x;
  bool stored = false;  // behind the loads of the work's first step there are kStores stores
  Work<T> work = workOf<T, MODE, BM, BN>(number, s_starts, longest, a, left, right);
  begin(work);
  while (number < a.works) {
    number += gridDim.x;
    const Work<T> following = workOf<T, MODE, BM, BN>(number, s_starts, longest, a, left, right);
    float4v acc[TM][TN] = {};
    const int steps = (work.depth + kDepth<T> - 1) / kDepth<T>;
    if (steps > 0) {
      fragment xs[kSlots + 2], ys[3][TN];
      if (stored)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kStores) : "memory");
      else
        stepBarrier();
      x.next(work.depth - kDepth<T>);
      y.next(work.depth - kDepth<T>);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        request(n, 1);
        xs[n] = left_fragment(n, 0);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) ys[0][j] = right_fragment(j, 0, 0);
      int buffer = 0, ahead = work.depth - kDepth<T>;
      for (int step = 0; step < steps; ++step) {
#pragma unroll
        for (int n = 0; n < kSlots; ++n) {
          if (n == kSlots - 2) {
            stepBarrier();
            ahead -= kDepth<T>;
            x.next(ahead);
            y.next(ahead);
          }
          if (n < kSlots - 2) {
            request(n + 2, buffer ^ 1);
            xs[n + 2] = left_fragment(n + 2, buffer);
#pragma unroll
            for (int j = 0; j < TN; ++j)
              if (j * TM / TN == n) ys[1][j] = right_fragment(j, 1, buffer);
          } else {
            request(n + 2 - kSlots, buffer);
            xs[n + 2] = left_fragment(n + 2 - kSlots, buffer ^ 1);
#pragma unroll
            for (int j = 0; j < TN; ++j)
              if (j * 2 / TN == n + 2 - kSlots) ys[2][j] = right_fragment(j, 0, buffer ^ 1);
          }
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[n % TM][j] = Fragment<T>::mma(ys[n / TM][j], xs[n], acc[n % TM][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
        xs[0] = xs[kSlots];
        xs[1] = xs[kSlots + 1];
#pragma unroll
        for (int j = 0; j < TN; ++j) ys[0][j] = ys[2][j];
        buffer ^= 1;
      }
    }
    // (the last steps' loads give zeros, but they too write LDS: the next work's, or another workgroup's when this one has
    // ended)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    begin(following);
    const bool partial = kFilter && a.slice_rows > 0;
    const int size = partial ? 4 : (int)sizeof(T);
    // (stores outside of the results go nowhere: the same number of them for every work)
    const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(
        partial ? static_cast<void *>(a.partial + work.out) : static_cast<void *>(out + work.out), 0,
        work.there ? (int)(((min(work.extent, BM) - 1) * columns + work.width) * size) : 0, 0x00020000);
    const int sub = lane & 15, quarter = lane >> 4;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = wm + i * 16 + sub;
      if (partial || sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int n = wn + j * 16 + quarter * 4;
          const int at = m < work.extent && n < work.width ? (m * columns + n) * 4 : (int)kNowhere;
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[i][j]), to, at, 0, 0);
        }
        continue;
      }
      if constexpr (sizeof(T) == 2)
      // Two blocks of columns at once: the odd quarters of the first change places with the even ones of the second, and a
      // lane has eight columns side by side.
#pragma unroll
      for (int j = 0; j < TN; j += 2) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        Vector<T, 4> v[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[0].v[e] = (T)acc[i][j][e];
          v[1].v[e] = (T)acc[i][j + 1][e];
        }
        const u32x2 one = __builtin_bit_cast(u32x2, v[0]), two = __builtin_bit_cast(u32x2, v[1]);
        const u32x2 lo = __builtin_amdgcn_permlane16_swap(one.x, two.x, false, false);
        const u32x2 hi = __builtin_amdgcn_permlane16_swap(one.y, two.y, false, false);
        const int n = wn + (j + (quarter & 1)) * 16 + (quarter >> 1) * 8;
        const int at = m < work.extent && n < work.width ? (m * columns + n) * 2 : (int)kNowhere;
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{lo.x, hi.x, lo.y, hi.y}, to, at, 0, 0);
      }
    }
    stored = true;
    work = following;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Few rows a group: the filters are what is read, and every workgroup keeps kFewStages steps of its 64 columns on their way.
// Four waves have 16 columns each.  (The kernel above has one step under way, which a product of a few steps waits for
// again and again.)
constexpr int kFewColumns = 64, kFewStages = 6, kFewWaves = 4;

template <typename T, int MODE, int BM>
__global__ __launch_bounds__(kFewWaves * 64) void groupedFew(const T *__restrict__ left, const T *__restrict__ right, Args a,
                                                             T *__restrict__ out) {
  typedef Operand<T, true, BM, kFewWaves> Left;
  typedef Operand<T, MODE == kBackwardData, kFewColumns, kFewWaves> Right;
  typedef typename Fragment<T>::type fragment;
  constexpr int TM = BM / 16, kLoads = Left::kLoads + Right::kLoads;
  static_assert((kFewStages - 2) * kLoads <= 63, "what a wait can count");
  extern __shared__ __attribute__((aligned(1024))) char s_tiles[];

  const int columns = MODE == kBackwardData ? a.ci : a.co;
  int n0;
  const RaggedTile t = tileOfRows<BM>(blockIdx.x, a.starts, a, (columns + kFewColumns - 1) / kFewColumns, &n0);
  if (t.segment < 0) return;
  n0 *= kFewColumns;
  const int group = t.segment - 1, width = columns - n0;
  const bool inside = group >= 0 && group < a.groups;
  const int depth = inside ? (MODE == kForward ? a.ci : a.co) : 0;
  Left x(left + t.first * a.left_stride, a.left_stride, t.rows, s_tiles);
  Right y(right + (int64_t)(inside ? group : 0) * a.ci * a.co + (MODE == kForward ? (int64_t)n0 : (int64_t)n0 * a.co),
          a.right_stride, width, s_tiles + kFewStages * Left::kBytes);
  auto request = [&](int left_over, int buffer) {
    x.next(left_over);
    y.next(left_over);
#pragma unroll
    for (int u = 0; u < Left::kLoads; ++u) x.request(u, buffer);
#pragma unroll
    for (int u = 0; u < Right::kLoads; ++u) y.request(u, buffer);
  };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float4v acc[TM] = {};
  if (depth > 0) {
#pragma unroll
    for (int s = 0; s < kFewStages - 1; ++s) request(depth - s * kDepth<T>, s);
    int buffer = 0, fill = kFewStages - 1;
    for (int k0 = 0; k0 < depth; k0 += kDepth<T>) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kFewStages - 2) * kLoads) : "memory");
      // (past the end the loads give zeros, so that their number stays what is waited for)
      request(depth - k0 - (kFewStages - 1) * kDepth<T>, fill);
      const char *x_tile = s_tiles + buffer * Left::kBytes, *y_tile = s_tiles + kFewStages * Left::kBytes + buffer * Right::kBytes;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const fragment ys = Right::fragment(y_tile + Right::place(wave * 16, half));
#pragma unroll
        for (int i = 0; i < TM; ++i)
          acc[i] = Fragment<T>::mma(ys, Left::fragment(x_tile + Left::place(i * 16, half)), acc[i]);
      }
      buffer = buffer + 1 == kFewStages ? 0 : buffer + 1;
      fill = fill + 1 == kFewStages ? 0 : fill + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  const int n = wave * 16 + (lane >> 4) * 4;
  if (n >= width) return;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = i * 16 + (lane & 15);
    const float v[4] = {acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
    if (m < t.rows) storeFloats<T, 4>(out + (int64_t)(t.first + m) * columns + n0 + n, v);
  }
}

// Adds up the slices of every group: a workgroup has 64 V results, whose slices its four waves share.
template <typename T, int V>
__global__ __launch_bounds__(256) void groupedSumSlices(Args a, T *__restrict__ out) {
  constexpr int kShares = 4, kAhead = 4;
  __shared__ float s_sum[kShares][64 * V];
  const int64_t filter = (int64_t)a.ci * a.co;
  const int group = blockIdx.y, lane = threadIdx.x & 63, share = threadIdx.x >> 6;
  int first, count;
  const int slices = raggedTilesOf(a.starts, a.rows, group, a.slice_rows, a.most_slices, &first, &count);
  const int64_t at = ((int64_t)blockIdx.x * 64 + lane) * V;
  const bool there = at < filter;
  float sum[V] = {};
  if (there) {
    const float *from = a.partial + first * filter + at;
    for (int s0 = share; s0 < slices; s0 += kShares * kAhead) {
      Vector<float, V> v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        v[j] = *reinterpret_cast<const Vector<float, V> *>(from + min(s0 + j * kShares, slices - 1) * filter);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (s0 + j * kShares >= slices) break;
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += v[j].v[e];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) s_sum[share][lane * V + e] = sum[e];
  __syncthreads();
  if (share != 0 || !there) return;
#pragma unroll
  for (int e = 0; e < V; ++e)
    for (int o = 1; o < kShares; ++o) sum[e] += s_sum[o][lane * V + e];
  storeFloats<T, V>(out + group * filter + at, sum);
}

// ---- host side -----------------------------------------------------------------------------

int tilesOf(int64_t n, int tile) { return (int)((n + tile - 1) / tile); }

// A kernel's tile, and what it takes (us): a step of 64 of the reduction where its workgroups are few and where they fill the
// GPU, and a tile's beginning and end.
struct Tile {
  const char *name;
  int m, n, per_cu;
  double few, full, end;
  double forward, data;  // TB/s at which filters come in, forward and for backward data
};
// The first three are groupedTiles, the others groupedFew.  Measured (bf16, us at 256 x 256 / 128 x 128 / 64 x 128 / 32 x 64 / 16 x 64):
// 16 rows of a 2048 x 2048 filter 39 / 19 / 14 / 9 / 8.5, 1000 rows 43 / 24 / 21 / 27 / 43, 4000 rows 47 / 36 / 48 / 95 / 158, 40 000
// rows 288 / 365 / 524 / 895 / 1480.
constexpr int kTileKinds = 3;
// 64 filters of 2048 x 2048 for a row each: 121 / 95 / 97 / 119 / 119, and backward data, which reads their rows, 136 / 125 / 122 /
// 102 / 102.
constexpr Tile kTiles[] = {{"groupedTiles256", 256, 256, 1, 1.25, 1.65, 5.0, 4.4, 3.9},
                           {"groupedTiles128", 128, 128, 2, 0.59, 1.06, 2.5, 5.6, 4.3},
                           {"groupedTiles64", 64, 128, 2, 0.43, 0.76, 2.0, 5.6, 4.3},
                           {"groupedFew32", 32, kFewColumns, 2, 0.25, 0.40, 1.5, 5.2, 5.2},
                           {"groupedFew16", 16, kFewColumns, 2, 0.22, 0.36, 1.5, 5.2, 5.2}};
// the kernel of any shape: a step of 64 is two of its own
// fp32, whose steps are 32 deep: bound by the multiplies.  Forward of 2048 x 2048, us as above: 1000 rows 464 / 155 / 82 / 85 / 104,
// 4000 rows 469 / 292 / 269 / 323 / 401, 16 000 rows 949 / 1077 / 1060 / 1258 / 1558 (141 TFLOP/s; a large library product has 154).
constexpr Tile kFloatTiles[] = {{"groupedTiles256", 256, 256, 1, 7.2, 7.0, 5.0, 4.4, 3.9},
                                {"groupedTiles128", 128, 128, 2, 2.3, 4.3, 2.5, 5.6, 4.3},
                                {"groupedTiles64", 64, 128, 2, 1.17, 2.1, 2.0, 5.6, 4.3},
                                {"groupedFew32", 32, kFewColumns, 2, 0.42, 0.63, 1.5, 5.2, 5.2},
                                {"groupedFew16", 16, kFewColumns, 2, 0.29, 0.39, 1.5, 5.2, 5.2}};
constexpr int kAllKinds = sizeof(kTiles) / sizeof(kTiles[0]);
// the kernel of any shape
constexpr Tile kAny = {"groupedAny", kAnyTile, kAnyTile, 4, 1.6, 2.2, 2.0, 3.0, 3.0};

// (how many tiles there are is known nearly: a last round that they fill a little is counted by its chance)
double timeOf(const Tile &t, double tiles, double steps, int cu_count) {
  const double rounds = tiles / (t.per_cu * (double)cu_count);
  return rounds <= 1.0 ? steps * (t.few + (t.full - t.few) * rounds) + t.end : (rounds + 0.3) * (steps * t.full + t.end);
}

struct Plan {
  int tile;        // of kTiles, or of kAnyTiles
  int slice_rows;  // backward filter; 0: whole groups
};

// Tiles of `m` rows that rows in groups will make, more or less: half a tile is lost in every group that has rows.
double rowTiles(const Problem &p, int m) {
  const double filled = std::min(p.rows, p.groups);
  return std::max(filled, (double)p.rows / m + 0.5 * filled);
}

// The tile of `kinds` that takes least, forward or for backward data.
int planRows(const Problem &p, const Tile *tiles, int kinds, int cu_count) {
  const bool forward = p.which == MLUOP_EXT_GROUPED_FORWARD;
  const int depth = forward ? p.ci : p.co, columns = forward ? p.co : p.ci;
  const double bytes = (double)std::min(p.rows, p.groups) * p.ci * p.co * elementBytes(p.type);
  const int step = 128 / elementBytes(p.type);
  int best = 0;
  double least = 0;
  for (int i = 0; i < kinds; ++i) {
    const Tile &t = tiles[i];
    const double us =
        std::max(timeOf(t, rowTiles(p, t.m) * tilesOf(columns, t.n), tilesOf(depth, step), cu_count),
                 bytes * 1e-6 / (forward ? t.forward : t.data));
    if (i == 0 || us < least) {
      least = us;
      best = i;
    }
  }
  return best;
}

// Tile and slices of the backward filter: more slices fill the GPU, and cost their partial sums a way to memory and back.
double planSlices(const Problem &p, const Tile &t, int cu_count, int *slice_rows) {
  const double tiles = (double)tilesOf(p.ci, t.m) * tilesOf(p.co, t.n);
  const double mean = (double)p.rows / p.groups;
  const int step = 128 / elementBytes(p.type);
  double least = timeOf(t, tiles * p.groups, mean / step + 0.5, cu_count);
  *slice_rows = 0;
  for (int64_t slices = 2; slices <= 1024; slices *= 2) {
    const int64_t rows = (p.rows / slices + step) / step * step;
    if (rows < 2 * step || rows >= p.rows) break;
    const double all = (double)mostRaggedTiles(p.rows, p.groups, rows);
    const double bytes = all * p.ci * p.co * 8.0;
    if (bytes > 2.5e9) break;
    const double us = timeOf(t, tiles * all, (double)rows / step, cu_count) + bytes / 4.0e6 + 5.0;
    if (us < least) {
      least = us;
      *slice_rows = (int)rows;
    }
  }
  return least;
}

Plan planFilter(const Problem &p, const Tile *tiles, int kinds, int cu_count) {
  Plan best = {0, 0};
  double least = 0;
  for (int i = 0; i < kinds; ++i) {
    int slice;
    const double us = planSlices(p, tiles[i], cu_count, &slice);
    if (i == 0 || us < least) {
      least = us;
      best = {i, slice};
    }
  }
  return best;
}

// Whether the kernels of whole 16-byte pieces take this, as far as its sizes say: then its plan does not depend on its
// addresses, and neither does its workspace.
int pieceOf(const Problem &p) { return 16 / elementBytes(p.type); }
bool wholeSizes(const Problem &p) {
  return p.groups < kStartsInLds && p.ci % pieceOf(p) == 0 && p.co % pieceOf(p) == 0;
}
bool wholePieces(const Problem &p) {
  auto whole = [&](const void *at, int64_t stride) {
    return alignedTo(at, 16) && stride % pieceOf(p) == 0 && stride < ((int64_t)1 << 20);
  };
  return wholeSizes(p) && whole(p.left, p.left_stride) && whole(p.right, p.right_stride) && alignedTo(p.out, 16);
}

Plan planFilter(const Problem &p, int cu_count) {
  if (!wholeSizes(p)) return planFilter(p, &kAny, 1, cu_count);
  return planFilter(p, p.type == MLUOP_DTYPE_FLOAT ? kFloatTiles : kTiles, kTileKinds, cu_count);
}

template <typename T>
hipError_t sumSlices(const LaunchCtx &lc, const Problem &p, const Args &a) {
  const int64_t filter = (int64_t)p.ci * p.co;
  T *out = static_cast<T *>(p.out);
  lc.begin("groupedSumSlices");
  if (filter % 4 == 0 && alignedTo(out, 16))
    groupedSumSlices<T, 4><<<dim3((unsigned)((filter + 255) / 256), p.groups), 256, 0, lc.stream>>>(a, out);
  else
    groupedSumSlices<T, 1><<<dim3((unsigned)((filter + 63) / 64), p.groups), 256, 0, lc.stream>>>(a, out);
  lc.end();
  return hipGetLastError();
}

template <typename T, int MODE>
hipError_t launchAny(const LaunchCtx &lc, const Problem &p, const Args &a) {
  const unsigned across = tilesOf(MODE == kBackwardData ? p.ci : p.co, kAnyTile);
  const dim3 grid = MODE == kBackwardFilter ? dim3((unsigned)a.blocks, across, tilesOf(p.ci, kAnyTile))
                                            : dim3((unsigned)mostRaggedTiles(p.rows, p.groups + 2, kAnyTile), across, 1);
  lc.begin(kAny.name);
  groupedAny<T, MODE><<<grid, kAnyThreads, 0, lc.stream>>>(static_cast<const T *>(p.left), static_cast<const T *>(p.right), a,
                                                           static_cast<T *>(p.out));
  lc.end();
  if (MODE == kBackwardFilter && a.slice_rows > 0) return sumSlices<T>(lc, p, a);
  return hipGetLastError();
}

template <typename T, int MODE, int TILE, int WM, int WN>
hipError_t launchTiles(const LaunchCtx &lc, const Problem &p, Args a, int cu_count) {
  constexpr int BM = kTiles[TILE].m, BN = kTiles[TILE].n;
  constexpr size_t kLds = (size_t)2 * (BM + BN) * 128;
  static_assert((kLds + kStartsInLds * 4 + kRankedGroups * 2) * kTiles[TILE].per_cu <= 160 * 1024, "LDS of a CU");
  auto kernel = groupedTiles<T, MODE, BM, BN, WM, WN>;
  const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds);
  if (allowed != hipSuccess) return allowed;
  const int64_t tiles_n = tilesOf(MODE == kBackwardData ? p.ci : p.co, BN);
  int64_t works;
  if (MODE == kBackwardFilter) {
    const int64_t per_block = tilesOf(p.ci, BM) * tiles_n;
    works = per_block >= 8 ? (per_block + 7) / 8 * 8 * a.blocks : per_block * a.blocks;
  } else {
    works = (mostRaggedTiles(p.rows, p.groups + 2, BM) * tiles_n + 7) / 8 * 8;
  }
  if (works > INT32_MAX / 2) return hipErrorInvalidValue;
  a.works = (int)works;
  // as many workgroups as the GPU holds at once, in whole rounds of the XCDs
  const int64_t stay = std::max<int64_t>((int64_t)kTiles[TILE].per_cu * cu_count / 8, 1) * 8;
  lc.begin(kTiles[TILE].name);
  kernel<<<(unsigned)std::min((works + 7) / 8 * 8, stay), WM * WN * 64, kLds, lc.stream>>>(
      static_cast<const T *>(p.left), static_cast<const T *>(p.right), a, static_cast<T *>(p.out));
  lc.end();
  if (MODE == kBackwardFilter && a.slice_rows > 0) return sumSlices<T>(lc, p, a);
  return hipGetLastError();
}

template <typename T, int MODE, int BM>
hipError_t launchFew(const LaunchCtx &lc, const Problem &p, const Args &a) {
  constexpr size_t kLds = (size_t)kFewStages * (BM + kFewColumns) * 128;
  auto kernel = groupedFew<T, MODE, BM>;
  const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds);
  if (allowed != hipSuccess) return allowed;
  const int64_t tiles_n = tilesOf(MODE == kBackwardData ? p.ci : p.co, kFewColumns);
  lc.begin(BM == 32 ? kTiles[3].name : kTiles[4].name);
  const int64_t works = (mostRaggedTiles(p.rows, p.groups + 2, BM) * tiles_n + 7) / 8 * 8;
  if (works > INT32_MAX / 2) return hipErrorInvalidValue;
  kernel<<<(unsigned)works, kFewWaves * 64, kLds, lc.stream>>>(
      static_cast<const T *>(p.left), static_cast<const T *>(p.right), a, static_cast<T *>(p.out));
  lc.end();
  return hipGetLastError();
}

template <typename T, int MODE>
hipError_t launchPieces(const LaunchCtx &lc, const Problem &p, const Args &a, int cu_count) {
  const int tile = MODE == kBackwardFilter ? planFilter(p, cu_count).tile
                                           : planRows(p, sizeof(T) == 4 ? kFloatTiles : kTiles, kAllKinds, cu_count);
  if constexpr (MODE != kBackwardFilter) {
    if (tile == 3) return launchFew<T, MODE, 32>(lc, p, a);
    if (tile == 4) return launchFew<T, MODE, 16>(lc, p, a);
  }
  switch (tile) {
    case 0: return launchTiles<T, MODE, 0, 2, 4>(lc, p, a, cu_count);
    case 1: return launchTiles<T, MODE, 1, 2, 2>(lc, p, a, cu_count);
    default: return launchTiles<T, MODE, 2, 2, 2>(lc, p, a, cu_count);
  }
}

template <typename T>
hipError_t launchOf(const LaunchCtx &lc, const Problem &p, const Args &a, int cu_count) {
  if (wholePieces(p)) switch (p.which) {
      case MLUOP_EXT_GROUPED_FORWARD: return launchPieces<T, kForward>(lc, p, a, cu_count);
      case MLUOP_EXT_GROUPED_BACKWARD_DATA: return launchPieces<T, kBackwardData>(lc, p, a, cu_count);
      default: return launchPieces<T, kBackwardFilter>(lc, p, a, cu_count);
    }
  switch (p.which) {
    case MLUOP_EXT_GROUPED_FORWARD: return launchAny<T, kForward>(lc, p, a);
    case MLUOP_EXT_GROUPED_BACKWARD_DATA: return launchAny<T, kBackwardData>(lc, p, a);
    default: return launchAny<T, kBackwardFilter>(lc, p, a);
  }
}

}  // namespace

size_t workspaceBytes(const Problem &p, int cu_count) {
  if (p.which != MLUOP_EXT_GROUPED_BACKWARD_FILTER) return 0;
  const int slice = planFilter(p, cu_count).slice_rows;
  if (slice == 0) return 0;
  return (size_t)mostRaggedTiles(p.rows, p.groups, slice) * p.ci * p.co * sizeof(float);
}

hipError_t launch(const LaunchCtx &lc, const Problem &p, int cu_count, void *workspace) {
  Args a = {p.rows, p.groups, p.ci, p.co, p.starts, p.left_stride, p.right_stride, 0, 0, 0, 0, nullptr};
  if (p.which == MLUOP_EXT_GROUPED_BACKWARD_FILTER) {
    a.slice_rows = planFilter(p, cu_count).slice_rows;
    a.most_slices = a.slice_rows > 0 ? (int)mostRaggedTiles(p.rows, p.groups, a.slice_rows) : 0;
    a.blocks = a.slice_rows > 0 ? a.most_slices : p.groups;
    a.partial = static_cast<float *>(workspace);
  }
  if (p.type == MLUOP_DTYPE_HALF) return launchOf<_Float16>(lc, p, a, cu_count);
  if (p.type == MLUOP_DTYPE_BFLOAT16) return launchOf<__bf16>(lc, p, a, cu_count);
  return launchOf<float>(lc, p, a, cu_count);
}

}  // namespace grouped_matmul
}  // namespace mluop
