// Kernels of the products grouped by expert: y_r = x_r W_g, dx_r = dy_r W_g^T and dW_g = sum over the rows r of a group of
// x_r^T dy_r, on matrix cores with fp32 sums and one rounding.  A tile of rows never crosses a group's end.
//   groupedTiles  rows in whole 16-byte pieces; bound by the matrix cores and, long and large, by the power they draw (the same
//                 product of zeros is faster).  32 768 rows, 8 x 2048 x 8192 bf16: forward 1.00 ms (1.10 PFLOP/s), backward data
//                 0.95 (1.16), filter gradient 0.87 (1.26), where a large library product has 1.24.
//   groupedFew    the same with few rows a group or few tiles; bound by the filters' way from memory: 12 rows of ten of 32
//                 experts, 1024 x 2048 bf16 (42 MB) 9.6 us, 4.4 TB/s with what a launch costs.
//   groupedAny    any shape and stride; bound by the step from load to LDS to multiply, some 2 us of 64.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

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
  int slice_rows;   // backward filter: rows of a slice; 0: a group's rows are one slice
  int blocks;       // backward filter: slices there can be,
  int slots;        // and how many there can be of groups of more than one, whose sums go to `partial`
  int works;        // numbers of works (some of which may not be there)
  int first_block;  // of the launch, of all that its kernel has
  int wide;         // of tiles of rows: an XCD's workgroups, whose last round is left for smaller tiles where they fill a quarter
                    // of it or less; or 0
  bool streamed;    // results go past the caches
  float *partial;   // backward filter: sums [slot, ci, co]
};

// A slice of a group's rows.  A group of few rows, or none, is one slice, whose sums are its result; the slices of the others
// have slots of partial sums, side by side, which groupedSumSlices adds up.
struct Slice {
  int group;  // -1: there is no such slice
  int first, rows;
  int slot;   // -1: the result
};
__device__ __forceinline__ int slicesOf(int rows, int slice_rows) {
  return rows <= slice_rows ? 1 : (rows - 1) / slice_rows + 1;
}
// By whole waves; the answer is the same in all lanes.
__device__ __forceinline__ Slice findSlice(const int32_t *starts, const Args &a, int number) {
  Slice s = {-1, 0, 0, -1};
  if (a.slice_rows == 0) {
    if (number >= a.groups) return s;
    s.group = number;
    segmentRows(starts, a.rows, number, &s.first, &s.rows);
    return s;
  }
  const int lane = threadIdx.x & 63;
  int before = 0, slots_before = 0;
  for (int base = 0; base < a.groups; base += 64) {
    int first = 0, count = 0, slices = 0;
    if (base + lane < a.groups) {
      segmentRows(starts, a.rows, base + lane, &first, &count);
      slices = slicesOf(count, a.slice_rows);
    }
    const int slots = slices > 1 ? slices : 0;
    const int upto = before + waveInclusiveScan(slices), slots_upto = slots_before + waveInclusiveScan(slots);
    const unsigned long long behind = __ballot(number < upto);
    if (behind != 0) {
      const int l = __ffsll((long long)behind) - 1;
      const int own = __builtin_amdgcn_readlane(slices, l), in_group = number - (__builtin_amdgcn_readlane(upto, l) - own);
      const int slot = __builtin_amdgcn_readlane(slots_upto, l) - own + in_group;
      // (starts that overlap can add up to more than an int holds, or than there are slots)
      if ((uint32_t)in_group >= (uint32_t)own || (own > 1 && (uint32_t)slot >= (uint32_t)a.slots)) return s;
      s.group = base + l;
      s.first = __builtin_amdgcn_readlane(first, l) + in_group * a.slice_rows;
      s.rows = __builtin_amdgcn_readlane(count, l) - in_group * a.slice_rows;
      if (s.rows > a.slice_rows) s.rows = a.slice_rows;
      if (own > 1) s.slot = slot;
      return s;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
    slots_before = __builtin_amdgcn_readlane(slots_upto, 63);
  }
  return s;
}

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
  bool result = true;  // and not partial sums
  if (kFilter) {
    m0 = blockIdx.z * kAnyTile;
    extent = a.ci - m0;
    const Slice slice = findSlice(a.starts, a, a.first_block + (int)blockIdx.x);
    if (slice.group < 0) return;
    group = slice.group;
    result = slice.slot < 0;
    out_row = (int64_t)(result ? group : slice.slot) * a.ci + m0;
    depth = slice.rows;
    l = left + slice.first * a.left_stride + m0;
    r = right + slice.first * a.right_stride + n0;
  } else {
    const RaggedTile t = findRaggedTile<true>(a.starts, a.rows, a.groups, kAnyTile, a.first_block + (int)blockIdx.x);
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
// reduction's part i / 4, and lane j receives result j of the four parts), fp32 ones are read one by one.  Either way rows are a
// multiple of the banks apart, and their 16-byte pieces are permuted by row so that the lanes of a read meet all banks; the
// loads permute, since a lane's place in LDS is fixed.

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
  bool there, partial;       // partial: sums of a slice
  int extent, width, depth;  // results of the tile that there are, and the reduction
  const T *left, *right;
  int64_t out;               // element of the result's (or the partial sums') first
};

// Tile number `tile` of total_m by tiles_n: bands of four by all columns, so that tiles side by side in number share operands.
__device__ __forceinline__ void placeOfTile(int tile, int total_m, int tiles_n, int *row, int *column) {
  constexpr int kBand = 4;
  const int band = tile / (kBand * tiles_n), in_band = tile - band * (kBand * tiles_n);
  const int height = min(total_m - band * kBand, kBand);
  *column = in_band / height;
  *row = band * kBand + in_band % height;
}

// Tiles of rows: workgroups go to the eight XCDs in turn, and so do the numbers; an XCD has a run of tiles that share
// operands in its L2.
struct RowTiles {
  int total_m, tiles_n;
  int each, kept;  // numbers of an XCD: all, and those in front of a last round that is left for smaller tiles
};
template <int BM>
__device__ __forceinline__ RowTiles rowTilesOf(const int32_t *starts, const Args &a, int tiles_n) {
  RowTiles all;
  all.total_m = raggedTiles<true>(starts, a.rows, a.groups, BM);
  all.tiles_n = tiles_n;
  all.each = all.kept = (all.total_m * tiles_n + 7) / 8;
  if (a.wide > 0 && all.each % a.wide <= a.wide / 4) all.kept -= all.each % a.wide;
  return all;
}
// Number `in_xcd` of an XCD, and which of the tiles of columns.
template <int BM>
__device__ __forceinline__ RaggedTile tileOfRows(const RowTiles &all, int xcd, int in_xcd, const int32_t *starts, const Args &a,
                                                 int *column) {
  const int tile = xcd * all.each + in_xcd;
  if (in_xcd >= all.each || tile >= all.total_m * all.tiles_n) {
    RaggedTile none = {};
    none.segment = -1;
    return none;
  }
  int row;
  placeOfTile(tile, all.total_m, all.tiles_n, &row, column);
  return findRaggedTile<true>(starts, a.rows, a.groups, BM, row);
}

// In which order a workgroup takes its works (in LDS; NULL: by number).
struct Order {
  const uint16_t *longest;  // blocks (groups, or slices of their rows) by falling length
  const uint16_t *taken;    // or NULL: this workgroup's share of what does not fill a round of its XCD, pairs of a place in
                            // `longest` and a tile of the XCD's
  int whole;                // rounds that an XCD's tiles of every block make
  int blocks;               // that there are
};
// Of `tiles` tiles of a block every XCD has an eighth, tiles that lie side by side;
// where eighths are of different sizes, the next block has them turned by one XCD.
__device__ __forceinline__ int eighthFrom(int tiles, int eighth) { return (int)((int64_t)tiles * eighth >> 3); }
__device__ __forceinline__ int eighthOf(int xcd, int block) { return (xcd + block) & 7; }

constexpr int kStartsInLds = 2048, kRanked = 256, kSharedBlocks = 64, kEndSteps = 3;
constexpr int kShared = 1024;  // blocks x workgroups of an XCD

// Groups are of very different lengths, and rounds of works of different lengths wait for whoever has most of the long ones.
// So every workgroup works out who takes what: block by block, the longest first, whose tiles go to those workgroups of
// the XCD that have least.  A lane stands for a workgroup; keys are steps of work so far (a tile's beginning and end take some
// kEndSteps) above the lane's number, so that no two are the same.  To `taken`; returns how many.
__device__ __forceinline__ int shareOut(const Order &order, const int *lengths, int step, int tiles, int wide, uint16_t *taken) {
  const int lane = threadIdx.x & 63, own = blockIdx.x >> 3, xcd = blockIdx.x & 7, behind = order.whole * wide;
  const int rows = lane < order.blocks ? lengths[order.longest[lane]] : 0;
  const uint32_t cost = (uint32_t)((rows + step - 1) / step + kEndSteps) << 6;
  uint32_t key = lane < wide ? (uint32_t)lane : ~0u;
  auto rankAmong = [&](auto n) {
    int rank = 0;
#pragma unroll
    for (int o = 0; o < decltype(n)::value; ++o) rank += (uint32_t)__builtin_amdgcn_readlane((int)key, o) < key ? 1 : 0;
    return rank;
  };
  int count = 0;
  for (int b = 0; b < order.blocks; ++b) {
    const int rank = wide > 32 ? rankAmong(std::integral_constant<int, 64>()) : rankAmong(std::integral_constant<int, 32>());
    const int eighth = eighthOf(xcd, b);
    const bool takes = lane < wide && behind + rank < eighthFrom(tiles, eighth + 1) - eighthFrom(tiles, eighth);
    if (takes && lane == own) {
      taken[2 * count] = (uint16_t)b;
      taken[2 * count + 1] = (uint16_t)(behind + rank);
    }
    count += __builtin_amdgcn_readlane(takes ? 1 : 0, own);
    if (takes) key += (uint32_t)__builtin_amdgcn_readlane((int)cost, b);
  }
  return count;
}

// Work number `number` of args.works, from the starts in LDS.  Workgroups go to the eight XCDs in turn, and so do the
// numbers; those of an XCD take tiles that share operands in its L2.
template <typename T, int MODE, int BM, int BN>
__device__ __forceinline__ Work<T> workOf(int number, int works, const int32_t *starts, const Order &order, const RowTiles &tiles,
                                          const Args &a, const T *left, const T *right) {
  Work<T> w;
  w.there = w.partial = false;
  w.extent = w.width = w.depth = 0;
  w.left = left;
  w.right = right;
  w.out = 0;
  if (number >= works) return w;
  const int columns = MODE == kBackwardData ? a.ci : a.co;
  int in_xcd = number >> 3, n0;
  if (MODE == kBackwardFilter) {
    const int tiles_n = (columns + BN - 1) / BN, per_block = (a.ci + BM - 1) / BM * tiles_n;
    const int xcd = blockIdx.x & 7, wide = gridDim.x >> 3;
    int block, tile;
    if (order.taken != nullptr) {
      const int in_rest = number - order.blocks * order.whole;
      if (in_rest < 0) {
        block = number / order.whole;
        tile = (number - block * order.whole) * wide + (blockIdx.x >> 3);
      } else {
        block = __builtin_amdgcn_readfirstlane(order.taken[2 * in_rest]);
        tile = __builtin_amdgcn_readfirstlane(order.taken[2 * in_rest + 1]);
      }
      tile += eighthFrom(per_block, eighthOf(xcd, block));
    } else {
      // (every second round of the workgroups backwards: who had a long one has a short one next)
      const int round = in_xcd / wide;
      if (order.longest != nullptr && (round & 1) != 0)
        in_xcd = 2 * round * wide + min(wide, (works >> 3) - round * wide) - 1 - in_xcd;
      // (of eight blocks an XCD has as many tiles as there are of one: from its own eighth on, and around)
      const int eight = in_xcd / per_block;
      tile = eighthFrom(per_block, xcd) + in_xcd - eight * per_block;
      if (tile >= per_block) tile -= per_block;
      const int eighth = (int)((8 * (int64_t)tile + 7) / per_block);
      block = 8 * eight + ((eighth - xcd) & 7);
    }
    if (block >= a.blocks) return w;
    if (order.longest != nullptr) block = __builtin_amdgcn_readfirstlane(order.longest[block]);
    Slice slice = findSlice(starts, a, block);
    if (slice.group < 0) return w;
    if (a.slice_rows == 0) {  // (read from LDS, and the same in all lanes)
      slice.first = __builtin_amdgcn_readfirstlane(slice.first);
      slice.rows = __builtin_amdgcn_readfirstlane(slice.rows);
    }
    int m0;
    placeOfTile(tile, (a.ci + BM - 1) / BM, tiles_n, &m0, &n0);
    m0 *= BM;
    n0 *= BN;
    w.depth = slice.rows;
    w.extent = a.ci - m0;
    w.left += slice.first * a.left_stride + m0;
    w.right += slice.first * a.right_stride + n0;
    w.partial = slice.slot >= 0;
    w.out = ((int64_t)(w.partial ? slice.slot : slice.group) * a.ci + m0) * columns + n0;
  } else {
    const RaggedTile t = tileOfRows<BM>(tiles, number & 7, in_xcd, starts, a, &n0);
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

template <int BM>
__device__ __forceinline__ void storeResults(u32x4 v, __amdgpu_buffer_rsrc_t to, int at, bool streamed) {
  constexpr int kPastTheCaches = 2;
  if (BM == 256 && streamed)
    __builtin_amdgcn_raw_buffer_store_b128(v, to, at, 0, kPastTheCaches);
  else
    __builtin_amdgcn_raw_buffer_store_b128(v, to, at, 0, 0);
}

// A workgroup has one tile and its two steps in LDS (256 x 256: 128 KB, one a CU): operands are read once for 256 results a
// side, which leaves L2 at 10 TB/s in all; 128 x 128 tiles of the same product need twice that and reach 0.8 of the rate.
// Workgroups stay: each takes the works blockIdx.x, blockIdx.x + gridDim.x, ... (or those of its order).  The first loads of
// the next are under way while the results of this one are stored.
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
  const int columns = MODE == kBackwardData ? a.ci : a.co;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Order order = {nullptr, nullptr, 0, 0};
  RowTiles tiles = {};
  int number = blockIdx.x, ahead = gridDim.x, works = a.works;
  const int per_block = (a.ci + BM - 1) / BM * ((columns + BN - 1) / BN), wide = gridDim.x >> 3;
  if (kFilter && a.blocks * (int64_t)per_block > gridDim.x && a.blocks <= (a.slice_rows == 0 ? kRanked : kSharedBlocks)) {
    // more than one round, and few enough blocks for everybody to rank them
    __shared__ int s_lengths[kRanked], s_count;
    __shared__ uint16_t s_longest[kRanked], s_taken[2 * kSharedBlocks];
    for (int b = wave; b < a.blocks; b += kWaves) {
      const Slice slice = findSlice(s_starts, a, b);
      if (lane == 0) s_lengths[b] = slice.group >= 0 ? slice.rows : -1;
    }
    __syncthreads();
    int there = 0;
    for (int base = 0; base < a.blocks; base += kWaves * 64) {
      const int b = base + threadIdx.x;
      const int length = b < a.blocks ? s_lengths[b] : -1;
      int place = 0;
      there = 0;
      for (int o = 0; o < a.blocks; ++o) {
        const int other = s_lengths[o];
        place += other > length || (other == length && o < b) ? 1 : 0;
        there += other >= 0 ? 1 : 0;
      }
      if (b < a.blocks) s_longest[place] = (uint16_t)b;
    }
    __syncthreads();
    order.longest = s_longest;
    order.blocks = __builtin_amdgcn_readfirstlane(there);
    if (wide <= 64 && a.blocks <= kSharedBlocks && a.blocks * wide <= kShared) {
      order.whole = per_block / 8 / wide;
      if (threadIdx.x < 64) {
        const int count = per_block % (8 * wide) == 0 ? 0 : shareOut(order, s_lengths, kDepth<T>, per_block, wide, s_taken);
        if (threadIdx.x == 0) s_count = count;
      }
      __syncthreads();
      order.taken = s_taken;
      number = 0;
      ahead = 1;
      works = order.blocks * order.whole + __builtin_amdgcn_readfirstlane(s_count);
    }
  }
  if (!kFilter) {
    tiles = rowTilesOf<BM>(s_starts, a, (columns + BN - 1) / BN);
    works = min(works, 8 * tiles.kept);
  }
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const char *x_tile = s_tiles, *y_tile = s_tiles + 2 * Left::kBytes;

  // A step has kSlots slots of TN multiplies each.  In slot n the left fragment of slot n + 2 is read, and in the first half
  // the right ones of the second.  In the last two slots they are those of the next step: in front of them everybody's
  // loads are waited for and everybody has read this step's buffer, which the loads of the step after next then
  // fill, kAtOnce a slot.
  constexpr int kSlots = 2 * TM, kLoads = Left::kLoads + Right::kLoads, kAtOnce = (2 * kLoads + kSlots - 1) / kSlots;
  static_assert(TM >= 2 && kAtOnce * (kSlots - 2) >= kLoads, "all loads are requested in front of the slots that wait for them");
  static_assert(TN % 2 == 0, "columns are stored two blocks at once");
  // (partial sums of 2-byte types take twice as many: the wait is for some of them too)
  constexpr int kStores = sizeof(T) == 2 ? TM * TN / 2 : TM * TN;
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

  bool stored = false;  // behind the loads of the work's first step there are kStores stores
  Work<T> work = workOf<T, MODE, BM, BN>(number, works, s_starts, order, tiles, a, left, right);
  begin(work);
  while (work.there) {
    number += ahead;
    const Work<T> following = workOf<T, MODE, BM, BN>(number, works, s_starts, order, tiles, a, left, right);
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
      int buffer = 0, left_over = work.depth - kDepth<T>;
      for (int step = 0; step < steps; ++step) {
#pragma unroll
        for (int n = 0; n < kSlots; ++n) {
          if (n == kSlots - 2) {
            stepBarrier();
            left_over -= kDepth<T>;
            x.next(left_over);
            y.next(left_over);
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
    const bool partial = kFilter && work.partial;
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
          storeResults<BM>(__builtin_bit_cast(u32x4, acc[i][j]), to, at, a.streamed && !partial);
        }
        continue;
      }
      if constexpr (sizeof(T) == 2) {
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
          storeResults<BM>(u32x4{lo.x, hi.x, lo.y, hi.y}, to, at, a.streamed);
        }
      }
    }
    stored = true;
    work = following;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// One tile a workgroup, and STAGES steps of both sides on their way: for few rows or tiles, where the filters are what is read,
// and for the last round that 256 x 256 tiles leave (REST: a quarter of such a tile each).  The kernel above has one step under
// way, which a product that takes less than a way from memory for a step waits for again and again: 48 tiles of 64 steps left
// over took 60 us in tiles of 128 x 128 of its own.
constexpr int kRestStages = 4, kFewWaves = 4;

template <typename T, int MODE, int BM, int BN, int WM, int WN, int STAGES, bool REST>
__global__ __launch_bounds__(kFewWaves * 64) void groupedFew(const T *__restrict__ left, const T *__restrict__ right, Args a,
                                                             T *__restrict__ out) {
  static_assert(WM * WN == kFewWaves, "waves");
  typedef Operand<T, true, BM, kFewWaves> Left;
  typedef Operand<T, MODE == kBackwardData, BN, kFewWaves> Right;
  typedef typename Fragment<T>::type fragment;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16, kLoads = Left::kLoads + Right::kLoads, kWhole = REST ? 2 : 1;
  static_assert((STAGES - 2) * kLoads <= 63, "what a wait can count");
  extern __shared__ __attribute__((aligned(1024))) char s_tiles[];

  const int columns = MODE == kBackwardData ? a.ci : a.co;
  const int block = a.first_block + (int)blockIdx.x;  // (of an XCD as blockIdx.x is: launches begin at multiples of eight)
  int n0, in_xcd = block >> 3;
  const RowTiles tiles = rowTilesOf<BM * kWhole>(a.starts, a, (columns + BN * kWhole - 1) / (BN * kWhole));
  if (REST) in_xcd = tiles.kept + in_xcd / 4;
  RaggedTile t = tileOfRows<BM * kWhole>(tiles, block & 7, in_xcd, a.starts, a, &n0);
  if (t.segment < 0) return;
  n0 *= BN * kWhole;
  if (REST) {
    const int quarter = block >> 3 & 3, down = (quarter >> 1) * BM;
    n0 += (quarter & 1) * BN;
    if (down >= t.rows || n0 >= columns) return;
    t.first += down;
    t.rows = min(t.rows - down, BM);
  }
  const int group = t.segment - 1, width = columns - n0;
  const bool inside = group >= 0 && group < a.groups;
  const int depth = inside ? (MODE == kForward ? a.ci : a.co) : 0;
  Left x(left + t.first * a.left_stride, a.left_stride, t.rows, s_tiles);
  Right y(right + (int64_t)(inside ? group : 0) * a.ci * a.co + (MODE == kForward ? (int64_t)n0 : (int64_t)n0 * a.co),
          a.right_stride, width, s_tiles + STAGES * Left::kBytes);
  auto request = [&](int left_over, int buffer) {
    x.next(left_over);
    y.next(left_over);
#pragma unroll
    for (int u = 0; u < Left::kLoads; ++u) x.request(u, buffer);
#pragma unroll
    for (int u = 0; u < Right::kLoads; ++u) y.request(u, buffer);
  };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  float4v acc[TM][TN] = {};
  if (depth > 0) {
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) request(depth - s * kDepth<T>, s);
    int buffer = 0, fill = STAGES - 1;
    for (int k0 = 0; k0 < depth; k0 += kDepth<T>) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * kLoads) : "memory");
      // (past the end the loads give zeros, so that their number stays what is waited for)
      request(depth - k0 - (STAGES - 1) * kDepth<T>, fill);
      const char *x_tile = s_tiles + buffer * Left::kBytes, *y_tile = s_tiles + STAGES * Left::kBytes + buffer * Right::kBytes;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        fragment ys[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) ys[j] = Right::fragment(y_tile + Right::place(wn + j * 16, half));
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const fragment xs = Left::fragment(x_tile + Left::place(wm + i * 16, half));
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = Fragment<T>::mma(ys[j], xs, acc[i][j]);
        }
      }
      buffer = buffer + 1 == STAGES ? 0 : buffer + 1;
      fill = fill + 1 == STAGES ? 0 : fill + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = wm + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = wn + j * 16 + (lane >> 4) * 4;
      const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      if (m < t.rows && n < width) storeFloats<T, 4>(out + (int64_t)(t.first + m) * columns + n0 + n, v);
    }
  }
}

// Adds up the slices of every group that has several: a workgroup has 64 V results, whose slices its four waves share.
template <typename T, int V>
__global__ __launch_bounds__(256) void groupedSumSlices(Args a, T *__restrict__ out) {
  constexpr int kShares = 4, kAhead = 4;
  __shared__ float s_sum[kShares][64 * V];
  const int64_t filter = (int64_t)a.ci * a.co;
  const int group = blockIdx.y, lane = threadIdx.x & 63, share = threadIdx.x >> 6;
  int in_group, rows, first = 0;
  segmentRows(a.starts, a.rows, group, &in_group, &rows);
  if (rows <= a.slice_rows) return;
  for (int base = 0; base < group; base += 64) {
    int other_first, other_rows = 0;
    if (base + lane < group) segmentRows(a.starts, a.rows, base + lane, &other_first, &other_rows);
    const int slots = other_rows <= a.slice_rows ? 0 : slicesOf(other_rows, a.slice_rows);
    first += __builtin_amdgcn_readlane(waveInclusiveScan(slots), 63);
  }
  // (inside the slots, whatever the starts hold)
  first = first < 0 || first > a.slots ? a.slots : first;
  const int slices = min(slicesOf(rows, a.slice_rows), a.slots - first);
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

// ---- rows of other lengths, padded ---------------------------------------------------------
//
// Matrices of rows that are no whole 16-byte pieces, copied to such that are: blocks of from_rows x from_width elements to
// blocks of to_rows x to_width, zeros where there is nothing to copy.  A thread has 16 bytes of the destination.

struct Copy {
  const char *from;
  char *to;
  int64_t from_stride;       // bytes
  int from_rows, to_rows;    // of a block
  int from_bytes, to_bytes;  // of a row
  uint32_t pieces;           // 16 bytes each, of all the destination's rows
  bool of_groups;            // blocks are groups' filters, and those of groups without rows are not looked at
};

// `bytes` of sixteen from `from` to `to`, by the widest accesses that both are aligned for.
template <typename T>
__device__ __forceinline__ void copyBytes(char *to, const char *from, int bytes) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(to) | reinterpret_cast<uintptr_t>(from);
  if (bytes >= 16 && (all & 7) == 0) {
    reinterpret_cast<uint2 *>(to)[0] = reinterpret_cast<const uint2 *>(from)[0];
    reinterpret_cast<uint2 *>(to)[1] = reinterpret_cast<const uint2 *>(from)[1];
    return;
  }
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i)
    if (i * (int)sizeof(T) < bytes) reinterpret_cast<T *>(to)[i] = reinterpret_cast<const T *>(from)[i];
}

template <typename T>
__global__ __launch_bounds__(256) void groupedPad(Copy one, Copy two, uint32_t one_blocks, const int32_t *starts, int rows) {
  const bool second = blockIdx.x >= one_blocks;
  const Copy &c = second ? two : one;
  const uint32_t piece = (blockIdx.x - (second ? one_blocks : 0u)) * 256u + threadIdx.x, per_row = (uint32_t)c.to_bytes / 16;
  if (piece >= c.pieces) return;
  const uint32_t row = piece / per_row, at = (piece - row * per_row) * 16, block = row / (uint32_t)c.to_rows,
                 in_block = row - block * (uint32_t)c.to_rows;
  if (c.of_groups) {
    int first, count;
    segmentRows(starts, rows, (int)block, &first, &count);
    if (count == 0) return;
  }
  Vector<T, 16 / (int)sizeof(T)> v = {};
  if (in_block < (uint32_t)c.from_rows && at < (uint32_t)c.from_bytes)
    copyBytes<T>(reinterpret_cast<char *>(&v), c.from + ((int64_t)block * c.from_rows + in_block) * c.from_stride + at,
                 c.from_bytes - (int)at);
  *reinterpret_cast<Vector<T, 16 / (int)sizeof(T)> *>(c.to + (int64_t)piece * 16) = v;
}

// The results without what was padded; from and to as above, the other way round.
template <typename T>
__global__ __launch_bounds__(256) void groupedUnpad(Copy c) {
  const uint32_t piece = blockIdx.x * 256u + threadIdx.x, per_row = (uint32_t)c.to_bytes / 16;
  if (piece >= c.pieces) return;
  const uint32_t row = piece / per_row, at = (piece - row * per_row) * 16, block = row / (uint32_t)c.to_rows,
                 in_block = row - block * (uint32_t)c.to_rows;
  if (in_block >= (uint32_t)c.from_rows || at >= (uint32_t)c.from_bytes) return;
  const Vector<T, 16 / (int)sizeof(T)> v = *reinterpret_cast<const Vector<T, 16 / (int)sizeof(T)> *>(c.to + (int64_t)piece * 16);
  copyBytes<T>(const_cast<char *>(c.from) + ((int64_t)block * c.from_rows + in_block) * c.from_stride + at,
               reinterpret_cast<const char *>(&v), c.from_bytes - (int)at);
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
// The first two are groupedTiles, the others groupedFew; filter gradients take the first three, all of them groupedTiles.
// Measured (fp16 forward of a 2048 x 2048 filter, us in this order): 16 rows 39 / 18 / 15 / 12 / 12 / 8.7 / 8.5, 500 rows 42 /
// 19 / 17 / 12.5 / 13 / 15 / 24, 1000 rows 43 / 22 / 17.6 / 18.5 / 22 / 27 / 42, 4000 rows 50 / 38 / 51 / 68 / 70 / 89 / 148;
// bf16 40 000 rows 288 / 365 / 524 / - / - / 895 / 1480.
constexpr int kTileKinds = 3;
// Steps of the reduction from which on a last round that 256 x 256 tiles fill to a quarter or less is left for 128 x 128 ones.
// Its tiles take a whole round's time otherwise; an empty launch takes 2 us.  2048 columns of fp16, us of 33 / 40 / 48 tiles an
// XCD (32 workgroups) without and with this: 8 steps 37 / 36 / 38 either way, 16 steps 58 / 57 / 59 and 52 / 54 / 58, 64 steps
// 180 / 180 / 182 and 153 / 156 / 183.
constexpr int kRestSteps = 16;
// Bytes of results from which on 256 x 256 tiles are stored past the caches, which then keep the operands: 82 MB 177 -> 158 us,
// 134 MB 268 -> 250; 31 MB 34 -> 38.
constexpr double kStreamedResults = 64e6;
// Padded copies, us without and with them: 25 973 rows of 2048 x 100 fp16 112 / 35, 229 rows of 64 x 2048 x 100 99 / 32; one
// row of 16 x 1024 x 100 32 / 12, where the filter is all there is to copy; twelve rows of 32 x 100 x 2048 stay at 6.6, which
// two launches take.  Bytes a us of padded copies, and a launch of them:
constexpr double kCopied = 3.0e6, kCopyLaunch = 4.0;
// 64 filters of 2048 x 2048 for a row each: 122 / 95 / 100 / 122 / 103 / 119 / 119, and backward data, which reads their rows,
// 136 / 125 / 116 / 111 / 104 / 102 / 101.
constexpr Tile kTiles[] = {{"groupedTiles256", 256, 256, 1, 1.25, 1.65, 5.0, 4.4, 3.9},
                           {"groupedTiles128", 128, 128, 2, 0.59, 1.06, 2.5, 5.6, 4.3},
                           {"groupedTiles64", 64, 128, 2, 0.43, 0.76, 2.0, 5.4, 4.6},
                           {"groupedFew64x64", 64, 64, 2, 0.25, 0.55, 1.5, 4.4, 4.8},
                           {"groupedFew32x128", 32, 128, 2, 0.28, 0.64, 1.5, 5.2, 5.1},
                           {"groupedFew32", 32, 64, 2, 0.25, 0.40, 1.5, 4.5, 5.25},
                           {"groupedFew16", 16, 64, 2, 0.22, 0.36, 1.5, 4.5, 5.3}};
// fp32, whose steps are 32 deep: bound by the multiplies.  Forward of 2048 x 2048, us as above: 16 rows 460 / 149 / 74 / 45 /
// 44 / 27 / 19, 1000 rows 461 / 149 / 81 / 79 / 78 / 83 / 103, 4000 rows 469 / 269 / 271 / 289 / 293 / 320 / 403; 16 000 rows
// 949 in the first (141 TFLOP/s; a large library product has 154), 1077 in the second.  64 filters for a row each 931 / 527 /
// 277 / 295 / 207 / 233 / 216, backward data 927 / 519 / 269 / 285 / 220 / 239 / 216.
constexpr Tile kFloatTiles[] = {{"groupedTiles256", 256, 256, 1, 7.2, 7.0, 5.0, 4.4, 3.9},
                                {"groupedTiles128", 128, 128, 2, 2.3, 4.3, 2.5, 5.6, 4.3},
                                {"groupedTiles64", 64, 128, 2, 1.17, 2.1, 2.0, 5.4, 4.6},
                                {"groupedFew64x64", 64, 64, 2, 0.6, 1.1, 1.5, 4.4, 4.8},
                                {"groupedFew32x128", 32, 128, 2, 0.7, 1.2, 1.5, 5.1, 4.9},
                                {"groupedFew32", 32, 64, 2, 0.42, 0.63, 1.5, 4.6, 4.5},
                                {"groupedFew16", 16, 64, 2, 0.29, 0.39, 1.5, 5.0, 5.0}};
constexpr int kAllKinds = sizeof(kTiles) / sizeof(kTiles[0]);
// the kernel of any shape
constexpr Tile kAny = {"groupedAny", kAnyTile, kAnyTile, 4, 2.0, 3.3, 2.0, 3.0, 3.0};

// (how many tiles there are is known nearly: a last round that they fill a little is counted by its chance)
double timeOf(const Tile &t, double tiles, double steps, int cu_count) {
  const double rounds = tiles / (t.per_cu * (double)cu_count);
  return rounds <= 1.0 ? steps * (t.few + (t.full - t.few) * rounds) + t.end : (rounds + 0.3) * (steps * t.full + t.end);
}

struct Plan {
  int tile;        // of the tiles that were asked for
  int slice_rows;  // backward filter; 0: whole groups
};

// Tiles of `m` rows that rows in groups will make, more or less: half a tile is lost in every group that has rows.
double rowTiles(const Problem &p, int m) {
  const double filled = std::min(p.rows, p.groups);
  return std::max(filled, (double)p.rows / m + 0.5 * filled);
}

// The tile of `kinds` that takes least, forward or for backward data.
int planRows(const Problem &p, const Tile *tiles, int kinds, int cu_count, double *us_of_best = nullptr) {
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
  if (us_of_best != nullptr) *us_of_best = least;
  return best;
}

// Slots that groups of more than slice_rows rows can have: fewer than twice as many as slices that their rows fill.
int64_t mostSlots(const Problem &p, int64_t slice_rows) { return 2 * (int64_t)p.rows / slice_rows; }

// Tile and slices of the backward filter.  How long the groups are is not known here, but as a rule some are several times as
// long as the mean: a group of kLongest times that is counted with, whose tiles the end waits for.  Shorter slices take less
// time, and the sums of groups of several a way to memory and back.
double planSlices(const Problem &p, const Tile &t, int cu_count, int *slice_rows) {
  constexpr double kLongest = 3.0;
  const double tiles = (double)tilesOf(p.ci, t.m) * tilesOf(p.co, t.n), filter = (double)p.ci * p.co;
  const double filled = std::max(std::min(p.rows, p.groups), 1), mean = p.rows / filled;
  const double longest = p.groups > 1 ? std::min(kLongest * mean, (double)p.rows) : p.rows;
  const int step = 128 / elementBytes(p.type);
  auto micros = [&](double rows) {
    const double blocks = 0.5 * filled + std::max(0.5 * filled, p.rows / rows);
    const double rate = tiles * blocks > t.per_cu * 0.5 * cu_count ? t.full : t.few;
    return std::max(timeOf(t, tiles * blocks, p.rows / blocks / step + 0.5, cu_count),
                    std::min(rows, longest) / step * rate + t.end);
  };
  double least = micros(p.rows);
  *slice_rows = 0;
  for (double slices = 1.0 / 4; slices <= 1024; slices *= 2) {  // of a group of the mean length
    const int64_t rows = ((int64_t)(mean / slices) + step) / step * step;
    if (rows < 2 * step) break;
    if (rows >= p.rows) continue;
    if (mostSlots(p, rows) * filter * 4.0 > 1.5e9) break;
    const double slots = p.rows / (double)rows * std::min(1.0, mean / rows);
    const double us = micros((double)rows) + slots * filter * 8.0 / 4.0e6 + 5.0;
    if (us < least) {
      least = us;
      *slice_rows = (int)rows;
    }
  }
  return least;
}

Plan planFilter(const Problem &p, const Tile *tiles, int kinds, int cu_count, double *us_of_best = nullptr) {
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
  if (us_of_best != nullptr) *us_of_best = least;
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
  const int64_t blocks = MODE == kBackwardFilter ? a.blocks : mostRaggedTiles(p.rows, p.groups + 2, kAnyTile);
  const unsigned down = MODE == kBackwardFilter ? tilesOf(p.ci, kAnyTile) : 1;
  inLaunches(blocks, kAnyThreads, [&](int64_t first, unsigned count) {
    Args part = a;
    part.first_block = (int)first;
    lc.begin(kAny.name);
    groupedAny<T, MODE><<<dim3(count, across, down), kAnyThreads, 0, lc.stream>>>(
        static_cast<const T *>(p.left), static_cast<const T *>(p.right), part, static_cast<T *>(p.out));
    lc.end();
  });
  if (MODE == kBackwardFilter && a.slice_rows > 0) return sumSlices<T>(lc, p, a);
  return hipGetLastError();
}

// Whether tiles of m rows, as many as the groups' lengths make of them, may fill a quarter or less of an XCD's last round.
bool restMayBe(const Problem &p, int m, int64_t tiles_n, int wide) {
  const int64_t least = ((p.rows + m - 1) / m * tiles_n + 7) / 8, most = (mostRaggedTiles(p.rows, p.groups, m) * tiles_n + 7) / 8;
  const int64_t last = most / wide;  // round that may begin
  for (int64_t round = std::max<int64_t>(last - 1, 1); round <= last; ++round)
    if (std::max(least, round * wide + 1) <= std::min(most, round * wide + wide / 4)) return true;
  return false;
}

template <typename T, int MODE, int TILE, int WM, int WN>
hipError_t launchTiles(const LaunchCtx &lc, const Problem &p, Args a, int cu_count) {
  constexpr int BM = kTiles[TILE].m, BN = kTiles[TILE].n;
  constexpr size_t kLds = (size_t)2 * (BM + BN) * 128;
  static_assert((kLds + kStartsInLds * 4 + kRanked * 6 + kSharedBlocks * 4 + 4) * kTiles[TILE].per_cu <= 160 * 1024,
                "LDS of a CU");
  auto kernel = groupedTiles<T, MODE, BM, BN, WM, WN>;
  const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds);
  if (allowed != hipSuccess) return allowed;
  const int64_t tiles_n = tilesOf(MODE == kBackwardData ? p.ci : p.co, BN);
  int64_t works;
  if (MODE == kBackwardFilter) {
    works = tilesOf(p.ci, BM) * tiles_n * ((a.blocks + 7) / 8 * 8);
  } else {
    works = (mostRaggedTiles(p.rows, p.groups + 2, BM) * tiles_n + 7) / 8 * 8;
  }
  if (works > INT32_MAX / 2) return hipErrorInvalidValue;
  a.works = (int)works;
  // as many workgroups as the GPU holds at once, in whole rounds of the XCDs
  const int64_t stay = std::max<int64_t>((int64_t)kTiles[TILE].per_cu * cu_count / 8, 1) * 8;
  const int grid = (int)std::min(works, stay);
  const double results = MODE == kBackwardFilter ? (double)p.groups * p.ci * p.co
                                                 : (double)p.rows * (MODE == kForward ? p.co : p.ci);
  a.streamed = TILE == 0 && results * sizeof(T) >= kStreamedResults;
  if constexpr (MODE != kBackwardFilter && TILE == 0) {
    const int depth = MODE == kForward ? p.ci : p.co, wide = (int)(stay / 8);
    if (depth >= kRestSteps * kDepth<T> && restMayBe(p, BM, tiles_n, wide)) a.wide = wide;
  }
  lc.begin(kTiles[TILE].name);
  kernel<<<grid, WM * WN * 64, kLds, lc.stream>>>(static_cast<const T *>(p.left), static_cast<const T *>(p.right), a,
                                                  static_cast<T *>(p.out));
  lc.end();
  if constexpr (MODE != kBackwardFilter && TILE == 0) {
    if (a.wide > 0) {
      constexpr size_t kRestLds = (size_t)kRestStages * (BM + BN) / 2 * 128;
      auto rest = groupedFew<T, MODE, BM / 2, BN / 2, 2, 2, kRestStages, true>;
      const hipError_t fits = hipFuncSetAttribute(reinterpret_cast<const void *>(rest),
                                                  hipFuncAttributeMaxDynamicSharedMemorySize, (int)kRestLds);
      if (fits != hipSuccess) return fits;
      a.works = (int)std::min<int64_t>(4 * works, 8 * 4 * (a.wide / 4));
      lc.begin("groupedRest");
      rest<<<a.works, kFewWaves * 64, kRestLds, lc.stream>>>(static_cast<const T *>(p.left), static_cast<const T *>(p.right), a,
                                                  static_cast<T *>(p.out));
      lc.end();
    }
  }
  if (MODE == kBackwardFilter && a.slice_rows > 0) return sumSlices<T>(lc, p, a);
  return hipGetLastError();
}

template <typename T, int MODE, int BM, int BN, int WM, int WN, int STAGES>
hipError_t launchFew(const LaunchCtx &lc, const char *name, const Problem &p, const Args &a) {
  constexpr size_t kLds = (size_t)STAGES * (BM + BN) * 128;
  static_assert(kLds * 2 <= 160 * 1024, "two a CU");
  auto kernel = groupedFew<T, MODE, BM, BN, WM, WN, STAGES, false>;
  const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds);
  if (allowed != hipSuccess) return allowed;
  const int64_t tiles_n = tilesOf(MODE == kBackwardData ? p.ci : p.co, BN);
  const int64_t works = (mostRaggedTiles(p.rows, p.groups + 2, BM) * tiles_n + 7) / 8 * 8;
  if (works > INT32_MAX / 2) return hipErrorInvalidValue;
  inLaunches(works, kFewWaves * 64, [&](int64_t first, unsigned count) {
    Args part = a;
    part.first_block = (int)first;
    lc.begin(name);
    kernel<<<count, kFewWaves * 64, kLds, lc.stream>>>(
        static_cast<const T *>(p.left), static_cast<const T *>(p.right), part, static_cast<T *>(p.out));
    lc.end();
  });
  return hipGetLastError();
}

template <typename T, int MODE>
hipError_t launchPieces(const LaunchCtx &lc, const Problem &p, const Args &a, int cu_count) {
  const int tile = MODE == kBackwardFilter ? planFilter(p, cu_count).tile
                                           : planRows(p, sizeof(T) == 4 ? kFloatTiles : kTiles, kAllKinds, cu_count);
  if (tile == 0) return launchTiles<T, MODE, 0, 2, 4>(lc, p, a, cu_count);
  if (tile == 1) return launchTiles<T, MODE, 1, 2, 2>(lc, p, a, cu_count);
  if constexpr (MODE == kBackwardFilter) {
    return launchTiles<T, MODE, 2, 2, 2>(lc, p, a, cu_count);
  } else {
    switch (tile) {
      case 2: return launchFew<T, MODE, 64, 128, 2, 2, 3>(lc, "groupedFew64x128", p, a);
      case 3: return launchFew<T, MODE, 64, 64, 2, 2, 4>(lc, kTiles[3].name, p, a);
      case 4: return launchFew<T, MODE, 32, 128, 1, 4, 4>(lc, kTiles[4].name, p, a);
      case 5: return launchFew<T, MODE, 32, 64, 1, 4, 6>(lc, kTiles[5].name, p, a);
      default: return launchFew<T, MODE, 16, 64, 1, 4, 6>(lc, kTiles[6].name, p, a);
    }
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

// The problem with both numbers of channels in whole pieces: which of its matrices are copies, and how large.
struct Padded {
  bool takes;  // it takes less time
  Problem q;
  bool left, right, out;
  size_t left_bytes, right_bytes, out_bytes;  // in multiples of 256
};

Padded padded(const Problem &p, int cu_count) {
  Padded d = {};
  const int piece = pieceOf(p), size = elementBytes(p.type);
  d.q = p;
  d.q.ci = (p.ci + piece - 1) / piece * piece;
  d.q.co = (p.co + piece - 1) / piece * piece;
  const bool ci = d.q.ci != p.ci, co = d.q.co != p.co;
  if (wholeSizes(p) || !wholeSizes(d.q) || p.rows == 0) return d;
  const bool filter = p.which == MLUOP_EXT_GROUPED_BACKWARD_FILTER, forward = p.which == MLUOP_EXT_GROUPED_FORWARD;
  const size_t x = (size_t)p.rows * d.q.ci * size, y = (size_t)p.rows * d.q.co * size,
               w = (size_t)p.groups * d.q.ci * d.q.co * size;
  auto bytes = [](bool there, size_t n) { return there ? (n + 255) / 256 * 256 : 0; };
  d.left = filter || forward ? ci : co;
  d.right = filter ? co : true;
  d.out = filter ? true : (forward ? co : ci);
  d.left_bytes = bytes(d.left, filter || forward ? x : y);
  d.right_bytes = bytes(d.right, filter ? y : w);
  d.out_bytes = bytes(d.out, filter ? w : (forward ? y : x));
  const double moved = (double)d.left_bytes + d.out_bytes +
                       (filter ? d.right_bytes : (double)d.right_bytes * std::min(p.rows, p.groups) / p.groups);
  if (moved > 4e9 || (double)d.right_bytes > 4e9) return d;
  const Tile *tiles = p.type == MLUOP_DTYPE_FLOAT ? kFloatTiles : kTiles;
  double any, whole;
  if (filter) {
    planFilter(p, &kAny, 1, cu_count, &any);
    planFilter(d.q, tiles, kTileKinds, cu_count, &whole);
  } else {
    planRows(p, &kAny, 1, cu_count, &any);
    planRows(d.q, tiles, kAllKinds, cu_count, &whole);
  }
  // (read and written, and a launch for what is copied in front and behind)
  d.takes = whole + 2.0 * moved / kCopied + kCopyLaunch * ((d.left || d.right ? 1 : 0) + (d.out ? 1 : 0)) < any;
  return d;
}

// `blocks` blocks of rows x width elements at `at` and their padded copy.
Copy copyOf(const void *at, void *copy, int64_t stride, int64_t blocks, int rows, int padded_rows, int width,
            int padded_width, int size, bool of_groups) {
  Copy c = {};
  c.from = static_cast<const char *>(at);
  c.to = static_cast<char *>(copy);
  c.from_stride = stride * size;
  c.from_rows = rows;
  c.to_rows = padded_rows;
  c.from_bytes = width * size;
  c.to_bytes = padded_width * size;
  c.pieces = (uint32_t)(blocks * padded_rows * (c.to_bytes / 16));
  c.of_groups = of_groups;
  return c;
}

Args argsOf(const Problem &p, int cu_count, void *partial) {
  Args a = {p.rows, p.groups, p.ci, p.co, p.starts, p.left_stride, p.right_stride, 0, 0, 0, 0, 0, 0, false, nullptr};
  if (p.which == MLUOP_EXT_GROUPED_BACKWARD_FILTER) {
    a.slice_rows = planFilter(p, cu_count).slice_rows;
    a.blocks = p.groups + (a.slice_rows > 0 ? p.rows / a.slice_rows : 0);
    a.slots = a.slice_rows > 0 ? (int)mostSlots(p, a.slice_rows) : 0;
    a.partial = static_cast<float *>(partial);
  }
  return a;
}

template <typename T>
hipError_t launchPadded(const LaunchCtx &lc, const Problem &p, Padded d, int cu_count, char *workspace) {
  constexpr int kSize = (int)sizeof(T);
  const bool filter = p.which == MLUOP_EXT_GROUPED_BACKWARD_FILTER, forward = p.which == MLUOP_EXT_GROUPED_FORWARD;
  Problem &q = d.q;
  Copy copies[2] = {};
  int count = 0;
  if (d.left) {
    const bool x = filter || forward;
    q.left = workspace;
    q.left_stride = x ? q.ci : q.co;
    copies[count++] = copyOf(p.left, workspace, p.left_stride, 1, p.rows, p.rows, x ? p.ci : p.co, (int)q.left_stride, kSize,
                             false);
    workspace += d.left_bytes;
  }
  if (d.right) {
    q.right = workspace;
    q.right_stride = q.co;
    copies[count++] = filter ? copyOf(p.right, workspace, p.right_stride, 1, p.rows, p.rows, p.co, q.co, kSize, false)
                             : copyOf(p.right, workspace, p.right_stride, p.groups, p.ci, q.ci, p.co, q.co, kSize, true);
    workspace += d.right_bytes;
  }
  Copy back = {};
  if (d.out) {
    back = filter ? copyOf(p.out, workspace, p.co, p.groups, p.ci, q.ci, p.co, q.co, kSize, false)
                  : copyOf(p.out, workspace, forward ? p.co : p.ci, 1, p.rows, p.rows, forward ? p.co : p.ci,
                           forward ? q.co : q.ci, kSize, false);
    q.out = workspace;
    workspace += d.out_bytes;
  }
  if (count > 0) {
    const uint32_t one = (copies[0].pieces + 255) / 256, two = (copies[1].pieces + 255) / 256;
    lc.begin("groupedPad");
    groupedPad<T><<<one + two, 256, 0, lc.stream>>>(copies[0], copies[1], one, p.starts, p.rows);
    lc.end();
  }
  const hipError_t status = launchOf<T>(lc, q, argsOf(q, cu_count, workspace), cu_count);
  if (status != hipSuccess) return status;
  if (d.out) {
    lc.begin("groupedUnpad");
    groupedUnpad<T><<<(back.pieces + 255) / 256, 256, 0, lc.stream>>>(back);
    lc.end();
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launchAs(const LaunchCtx &lc, const Problem &p, int cu_count, void *workspace) {
  const Padded d = padded(p, cu_count);
  // (the matrices that are no copies have to be whole pieces as they are)
  auto whole = [&](const void *at, int64_t stride) {
    return alignedTo(at, 16) && stride % pieceOf(p) == 0 && stride < ((int64_t)1 << 20);
  };
  if (d.takes && (d.left || whole(p.left, p.left_stride)) && (d.right || whole(p.right, p.right_stride)) &&
      (d.out || alignedTo(p.out, 16)))
    return launchPadded<T>(lc, p, d, cu_count, static_cast<char *>(workspace));
  return launchOf<T>(lc, p, argsOf(p, cu_count, workspace), cu_count);
}

size_t partialBytes(const Problem &p, int cu_count) {
  if (p.which != MLUOP_EXT_GROUPED_BACKWARD_FILTER) return 0;
  const int slice = planFilter(p, cu_count).slice_rows;
  if (slice == 0) return 0;
  return (size_t)mostSlots(p, slice) * p.ci * p.co * sizeof(float);
}

}  // namespace

size_t workspaceBytes(const Problem &p, int cu_count) {
  const Padded d = padded(p, cu_count);
  const size_t as_it_is = partialBytes(p, cu_count);
  if (!d.takes) return as_it_is;
  return std::max(as_it_is, d.left_bytes + d.right_bytes + d.out_bytes + partialBytes(d.q, cu_count));
}

hipError_t launch(const LaunchCtx &lc, const Problem &p, int cu_count, void *workspace) {
  if (p.type == MLUOP_DTYPE_HALF) return launchAs<_Float16>(lc, p, cu_count, workspace);
  if (p.type == MLUOP_DTYPE_BFLOAT16) return launchAs<__bf16>(lc, p, cu_count, workspace);
  return launchAs<float>(lc, p, cu_count, workspace);
}

}  // namespace grouped_matmul
}  // namespace mluop
