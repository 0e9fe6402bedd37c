// Elements of the three floating types in memory and as fp32 in registers, singly and as vectors of up to 16 bytes, for
// kernels that compute in fp32 and round once when they store.
#ifndef MLUOP_AMD_CORE_ELEMENTS_H_
#define MLUOP_AMD_CORE_ELEMENTS_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "mlu_op.h"

namespace mluop {

// (in memory a vector is aligned to its own length, at most 16 bytes)
template <typename T, int V>
struct alignas(sizeof(T) * V <= 16 ? sizeof(T) * V : 16) Vector {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void loadFloats(const T *from, float (&to)[V]) {
  const Vector<T, V> packed = *reinterpret_cast<const Vector<T, V> *>(from);
#pragma unroll
  for (int i = 0; i < V; ++i) to[i] = (float)packed.v[i];
}

template <typename T, int V>
__device__ __forceinline__ void storeFloats(T *to, const float (&from)[V]) {
  Vector<T, V> packed;
#pragma unroll
  for (int i = 0; i < V; ++i) packed.v[i] = (T)from[i];
  *reinterpret_cast<Vector<T, V> *>(to) = packed;
}

// The same past the caches (16-byte pieces of it): for results that the kernel behind this one does not read at once.
template <typename T, int V>
__device__ __forceinline__ void streamFloats(T *to, const float (&from)[V]) {
  if constexpr (sizeof(T) * V % 16 == 0) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    struct alignas(16) Pieces {
      u32x4 piece[sizeof(T) * V / 16];
    };
    Vector<T, V> packed;
#pragma unroll
    for (int i = 0; i < V; ++i) packed.v[i] = (T)from[i];
    const Pieces pieces = __builtin_bit_cast(Pieces, packed);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * V / 16); ++i)
      __builtin_nontemporal_store(pieces.piece[i], reinterpret_cast<u32x4 *>(to) + i);
  } else {
    storeFloats<T, V>(to, from);
  }
}

// Results of so many bytes are streamed: fewer stay where the next kernel finds them in a cache.
constexpr size_t kStreamedBytes = (size_t)32 << 20;

template <typename T, int V>
__device__ __forceinline__ void storeFloats(T *to, const float (&from)[V], bool streamed) {
  if (streamed)
    streamFloats<T, V>(to, from);
  else
    storeFloats<T, V>(to, from);
}

// How the threads of a workgroup lie over rows of `channels`: V channels each, row after row; a slab of channels where a row
// has more than they take at once (blockIdx.y).
template <int V, int THREADS>
struct RowLanes {
  int across, row, rows_at_once, channel;  // row < 0: a thread without work
  __device__ explicit RowLanes(int channels) {
    const int left = channels / V - (int)blockIdx.y * THREADS;
    across = left < THREADS ? left : THREADS;
    rows_at_once = THREADS / across;
    row = (int)threadIdx.x / across;
    channel = ((int)blockIdx.y * THREADS + (int)threadIdx.x - row * across) * V;
    if (row >= rows_at_once) row = -1;
  }
};

inline bool isFloating(mluOpDataType_t t) {
  return t == MLUOP_DTYPE_FLOAT || t == MLUOP_DTYPE_HALF || t == MLUOP_DTYPE_BFLOAT16;
}
inline int elementBytes(mluOpDataType_t t) { return t == MLUOP_DTYPE_FLOAT ? 4 : 2; }

inline bool alignedTo(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace mluop

#endif  // MLUOP_AMD_CORE_ELEMENTS_H_
