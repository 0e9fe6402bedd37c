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
