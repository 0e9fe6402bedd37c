// The weight and the bias of a norm, a value of each for every channel, in one of the floating types or left out, and where
// their gradients go.
#ifndef MLUOP_AMD_CORE_CHANNEL_PARAMS_H_
#define MLUOP_AMD_CORE_CHANNEL_PARAMS_H_

#include <hip/hip_runtime.h>

#include "core/elements.h"

namespace mluop {

struct ChannelParams {
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

}  // namespace mluop

#endif  // MLUOP_AMD_CORE_CHANNEL_PARAMS_H_
