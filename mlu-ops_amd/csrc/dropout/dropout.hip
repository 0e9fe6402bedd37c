// mluOpExtDropoutAdd (no counterpart in the reference): elements dropped at random, the others scaled and added to a residual.
// The mask is never stored: it is computed again wherever it is needed, from the seed, the call and the element's number.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "core/core.h"
#include "core/elements.h"
#include "mlu_op_ext.h"

namespace {

using namespace mluop;

constexpr int kThreads = 256;
constexpr int kShared = 8;         // elements that share a counter: half a word of its four each
constexpr uint32_t kSteps = 1 << 16;
constexpr int kGroups = 2;         // counters of a thread, whose elements are on their way together

// Four words for a counter of four under a key of two: Philox4x32 with ten rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011).  A round is two products of 64 bits and four exclusive ors; the
// keys are the same for all lanes and cost no vector operation.
__device__ __forceinline__ void randomWords(uint64_t low, uint64_t high, uint64_t key, uint32_t (&word)[4]) {
  uint32_t c0 = (uint32_t)low, c1 = (uint32_t)(low >> 32), c2 = (uint32_t)high, c3 = (uint32_t)(high >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)q;
    c3 = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  word[0] = c0;
  word[1] = c1;
  word[2] = c2;
  word[3] = c3;
}

// Bound by memory: 65 536 x 2048 bf16 onto a residual (805 MB) 141 us, 5.7 TB/s; 248 636 x 128 fp32 (382 MB) 68 us, its gradient
// (255 MB) 46.  Ten rounds are some 60 operations for each of 8 elements' numbers and hide behind the loads; a number of 32 bits
// for each element would be twice that.  ADD: onto the residual.  WIDE: addresses are multiples of 16 bytes.  Elements that are
// dropped are zero whatever they hold.
template <typename T, bool ADD, bool WIDE>
__global__ __launch_bounds__(kThreads) void dropoutAdd(const T *__restrict__ x, const T *__restrict__ residual, int64_t n,
                                                       uint32_t threshold, float scale, const uint64_t *__restrict__ state,
                                                       int64_t first_block, bool streamed, T *__restrict__ out) {
  const uint64_t seed = state[0], call = state[1];
  const int64_t group = (first_block + blockIdx.x) * kThreads * kGroups + threadIdx.x;
  float v[kGroups][kShared], r[kGroups][kShared];
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    const int64_t at = (group + j * kThreads) * kShared;
#pragma unroll
    for (int i = 0; i < kShared; ++i) v[j][i] = r[j][i] = 0.f;
    if (WIDE && at + kShared <= n) {
      loadFloats<T, kShared>(x + at, v[j]);
      if (ADD) loadFloats<T, kShared>(residual + at, r[j]);
    } else {
#pragma unroll
      for (int i = 0; i < kShared; ++i) {
        if (at + i < n) {
          v[j][i] = (float)x[at + i];
          if (ADD) r[j][i] = (float)residual[at + i];
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    const int64_t at = (group + j * kThreads) * kShared;
    if (at >= n) break;
    uint32_t word[4];
    randomWords((uint64_t)(group + j * kThreads), call, seed, word);
#pragma unroll
    for (int i = 0; i < kShared; ++i) {
      const uint32_t half = i % 2 == 0 ? word[i / 2] & 0xffffu : word[i / 2] >> 16;
      v[j][i] = half >= threshold ? fmaf(v[j][i], scale, r[j][i]) : r[j][i];
    }
    if (WIDE && at + kShared <= n) {
      storeFloats<T, kShared>(out + at, v[j], streamed);
    } else {
#pragma unroll
      for (int i = 0; i < kShared; ++i)
        if (at + i < n) out[at + i] = (T)v[j][i];
    }
  }
}

}  // namespace

mluOpStatus_t MLUOP_WIN_API mluOpExtDropoutAdd(mluOpHandle_t handle, mluOpDataType_t type, const void *features,
                                               const void *residual, int64_t count, double p, const int64_t *state,
                                               void *out) {
  const char *api = "[mluOpExtDropoutAdd]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  PARAM_CHECK(api, count >= 0);
  PARAM_CHECK(api, p >= 0.0 && p <= 1.0);
  if (count > ((int64_t)1 << 46)) {
    MLUOP_LOG(ERROR) << api << " At most 2^46 values are supported.";
    return MLUOP_STATUS_NOT_SUPPORTED;
  }
  PARAM_CHECK(api, count == 0 || (features != NULL && out != NULL));
  PARAM_CHECK(api, state != NULL && alignedTo(state, sizeof(int64_t)));
  DEVICE_HANDLE_CHECK(api, handle);
  if (count == 0) return MLUOP_STATUS_SUCCESS;
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  const size_t bytes = (size_t)count * elementBytes(type);
  handle->forgetNotesIn(out, bytes);
  const uint32_t threshold = (uint32_t)std::floor(p * kSteps + 0.5);
  const float scale = threshold < kSteps ? (float)((double)kSteps / (kSteps - threshold)) : 0.f;
  const mluop::LaunchCtx lc = handle->launchCtx();
  auto run = [&](auto zero, auto add, auto wide) {
    typedef decltype(zero) T;
    constexpr int64_t kBlock = kThreads * kGroups * kShared;
    inLaunches((count + kBlock - 1) / kBlock, kThreads, [&](int64_t first, unsigned blocks) {
      lc.begin("dropoutAdd");
      dropoutAdd<T, decltype(add)::value, decltype(wide)::value><<<blocks, kThreads, 0, lc.stream>>>(
          static_cast<const T *>(features), static_cast<const T *>(residual), count, threshold, scale,
          reinterpret_cast<const uint64_t *>(state), first, bytes >= kStreamedBytes, static_cast<T *>(out));
      lc.end();
    });
  };
  auto byType = [&](auto add, auto wide) {
    if (type == MLUOP_DTYPE_HALF)
      run((_Float16)0, add, wide);
    else if (type == MLUOP_DTYPE_BFLOAT16)
      run((__bf16)0.f, add, wide);
    else
      run(0.f, add, wide);
  };
  const bool wide = alignedTo(features, 16) && alignedTo(residual, 16) && alignedTo(out, 16);
  auto byWidth = [&](auto add) {
    if (wide)
      byType(add, std::true_type());
    else
      byType(add, std::false_type());
  };
  if (residual != nullptr)
    byWidth(std::true_type());
  else
    byWidth(std::false_type());
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
