// mluOpExtAdamWStep (no counterpart in the reference): one AdamW step over many tensors.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "core/core.h"
#include "core/elements.h"
#include "mlu_op_ext.h"

// A product and a sum stay two roundings, so that a step gives the bits of the same operations made one after the other.
#pragma clang fp contract(off)

namespace {

using namespace mluop;

constexpr int kThreads = 256;
constexpr int kPerThread = 8;                        // consecutive elements of a thread
constexpr int kRound = kThreads * kPerThread;        // of a workgroup at once
constexpr int kChunk = kRound;                       // elements of a workgroup
constexpr int kStateBlock = MLUOP_EXT_ADAMW_BLOCK;   // elements that share a scale: 32 lanes
constexpr int kLanesPerBlock = kStateBlock / kPerThread;
constexpr float kMostCode = 448.f, kLeastCode = 0x1p-9f;  // of e4m3
struct Hyper {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, decay, step_size, inv_root2, eps, grad_scale;
};

// Tensors of a launch: as many as 4 KB of kernel arguments hold, 65 to 106, so that only the addresses that there are have a
// place and a length is its number of chunks and what the last of them has.  (A launch of small tensors takes some 7 us: 288
// bf16 tensors of 85 000 elements in all 42 us at 56 a launch, 23 now.  A table in device memory would have to be copied
// there in front of every step, since gradients are new tensors each time.)
template <bool MASTER, bool EIGHT>
struct Tensors {
  enum { kParam, kGrad, kM, kV, kMaster, kMScale = kMaster + (MASTER ? 1 : 0), kVScale, kAddresses = kMScale + (EIGHT ? 2 : 0) };
  static constexpr int kTensors = (4096 - (int)sizeof(Hyper) - 16) / (kAddresses * 8 + 6);
  static_assert(kTensors <= 128, "two to a lane");
  void *address[kAddresses][kTensors];
  uint32_t first[kTensors + 1];  // chunk of the launch; behind the last tensor's: the number of chunks
  uint16_t last[kTensors];       // elements of the last chunk
};

template <typename T>
__device__ __forceinline__ void loadEight(const T *from, int64_t at, int n, bool whole, float (&to)[kPerThread]) {
  if (whole) {
    loadFloats<T, kPerThread>(from + at, to);
  } else {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) to[i] = i < n ? (float)from[at + i] : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void storeEight(T *to, int64_t at, int n, bool whole, const float (&from)[kPerThread]) {
  if (whole) {
    streamFloats<T, kPerThread>(to + at, from);
  } else {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (i < n) to[at + i] = (T)from[i];
  }
}

// e4m3 codes of eight elements.
__device__ __forceinline__ uint2 loadCodes(const uint8_t *from, int64_t at, int n, bool whole) {
  if (whole) return *reinterpret_cast<const uint2 *>(from + at);
  uint2 codes = make_uint2(0, 0);
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const uint32_t c = i < n ? from[at + i] : 0u;
    (i < 4 ? codes.x : codes.y) |= c << (8 * (i & 3));
  }
  return codes;
}

__device__ __forceinline__ void storeCodes(uint8_t *to, int64_t at, int n, bool whole, uint2 codes) {
  if (whole) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    __builtin_nontemporal_store(u32x2{codes.x, codes.y}, reinterpret_cast<u32x2 *>(to + at));
  } else {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (i < n) to[at + i] = (uint8_t)((i < 4 ? codes.x : codes.y) >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ void decode(uint2 codes, float scale, float (&to)[kPerThread]) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  const float2v a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.x, false);
  const float2v b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.x, true);
  const float2v c = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.y, false);
  const float2v d = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.y, true);
  const float v[kPerThread] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) to[i] = v[i] * scale;
}

// (of values that lie inside the type's range: rounded to nearest, ties to even)
__device__ __forceinline__ uint2 encode(const float (&v)[kPerThread]) {
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// Largest value of a state block's 32 lanes, in all of them.
__device__ __forceinline__ float blockMost(float v) {
  static_assert(kLanesPerBlock == 32, "half a wavefront");
  auto moved = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v = fmaxf(v, moved(v, std::integral_constant<int, 0xb1>()));   // the other of a pair
  v = fmaxf(v, moved(v, std::integral_constant<int, 0x4e>()));   // the other pair of four
  v = fmaxf(v, moved(v, std::integral_constant<int, 0x141>()));  // the other four of eight
  v = fmaxf(v, moved(v, std::integral_constant<int, 0x140>()));  // the other eight of a row of 16
  return fmaxf(v, __shfl_xor(v, 16, 64));
}

// m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g g;
// p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps), in fp32.
// States in 8 bits are e4m3 codes of m and of sqrt(v), 256 of them with one fp32 scale, (the largest magnitude) / 448:
// the root has half of v's range of exponents, so that four bits hold it.  A root that is not zero keeps the least code: as
// zero it would leave eps alone in the denominator of the next step.  The parameters take the values in front of this rounding.
// Bound by memory: 28 bytes an element with fp32 parameters, 10 with 16-bit parameters and 8-bit states.  Results go past the
// caches (nobody reads a state before the next step): 130 M bf16 parameters with masters 757 -> 676 us (5.4 TB/s, where
// a copy has 5.1), 250 M with 8-bit states 472 -> 450 us (5.6 TB/s), 33 fp32 tensors of 1.9 M elements in all 12.3 -> 10.8.
// TINY: a root below the smallest normal number counts.  The hardware's own root and reciprocal take such numbers for zero: that
// root is below 2^-63, and corrected it is lost beside an eps of 2^25 times that.  With a smaller eps (1.1e-10 in the first
// step with beta2 = 0.999, 3.6e-12 later on) root and quotient are those that are defined.  us without / with: 250 M bf16
// parameters with 8-bit states 454 / 467, 33 fp32 tensors of 1.9 M elements in all 9.7 / 10.2, 130 M with masters 676 / 679.
template <typename P, typename G, bool MASTER, bool EIGHT, bool TINY>
__global__ __launch_bounds__(kThreads) void adamwStep(Tensors<MASTER, EIGHT> t, Hyper h) {
  typedef Tensors<MASTER, EIGHT> Table;
  const int lane = threadIdx.x & 63;
  const uint32_t one = t.first[lane], two = lane + 64 < Table::kTensors ? t.first[lane + 64] : 0xffffffffu;
  const int which =
      __builtin_amdgcn_readfirstlane(__popcll(__ballot(one <= blockIdx.x)) + __popcll(__ballot(two <= blockIdx.x)) - 1);
  const uint32_t begin = t.first[which], chunk = blockIdx.x - begin;
  const int in_chunk = chunk + 1 == t.first[which + 1] - begin ? t.last[which] : kChunk;
  P *param = static_cast<P *>(t.address[Table::kParam][which]);
  const G *grad = static_cast<const G *>(t.address[Table::kGrad][which]);
  void *const m_at = t.address[Table::kM][which], *const v_at = t.address[Table::kV][which];
  float *master = nullptr, *m_scales = nullptr, *v_scales = nullptr;
  if constexpr (MASTER) master = static_cast<float *>(t.address[Table::kMaster][which]);
  if constexpr (EIGHT) {
    m_scales = static_cast<float *>(t.address[Table::kMScale][which]);
    v_scales = static_cast<float *>(t.address[Table::kVScale][which]);
  }
  const uintptr_t wide = reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad) |
                         (MASTER ? reinterpret_cast<uintptr_t>(master) : 0);
  const uintptr_t states = reinterpret_cast<uintptr_t>(m_at) | reinterpret_cast<uintptr_t>(v_at);
  const bool aligned = (wide & 15) == 0 && (states & (EIGHT ? 7 : 15)) == 0;
  const int64_t at = (int64_t)chunk * kChunk + threadIdx.x * kPerThread;
  const int left = in_chunk - (int)threadIdx.x * kPerThread;
  const int n = left >= kPerThread ? kPerThread : (left > 0 ? left : 0);
  const bool whole = aligned && n == kPerThread;

  float g[kPerThread], p[kPerThread], m[kPerThread], r[kPerThread];
  uint2 m_codes, v_codes;
  float m_scale = 0.f, v_scale = 0.f;
  loadEight(grad, at, n, whole, g);
  if constexpr (MASTER)
    loadEight(master, at, n, whole, p);
  else
    loadEight(param, at, n, whole, p);
  if constexpr (EIGHT) {
    m_codes = loadCodes(static_cast<const uint8_t *>(m_at), at, n, whole);
    v_codes = loadCodes(static_cast<const uint8_t *>(v_at), at, n, whole);
    if (n > 0) {
      m_scale = m_scales[at / kStateBlock];
      v_scale = v_scales[at / kStateBlock];
    }
    decode(m_codes, m_scale, m);
    decode(v_codes, v_scale, r);
  } else {
    loadEight(static_cast<const float *>(m_at), at, n, whole, m);
    loadEight(static_cast<const float *>(v_at), at, n, whole, r);
  }
  float v[kPerThread];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const float gi = g[i] * h.grad_scale;
    m[i] = m[i] * h.beta1 + gi * h.one_minus_beta1;
    v[i] = (EIGHT ? r[i] * r[i] : r[i]) * h.beta2 + gi * gi * h.one_minus_beta2;
    // (the hardware's own reciprocal, one unit in the last place; and its own root too, but where codes are made of it: half a
    // code on from there a unit decides between two of them, and the next step starts from it)
    r[i] = EIGHT || TINY ? sqrtf(v[i]) : __builtin_amdgcn_sqrtf(v[i]);
    const float below = r[i] * h.inv_root2 + h.eps;
    p[i] = p[i] * h.decay - h.step_size * (TINY ? m[i] / below : m[i] * __builtin_amdgcn_rcpf(below));
  }
  if constexpr (MASTER) storeEight(master, at, n, whole, p);
  storeEight(param, at, n, whole, p);
  if constexpr (EIGHT) {
    float most_m = 0.f, most_r = 0.f;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      // (behind a tensor's end everything is zero; a root of the gradient alone too)
      most_m = fmaxf(most_m, fabsf(m[i]));
      most_r = fmaxf(most_r, r[i]);
    }
    most_m = blockMost(most_m);
    most_r = blockMost(most_r);
    const float by_m = most_m > 1e-30f ? 1.f / most_m * kMostCode : 0.f;
    const float by_r = most_r > 1e-30f ? 1.f / most_r * kMostCode : 0.f;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      m[i] = m[i] * by_m;
      const float root = r[i] * by_r;
      // (a NaN stays one)
      r[i] = r[i] == 0.f ? 0.f : (root < kLeastCode ? kLeastCode : root);
    }
    storeCodes(static_cast<uint8_t *>(m_at), at, n, whole, encode(m));
    storeCodes(static_cast<uint8_t *>(v_at), at, n, whole, encode(r));
    if (n > 0 && lane % kLanesPerBlock == 0) {
      m_scales[at / kStateBlock] = most_m * (1.f / kMostCode);
      v_scales[at / kStateBlock] = most_r * (1.f / kMostCode);
    }
  } else {
    storeEight(static_cast<float *>(m_at), at, n, whole, m);
    storeEight(static_cast<float *>(v_at), at, n, whole, v);
  }
}

struct Step {
  const char *api;
  mluOpHandle_t handle;
  const mluOpExtAdamWTensor_t *tensors;
  int count;
  bool tiny;
  Hyper h;
};
constexpr int64_t kMostChunks = mostBlocks(kThreads);  // of a launch

template <typename P, typename G, bool MASTER, bool EIGHT>
mluOpStatus_t launchStep(const Step &step) {
  typedef Tensors<MASTER, EIGHT> Table;
  static_assert(sizeof(Table) + sizeof(Hyper) <= 4096, "kernel arguments");
  const LaunchCtx lc = step.handle->launchCtx();
  const bool notes = step.handle->hasNotes();
  Table t;
  int held = 0;
  uint32_t chunks = 0;
  auto launch = [&]() -> hipError_t {
    if (held == 0) return hipSuccess;
    t.first[held] = chunks;
    for (int i = held; i < Table::kTensors; ++i) {
      for (auto &of : t.address) of[i] = nullptr;
      t.first[i + 1] = 0xffffffffu;
      t.last[i] = 0;
    }
    lc.begin("adamwStep");
    auto kernel = step.tiny ? adamwStep<P, G, MASTER, EIGHT, true> : adamwStep<P, G, MASTER, EIGHT, false>;
    kernel<<<chunks, kThreads, 0, lc.stream>>>(t, step.h);
    lc.end();
    held = 0;
    chunks = 0;
    return hipGetLastError();
  };
  for (int i = 0; i < step.count; ++i) {
    const mluOpExtAdamWTensor_t &x = step.tensors[i];
    if (x.count == 0) continue;
    if (notes) {
      const int64_t blocks = (x.count + kStateBlock - 1) / kStateBlock;
      step.handle->forgetNotesIn(x.param, (size_t)x.count * sizeof(P));
      step.handle->forgetNotesIn(x.exp_avg, (size_t)x.count * (EIGHT ? 1 : 4));
      step.handle->forgetNotesIn(x.exp_avg_sq, (size_t)x.count * (EIGHT ? 1 : 4));
      if (MASTER) step.handle->forgetNotesIn(x.master, (size_t)x.count * 4);
      if (EIGHT) {
        step.handle->forgetNotesIn(x.exp_avg_scale, (size_t)blocks * 4);
        step.handle->forgetNotesIn(x.exp_avg_sq_scale, (size_t)blocks * 4);
      }
    }
    // (a tensor of more chunks than a launch takes goes in several)
    for (int64_t from = 0; from < x.count; from += kMostChunks * kChunk) {
      const int64_t count = std::min(x.count - from, kMostChunks * kChunk), own = (count + kChunk - 1) / kChunk;
      if (held == Table::kTensors || chunks + own > kMostChunks) HIP_CHECK_RETURN(step.api, launch());
      auto at = [&](const void *p, size_t size) { return static_cast<char *>(const_cast<void *>(p)) + from * size; };
      t.address[Table::kParam][held] = at(x.param, sizeof(P));
      t.address[Table::kGrad][held] = at(x.grad, sizeof(G));  // (only read)
      t.address[Table::kM][held] = at(x.exp_avg, EIGHT ? 1 : 4);
      t.address[Table::kV][held] = at(x.exp_avg_sq, EIGHT ? 1 : 4);
      if constexpr (MASTER) t.address[Table::kMaster][held] = at(x.master, 4);
      if constexpr (EIGHT) {
        t.address[Table::kMScale][held] = x.exp_avg_scale + from / kStateBlock;
        t.address[Table::kVScale][held] = x.exp_avg_sq_scale + from / kStateBlock;
      }
      t.first[held] = chunks;
      t.last[held] = (uint16_t)(count - (own - 1) * kChunk);
      chunks += (uint32_t)own;
      ++held;
    }
  }
  HIP_CHECK_RETURN(step.api, launch());
  return MLUOP_STATUS_SUCCESS;
}

template <typename P, typename G, bool MASTER>
mluOpStatus_t ofStates(const Step &step, bool eight) {
  return eight ? launchStep<P, G, MASTER, true>(step) : launchStep<P, G, MASTER, false>(step);
}

template <typename P>
mluOpStatus_t ofSixteen(const Step &step, bool float_grads, bool masters, bool eight) {
  if (float_grads) return masters ? ofStates<P, float, true>(step, eight) : ofStates<P, float, false>(step, eight);
  return masters ? ofStates<P, P, true>(step, eight) : ofStates<P, P, false>(step, eight);
}

mluOpStatus_t launchOf(const Step &step, mluOpDataType_t param_type, bool float_grads, bool masters, bool eight) {
  if (param_type == MLUOP_DTYPE_FLOAT) return ofStates<float, float, false>(step, eight);
  return param_type == MLUOP_DTYPE_HALF ? ofSixteen<_Float16>(step, float_grads, masters, eight)
                                        : ofSixteen<__bf16>(step, float_grads, masters, eight);
}

}  // namespace

mluOpStatus_t MLUOP_WIN_API mluOpExtAdamWStep(mluOpHandle_t handle, const mluOpExtAdamWTensor_t tensors[],
                                              int num_tensors, mluOpDataType_t param_type, mluOpDataType_t grad_type,
                                              mluOpDataType_t state_type, int64_t step, double lr, double beta1,
                                              double beta2, double eps, double weight_decay, double grad_scale) {
  const char *api = "[mluOpExtAdamWStep]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, num_tensors >= 0);
  PARAM_CHECK(api, num_tensors == 0 || tensors != NULL);
  PARAM_CHECK(api, isFloating(param_type));
  PARAM_CHECK(api, grad_type == param_type || grad_type == MLUOP_DTYPE_FLOAT);
  PARAM_CHECK(api, state_type == MLUOP_DTYPE_FLOAT || state_type == MLUOP_DTYPE_UINT8);
  PARAM_CHECK(api, step >= 1);
  PARAM_CHECK(api, std::isfinite(lr) && std::isfinite(weight_decay) && std::isfinite(grad_scale));
  PARAM_CHECK(api, beta1 >= 0.0 && beta1 < 1.0);
  PARAM_CHECK(api, beta2 >= 0.0 && beta2 < 1.0);
  PARAM_CHECK(api, eps >= 0.0 && std::isfinite(eps));
  const bool eight = state_type == MLUOP_DTYPE_UINT8;
  bool masters = false, any = false;
  for (int i = 0; i < num_tensors; ++i) {
    const mluOpExtAdamWTensor_t &t = tensors[i];
    PARAM_CHECK(api, t.count >= 0);
    if (t.count == 0) continue;  // (a tensor of nothing has no addresses)
    if (!any) masters = t.master != NULL;
    any = true;
    PARAM_CHECK(api, masters == (t.master != NULL));
    PARAM_CHECK(api, t.param != NULL && t.grad != NULL && t.exp_avg != NULL && t.exp_avg_sq != NULL);
    PARAM_CHECK(api, !eight || (t.exp_avg_scale != NULL && t.exp_avg_sq_scale != NULL));
    if (t.count > ((int64_t)1 << 46)) {
      MLUOP_LOG(ERROR) << api << " At most 2^46 elements of a tensor are supported.";
      return MLUOP_STATUS_NOT_SUPPORTED;
    }
  }
  PARAM_CHECK(api, !masters || param_type != MLUOP_DTYPE_FLOAT);
  DEVICE_HANDLE_CHECK(api, handle);
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));

  Step all = {api, handle, tensors, num_tensors, false, {}};
  Hyper &h = all.h;
  h.beta1 = (float)beta1;
  h.one_minus_beta1 = (float)(1.0 - beta1);
  h.beta2 = (float)beta2;
  h.one_minus_beta2 = (float)(1.0 - beta2);
  h.decay = (float)(1.0 - lr * weight_decay);
  h.step_size = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
  h.inv_root2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
  h.eps = (float)eps;
  all.tiny = h.eps < h.inv_root2 * 0x1p-38f;
  h.grad_scale = (float)grad_scale;

  return launchOf(all, param_type, grad_type == MLUOP_DTYPE_FLOAT, masters, eight);
}
