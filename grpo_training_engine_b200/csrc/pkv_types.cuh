// pkv_types.cuh — rounding to an element type, NaN-propagating maxima and the
// dispatch over element types of the scoring and update kernels.
#pragma once

#include <initializer_list>

#include "pkv_common.cuh"

// Runs the statements with T the element type of `dtype` (a checked code).
#define PKV_BY_DTYPE(dtype, ...)                                          \
  switch (dtype) {                                                        \
    case PKV_DTYPE_BF16: { using T = __nv_bfloat16; __VA_ARGS__; break; } \
    case PKV_DTYPE_F16: { using T = __half; __VA_ARGS__; break; }         \
    default: { using T = float; __VA_ARGS__; break; }                     \
  }

namespace pkv {

// Whether every pointer (NULL ones too) is a multiple of `size`: a misaligned one would fault in the kernel.
inline bool all_aligned(size_t size, std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (!aligned_to(p, size)) return false;
  return true;
}

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

}  // namespace pkv
