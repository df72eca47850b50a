// pkv_fp8.cu — 8-bit (e4m3) values with a scale for each 128 of them: the
// residual add + RMSNorm that writes them, and the quantisers of activations
// (1 x 128 groups of a row) and weights (128 x 128 blocks).
//
//   s = x + r,  y = w s / sqrt(mean(s^2) + eps),
//   scale = max(max_group |y|, 2^-100) / 448,  q = e4m3(y / scale).
// Everything up to q is fp32: y is taken from the unrounded sum and is itself
// never rounded to 16 bits, so q carries one rounding; s is rounded once, to
// x's type, where it is stored as the next residual. 448 is the largest e4m3
// value; the floor of 2^-100 keeps the scale of a group of zeros normal.
#include <algorithm>

#include "pkv_types.cuh"

namespace pkv {
namespace {

constexpr int kGroup = 128;
constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;  // 2^-100

// e4m3 of two values (the first in the low byte), saturating; NaN stays NaN
__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float group_scale(float amax) { return max_nan(amax, kAmaxFloor) / kE4m3Max; }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

constexpr int kNormThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kNormThreads)
norm_fp8_kernel(const T *x, const T *res, const T *w, T *sum_out, uint8_t *q, float *scales, int H, int64_t xs,
                int64_t rs, int64_t ss, int64_t qs, int64_t cs, float eps) {
  __shared__ float red[kNormThreads / 32];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float acc = 0.f;
  for (int i = tid; i < H; i += kNormThreads) {
    float s = Elem<T>::to_f32(x[b * xs + i]);
    if (res != nullptr) {
      s += Elem<T>::to_f32(res[b * rs + i]);
      sum_out[b * ss + i] = from_f32<T>(s);
    }
    acc += s * s;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) red[warp] = acc;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int k = 0; k < kNormThreads / 32; ++k) tot += red[k];
  const float r = rsqrtf(tot / (float)H + eps);
  // one warp per group, 4 values per lane
  for (int g = warp; g * kGroup < H; g += kNormThreads / 32) {
    float y[4], amax = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = g * kGroup + lane * 4 + e;
      y[e] = 0.f;
      if (i < H) {
        float s = Elem<T>::to_f32(x[b * xs + i]);
        if (res != nullptr) s += Elem<T>::to_f32(res[b * rs + i]);
        y[e] = s * r * Elem<T>::to_f32(w[i]);
      }
      amax = max_nan(amax, fabsf(y[e]));
    }
    const float scale = group_scale(warp_max(amax)), inv = 1.f / scale;
    if (lane == 0) scales[b * cs + g] = scale;
    const uint32_t p = e4m3x2(y[0] * inv, y[1] * inv) | ((uint32_t)e4m3x2(y[2] * inv, y[3] * inv) << 16);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (g * kGroup + lane * 4 + e < H) q[b * qs + g * kGroup + lane * 4 + e] = (uint8_t)(p >> (8 * e));
  }
}

// One block of 8 warps per (group of `block_rows` rows, group of 128 columns).
template <typename T>
__global__ void __launch_bounds__(256)
quantize_kernel(const T *x, uint8_t *q, float *scales, int64_t rows, int cols, int64_t xs, int64_t qs, int64_t cs,
                int block_rows, int groups) {
  __shared__ float red[8];
  const int64_t br = blockIdx.x / groups;
  const int g = (int)(blockIdx.x % groups), c0 = g * kGroup, n = min(kGroup, cols - c0);
  const int64_t r0 = br * block_rows;
  const int nr = (int)min((int64_t)block_rows, rows - r0);
  float amax = 0.f;
  for (int i = threadIdx.x; i < nr * n; i += 256)
    amax = max_nan(amax, fabsf(Elem<T>::to_f32(x[(r0 + i / n) * xs + c0 + i % n])));
  amax = warp_max(amax);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();
  for (int i = 0; i < 8; ++i) amax = max_nan(amax, red[i]);
  const float scale = group_scale(amax), inv = 1.f / scale;
  if (threadIdx.x == 0) scales[br * cs + g] = scale;
  for (int i = threadIdx.x; i < nr * n; i += 256)
    q[(r0 + i / n) * qs + c0 + i % n] =
        (uint8_t)e4m3x2(Elem<T>::to_f32(x[(r0 + i / n) * xs + c0 + i % n]) * inv, 0.f);
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_add_rmsnorm_fp8(const void *x, const void *residual, const void *weight, void *sum_out,
                                   void *q_out, float *scales, int32_t rows, int32_t hidden, int64_t x_stride,
                                   int64_t residual_stride, int64_t sum_stride, int64_t q_stride,
                                   int64_t scale_stride, float eps, int32_t dtype, void *stream) {
  const int es = dtype_size(dtype);
  if (es == 0) return PKV_ERR_UNSUPPORTED;
  if (rows < 0 || hidden <= 0 || (rows > 0 && (!x || !weight || !q_out || !scales)) ||
      (residual == nullptr) != (sum_out == nullptr)) {
    set_error_detail("pkv_add_rmsnorm_fp8: rows %d, hidden %d, a NULL pointer, or one of residual and sum_out", rows,
                     hidden);
    return PKV_ERR_INVALID_ARG;
  }
  if (rows == 0) return PKV_OK;
  const void *ptrs[] = {x, residual, weight, sum_out};
  for (const void *p : ptrs)
    if (!aligned_to(p, es)) return PKV_ERR_ALIGNMENT;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PKV_BY_DTYPE(dtype, (norm_fp8_kernel<T><<<rows, kNormThreads, 0, st>>>(
                          (const T *)x, (const T *)residual, (const T *)weight, (T *)sum_out, (uint8_t *)q_out, scales,
                          hidden, x_stride, residual_stride, sum_stride, q_stride, scale_stride, eps)))
  return check_launch("pkv_add_rmsnorm_fp8");
}

extern "C" int pkv_quantize_fp8(const void *x, void *q_out, float *scales, int64_t rows, int32_t cols,
                                int32_t block_rows, int64_t x_stride, int64_t q_stride, int64_t scale_stride,
                                int32_t dtype, void *stream) {
  const int es = dtype_size(dtype);
  if (es == 0) return PKV_ERR_UNSUPPORTED;
  const int64_t groups = ((int64_t)cols + kGroup - 1) / kGroup;
  if (rows < 0 || cols <= 0 || (block_rows != 1 && block_rows != kGroup) ||
      (rows > 0 && (!x || !q_out || !scales)) || (rows + block_rows - 1) / block_rows * groups > INT32_MAX) {
    set_error_detail("pkv_quantize_fp8: rows %lld, cols %d, blocks of %d rows (1 or 128), or a NULL pointer",
                     (long long)rows, cols, block_rows);
    return PKV_ERR_INVALID_ARG;
  }
  if (rows == 0) return PKV_OK;
  if (!aligned_to(x, es)) return PKV_ERR_ALIGNMENT;
  const unsigned blocks = (unsigned)((rows + block_rows - 1) / block_rows * groups);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PKV_BY_DTYPE(dtype, (quantize_kernel<T><<<blocks, 256, 0, st>>>((const T *)x, (uint8_t *)q_out, scales, rows, cols,
                                                                  x_stride, q_stride, scale_stride, block_rows,
                                                                  (int)groups)))
  return check_launch("pkv_quantize_fp8");
}
