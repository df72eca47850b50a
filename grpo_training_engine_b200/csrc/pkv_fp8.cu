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

// 16 bytes as N fp32 values, and back.
template <typename T> struct alignas(16) Vec16 {
  static constexpr int kN = 16 / (int)sizeof(T);
  T e[kN];
};

__device__ __forceinline__ float sum_block(float v, float *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int k = 0; k < (int)blockDim.x / 32; ++k) v += red[k];
  return v;
}

struct NormArgs {
  const void *x, *res, *w;
  void *sum;
  uint8_t *q;
  float *scales;
  int64_t xs, rs, ss, qs, cs;
  int hidden;
  float eps;
};

// One block per row, NV vectors of 16 bytes per thread, the row held in
// registers between the sum of squares and the quotient: x, the residual and
// their sum cross HBM once. A group of 128 values is the vectors of 32 (fp32)
// or 16 neighbouring lanes, so its maximum takes four or five shuffles. Bound by
// HBM: 16384 rows of 3584 bf16 with a residual take 69 us, 6.0 TB/s of the 6.5
// that a copy reaches (200 us element by element; 92 with loads that keep the
// inputs in L2). One row of 1536: 2.3 us, a launch and two round trips to memory.
template <typename T, int NV, bool Res>
__global__ void __launch_bounds__(NV == 4 ? 512 : 1024) norm_fp8_kernel(NormArgs a) {
  using V = Vec16<T>;
  constexpr int N = V::kN, kLanes = kGroup / N;
  __shared__ float red[32];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, nt = blockDim.x, nv = a.hidden / N;
  const V *x = reinterpret_cast<const V *>(reinterpret_cast<const T *>(a.x) + b * a.xs);
  const V *res = reinterpret_cast<const V *>(reinterpret_cast<const T *>(a.res) + b * a.rs);
  V *sum = reinterpret_cast<V *>(reinterpret_cast<T *>(a.sum) + b * a.ss);
  const V *w = reinterpret_cast<const V *>(a.w);
  V xv[NV], rv[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (tid + j * nt < nv) {
      // read for the last time: what is read again is their sum
      *reinterpret_cast<uint4 *>(&xv[j]) = __ldcs(reinterpret_cast<const uint4 *>(x + tid + j * nt));
      if (Res) *reinterpret_cast<uint4 *>(&rv[j]) = __ldcs(reinterpret_cast<const uint4 *>(res + tid + j * nt));
    }
  float s[NV][N], acc = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const bool in = tid + j * nt < nv;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      s[j][e] = in ? Elem<T>::to_f32(xv[j].e[e]) : 0.f;
      if (Res && in) {
        s[j][e] += Elem<T>::to_f32(rv[j].e[e]);
        xv[j].e[e] = from_f32<T>(s[j][e]);
      }
      acc += s[j][e] * s[j][e];
    }
    if (Res && in) sum[tid + j * nt] = xv[j];
  }
  const float r = rsqrtf(sum_block(acc, red) / (float)a.hidden + a.eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = tid + j * nt;
    const bool in = i < nv;
    float amax = 0.f;
    if (in) {
      const V wv = w[i];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        s[j][e] *= r * Elem<T>::to_f32(wv.e[e]);
        amax = max_nan(amax, fabsf(s[j][e]));
      }
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float scale = group_scale(amax), inv = 1.f / scale;
    if (!in) continue;
    if (i % kLanes == 0) a.scales[b * a.cs + i / kLanes] = scale;
    uint32_t o[N / 4];
#pragma unroll
    for (int e = 0; e < N; e += 4)
      o[e / 4] = e4m3x2(s[j][e] * inv, s[j][e + 1] * inv) |
                 ((uint32_t)e4m3x2(s[j][e + 2] * inv, s[j][e + 3] * inv) << 16);
    uint8_t *q = a.q + b * a.qs + (int64_t)i * N;
    if (N == 8)
      *reinterpret_cast<uint2 *>(q) = make_uint2(o[0], o[N / 4 - 1]);
    else
      *reinterpret_cast<uint32_t *>(q) = o[0];
  }
}

// Rows of any length and alignment, element by element (the second read: L1/L2).
constexpr int kAnyThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kAnyThreads) norm_fp8_any_kernel(NormArgs a) {
  __shared__ float red[32];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, H = a.hidden;
  const T *x = reinterpret_cast<const T *>(a.x) + b * a.xs;
  const T *res = a.res != nullptr ? reinterpret_cast<const T *>(a.res) + b * a.rs : nullptr;
  T *sum = reinterpret_cast<T *>(a.sum) + b * a.ss;
  const T *w = reinterpret_cast<const T *>(a.w);
  // a warp's groups in both passes: what it reads again it has read itself, before it stored the sum
  constexpr int kHeld = 4;  // groups per warp that stay in registers
  float held[kHeld][4], acc = 0.f;
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = (warp + j * (kAnyThreads / 32)) * kGroup + lane + 32 * e;
      held[j][e] = 0.f;
      if (i < H) {
        held[j][e] = Elem<T>::to_f32(x[i]) + (res != nullptr ? Elem<T>::to_f32(res[i]) : 0.f);
        acc += held[j][e] * held[j][e];
      }
    }
  for (int g = warp + kHeld * (kAnyThreads / 32); g * kGroup < H; g += kAnyThreads / 32)
    for (int i = g * kGroup + lane; i < min(H, (g + 1) * kGroup); i += 32) {
      const float s = Elem<T>::to_f32(x[i]) + (res != nullptr ? Elem<T>::to_f32(res[i]) : 0.f);
      acc += s * s;
    }
  const float r = rsqrtf(sum_block(acc, red) / (float)H + a.eps);
  auto write = [&](int g, const float (&s)[4]) {
    float y[4], amax = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = g * kGroup + lane + 32 * e;
      y[e] = i < H ? s[e] * (r * Elem<T>::to_f32(w[i])) : 0.f;
      amax = max_nan(amax, fabsf(y[e]));
      if (res != nullptr && i < H) sum[i] = from_f32<T>(s[e]);
    }
    const float scale = group_scale(warp_max(amax)), inv = 1.f / scale;
    if (lane == 0) a.scales[b * a.cs + g] = scale;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = g * kGroup + lane + 32 * e;
      if (i < H) a.q[b * a.qs + i] = (uint8_t)e4m3x2(y[e] * inv, 0.f);
    }
  };
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if ((warp + j * (kAnyThreads / 32)) * kGroup < H) write(warp + j * (kAnyThreads / 32), held[j]);
  for (int g = warp + kHeld * (kAnyThreads / 32); g * kGroup < H; g += kAnyThreads / 32) {
    float s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = g * kGroup + lane + 32 * e;
      s[e] = i < H ? Elem<T>::to_f32(x[i]) + (res != nullptr ? Elem<T>::to_f32(res[i]) : 0.f) : 0.f;
    }
    write(g, s);
  }
}

// Activations: a warp per 128 values of a row, four per lane, read once.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T *x, uint8_t *q, float *scales, int64_t rows, int cols, int64_t xs, int64_t qs, int64_t cs,
                     int groups) {
  const int64_t at = blockIdx.x * 8ll + threadIdx.x / 32, r = at / groups;
  const int g = (int)(at - r * groups), lane = threadIdx.x & 31;
  if (r >= rows) return;
  float v[4], amax = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = g * kGroup + lane + 32 * e;
    v[e] = c < cols ? Elem<T>::to_f32(x[r * xs + c]) : 0.f;
    amax = max_nan(amax, fabsf(v[e]));
  }
  const float scale = group_scale(warp_max(amax)), inv = 1.f / scale;
  if (lane == 0) scales[r * cs + g] = scale;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = g * kGroup + lane + 32 * e;
    if (c < cols) q[r * qs + c] = (uint8_t)e4m3x2(v[e] * inv, 0.f);
  }
}

// Weights: a block per 128 x 128 values, 64 per thread, read once (a model's weights are laid out once).
template <typename T>
__global__ void __launch_bounds__(256)
quantize_block_kernel(const T *x, uint8_t *q, float *scales, int64_t rows, int cols, int64_t xs, int64_t qs, int64_t cs,
                      int groups) {
  __shared__ float red[8];
  const int64_t br = blockIdx.x / groups;
  const int g = (int)(blockIdx.x % groups);
  const int col = g * kGroup + (threadIdx.x & 127);
  const int64_t row = br * kGroup + (threadIdx.x >> 7);
  float v[64], amax = 0.f;
#pragma unroll
  for (int j = 0; j < 64; ++j) {
    v[j] = col < cols && row + 2 * j < rows ? Elem<T>::to_f32(x[(row + 2 * j) * xs + col]) : 0.f;
    amax = max_nan(amax, fabsf(v[j]));
  }
  amax = warp_max(amax);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();
  for (int i = 0; i < 8; ++i) amax = max_nan(amax, red[i]);
  const float scale = group_scale(amax), inv = 1.f / scale;
  if (threadIdx.x == 0) scales[br * cs + g] = scale;
#pragma unroll
  for (int j = 0; j < 64; ++j)
    if (col < cols && row + 2 * j < rows) q[(row + 2 * j) * qs + col] = (uint8_t)e4m3x2(v[j] * inv, 0.f);
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
  if (!all_aligned(es, {x, residual, weight, sum_out}) || !aligned_to(scales, 4)) return PKV_ERR_ALIGNMENT;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const NormArgs a{x, residual, weight, sum_out, (uint8_t *)q_out, scales, x_stride, residual_stride, sum_stride,
                   q_stride, scale_stride, hidden, eps};
  // 16-byte vectors where every row begins on one; q's rows take the vectors' 8-bit images
  const int n = 16 / es;
  const int64_t strides[] = {x_stride, residual ? residual_stride : 0, sum_out ? sum_stride : 0};
  bool vec = hidden % n == 0 && hidden / n <= 2 * 1024 && aligned_to(q_out, n) && q_stride % n == 0 &&
             all_aligned(16, {x, residual, weight, sum_out});
  for (int64_t v : strides) vec = vec && v % n == 0;
  if (!vec) {
    PKV_BY_DTYPE(dtype, (norm_fp8_any_kernel<T><<<rows, kAnyThreads, 0, st>>>(a)))
    return check_launch("pkv_add_rmsnorm_fp8");
  }
  // Few rows: one vector per thread, for the shortest chain. Many: four, for the most bytes in flight per
  // register and the fewest blocks.
  const int nv = hidden / n;
  const int per = std::max(rows <= 2 * 148 ? 1 : rows <= 16 * 148 ? 2 : 4, nv > 1024 ? 2 : 1);
  const int threads = ((nv + per - 1) / per + 31) / 32 * 32;
  PKV_BY_DTYPE(dtype, {
    auto k = residual ? (per == 1 ? norm_fp8_kernel<T, 1, true> : per == 2 ? norm_fp8_kernel<T, 2, true>
                                                                            : norm_fp8_kernel<T, 4, true>)
                      : (per == 1 ? norm_fp8_kernel<T, 1, false> : per == 2 ? norm_fp8_kernel<T, 2, false>
                                                                             : norm_fp8_kernel<T, 4, false>);
    k<<<rows, threads, 0, st>>>(a);
  })
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
  if (!aligned_to(x, es) || !aligned_to(scales, 4)) return PKV_ERR_ALIGNMENT;
  const int64_t blocks = (rows + block_rows - 1) / block_rows * groups;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PKV_BY_DTYPE(dtype, {
    if (block_rows == 1)
      quantize_rows_kernel<T><<<(unsigned)((blocks + 7) / 8), 256, 0, st>>>(
          (const T *)x, (uint8_t *)q_out, scales, rows, cols, x_stride, q_stride, scale_stride, (int)groups);
    else
      quantize_block_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(
          (const T *)x, (uint8_t *)q_out, scales, rows, cols, x_stride, q_stride, scale_stride, (int)groups);
  })
  return check_launch("pkv_quantize_fp8");
}
