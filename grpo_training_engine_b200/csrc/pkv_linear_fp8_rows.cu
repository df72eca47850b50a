// pkv_linear_fp8_rows.cu — 8-bit projections of a few activation rows.
//
// The product of pkv_linear_fp8.cu for up to 16 rows: the weights are read once
// and used for at most 16 multiply-adds each, so HBM is the bound, and what
// counts is bytes in flight. A tcgen05 tile of 128 rows would be half empty and
// every block of k would cross TMEM; here each warp loads its 16 rows of W
// straight into the registers that mma.sync (m16n8k32, e4m3) takes them from,
// three or four blocks of k ahead, with W's rows on M and the activations on N. All rows
// of x lie in shared memory for the whole (persistent) launch. k is permuted
// alike for both operands, so that a thread's 16 loaded bytes are its fragments
// of two MMAs. Each block's sum is added to fp32 sums times the block's scales.
// Measured: 1 x 2048 x 1536 3.3 us (8.6 on tcgen05 tiles), 1 x 151,936 x 1536 40
// us, 5.9 TB/s (66), 16 rows of it 49 us. Beyond 16 rows the fragments of x, read
// from shared memory for every block, take over (37 rows: 82 us), and the tiles
// are faster.
#include <algorithm>

#include "pkv_tc.cuh"
#include "pkv_types.cuh"

namespace pkv {
namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kBK = 128;    // values of k that share a scale
constexpr int kPad = 64;    // bytes between rows of x in shared memory: two rows of 64 bytes fill the banks

struct RowsArgs {
  const uint8_t *x, *w;
  const float *xs, *ws;
  const void *bias;
  void *out;
  int64_t x_stride, w_stride, xs_stride, ws_stride, out_stride;
  int32_t rows, n, k, kblocks;
};

__device__ __forceinline__ void mma_f8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_w(const uint8_t *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// NT: groups of 8 activation rows. KW: warps that share 16 rows of W, each with
// every KW-th block of k (the other factor of the 8 warps takes other rows).
template <typename T, int NT, int KW>
__global__ void __launch_bounds__(kThreads, 2) linear_rows_kernel(RowsArgs a) {
  constexpr int MW = kWarps / KW, kRows = 8 * NT;
  // Blocks of k in flight per warp, 16 registers each. At 2 blocks on an SM and 16 warps, four are 128 KB on an
  // SM: 151,936 x 1536 by one row takes 39 us (5.9 TB/s); two 44. With 16 rows the registers hold three.
  constexpr int kAhead = NT == 1 ? 4 : 3;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int mw = warp / KW, kw = warp % KW;
  const int stride = a.kblocks * kBK + kPad;
  float *xs = reinterpret_cast<float *>(smem + (size_t)kRows * stride);  // [kblocks][kRows]
  float *part_s = xs + a.kblocks * kRows;                               // [kWarps][16][kRows], with KW > 1
  const int groups = (a.n + 16 * MW - 1) / (16 * MW);                   // of a block's rows of W
  const int blocks = (a.kblocks - kw + KW - 1) / KW;                    // of k, of this warp; may be 0

  // the warp's sequence of (group of rows, block of k), loaded kAhead ahead
  struct Block {
    uint4 v[2][2];  // [row g, row g + 8][64-byte half]
    float ws;
  };
  int lg = blockIdx.x, lk = 0;  // what is loaded next
  auto load = [&](Block &b) {
    if (lg >= groups || blocks == 0) return;
    const int row = (lg * MW + mw) * 16, kb = kw + lk * KW;
    b.ws = a.ws[(int64_t)(min(row, a.n - 1) / 128) * a.ws_stride + kb];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t *p = a.w + (int64_t)min(row + g + 8 * r, a.n - 1) * a.w_stride + kb * kBK + 16 * t;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        b.v[r][h] = kb * kBK + 64 * h + 16 * t < a.k ? load_w(p + 64 * h) : make_uint4(0, 0, 0, 0);
    }
    if (++lk == blocks) {
      lk = 0;
      lg += gridDim.x;
    }
  };
  Block ring[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(ring[i]);

  // x and its scales, zeros where there are none
  const int vecs = a.kblocks * (kBK / 16);
#pragma unroll 4
  for (int i = tid; i < kRows * vecs; i += kThreads) {
    const int r = i / vecs, c = i - r * vecs;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < a.rows && 16 * c < a.k) v = __ldg(reinterpret_cast<const uint4 *>(a.x + r * a.x_stride) + c);
    *reinterpret_cast<uint4 *>(smem + (size_t)r * stride + 16 * c) = v;
  }
  for (int i = tid; i < kRows * a.kblocks; i += kThreads) {
    const int r = i / a.kblocks, kb = i - r * a.kblocks;
    xs[kb * kRows + r] = r < a.rows ? a.xs[r * a.xs_stride + kb] : 0.f;
  }
  __syncthreads();

  float acc[NT][4];
  auto multiply = [&](const Block &b, int kb) {
    float sum[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[j][e] = 0.f;
    const uint8_t *xp = smem + (size_t)g * stride + kb * kBK + 16 * t;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t a0[4] = {b.v[0][h].x, b.v[1][h].x, b.v[0][h].y, b.v[1][h].y};
      const uint32_t a1[4] = {b.v[0][h].z, b.v[1][h].z, b.v[0][h].w, b.v[1][h].w};
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint4 v = *reinterpret_cast<const uint4 *>(xp + (size_t)8 * j * stride + 64 * h);
        mma_f8(sum[j], a0, v.x, v.y);
        mma_f8(sum[j], a1, v.z, v.w);
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float2 s = *reinterpret_cast<const float2 *>(xs + kb * kRows + 8 * j + 2 * t);
      acc[j][0] = fmaf(sum[j][0], s.x * b.ws, acc[j][0]);
      acc[j][1] = fmaf(sum[j][1], s.y * b.ws, acc[j][1]);
      acc[j][2] = fmaf(sum[j][2], s.x * b.ws, acc[j][2]);
      acc[j][3] = fmaf(sum[j][3], s.y * b.ws, acc[j][3]);
    }
  };
  const T *bias = reinterpret_cast<const T *>(a.bias);
  auto store = [&](int r, int c, float v) {  // activation row r, column c
    if (r < a.rows && c < a.n)
      reinterpret_cast<T *>(a.out)[r * a.out_stride + c] =
          from_f32<T>(bias != nullptr ? v + Elem<T>::to_f32(bias[c]) : v);
  };

  // a group's sums are complete
  auto finish = [&](int grp) {
    const int row = (grp * MW + mw) * 16;
    if constexpr (KW == 1) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) store(8 * j + 2 * t + (e & 1), row + g + 8 * (e >> 1), acc[j][e]);
    } else {
      // the warps that share the rows add their sums in order
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          part_s[(warp * kRows + 8 * j + 2 * t + (e & 1)) * 16 + g + 8 * (e >> 1)] = acc[j][e];
      __syncthreads();
      for (int i = tid; i < MW * kRows * 16; i += kThreads) {
        const int m = i / (kRows * 16), r = i / 16 % kRows, c = i % 16;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < KW; ++q) v += part_s[((m * KW + q) * kRows + r) * 16 + c];
        store(r, (grp * MW + m) * 16 + c, v);
      }
      __syncthreads();
    }
  };
  auto clear = [&] {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
  };

  int grp = blockIdx.x, i = 0;
  clear();
  if (blocks == 0) {  // a warp beyond the blocks of k takes part in the additions
    for (; grp < groups; grp += gridDim.x) finish(grp);
    return;
  }
  while (grp < groups) {
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (grp >= groups) break;
      multiply(ring[q], kw + i * KW);
      load(ring[q]);
      if (++i == blocks) {
        finish(grp);
        clear();
        i = 0;
        grp += gridDim.x;
      }
    }
  }
}

size_t rows_smem(int nt, int kw, int kblocks) {
  return (size_t)8 * nt * (kblocks * kBK + kPad) + (size_t)4 * 8 * nt * kblocks +
         (kw > 1 ? (size_t)4 * kWarps * 16 * 8 * nt : 0);
}

template <typename T, int NT, int KW>
int rows_launch(const RowsArgs &a, void *stream) {
  const size_t smem = rows_smem(NT, KW, a.kblocks);
  auto kern = linear_rows_kernel<T, NT, KW>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return check_launch("cudaFuncSetAttribute(linear_rows)");
  const int64_t groups = ((int64_t)a.n + 16 * (kWarps / KW) - 1) / (16 * (kWarps / KW));
  const int per_sm = smem <= 100 * 1024 ? 2 : 1;
  kern<<<(unsigned)std::min<int64_t>(groups, lin_sms() * per_sm), kThreads, smem,
         reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return check_launch("linear_rows_kernel");
}

template <typename T, int NT>
int rows_dispatch_kw(const RowsArgs &a, int kw, void *stream) {
  if (kw == 1) return rows_launch<T, NT, 1>(a, stream);
  if (kw == 4) return rows_launch<T, NT, 4>(a, stream);
  return rows_launch<T, NT, 8>(a, stream);
}

// Warps that share rows of W: as many as give every SM some 16 warps.
int rows_kw(int64_t n) {
  const int64_t tiles = (n + 15) / 16;
  return tiles >= 16 * 148 ? 1 : tiles >= 4 * 148 ? 4 : 8;
}

}  // namespace

// Whether the kernel above takes these sizes: x in one SM's shared memory, whole 16-byte pieces of k.
bool linear_fp8_rows_fits(int32_t rows, int32_t n, int32_t k) {
  return rows <= 16 && k % 16 == 0 && rows_smem(rows <= 8 ? 1 : 2, rows_kw(n), (k - 1) / kBK + 1) <= 220 * 1024;
}

int linear_fp8_rows(const void *x, const float *x_scale, const void *w, const float *w_scale, const void *bias,
                    void *out, int32_t rows, int32_t n, int32_t k, int64_t x_stride, int64_t xs_stride,
                    int64_t w_stride, int64_t ws_stride, int64_t out_stride, int32_t out_dtype, void *stream) {
  const RowsArgs a{static_cast<const uint8_t *>(x), static_cast<const uint8_t *>(w), x_scale, w_scale, bias, out,
                   x_stride, w_stride, xs_stride, ws_stride, out_stride, rows, n, k, (k - 1) / kBK + 1};
  const int kw = rows_kw(n);
  auto run = [&](auto tag) {
    using T = decltype(tag);
    return rows <= 8 ? rows_dispatch_kw<T, 1>(a, kw, stream) : rows_dispatch_kw<T, 2>(a, kw, stream);
  };
  return out_dtype == PKV_DTYPE_BF16 ? run(__nv_bfloat16()) : run(__half());
}

}  // namespace pkv
