// pkv_linear_fp8.cu — projections of 8-bit activations by 8-bit weights on the
// tcgen05 tensor cores (sm_100a).
//
//   out[r, j] = sum_b xs[r, b] ws[j / 128, b] (sum_{k in block b} x[r, k] W[j, k])  (+ bias[j])
//
// x [rows, k] and W [n, k] (nn.Linear's layout) are e4m3 with a scale for each
// 128 values of a row of x and each 128 x 128 block of W. The scales differ
// from block to block of k, so a block's products cannot be added to the last
// block's inside the tensor core: the MMAs of one block of k fill a TMEM buffer
// of their own, and the epilogue warps add it, times the block's two scales,
// to fp32 accumulators in registers while the tensor core fills the next.
//
// One CTA computes a 128-row by BN-column tile (or one split of its k):
//   warp 0, one thread : TMA loads of 128-wide k blocks of x and W into an
//                        S-stage shared-memory ring (128-byte swizzle)
//   warp 1             : TMEM allocation; one thread issues the 4 MMAs (M 128,
//                        N BN, K 32) of each block
//   warps 2-9          : two warps per 32-lane TMEM group, half the columns
//                        each: accumulate block by block, then store.
// With few rows the tiles of one weight matrix are split along k over the CTAs
// of a cluster, which add their fp32 tiles in split order through distributed
// shared memory, so results do not depend on timing.
//
// Every wait is bounded; one that runs out sets PKV_DEV_WAIT_TIMEOUT, and the
// CTA waits (bounded) for its own copies and MMAs, frees its TMEM and returns.
#include <algorithm>
#include <type_traits>

#include "pkv_tc.cuh"
#include "pkv_types.cuh"

namespace pkv {
namespace {

constexpr int kBM = 128, kBK = 128;  // tile rows; k values of a block, the span of one scale
constexpr int kEpiWarps = 8, kThreads = 64 + 32 * kEpiWarps;
constexpr int kMaxSplits = 8;        // a portable cluster

struct Fp8Args {
  const float *xs, *ws;  // scales: rows of x, blocks of W
  const void *bias;      // [n], out's type, or nullptr
  void *out;
  int32_t *status;
  int64_t xs_stride, ws_stride, out_stride;
  int32_t rows, n, kblocks, tiles_m, tiles_n, splits;
  uint32_t max_polls;
};

// D[tmem] (+)= A[smem] B[smem]^T with e4m3 operands
__device__ __forceinline__ void tc_mma_f8(uint32_t tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}

// Instruction descriptor: fp32 accumulator, A and B e4m3 (0), both K-major, M 128, N n.
__host__ __device__ constexpr uint32_t f8_idesc(int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
}

__device__ __forceinline__ uint32_t bits16(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ uint32_t bits16(__half v) { return __half_as_ushort(v); }

template <int BN, int S>
struct Smem {
  static constexpr int kA = kBM * kBK, kB = BN * kBK;  // one stage of x and of W, bytes
  static constexpr int kBufs = BN <= 128 ? 4 : 2;      // TMEM buffers of BN fp32 columns
  static constexpr uint32_t kCols = kBufs * BN;        // a power of two, at most 512
  static constexpr size_t kW = (size_t)S * kA;
  static constexpr size_t kFull = kW + (size_t)S * kB;
  static constexpr size_t kEmpty = kFull + 8 * S;
  static constexpr size_t kAccFull = kEmpty + 8 * S;
  static constexpr size_t kAccEmpty = kAccFull + 8 * kBufs;
  static constexpr size_t kDone = kAccEmpty + 8 * kBufs;
  static constexpr size_t kTmem = kDone + 8;
  static constexpr size_t kBytes = kTmem + 8 + 1024;  // + alignment slack
};

// NC results of one row from column col on: bias, rounding, store.
template <typename T, int NC>
__device__ __forceinline__ void store_cols(const Fp8Args &a, int row, int col, const float *v) {
  T *out = reinterpret_cast<T *>(a.out) + row * a.out_stride + col;
  const T *bias = reinterpret_cast<const T *>(a.bias);
  T o[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j)
    o[j] = from_f32<T>(bias != nullptr && col + j < a.n ? v[j] + Elem<T>::to_f32(bias[col + j]) : v[j]);
  if (NC == 8 && col + NC <= a.n && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
    uint4 w;
    w.x = bits16(o[0]) | (bits16(o[1]) << 16);
    w.y = bits16(o[2]) | (bits16(o[3]) << 16);
    w.z = bits16(o[4]) | (bits16(o[5]) << 16);
    w.w = bits16(o[6]) | (bits16(o[7]) << 16);
    *reinterpret_cast<uint4 *>(out) = w;
  } else {
#pragma unroll
    for (int j = 0; j < NC; ++j)
      if (col + j < a.n) out[j] = o[j];
  }
}

template <typename T, int BN, int S>
__global__ void __launch_bounds__(kThreads, 1)
linear_fp8_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, Fp8Args a) {
  using L = Smem<BN, S>;
  constexpr int NB = L::kBufs, kPart = BN / 2;  // columns of one epilogue warp
  extern __shared__ uint8_t raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *sa = smem, *sb = smem + L::kW;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kFull);
  uint64_t *empty = reinterpret_cast<uint64_t *>(smem + L::kEmpty);
  uint64_t *acc_full = reinterpret_cast<uint64_t *>(smem + L::kAccFull);
  uint64_t *acc_empty = reinterpret_cast<uint64_t *>(smem + L::kAccEmpty);
  uint64_t *done = reinterpret_cast<uint64_t *>(smem + L::kDone);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::kTmem);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / a.splits, split = blockIdx.x - tile * a.splits;
  const int m0 = (tile % a.tiles_m) * kBM, n0 = (tile / a.tiles_m) * BN;
  const int kb0 = (int)((int64_t)split * a.kblocks / a.splits);
  const int nkb = (int)((int64_t)(split + 1) * a.kblocks / a.splits) - kb0;  // >= 1

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < NB; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], kEpiWarps);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(L::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < nkb; ++i) {
        const int s = i % S, use = i / S;
        if (use > 0 && !mbar_wait_bounded(&empty[s], (use - 1) & 1, a.max_polls)) {
          flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
          break;
        }
        mbar_expect_tx(&full[s], L::kA + L::kB);
        tma_load_2d(sa + s * L::kA, &tx, (kb0 + i) * kBK, m0, &full[s]);
        tma_load_2d(sb + s * L::kB, &tw, (kb0 + i) * kBK, n0, &full[s]);
        ++issued;
      }
      // the last load of each stage has landed before the shared memory goes away
      for (int i = issued > S ? issued - S : 0; i < issued; ++i)
        if (!mbar_wait_bounded(&full[i % S], (i / S) & 1, a.max_polls)) flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = f8_idesc(BN);
      for (int i = 0; i < nkb; ++i) {
        const int s = i % S, buf = i % NB, use = i / NB;
        if ((use > 0 && !mbar_wait_bounded(&acc_empty[buf], (use - 1) & 1, a.max_polls)) ||
            !mbar_wait_bounded(&full[s], (i / S) & 1, a.max_polls)) {
          flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
          break;
        }
        tc_fence_after();
        const uint64_t ad = sw128_desc(sa + s * L::kA), bd = sw128_desc(sb + s * L::kB);
#pragma unroll
        for (int kk = 0; kk < kBK / 32; ++kk)  // 32 bytes of k per MMA along the swizzled rows
          tc_mma_f8(tmem + buf * BN, ad + 2 * kk, bd + 2 * kk, idesc, kk > 0 ? 1u : 0u);
        tc_commit(&empty[s]);
        tc_commit(&acc_full[buf]);
      }
      tc_commit(done);
    }
  } else {
    const int lg = warp & 3, part = (warp - 2) >> 2;  // TMEM lanes 32 lg ..; half of the columns
    const int row = m0 + lg * 32 + lane, col = part * kPart;
    const float *xs = a.xs + (int64_t)min(row, a.rows - 1) * a.xs_stride + kb0;
    const float *ws = a.ws + (int64_t)(n0 / 128) * a.ws_stride + kb0;
    float acc[kPart];
#pragma unroll
    for (int j = 0; j < kPart; ++j) acc[j] = 0.f;
    float scale = xs[0] * ws[0];
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const int buf = i % NB;
      const float sc = scale;
      if (i + 1 < nkb) scale = xs[i + 1] * ws[i + 1];
      if (!mbar_wait_bounded(&acc_full[buf], (i / NB) & 1, a.max_polls)) {
        ok = false;
        flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t t = tmem + ((uint32_t)(lg * 32) << 16) + buf * BN + col;
#pragma unroll
      for (int c = 0; c < kPart; c += 32) {
        uint32_t v[32];
        tmem_ld<32>(t + c, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[c + j] = fmaf(__uint_as_float(v[j]), sc, acc[c + j]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[buf]);
    }
    if (a.splits == 1) {
      if (ok && row < a.rows)
#pragma unroll
        for (int c = 0; c < kPart; c += 8)
          if (n0 + col + c < a.n) store_cols<T, 8>(a, row, n0 + col + c, acc + c);
    } else {
      // every MMA has read the stages before they are overwritten: this warp saw the last block's results
      float *tile_s = reinterpret_cast<float *>(smem) + (lg * 32 + lane) * (BN + 4) + col;
#pragma unroll
      for (int c = 0; c < kPart; c += 4)
        if (ok) *reinterpret_cast<float4 *>(tile_s + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
    }
  }
  __syncwarp();
  __syncthreads();
  if (a.splits > 1) {
    cluster_sync();
    const uint32_t base = smem_u32(smem);
    constexpr int kC4 = BN / 4;
    const int my_rows = (kBM - split + a.splits - 1) / a.splits;
    for (int it = threadIdx.x; it < my_rows * kC4; it += kThreads) {
      const int r = split + (it / kC4) * a.splits, c4 = it % kC4;
      if (m0 + r >= a.rows || n0 + 4 * c4 >= a.n) continue;
      const uint32_t off = (uint32_t)((r * (BN + 4) + 4 * c4) * sizeof(float));
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      for (int sp = 0; sp < a.splits; ++sp) {
        const float4 p = ld_cluster_f4(map_cluster(base + off, sp));
        v[0] += p.x;
        v[1] += p.y;
        v[2] += p.z;
        v[3] += p.w;
      }
      store_cols<T, 4>(a, m0 + r, n0 + 4 * c4, v);
    }
    cluster_sync();
  }
  if (warp == 1) {
    if (lane == 0 && !mbar_wait_bounded(done, 0, a.max_polls)) flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kCols) : "memory");
  }
}

// 2-D map of a row-major [rows, k] byte matrix, boxes of 128 (k) by box_rows
// rows, 128-byte swizzle, zero fill outside the matrix.
int encode_bytes(CUtensorMap *map, const void *base, int64_t k, int64_t rows, int64_t row_stride,
                 uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) {
    set_error_detail("pkv_linear_fp8: cuTensorMapEncodeTiled is not available from the driver");
    return PKV_ERR_TENSOR_MAP;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)row_stride};
  const cuuint32_t box[2] = {(cuuint32_t)kBK, box_rows}, elem[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, elem,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error_detail("pkv_linear_fp8: cuTensorMapEncodeTiled failed (%d) for a [%lld, %lld] matrix", (int)r,
                     (long long)rows, (long long)k);
    return PKV_ERR_TENSOR_MAP;
  }
  return PKV_OK;
}

template <typename T, int BN, int S>
int fp8_launch(const CUtensorMap &tx, const CUtensorMap &tw, const Fp8Args &a, cudaStream_t st) {
  using L = Smem<BN, S>;
  static_assert(L::kBytes <= 227 * 1024, "shared memory");
  static_assert(kBM * (BN + 4) * sizeof(float) <= L::kFull, "the split tile fits the ring");
  auto kern = linear_fp8_kernel<T, BN, S>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes) != cudaSuccess)
    return check_launch("cudaFuncSetAttribute(linear_fp8)");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.tiles_m * a.tiles_n * a.splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.splits > 1 ? 1 : 0;
  (void)cudaLaunchKernelEx(&cfg, kern, tx, tw, a);
  return check_launch("linear_fp8_kernel");
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_linear_fp8(const void *x, const float *x_scale, const void *w, const float *w_scale,
                              const void *bias, void *out, int32_t rows, int32_t n, int32_t k, int64_t x_stride,
                              int64_t xs_stride, int64_t w_stride, int64_t ws_stride, int64_t out_stride,
                              int32_t out_dtype, int32_t *status, void *stream) {
  if (rows < 0 || n <= 0 || k <= 0) {
    set_error_detail("pkv_linear_fp8: rows %d, n %d, k %d", rows, n, k);
    return PKV_ERR_INVALID_ARG;
  }
  if (out_dtype != PKV_DTYPE_BF16 && out_dtype != PKV_DTYPE_F16) {
    set_error_detail("pkv_linear_fp8: out must be bf16 or fp16");
    return PKV_ERR_UNSUPPORTED;
  }
  if (rows == 0) return PKV_OK;
  const int32_t kblocks = (k - 1) / kBK + 1;
  if (!x || !x_scale || !w || !w_scale || !out || xs_stride < kblocks || ws_stride < kblocks || out_stride < n) {
    set_error_detail("pkv_linear_fp8: NULL tensor pointer, or a row stride below the row's length");
    return PKV_ERR_INVALID_ARG;
  }
  if (!aligned_to(x, 16) || !aligned_to(w, 16) || x_stride < k || w_stride < k || x_stride % 16 != 0 ||
      w_stride % 16 != 0 || !aligned_to(x_scale, 4) || !aligned_to(w_scale, 4) || !aligned_to(out, 2) ||
      !aligned_to(bias, 2)) {
    set_error_detail("pkv_linear_fp8: x and W need 16-byte aligned bases and row strides (x %lld, W %lld)",
                     (long long)x_stride, (long long)w_stride);
    return PKV_ERR_ALIGNMENT;
  }
  Fp8Args a{};
  a.xs = x_scale;
  a.ws = w_scale;
  a.bias = bias;
  a.out = out;
  a.status = status;
  a.xs_stride = xs_stride;
  a.ws_stride = ws_stride;
  a.out_stride = out_stride;
  a.rows = rows;
  a.n = n;
  a.kblocks = kblocks;
  constexpr int BN = 128;
  a.tiles_m = (rows - 1) / kBM + 1;
  a.tiles_n = (n - 1) / BN + 1;
  a.splits = (int)std::max<int64_t>(
      1, std::min<int64_t>({(int64_t)kblocks, (int64_t)kMaxSplits, lin_sms() / ((int64_t)a.tiles_m * a.tiles_n)}));
  a.max_polls = kMaxPolls;
  if ((int64_t)a.tiles_m * a.tiles_n * a.splits > INT32_MAX) {
    set_error_detail("pkv_linear_fp8: too many tiles");
    return PKV_ERR_UNSUPPORTED;
  }
  CUtensorMap tx, tw;
  int rc = encode_bytes(&tx, x, k, rows, x_stride, kBM);
  if (rc) return rc;
  rc = encode_bytes(&tw, w, k, n, w_stride, BN);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return out_dtype == PKV_DTYPE_BF16 ? fp8_launch<__nv_bfloat16, BN, 6>(tx, tw, a, st)
                                     : fp8_launch<__half, BN, 6>(tx, tw, a, st);
}
