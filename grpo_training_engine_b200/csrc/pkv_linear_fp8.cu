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
// A persistent grid; a CTA (G = 1), or a pair of CTAs on one MMA (G = 2, twice
// the rows, each loading half of the columns), takes tiles of 128 G rows by BN
// columns in turn:
//   warp 0, one thread : TMA loads of 128-wide k blocks of x and W into an
//                        S-stage shared-memory ring (128-byte swizzle)
//   warp 1             : TMEM allocation; one thread (of the pair's first CTA)
//                        issues the 4 MMAs (M 128 G, N BN, K 32) of each block
//   warp 2             : the products of the two scales for each row and block,
//                        beside the TMEM buffers: straight from global memory
//                        every epilogue thread's load would be a line of its own
//   warps 4-11         : two warps per 32-lane TMEM group, half of the columns
//                        each: accumulate block by block, then store through
//                        shared memory by TMA, while the next tile's blocks are
//                        loaded and multiplied. They take the registers that the
//                        first four warps give up.
// With few rows the tiles of one weight matrix are split along k over the CTAs
// of a cluster, which add their fp32 tiles in split order through distributed
// shared memory, so results do not depend on timing.
//
// Bounds. 4096 x 18944 x 3584: 322 us, 1730 TFLOP/s (a bf16 library product of
// 8192^3 reaches 1634 here). The tensor pipe is busy 38% of the time: a block's
// sums have to be out of TMEM before its buffer is filled again, and all 512
// columns hold two blocks of a pair's tile. Measured in an earlier form of 339
// us: leaving the epilogue's reads out gave 0.64 us a block instead of 0.67,
// adding 28 blocks up inside the tensor core (wrong scales) 0.52; 128 x 128
// tiles by single CTAs stopped at 426 us, 10 TB/s out of L2; two MMAs of 128
// columns per block took 0.88 us a block; 16 epilogue warps of 64 columns 433 us
// (96 registers each). 37 x 151,936 x 1536: 54 us, 4.3 TB/s of weights: 594
// tiles of 12 blocks, two more than four rounds, each with the same hand-over.
// 128 x 1536 x 8960: 11.8 us; with k = 1024, one block per split, 8.3.
//
// Every wait is bounded; one that runs out sets PKV_DEV_WAIT_TIMEOUT, and the
// CTA waits (bounded) for its own copies and MMAs, frees its TMEM and returns.
#include <algorithm>
#include <type_traits>

#include "pkv_tc.cuh"
#include "pkv_types.cuh"

namespace pkv {

// pkv_linear_fp8_rows.cu: the product for a few rows
bool linear_fp8_rows_fits(int32_t rows, int32_t n, int32_t k);
int linear_fp8_rows(const void *x, const float *x_scale, const void *w, const float *w_scale, const void *bias,
                    void *out, int32_t rows, int32_t n, int32_t k, int64_t x_stride, int64_t xs_stride,
                    int64_t w_stride, int64_t ws_stride, int64_t out_stride, int32_t out_dtype, void *stream);

namespace {

constexpr int kBM = 128, kBK = 128;  // tile rows; k values of a block, the span of one scale
constexpr int kMaxSplits = 8;        // a portable cluster
constexpr int kFirstEpi = 4;         // first epilogue warp: its warpgroup is all epilogue
constexpr int kEpiWarps = 8, kThreads = 32 * (kFirstEpi + kEpiWarps);
// registers per thread: 384 threads start with 168 each, 64512 in all = 128 x 72 + 256 x 216
constexpr int kRegsOther = 72, kRegsEpi = 216;

struct Fp8Args {
  const float *xs, *ws;  // scales: rows of x, blocks of W
  const void *bias;      // [n], out's type, or nullptr
  void *out;
  int32_t *status;
  int64_t xs_stride, ws_stride, out_stride;
  int32_t rows, n, kblocks, tiles_m, tiles_n, splits;
  int32_t x_rows;   // rows of x that a tile loads (the MMA's others hold what they hold: their sums go nowhere)
  int32_t tma_out;  // out can be stored by TMA: 16-byte aligned base and rows
  uint32_t max_polls;
};

// D[tmem] (+)= A[smem] B[smem]^T with e4m3 operands, by one CTA or a pair
template <int G>
__device__ __forceinline__ void tc_mma_f8(uint32_t tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t acc) {
  if constexpr (G == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}

// Arrive on `bar` (of both CTAs of a pair) once every MMA issued before has completed.
template <int G>
__device__ __forceinline__ void tc_commit_group(uint64_t *bar) {
  if constexpr (G == 1)
    tc_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}

// TMA load into this CTA's shared memory that completes on a barrier of the
// pair's first CTA (`bar`: its cluster address).
template <int G>
__device__ __forceinline__ void tma_load_group(void *dst, const CUtensorMap *map, int32_t x, int32_t y, uint32_t bar) {
  if constexpr (G == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// One lane of the (converged) warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// Bounded wait of a thread that others wait for in turn: it looks again at once.
__device__ __forceinline__ bool mbar_wait_spin(uint64_t *bar, uint32_t parity, uint32_t max_polls) {
  for (uint32_t i = 0; i < max_polls; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return false;
}

// Instruction descriptor: fp32 accumulator, A and B e4m3 (0), both K-major, M m, N n.
__host__ __device__ constexpr uint32_t f8_idesc(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// 32 columns of this thread's TMEM lane; the values are there after tmem_wait.
__device__ __forceinline__ void tmem_ld_async(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
// Waits for this thread's loads; passing the registers through keeps their uses behind it.
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                 "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                 "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                 "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}

// acc += v * s, two columns per instruction
template <int N>
__device__ __forceinline__ void fma_cols(float2 (&acc)[N / 2], const uint32_t (&v)[N], float s) {
#pragma unroll
  for (int j = 0; j < N / 2; ++j)
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%0, %1};\n\t"
        "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "+f"(acc[j].x), "+f"(acc[j].y)
        : "r"(v[2 * j]), "r"(v[2 * j + 1]), "f"(s));
}

__device__ __forceinline__ uint32_t bits16(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ uint32_t bits16(__half v) { return __half_as_ushort(v); }

template <int BN, int S, int G>
struct Smem {
  static constexpr int kA = kBM * kBK, kB = BN / G * kBK;  // one stage of x and of W, bytes
  static constexpr int kCols = 512;                        // TMEM columns: all
  static constexpr int kBufs = kCols / BN;                 // TMEM buffers of BN fp32 columns
  static constexpr int kCW = BN / 2;                       // columns of an epilogue warp
  static constexpr int kBlocks = (BN + 127) / 128;         // blocks of W's scales across a tile
  static constexpr size_t kW = (size_t)S * kA;
  static constexpr size_t kOut = kW + (size_t)S * kB;      // 32 rows x kCW 16-bit results of each epilogue warp
  static constexpr size_t kSc = kOut + kEpiWarps * 32 * kCW * 2;  // [kBufs][kBlocks][kBM] fp32
  static constexpr size_t kFull = kSc + 4 * kBufs * kBlocks * kBM;
  static constexpr size_t kEmpty = kFull + 8 * S;
  static constexpr size_t kAccFull = kEmpty + 8 * S;
  static constexpr size_t kAccEmpty = kAccFull + 8 * kBufs;
  static constexpr size_t kDone = kAccEmpty + 8 * kBufs;
  static constexpr size_t kTmem = kDone + 8;
  static constexpr size_t kBytes = kTmem + 8 + 1024;  // + alignment slack
};

// NC results of one row, rounded.
template <typename T, int NC>
__device__ __forceinline__ void round_cols(const float *v, T (&o)[NC]) {
#pragma unroll
  for (int j = 0; j < NC; ++j) o[j] = from_f32<T>(v[j]);
}
template <typename T>
__device__ __forceinline__ uint4 pack_8(const T (&o)[8]) {
  return make_uint4(bits16(o[0]) | (bits16(o[1]) << 16), bits16(o[2]) | (bits16(o[3]) << 16),
                    bits16(o[4]) | (bits16(o[5]) << 16), bits16(o[6]) | (bits16(o[7]) << 16));
}

// ... and stored.
template <typename T, int NC>
__device__ __forceinline__ void store_cols(const Fp8Args &a, int row, int col, const float *v) {
  T *out = reinterpret_cast<T *>(a.out) + row * a.out_stride + col;
  T o[NC];
  round_cols<T, NC>(v, o);
  if constexpr (NC == 8) {
    if (col + NC <= a.n && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
      *reinterpret_cast<uint4 *>(out) = pack_8(o);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < NC; ++j)
    if (col + j < a.n) out[j] = o[j];
}

template <typename T, int BN, int S, int G>
__global__ void __launch_bounds__(kThreads, 1)
linear_fp8_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw,
                  const __grid_constant__ CUtensorMap to, Fp8Args a) {
  using L = Smem<BN, S, G>;
  constexpr int NB = L::kBufs, CW = L::kCW, ST = 32;
  constexpr bool kSplitRegs = CW == 128;  // 128 sums per epilogue thread
  extern __shared__ uint8_t raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *sa = smem, *sb = smem + L::kW;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kFull);
  uint64_t *empty = reinterpret_cast<uint64_t *>(smem + L::kEmpty);
  uint64_t *acc_full = reinterpret_cast<uint64_t *>(smem + L::kAccFull);
  uint64_t *acc_empty = reinterpret_cast<uint64_t *>(smem + L::kAccEmpty);
  uint64_t *done = reinterpret_cast<uint64_t *>(smem + L::kDone);
  float *sc = reinterpret_cast<float *>(smem + L::kSc);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::kTmem);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = G == 2 ? (int)(blockIdx.x & 1) : 0;  // in the pair
  const int split = G == 1 ? (int)(blockIdx.x % a.splits) : 0;
  const int first = G == 2 ? (int)(blockIdx.x >> 1) : (int)(blockIdx.x / a.splits);
  const int step = G == 2 ? (int)(gridDim.x >> 1) : (int)(gridDim.x / a.splits);
  const int tiles = a.tiles_m * a.tiles_n;
  const int kb0 = (int)((int64_t)split * a.kblocks / a.splits);
  const int nkb = (int)((int64_t)(split + 1) * a.kblocks / a.splits) - kb0;  // >= 1

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < NB; ++s) {
      mbar_init(&acc_full[s], 2);  // the MMAs, the scales
      mbar_init(&acc_empty[s], rank == 0 ? kEpiWarps * G : kEpiWarps);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tx)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tw)) : "memory");
  }
  if (warp == 1) {
    if constexpr (G == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(L::kCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(L::kCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (G == 2) cluster_sync();  // the pair's barriers and TMEM are ready in both CTAs
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto tile_m = [&](int t) { return (t % a.tiles_m) * (kBM * G) + rank * kBM; };  // this CTA's first row
  auto tile_n = [&](int t) { return (t / a.tiles_m) * BN; };

  if (warp < kFirstEpi) {
    if constexpr (kSplitRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    // (Warps 0 and 1 run their loops whole, one lane issues: the descriptors then are uniform values.)
    if (warp == 0) {
      int i = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        const int m0 = tile_m(t), n0 = tile_n(t) + rank * (BN / G);
        for (int k = 0; k < nkb; ++k, ++i) {
          const int s = i % S, use = i / S;
          ok = __all_sync(0xffffffffu, use == 0 || mbar_wait_spin(&empty[s], (use - 1) & 1, a.max_polls));
          if (!ok) break;
          if (elect_one()) {
            uint32_t bar = smem_u32(&full[s]);
            if (G == 2) bar = map_cluster(bar, 0);
            if (rank == 0) mbar_expect_tx(&full[s], G * (a.x_rows * kBK + L::kB));
            tma_load_group<G>(sa + s * L::kA, &tx, (kb0 + k) * kBK, m0, bar);
            tma_load_group<G>(sb + s * L::kB, &tw, (kb0 + k) * kBK, n0, bar);
          }
          __syncwarp();
        }
      }
      if (!ok) flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
      // the last load of each stage has landed before the shared memory goes away (in the pair's second
      // CTA: the MMAs that read it are waited for)
      if (rank == 0)
        for (int j = i > S ? i - S : 0; j < i; ++j)
          if (!mbar_wait_spin(&full[j % S], (j / S) & 1, a.max_polls)) flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
    } else if (warp == 1) {
      if (rank == 0) {
        constexpr uint32_t idesc = f8_idesc(kBM * G, BN);
        int i = 0;
        bool ok = true;
        for (int t = first; t < tiles && ok; t += step) {
          for (int k = 0; k < nkb; ++k, ++i) {
            const int s = i % S, buf = i % NB, use = i / NB;
            ok = mbar_wait_spin(&full[s], (i / S) & 1, a.max_polls) &&
                 (use == 0 || mbar_wait_spin(&acc_empty[buf], (use - 1) & 1, a.max_polls));
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint64_t ad = sw128_desc(sa + s * L::kA), bd = sw128_desc(sb + s * L::kB);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < kBK / 32; ++kk)  // 32 bytes of k per MMA along the swizzled rows
                tc_mma_f8<G>(tmem + buf * BN, ad + 2 * kk, bd + 2 * kk, idesc, kk > 0 ? 1u : 0u);
              tc_commit_group<G>(&acc_full[buf]);
              tc_commit_group<G>(&empty[s]);
            }
            __syncwarp();
          }
        }
        if (!ok) flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
        if (elect_one()) tc_commit_group<G>(done);
        __syncwarp();
      }
    } else if (warp == 2) {
      // four blocks at a time, the next four's loads in flight while these are handed out
      struct Group {
        float x[4][4], w[4][L::kBlocks];  // [block][32 rows], [block][128 columns]
      };
      auto load = [&](int t, int k0, Group &g) {
        const int m0 = tile_m(t), nb0 = tile_n(t) / 128, nb_last = (a.n - 1) / 128;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int k = kb0 + min(k0 + q, nkb - 1);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            g.x[q][j] = m0 + 32 * j < a.rows ? a.xs[min(m0 + lane + 32 * j, a.rows - 1) * a.xs_stride + k] : 0.f;
#pragma unroll
          for (int b = 0; b < L::kBlocks; ++b) g.w[q][b] = a.ws[min(nb0 + b, nb_last) * a.ws_stride + k];
        }
      };
      int i = 0, t = first, k0 = 0;
      bool ok = true;
      Group now, next;
      if (t < tiles) load(t, 0, now);
      while (t < tiles && ok) {
        const int kn = k0 + 4 < nkb ? k0 + 4 : 0, tn = kn > 0 ? t : t + step;
        if (tn < tiles) load(tn, kn, next);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (k0 + q >= nkb || !ok) break;
          const int slot = i % NB, use = i / NB;
          ok = __all_sync(0xffffffffu, use == 0 || mbar_wait_spin(&acc_empty[slot], (use - 1) & 1, a.max_polls));
#pragma unroll
          for (int b = 0; b < L::kBlocks; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[(slot * L::kBlocks + b) * kBM + lane + 32 * j] = now.x[q][j] * now.w[q][b];
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_full[slot]);
          ++i;
        }
        now = next;
        t = tn;
        k0 = kn;
      }
      if (!ok) flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
    }
  } else {
    if constexpr (kSplitRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    const int lg = warp & 3, part = (warp - kFirstEpi) >> 2;  // TMEM lanes 32 lg ..; half of the columns
    const uint32_t tcol = part * CW + ((uint32_t)(lg * 32) << 16);
    T *stage = reinterpret_cast<T *>(smem + L::kOut) + (warp - kFirstEpi) * 32 * CW;
    const float *my_sc = sc + part * CW / 128 * kBM + lg * 32 + lane;
    constexpr int kStretches = CW / ST;
    static_assert(kStretches % 2 == 0, "two buffers in turn");
    float2 acc[kStretches][ST / 2];
    // block i's sums and scales are there
    auto ready = [&](int i) {
      const bool ok = mbar_wait_spin(&acc_full[i % NB], (i / NB) & 1, a.max_polls);
      const bool all = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      return all;
    };
    int i = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      const int row = tile_m(t) + lg * 32 + lane, n0 = tile_n(t) + part * CW;
      // the sums begin at the bias (where k is split, it is added with the splits)
#pragma unroll
      for (int c = 0; c < kStretches; ++c)
#pragma unroll
        for (int j = 0; j < ST / 2; ++j) acc[c][j] = make_float2(0.f, 0.f);
      if (a.bias != nullptr && a.splits == 1) {
        const T *bias = reinterpret_cast<const T *>(a.bias) + n0;
#pragma unroll
        for (int c = 0; c < kStretches; ++c)
#pragma unroll
          for (int j = 0; j < ST / 2; ++j) {
            if (n0 + c * ST + 2 * j < a.n) acc[c][j].x = Elem<T>::to_f32(bias[c * ST + 2 * j]);
            if (n0 + c * ST + 2 * j + 1 < a.n) acc[c][j].y = Elem<T>::to_f32(bias[c * ST + 2 * j + 1]);
          }
      }
      // The loads of one stretch of ST columns are in flight while the last one is added up, and the next
      // block is waited for meanwhile.
      uint32_t v[2][ST];
      ok = ready(i);
      float scale = my_sc[i % NB * L::kBlocks * kBM], next = 0.f;
      if (ok) tmem_ld_async(tmem + i % NB * BN + tcol, v[0]);
      for (int k = 0; k < nkb && ok; ++k, ++i) {
        const int buf = i % NB;
#pragma unroll
        for (int c = 0; c < kStretches; ++c) {
          tmem_wait(v[c & 1]);
          if (c + 1 < kStretches) {
            tmem_ld_async(tmem + buf * BN + tcol + ST * (c + 1), v[(c + 1) & 1]);
          } else {
            // the buffer and the scale have been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&acc_empty[buf]);
              if (rank == 1)  // for the MMAs, which the pair's first CTA issues
                asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(
                                 map_cluster(smem_u32(&acc_empty[buf]), 0))
                             : "memory");
            }
            __syncwarp();  // (the loads are a whole warp's)
            if (k + 1 < nkb && ok) tmem_ld_async(tmem + (i + 1) % NB * BN + tcol, v[(c + 1) & 1]);
          }
          fma_cols<ST>(acc[c], v[c & 1], scale);
          if (c == kStretches - 2 && k + 1 < nkb) {
            ok = ready(i + 1);
            next = my_sc[(i + 1) % NB * L::kBlocks * kBM];
          }
        }
        scale = next;
      }
      if (!ok) flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
      if (a.splits == 1 && a.tma_out) {
        // 32 rows by 64 columns at a time, swizzled as TMA reads them, which clips what lies outside
        const int row0 = row - lane;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the last tile's have been read
        __syncwarp();
#pragma unroll
        for (int c = 0; c < CW / 8; ++c) {
          T o[8];
          round_cols<T, 8>(&acc[8 * c / ST][8 * c % ST / 2].x, o);
          uint4 *dst = reinterpret_cast<uint4 *>(stage + c / 8 * (32 * 64) + lane * 64);
          dst[(c % 8) ^ (lane & 7)] = pack_8(o);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && ok && row0 < a.rows) {
#pragma unroll
          for (int c = 0; c < CW / 64; ++c)
            if (n0 + 64 * c < a.n)
              asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                               reinterpret_cast<uint64_t>(&to)),
                           "r"(n0 + 64 * c), "r"(row0), "r"(smem_u32(stage + c * (32 * 64)))
                           : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      } else if (a.splits == 1) {
        if (ok && row < a.rows) {
#pragma unroll
          for (int c = 0; c < CW / 8; ++c)
            if (n0 + 8 * c < a.n) store_cols<T, 8>(a, row, n0 + 8 * c, &acc[8 * c / ST][8 * c % ST / 2].x);
        }
      } else {
        // every MMA has read the stages before they are overwritten: this warp saw the last block's results
        float *tile_s = reinterpret_cast<float *>(smem) + (lg * 32 + lane) * (BN + 4) + part * CW;
        if (ok) {
#pragma unroll
          for (int c = 0; c < CW / 4; ++c)
            *reinterpret_cast<float4 *>(tile_s + 4 * c) =
                make_float4(acc[4 * c / ST][4 * c % ST / 2].x, acc[4 * c / ST][4 * c % ST / 2].y,
                            acc[4 * c / ST][4 * c % ST / 2 + 1].x, acc[4 * c / ST][4 * c % ST / 2 + 1].y);
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  __syncthreads();
  if (G == 1 && a.splits > 1) {  // one tile per cluster
    cluster_sync();
    const int m0 = tile_m(first), n0 = tile_n(first);
    const uint32_t base = smem_u32(smem);
    constexpr int kC4 = BN / 4;
    const int my_rows = (min(kBM, a.rows - m0) - split + a.splits - 1) / a.splits;
    for (int it = threadIdx.x; it < my_rows * kC4; it += kThreads) {
      const int r = split + (it / kC4) * a.splits, c4 = it % kC4;
      if (n0 + 4 * c4 >= a.n) continue;
      const uint32_t off = (uint32_t)((r * (BN + 4) + 4 * c4) * sizeof(float));
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      for (int sp = 0; sp < a.splits; ++sp) {
        const float4 p = ld_cluster_f4(map_cluster(base + off, sp));
        v[0] += p.x;
        v[1] += p.y;
        v[2] += p.z;
        v[3] += p.w;
      }
      if (a.bias != nullptr) {
        const T *bias = reinterpret_cast<const T *>(a.bias) + n0 + 4 * c4;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n0 + 4 * c4 + j < a.n) v[j] += Elem<T>::to_f32(bias[j]);
      }
      store_cols<T, 4>(a, m0 + r, n0 + 4 * c4, v);
    }
    cluster_sync();
  }
  if (warp == 1) {
    if (lane == 0 && !mbar_wait_spin(done, 0, a.max_polls)) flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
    __syncwarp();
  }
  if (G == 2) cluster_sync();  // no MMA of the pair is in flight, nothing arrives at a CTA that has gone
  if (warp == 1) {
    tc_fence_after();
    if constexpr (G == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kCols) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kCols) : "memory");
  }
}

// 2-D map of a row-major [rows, cols] matrix of `type`, boxes of 128 bytes of a
// row by box_rows rows, 128-byte swizzle; loads read zeros outside the matrix.
int encode_rows(CUtensorMap *map, CUtensorMapDataType type, int size, const void *base, int64_t cols, int64_t rows,
                int64_t row_stride, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) {
    set_error_detail("pkv_linear_fp8: cuTensorMapEncodeTiled is not available from the driver");
    return PKV_ERR_TENSOR_MAP;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(row_stride * size)};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / size), box_rows}, elem[2] = {1, 1};
  const CUresult r = fn(map, type, 2, const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error_detail("pkv_linear_fp8: cuTensorMapEncodeTiled failed (%d) for a [%lld, %lld] matrix", (int)r,
                     (long long)rows, (long long)cols);
    return PKV_ERR_TENSOR_MAP;
  }
  return PKV_OK;
}

template <typename T, int BN, int S, int G>
int fp8_launch(const void *x, const void *w, int64_t k, int64_t x_stride, int64_t w_stride, Fp8Args a,
               cudaStream_t st) {
  using L = Smem<BN, S, G>;
  static_assert(L::kBytes <= 227 * 1024, "shared memory");
  static_assert(G == 2 || kBM * (BN + 4) * sizeof(float) <= L::kSc, "the split tile fits the ring");
  a.x_rows = std::min(kBM, (a.rows + 7) / 8 * 8);
  CUtensorMap tx, tw, to;
  int rc = encode_rows(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, k, a.rows, x_stride, a.x_rows);
  if (rc == PKV_OK) rc = encode_rows(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, k, a.n, w_stride, BN / G);
  to = tx;
  a.tma_out = aligned_to(a.out, 16) && a.out_stride % 8 == 0;
  if (rc == PKV_OK && a.tma_out)
    rc = encode_rows(&to, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, a.out, a.n, a.rows, a.out_stride, 32);
  if (rc != PKV_OK) return rc;
  auto kern = linear_fp8_kernel<T, BN, S, G>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes) != cudaSuccess)
    return check_launch("cudaFuncSetAttribute(linear_fp8)");
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
  const int cluster = G == 2 ? 2 : a.splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(tiles * cluster, lin_sms() / cluster * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  (void)cudaLaunchKernelEx(&cfg, kern, tx, tw, to, a);
  return check_launch("linear_fp8_kernel");
}

template <typename T>
int fp8_dispatch(const void *x, const void *w, int64_t k, int64_t x_stride, int64_t w_stride, Fp8Args a,
                 cudaStream_t st) {
  const int sms = lin_sms();
  auto tiles = [&](int bm, int bn) {
    a.tiles_m = (a.rows - 1) / bm + 1;
    a.tiles_n = (a.n - 1) / bn + 1;
    return (int64_t)a.tiles_m * a.tiles_n;
  };
  a.splits = 1;
  // Many rows: pairs, whose 256 x 256 tiles read least from L2 for what they multiply (4096 x 18944 x 3584: 322 us
  // against 426 with 128 x 128 tiles, which stop at 10 TB/s out of L2), from half a round of them on (512 x 8960 x
  // 1536: 15.6 us against 18.1).
  if (a.rows > kBM && tiles(256, 256) >= sms / 4)
    return fp8_launch<T, 256, 4, 2>(x, w, k, x_stride, w_stride, a, st);
  // Wide matrices: an MMA of 256 columns takes little longer than one of 64 (151,936 columns by 37 rows: 54 us
  // against 67).
  if (tiles(128, 256) >= 2 * sms) return fp8_launch<T, 256, 3, 1>(x, w, k, x_stride, w_stride, a, st);
  // The rest: 128-column tiles, k split until they fill the machine. (Twice as many of 64 columns, two CTAs on an SM,
  // took 12.0 us for 128 x 1536 x 8960 where this takes 11.7, 10.2 against 8.2 for 24 x 8960 x 1536.) Clusters of
  // more than 2 only where all of them fit at once: 16 of 8 did not and took a second round (2048 x 1536: 11.8 us, 6.7
  // in clusters of 4), nor 48 of 3 (512 x 1536 x 8960: 33 us).
  const int64_t t = tiles(128, 128);
  int64_t splits = std::min<int64_t>({(int64_t)a.kblocks, (int64_t)kMaxSplits, sms / t});
  if (splits > 4 && t * splits > 96) splits = 4;
  while (splits > 2 && t * splits > 120) --splits;
  a.splits = (int)std::max<int64_t>(1, splits);
  return fp8_launch<T, 128, 5, 1>(x, w, k, x_stride, w_stride, a, st);
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
      w_stride % 16 != 0 || !all_aligned(4, {x_scale, w_scale, status}) || !all_aligned(2, {out, bias})) {
    set_error_detail("pkv_linear_fp8: x and W need 16-byte aligned bases and row strides (x %lld, W %lld), the "
                     "others their elements' alignment",
                     (long long)x_stride, (long long)w_stride);
    return PKV_ERR_ALIGNMENT;
  }
  if (linear_fp8_rows_fits(rows, n, k))
    return linear_fp8_rows(x, x_scale, w, w_scale, bias, out, rows, n, k, x_stride, xs_stride, w_stride, ws_stride,
                           out_stride, out_dtype, stream);
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
  a.max_polls = kMaxPolls;
  if (((int64_t)(rows - 1) / kBM + 1) * ((n - 1) / 128 + 1) > INT32_MAX / 2) {
    set_error_detail("pkv_linear_fp8: too many tiles");
    return PKV_ERR_UNSUPPORTED;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return out_dtype == PKV_DTYPE_BF16 ? fp8_dispatch<__nv_bfloat16>(x, w, k, x_stride, w_stride, a, st)
                                     : fp8_dispatch<__half>(x, w, k, x_stride, w_stride, a, st);
}
