// pkv_loss.cu — from logits to the policy update: log-probabilities (and
// entropies) of given tokens, the clipped policy loss with a KL term, and the
// gradients of both.
//
// With z = x / T for one row x of logits, m = max x, c = log2(e) / T,
//   t_v = (x_v - m) c,  e_v = 2^t_v,  s = sum_v e_v,
//   log p_v = t_v ln2 - ln s,     H = ln s - ln2 (sum_v e_v t_v) / s.
// The difference to the maximum is taken before the scale, so rows of the
// type's lowest value, of -inf with one finite entry, or of huge logits need
// no special case; a row that is -inf throughout or holds NaN or +inf gives NaN.
// Both sums are kept per thread in fp32 with a running maximum (a thread that
// meets a new maximum rescales what it has) and joined over the block.
//
// Gradients, for g = dL/dlog p_token and h = dL/dH:
//   dL/dx_v = (g [v = token] - p_v (g + h (log p_v + H))) / T.
//
// Policy loss of one token, with r = exp(log p - old), d = ref - log p:
//   l = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (e^d - d - 1)
//   dl/dlog p = -r A [r A <= clip(r) A] + kl_coef (1 - e^d)
// and the loss is sum_tokens w l, w = mask / normaliser of the reduction.
#include <algorithm>
#include <cfloat>

#include "pkv_types.cuh"

namespace pkv {
namespace {

constexpr double kLog2e = 1.4426950408889634;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;  // CTAs that share a row: a portable cluster
constexpr int kUnroll = 4;      // 16-byte loads in flight per thread
constexpr int kMaxBlocks = 148 * 8;  // blocks of a policy launch that have sums to add

// Where row r of the logits begins: rows are (outer, inner) pairs.
struct Rows {
  int64_t outer_stride, row_stride;
  int32_t inner;
  __device__ __forceinline__ int64_t offset(int64_t r) const {
    return (r / inner) * outer_stride + (r % inner) * row_stride;
  }
};

// One row cut into 16-byte vectors of its aligned middle and the few elements
// before and after; CTA `rank` of the `ctas` that share the row has the vectors
// [lo, hi), the first one the head too and the last one the tail.
template <typename T>
struct Slice {
  static constexpr int kV = 16 / (int)sizeof(T);
  const T *x;
  int head, tail, tail0, lo, hi;  // tail0: first element of the tail
  __device__ __forceinline__ Slice(const T *row, int vocab, int rank, int ctas) : x(row) {
    const int peel = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    const int skip = min(vocab, peel), nvec = (vocab - skip) / kV;
    lo = (int)((int64_t)nvec * rank / ctas);
    hi = (int)((int64_t)nvec * (rank + 1) / ctas);
    tail0 = skip + nvec * kV;
    head = skip;
    tail = rank == ctas - 1 ? vocab - tail0 : 0;
    first = rank == 0;
  }
  bool first;
  __device__ __forceinline__ int at(int vec) const { return head + vec * kV; }  // first element of a vector
  __device__ __forceinline__ const uint4 *vecs() const { return reinterpret_cast<const uint4 *>(x + head); }
  // The head or tail element that thread t of those that share the slice has, or -1.
  __device__ __forceinline__ int edge(int t) const {
    if (first && t < head) return t;
    return t >= kV && t < kV + tail ? tail0 + t - kV : -1;
  }
};

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// The elements of a vector as fp32 pairs, their maximum (NaN if one is), and
// fp32 pairs rounded to a vector.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int kPairs = 2;
  static __device__ __forceinline__ void unpack(uint4 v, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ float max(uint4 v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)),
                   max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ uint4 max4(uint4 a, uint4 b) {
    return make_uint4(max2(a.x, b.x), max2(a.y, b.y), max2(a.z, b.z), max2(a.w, b.w));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[2]) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x),
                      __float_as_uint(f[1].y));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int kPairs = 4;
  static __device__ __forceinline__ float2 pair(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ void unpack(uint4 v, float2 (&f)[4]) {
    f[0] = pair(v.x), f[1] = pair(v.y), f[2] = pair(v.z), f[3] = pair(v.w);
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint4 max4(uint4 a, uint4 b) {
    return make_uint4(max2(a.x, b.x), max2(a.y, b.y), max2(a.z, b.z), max2(a.w, b.w));
  }
  static __device__ __forceinline__ float max(uint4 v) {
    const float2 m = pair(max2(max2(v.x, v.y), max2(v.z, v.w)));
    return max_nan(m.x, m.y);
  }
  static __device__ __forceinline__ uint32_t word(float2 f) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(f.y), "f"(f.x));
    return r;
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    return make_uint4(word(f[0]), word(f[1]), word(f[2]), word(f[3]));
  }
};
template <> struct Vec<__half> {
  static constexpr int kPairs = 4;
  static __device__ __forceinline__ float2 pair(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
  }
  static __device__ __forceinline__ void unpack(uint4 v, float2 (&f)[4]) {
    f[0] = pair(v.x), f[1] = pair(v.y), f[2] = pair(v.z), f[3] = pair(v.w);
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint4 max4(uint4 a, uint4 b) {
    return make_uint4(max2(a.x, b.x), max2(a.y, b.y), max2(a.z, b.z), max2(a.w, b.w));
  }
  static __device__ __forceinline__ float max(uint4 v) {
    const float2 m = pair(max2(max2(v.x, v.y), max2(v.z, v.w)));
    return max_nan(m.x, m.y);
  }
  static __device__ __forceinline__ uint32_t word(float2 f) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    return make_uint4(word(f[0]), word(f[1]), word(f[2]), word(f[3]));
  }
};

// Running maximum, sum of 2^t and sum of t 2^t of one thread (or of several, joined).
struct Soft {
  float m = -FLT_MAX, s = 0.f, w = 0.f;
};

// 0 * -inf is NaN: the weight of an entry with probability 0 in the entropy is 0
__device__ __forceinline__ float weighted(float e, float t) { return e * fmaxf(t, -1e4f); }

template <bool Entropy>
__device__ __forceinline__ void rescale(Soft &a, float m, float c) {
  const float d = (a.m - m) * c, f = fast_exp2(d);
  if (Entropy) a.w = f * a.w + weighted(f, d) * a.s;
  a.s *= f;
  a.m = m;
}

template <bool Entropy>
__device__ __forceinline__ void join(Soft &a, Soft b, float c) {
  const float m = max_nan(a.m, b.m);
  rescale<Entropy>(a, m, c);
  rescale<Entropy>(b, m, c);
  a.s += b.s;
  a.w += b.w;
}

template <bool Entropy>
__device__ __forceinline__ void add(Soft &a, float x, float c) {
  if (!(x <= a.m)) rescale<Entropy>(a, max_nan(a.m, x), c);
  const float t = (x - a.m) * c, e = fast_exp2(t);
  a.s += e;
  if (Entropy) a.w += weighted(e, t);
}

// N vectors: one look at the maximum, and their exponentials are added to each
// other before they are added to the running sum, which keeps what is small
// beside a dominant entry.
template <typename T, bool Entropy, int N>
__device__ __forceinline__ void add_vecs(Soft &a, const uint4 (&v)[N], float c) {
  constexpr int P = Vec<T>::kPairs;
  uint4 top = v[0];
#pragma unroll
  for (int n = 1; n < N; ++n) top = Vec<T>::max4(top, v[n]);
  const float vm = Vec<T>::max(top);
  if (!(vm <= a.m)) rescale<Entropy>(a, max_nan(a.m, vm), c);
  float2 s = make_float2(0.f, 0.f), w = s;
  const float2 nm = make_float2(-a.m, -a.m), cc = make_float2(c, c);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float2 f[P];
    Vec<T>::unpack(v[n], f);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 t = mul2(add2(f[i], nm), cc), e = make_float2(fast_exp2(t.x), fast_exp2(t.y));
      s = n + i == 0 ? e : add2(s, e);
      if (Entropy) w = fma2(e, make_float2(fmaxf(t.x, -1e4f), fmaxf(t.y, -1e4f)), w);
    }
  }
  a.s += s.x + s.y;
  if (Entropy) a.w += w.x + w.y;
}

__device__ __forceinline__ void mbar_expect(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// Barrier of the block's first NT threads.
template <int NT>
__device__ __forceinline__ void bar_sync() {
  __syncwarp();
  asm volatile("barrier.sync 1, %0;" ::"n"(NT) : "memory");
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

struct Joint {
  Soft warp[kWarps];
  Soft cta[kMaxCluster];  // written by the CTAs of the cluster
};

template <bool Entropy>
__device__ __forceinline__ void warp_join(Soft &a, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Soft b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.w = Entropy ? __shfl_xor_sync(0xffffffffu, a.w, o) : 0.f;
    join<Entropy>(a, b, c);
  }
}

// Joined over the block and over the CTAs that share the row (the caller has
// arrived at the cluster barrier once); every thread returns the same values.
template <bool Entropy>
__device__ __forceinline__ Soft row_join(Soft a, float c, Joint &red, int rank, int ctas) {
  warp_join<Entropy>(a, c);
  if ((threadIdx.x & 31) == 0) red.warp[threadIdx.x >> 5] = a;
  __syncthreads();
  a = red.warp[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) join<Entropy>(a, red.warp[i], c);
  if (ctas == 1) return a;
  cluster_wait();  // every CTA of the cluster runs: its shared memory may be written
  if (threadIdx.x < ctas) {
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(&red.cta[rank])), "r"(threadIdx.x));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(a.m) : "memory");
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(a.s) : "memory");
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(a.w) : "memory");
  }
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  a = red.cta[0];
  for (int i = 1; i < ctas; ++i) join<Entropy>(a, red.cta[i], c);
  return a;
}

// Thread tid's part (of NT) of n vectors in global (Ldg) or shared memory.
template <typename T, bool Entropy, int NT, bool Ldg>
__device__ __forceinline__ void add_range(Soft &a, const uint4 *p, int n, float c, int tid) {
  int i = tid;
  for (; i + (kUnroll - 1) * NT < n; i += kUnroll * NT) {
    uint4 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = Ldg ? __ldg(p + i + u * NT) : p[i + u * NT];
    add_vecs<T, Entropy, kUnroll>(a, v, c);
  }
  for (; i < n; i += NT) {
    const uint4 v[1] = {Ldg ? __ldg(p + i) : p[i]};
    add_vecs<T, Entropy, 1>(a, v, c);
  }
}

// ---------------------------------------------------------------------------
// token log-probabilities
// ---------------------------------------------------------------------------
struct LogprobArgs {
  const int64_t *tokens;
  float *logp, *entropy;  // entropy: with Entropy only
  float2 *stats;          // m and s of each row, or nullptr
  int32_t *status;
  int64_t rows;
  int32_t vocab, ctas;
  float inv_t, c;
};

// One thread per row, from the row's joined sums.
template <typename T, bool Entropy>
__device__ __forceinline__ void store_logprob(const LogprobArgs &p, const T *x, int64_t r, const Soft &a) {
  const int64_t tok = p.tokens[r];
  const bool in = tok >= 0 && tok < p.vocab;
  const float lns = logf(a.s);
  if (!in) flag_status(p.status, PKV_DEV_TOKEN_OUT_OF_RANGE);
  p.logp[r] = in ? (Elem<T>::to_f32(x[tok]) - a.m) * p.inv_t - lns : NAN;
  if (Entropy) p.entropy[r] = lns - kLn2 * (a.w / a.s);
  if (p.stats != nullptr) p.stats[r] = make_float2(a.m, a.s);
}

// A block, or the blocks of a cluster, per row: one read of the logits, four
// 16-byte loads in flight per thread. 4096 x 151,936 bf16 take 186 us, 6.7 TB/s,
// with the exponential unit 75% busy; one row 4.8 us in a cluster of 8 (17 us in
// one block).
template <typename T, bool Entropy>
__global__ void __launch_bounds__(kThreads) logprob_kernel(const T *logits, Rows rows, LogprobArgs p) {
  __shared__ Joint red;
  if (p.ctas > 1) cluster_arrive();
  const int64_t r = blockIdx.x / p.ctas;
  const int rank = blockIdx.x % p.ctas;
  const T *x = logits + rows.offset(r);
  const Slice<T> sl(x, p.vocab, rank, p.ctas);
  Soft a;
  add_range<T, Entropy, kThreads, true>(a, sl.vecs() + sl.lo, sl.hi - sl.lo, p.c, threadIdx.x);
  const int e = sl.edge(threadIdx.x);
  if (e >= 0) add<Entropy>(a, Elem<T>::to_f32(x[e]), p.c);
  a = row_join<Entropy>(a, p.c, red, rank, p.ctas);
  if (rank == 0 && threadIdx.x == 0) store_logprob<T, Entropy>(p, x, r, a);
}

// A warp per row, for rows that would leave most of a block idle: 65,536 rows of
// 200 fp32 take 25 us (181 with a block each).
template <typename T, bool Entropy>
__global__ void __launch_bounds__(kThreads) logprob_warp_kernel(const T *logits, Rows rows, LogprobArgs p) {
  const int64_t r = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  if (r >= p.rows) return;
  const T *x = logits + rows.offset(r);
  const Slice<T> sl(x, p.vocab, 0, 1);
  Soft a;
  add_range<T, Entropy, 32, true>(a, sl.vecs(), sl.hi, p.c, lane);
  const int e = sl.edge(lane);
  if (e >= 0) add<Entropy>(a, Elem<T>::to_f32(x[e]), p.c);
  __syncwarp();
  warp_join<Entropy>(a, p.c);
  if (lane == 0) store_logprob<T, Entropy>(p, x, r, a);
}

// Gradient of one element from t = (x - m) c and e = 2^t: e (a + b t), and `hot` more at the token.
struct Slope {
  float m, c, a, b, hot;
  int64_t tok;
};

template <bool Entropy>
__device__ __forceinline__ float grad_of(const Slope &g, float x, int v) {
  const float t = (x - g.m) * g.c, e = fast_exp2(t);
  const float d = Entropy ? e * fmaf(g.b, fmaxf(t, -1e4f), g.a) : e * g.a;
  return v == g.tok ? d + g.hot : d;
}

template <typename T, bool Entropy>
__device__ __forceinline__ uint4 grad_vec(const Slope &g, uint4 v) {
  constexpr int P = Vec<T>::kPairs;
  float2 f[P];
  Vec<T>::unpack(v, f);
  const float2 nm = make_float2(-g.m, -g.m), cc = make_float2(g.c, g.c), ga = make_float2(g.a, g.a),
               gb = make_float2(g.b, g.b);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float2 t = mul2(add2(f[i], nm), cc), e = make_float2(fast_exp2(t.x), fast_exp2(t.y));
    f[i] = Entropy ? mul2(e, fma2(gb, make_float2(fmaxf(t.x, -1e4f), fmaxf(t.y, -1e4f)), ga)) : mul2(e, ga);
  }
  return Vec<T>::pack(f);
}

// The gradient of the row's vectors [i0, i1), from `src` (i0's place, in global
// or shared memory). Where the vectors of the gradient's row do not begin where
// the logits' do, elements go one by one. The token's element gets its share
// from the thread that stored its vector.
template <typename T, bool Entropy, int NT>
__device__ __forceinline__ void grad_range(const Slice<T> &sl, const Slope &g, T *out, const uint4 *src, int i0,
                                           int i1, int tid) {
  if ((reinterpret_cast<uintptr_t>(out + sl.head) & 15) == 0) {
    uint4 *o = reinterpret_cast<uint4 *>(out + sl.head) + i0;
    const int n = i1 - i0;
    int i = tid;
    for (; i + (kUnroll - 1) * NT < n; i += kUnroll * NT) {
      uint4 v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) v[u] = src[i + u * NT];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        __stcs(o + i + u * NT, grad_vec<T, Entropy>(g, v[u]));
    }
    for (; i < n; i += NT) __stcs(o + i, grad_vec<T, Entropy>(g, src[i]));
    const int64_t k = g.tok - sl.at(i0);  // the token's place in the range
    if (k >= 0 && k < (int64_t)n * Slice<T>::kV && (int)(k / Slice<T>::kV) % NT == tid)
      out[g.tok] = from_f32<T>(grad_of<Entropy>(g, Elem<T>::to_f32(reinterpret_cast<const T *>(src)[k]), (int)g.tok));
  } else {
    const T *e = reinterpret_cast<const T *>(src);
    const int v0 = sl.at(i0), n = (i1 - i0) * Slice<T>::kV;
    for (int i = tid; i < n; i += NT)
      out[v0 + i] = from_f32<T>(grad_of<Entropy>(g, Elem<T>::to_f32(e[i]), v0 + i));
  }
}

template <typename T, bool Entropy>
__device__ __forceinline__ void grad_edge(const Slice<T> &sl, const Slope &g, T *out, int tid) {
  const int e = sl.edge(tid);
  if (e >= 0) out[e] = from_f32<T>(grad_of<Entropy>(g, Elem<T>::to_f32(sl.x[e]), e));
}

// NT threads per row or per share of a row (p.ctas of them): the logits are read
// once more and the gradient written. 515 x 32,003 fp32 with entropies: 19 us
// beside the forward pass's 20, of 20 for both from HBM alone (these 66 MB stay
// in L2).
template <typename T, bool Entropy, int NT>
__global__ void __launch_bounds__(kThreads)
logprob_grad_kernel(const T *logits, Rows rows, LogprobArgs p, const float *d_logp, const float *d_entropy, T *grad) {
  const int64_t at = (int64_t)blockIdx.x * (kThreads / NT) + threadIdx.x / NT, r = at / p.ctas;
  const int tid = threadIdx.x % NT;
  if (r >= p.rows) return;
  const Slice<T> sl(logits + rows.offset(r), p.vocab, (int)(at % p.ctas), p.ctas);
  const float2 st = p.stats[r];
  const float g = d_logp != nullptr ? d_logp[r] : 0.f, h = Entropy ? d_entropy[r] : 0.f, k = p.inv_t / st.y;
  // -p (g + h (log p + H)) / T with log p = t ln2 - ln s
  const Slope sp{st.x, p.c, Entropy ? -k * (g + h * (p.entropy[r] - logf(st.y))) : -k * g, -h * kLn2 * k,
                 g * p.inv_t, p.tokens[r]};
  T *out = grad + r * (int64_t)p.vocab;
  grad_range<T, Entropy, NT>(sl, sp, out, sl.vecs() + sl.lo, sl.lo, sl.hi, tid);
  grad_edge<T, Entropy>(sl, sp, out, tid);
}

// ---------------------------------------------------------------------------
// policy loss
// ---------------------------------------------------------------------------
struct PolicyArgs {
  const int64_t *tokens;   // [batch, length]
  const float *old_logp;   // [batch, length]
  const float *ref_logp;   // [batch, length] or nullptr
  const float *adv;        // strides adv_b, adv_t
  const uint8_t *mask;     // [batch, length] or nullptr
  float *out;              // loss, kl, clipped fraction
  float *logp;             // [batch, length]
  double *partial;         // workspace [3 * kMaxBlocks]: each block's sums
  int32_t *order;          // workspace [batch * length]: tokens with a weight first
  int32_t *before;         // workspace [batch + 1]: such tokens before each sequence
  int32_t *counts;         // workspace: [0] tokens with a weight, [1] blocks done
  float4 *slopes;          // workspace [batch * length]: what policy_grad_scaled_kernel takes of a row
  int32_t *status;
  int64_t adv_b, adv_t;
  int32_t batch, length, vocab, reduction;
  int32_t ctas, hold;  // CTAs of a row (loss alone); vectors of a row kept in shared memory (gradient)
  float inv_t, c, clip_low, clip_high, kl_coef;
  uint32_t max_polls;  // limit of each wait of the ring
  int32_t withhold;    // PKV_POLICY_TEST_WAIT_TIMEOUT: the first CTA leaves out its second row's last chunk
};

constexpr int kPrepThreads = 1024;

// Non-zero bytes among mask[0, n) that this thread of the block looks at.
__device__ __forceinline__ int count_mask(const uint8_t *mask, int64_t n) {
  int count = 0;
  int64_t i = threadIdx.x;
  if ((reinterpret_cast<uintptr_t>(mask) & 15) == 0) {
    for (; i < n / 16; i += kPrepThreads) {
      const uint4 v = __ldg(reinterpret_cast<const uint4 *>(mask) + i);
      count += __popc(__vsetne4(v.x, 0)) + __popc(__vsetne4(v.y, 0)) + __popc(__vsetne4(v.z, 0)) +
               __popc(__vsetne4(v.w, 0));
    }
    i = n / 16 * 16 + threadIdx.x;
  }
  for (; i < n; i += kPrepThreads) count += mask[i] != 0;
  return count;
}

// Sum over the block; every thread returns it.
__device__ __forceinline__ int block_sum(int v, int *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < kPrepThreads / 32; ++i) v += red[i];
  return v;
}

// The tokens with a weight in front, and how many of them there are before each
// sequence. One token per thread; each block counts what lies before and behind
// its tokens itself (a byte per token, from L2), so one launch does.
__global__ void __launch_bounds__(kPrepThreads) policy_prep_kernel(PolicyArgs a) {
  __shared__ int red[kPrepThreads / 32];
  const int64_t n = (int64_t)a.batch * a.length, base = (int64_t)blockIdx.x * kPrepThreads, i = base + threadIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool on = i < n && (a.mask == nullptr || a.mask[i] != 0);
  const uint32_t votes = __ballot_sync(0xffffffffu, on);
  int before = (int)base, total = (int)n;
  if (a.mask != nullptr) {
    before = block_sum(count_mask(a.mask, base), red);
    total = block_sum(count_mask(a.mask, n), red);
  }
  __syncthreads();
  if (lane == 0) red[warp] = __popc(votes);
  __syncthreads();
  for (int w = 0; w < warp; ++w) before += red[w];
  before += __popc(votes & ((1u << lane) - 1));
  if (i < n) {
    a.order[on ? before : total + (int)i - before] = (int32_t)i;
    if (i % a.length == 0) a.before[i / a.length] = before;
  }
  if (i == 0) {
    a.before[a.batch] = total;
    a.counts[0] = total;
    a.counts[1] = 0;
  }
}

// A token's inputs.
struct TokenIn {
  int64_t tok;
  float x, old, ref, adv;  // x: the token's logit
  int len;                 // tokens with a weight that share the token's weight's normaliser
  bool in;
};

template <typename T>
__device__ __forceinline__ TokenIn token_in(const PolicyArgs &a, const T *x, int64_t r) {
  TokenIn t;
  const int b = (int)r / a.length;
  t.tok = a.tokens[r];
  t.in = t.tok >= 0 && t.tok < a.vocab;
  t.old = a.old_logp[r];
  t.ref = a.ref_logp != nullptr ? a.ref_logp[r] : 0.f;
  t.adv = a.adv[b * a.adv_b + ((int)r - b * a.length) * a.adv_t];
  t.len = a.reduction == PKV_REDUCE_SEQUENCE ? a.before[b + 1] - a.before[b] : a.counts[0];
  t.x = t.in ? Elem<T>::to_f32(x[t.tok]) : 0.f;
  return t;
}

// Sums over a block's tokens: the weighted loss (its constant factor left out),
// the KL estimate, the clipped tokens.
struct Sums {
  double loss = 0, kl = 0, clipped = 0;
};

// What a row's gradient needs: the maximum, the factor of the exponentials, the
// slope at the token.
struct RowResult {
  float m, k, slope;
  int64_t tok;
};

// One thread per row, from the row's joined sums: its log-probability, its
// share of the sums, and what its gradient needs.
__device__ __forceinline__ RowResult token_result(const PolicyArgs &a, const TokenIn &t, const Soft &st, int64_t r,
                                                  Sums &sums) {
  const float lp = t.in ? (t.x - st.m) * a.inv_t - logf(st.s) : NAN;
  const float ratio = expf(lp - t.old);
  const float free = ratio * t.adv, clip = fminf(fmaxf(ratio, 1.f - a.clip_low), 1.f + a.clip_high) * t.adv;
  const bool clipped = clip < free;
  float l = clipped ? -clip : -free, slope = clipped ? 0.f : -free, kl = 0.f;
  if (a.ref_logp != nullptr) {
    const float d = t.ref - lp, em = expm1f(d);
    kl = em - d;
    l += a.kl_coef * kl;
    slope -= a.kl_coef * em;
  }
  if (!t.in) flag_status(a.status, PKV_DEV_TOKEN_OUT_OF_RANGE);
  a.logp[r] = lp;
  sums.loss += a.reduction == PKV_REDUCE_SEQUENCE ? (double)l / t.len : (double)l;
  sums.kl += kl;
  sums.clipped += clipped;
  const float w = a.reduction == PKV_REDUCE_SUM        ? 1.f
                  : a.reduction == PKV_REDUCE_SEQUENCE ? 1.f / ((float)t.len * (float)a.batch)
                                                       : 1.f / (float)t.len;
  slope *= w * a.inv_t;
  return RowResult{st.m, -slope / st.s, slope, t.tok};
}

// ... and in a gradient's kernel, kept for policy_grad_scaled_kernel.
__device__ __forceinline__ RowResult kept_result(const PolicyArgs &a, const TokenIn &t, const Soft &st, int64_t r,
                                                 Sums &sums) {
  const RowResult res = token_result(a, t, st, r, sums);
  a.slopes[r] = make_float4(res.m, res.k, res.slope, __int_as_float(t.in ? (int)t.tok : -1));
  return res;
}

// Called by the NT threads of a block with its sums in thread 0: the block that
// comes last of `blocks` adds the blocks' sums in their order. Each block's
// tokens and their order are fixed, so the result does not depend on timing.
template <int NT>
__device__ __forceinline__ void finish(const PolicyArgs &a, const Sums &mine, int block, int blocks) {
  __shared__ double sums[3][NT / 32];
  __shared__ int last_s;
  const int tid = threadIdx.x;
  if (tid == 0) {
    a.partial[3 * block] = mine.loss;
    a.partial[3 * block + 1] = mine.kl;
    a.partial[3 * block + 2] = mine.clipped;
    __threadfence();
    last_s = atomicAdd(&a.counts[1], 1) == blocks - 1;
  }
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  double v[3] = {0, 0, 0};
#pragma unroll 4
  for (int i = tid; i < blocks; i += NT) {
    v[0] += __ldcg(a.partial + 3 * i);
    v[1] += __ldcg(a.partial + 3 * i + 1);
    v[2] += __ldcg(a.partial + 3 * i + 2);
  }
#pragma unroll
  for (int j = 0; j < 3; ++j) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[j] += __shfl_xor_sync(0xffffffffu, v[j], o);
    if ((tid & 31) == 0) sums[j][tid >> 5] = v[j];
  }
  __syncthreads();
  if (tid < 3) {
    const double tokens = max(1, a.counts[0]);
    double t = 0;
    for (int i = 0; i < NT / 32; ++i) t += sums[tid][i];
    if (tid > 0 || a.reduction == PKV_REDUCE_TOKEN) t /= tokens;
    if (tid == 0 && a.reduction == PKV_REDUCE_SEQUENCE) t /= a.batch;
    a.out[tid] = (float)t;
  }
}

// The loss alone. A cluster takes every row_step-th row (one each where rows
// are shared), streamed.
template <typename T>
__global__ void __launch_bounds__(kThreads) policy_kernel(const T *logits, Rows rows, PolicyArgs a) {
  __shared__ Joint red;
  if (a.ctas > 1) cluster_arrive();
  const int64_t n = (int64_t)a.batch * a.length;
  const int rank = blockIdx.x % a.ctas, first = blockIdx.x / a.ctas, row_step = gridDim.x / a.ctas;
  const int active = a.counts[0];
  Sums sums;
  for (int64_t pos = first; pos < n; pos += row_step) {
    const int64_t r = a.order[pos];
    if (pos >= active) {
      if (a.ctas > 1) cluster_wait();
      if (rank == 0 && threadIdx.x == 0) a.logp[r] = 0.f;
      continue;
    }
    const T *x = logits + rows.offset(r);
    const Slice<T> sl(x, a.vocab, rank, a.ctas);
    Soft st;
    add_range<T, false, kThreads, true>(st, sl.vecs() + sl.lo, sl.hi - sl.lo, a.c, threadIdx.x);
    const int e = sl.edge(threadIdx.x);
    if (e >= 0) add<false>(st, Elem<T>::to_f32(x[e]), a.c);
    st = row_join<false>(st, a.c, red, rank, a.ctas);
    if (rank == 0 && threadIdx.x == 0) token_result(a, token_in(a, x, r), st, r, sums);
    if (a.ctas == 1) __syncthreads();  // every thread has read the warps' sums
  }
  if (rank == 0) finish<kThreads>(a, sums, first, row_step);
}

// A row without a weight: a gradient of zeros.
template <typename T, int NT>
__device__ __forceinline__ void zero_row(const PolicyArgs &a, T *grad, int64_t r, int tid) {
  T *out = grad + r * (int64_t)a.vocab;
  const Slice<T> sl(out, a.vocab, 0, 1);
  uint4 *o = reinterpret_cast<uint4 *>(out + sl.head);
#pragma unroll 4
  for (int v = tid; v < sl.hi; v += NT) __stcs(o + v, make_uint4(0, 0, 0, 0));
  const int e = sl.edge(tid);
  if (e >= 0) out[e] = from_f32<T>(0.f);
  if (tid == 0) a.logp[r] = 0.f;
}

// The loss and its gradient where a row fits in the registers of NT threads (a
// warp, of which a block has W, or a block), NV vectors each: loaded once,
// summed and turned into its gradient in place. The groups of threads take rows
// in turn; several on an SM overlap their phases. 16,384 rows of 1000 fp32 take
// 45 us (20 us of HBM traffic), 8192 of 16,000 bf16 121 (80).
template <typename T, int NT, int NV, int W, int PerSm>
__global__ void __launch_bounds__(NT * W, PerSm)
policy_row_kernel(const T *logits, Rows rows, T *grad, PolicyArgs a) {
  static_assert(NT == 32 || W == 1, "several rows per block: one warp each");
  __shared__ float2 part[NT / 32];
  __shared__ RowResult result[W];
  __shared__ Sums sums_s[W];
  const int tid = threadIdx.x % NT, group = threadIdx.x / NT, lane = tid & 31, warp = tid >> 5;
  const int64_t n = (int64_t)a.batch * a.length, step = (int64_t)gridDim.x * W;
  const int active = a.counts[0];
  auto sync = [] {
    if (NT == 32)
      __syncwarp();
    else
      __syncthreads();
  };
  Sums sums;
  int64_t pos = (int64_t)blockIdx.x * W + group;
  for (; pos < active; pos += step) {
    const int64_t r = a.order[pos];
    const T *x = logits + rows.offset(r);
    const Slice<T> sl(x, a.vocab, 0, 1);
    uint4 v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (tid + j * NT < sl.hi) v[j] = __ldg(sl.vecs() + tid + j * NT);
    TokenIn t;
    if (tid == 0) t = token_in(a, x, r);
    Soft st;
#pragma unroll
    for (int j = 0; j < NV; j += kUnroll) {
      if (tid + (j + kUnroll - 1) * NT < sl.hi) {
        const uint4 q[kUnroll] = {v[j], v[j + 1], v[j + 2], v[j + 3]};
        add_vecs<T, false, kUnroll>(st, q, a.c);
      } else {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (tid + (j + u) * NT < sl.hi) {
            const uint4 q[1] = {v[j + u]};
            add_vecs<T, false, 1>(st, q, a.c);
          }
      }
    }
    const int e = sl.edge(tid);
    if (e >= 0) add<false>(st, Elem<T>::to_f32(x[e]), a.c);
    __syncwarp();
    warp_join<false>(st, a.c);
    if (NT > 32) {
      if (lane == 0) part[warp] = make_float2(st.m, st.s);
      __syncthreads();
      if (warp == 0) {
        st = Soft();
        if (lane < NT / 32) {
          st.m = part[lane].x;
          st.s = part[lane].y;
        }
        warp_join<false>(st, a.c);
      }
    }
    if (tid == 0) result[group] = kept_result(a, t, st, r, sums);
    sync();
    const RowResult res = result[group];
    const Slope g{res.m, a.c, res.k, 0.f, res.slope, res.tok};
    T *out = grad + r * (int64_t)a.vocab;
    if ((reinterpret_cast<uintptr_t>(out + sl.head) & 15) == 0) {
      uint4 *o = reinterpret_cast<uint4 *>(out + sl.head);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (tid + j * NT < sl.hi) __stcs(o + tid + j * NT, grad_vec<T, false>(g, v[j]));
      const int64_t k = g.tok - sl.head;  // the token's share, from the thread that stored its vector
      if (k >= 0 && k < (int64_t)sl.hi * Slice<T>::kV && (int)(k / Slice<T>::kV) % NT == tid)
        out[g.tok] = from_f32<T>(grad_of<false>(g, Elem<T>::to_f32(x[g.tok]), (int)g.tok));
    } else {
      grad_range<T, false, NT>(sl, g, out, sl.vecs(), 0, sl.hi, tid);
    }
    grad_edge<T, false>(sl, g, out, tid);
    sync();  // the results may be overwritten
  }
  for (; pos < n; pos += step) zero_row<T, NT>(a, grad, a.order[pos], tid);
  if (W > 1) {
    if (tid == 0) sums_s[group] = sums;
    __syncthreads();
    if (threadIdx.x == 0)
      for (int i = 1; i < W; ++i) {
        sums.loss += sums_s[i].loss;
        sums.kl += sums_s[i].kl;
        sums.clipped += sums_s[i].clipped;
      }
  }
  finish<NT * W>(a, sums, blockIdx.x, gridDim.x);
}

// The loss and its gradient, a persistent grid; a CTA takes every gridDim-th
// row. The row is read from HBM once: its first K chunks (of kUnroll vectors per
// thread) are copied to shared memory, the rest is streamed to the sums and read
// again, from L2, for the gradient. The producer warp refills a chunk with the next
// row's as soon as its gradient has gone out, and the consumers add the refilled
// chunks up one chunk behind: reads, writes and arithmetic of two rows go on
// together, and only the join of a row's sums stands alone. Bound by HBM and, in
// that join, by latency: 2752 of 4096 rows of 151,936 bf16 take 400 us with all
// 4096 rows' gradients written, 5.2 TB/s of what has to cross; with every row
// 481 us. (Before: a block per row with two reads 1114 us; a cluster of 8 per row
// that holds it, 490; rows summed before the last one is written, 500; chunks
// of half the size 560.)
//
// Every wait is bounded. Where one runs out, its thread waits for nothing more,
// the consumers take no further row after the next join, the producer waits
// (bounded) for its copies in flight, and the status gets PKV_DEV_WAIT_TIMEOUT. For
// a caller without a status, the loss is NaN, and so are the log-probability and the
// first element of the gradient of each row that is left.
template <int NT, int K>
struct GradShared {
  uint64_t full[K], empty[K];  // a chunk has landed, has been used by every warp
  uint64_t info;                // token inputs are there
  TokenIn token[2];
  float2 part[NT / 32];
  RowResult result;
  volatile int dead;  // a wait ran out
  int stop;           // ... as every consumer sees it after the row's join
};

template <typename T, int NT, int K, int PerSm>
__global__ void __launch_bounds__(NT + 32, PerSm)
policy_grad_kernel(const T *logits, Rows rows, T *grad, PolicyArgs a) {
  extern __shared__ __align__(16) uint8_t held_raw[];
  __shared__ GradShared<NT, K> sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t n = (int64_t)a.batch * a.length;
  const int active = a.counts[0];
  uint4 *const hv = reinterpret_cast<uint4 *>(held_raw);
  if (tid == 0) {
    for (int k = 0; k < K; ++k) {
      mbar_init(&sh.full[k], 1);
      mbar_init(&sh.empty[k], NT / 32);
    }
    mbar_init(&sh.info, 1);
    sh.dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  auto chunk = [](int held, int k) { return min(held, k * NT * kUnroll); };
  bool ok = true;
  Sums sums;
  int it = 0, k = 0;  // this CTA's row; the producer's chunk of it, 0 once all have been issued

  if (warp == NT / 32) {
    // producer
    if (lane == 0) {
      for (int64_t pos = blockIdx.x; pos < active; pos += gridDim.x, ++it) {
        const int64_t r = a.order[pos];
        const T *x = logits + rows.offset(r);
        const Slice<T> sl(x, a.vocab, 0, 1);
        const int held = min(sl.hi, a.hold);
        for (k = 0; k < K; ++k) {
          if (it > 0) ok = mbar_wait_bounded(&sh.empty[k], (it - 1) & 1, a.max_polls);
          if (!ok) break;
          if (a.withhold && blockIdx.x == 0 && it == 1 && k == K - 1) continue;
          if (k == K / 2 && sl.hi > held)  // what is not held, on its way to L2 before the consumers stream it
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(sl.vecs() + held),
                         "r"((sl.hi - held) * 16)
                         : "memory");
          const int c0 = chunk(held, k), bytes = (chunk(held, k + 1) - c0) * 16;
          mbar_expect(&sh.full[k], bytes);
          if (bytes > 0)
            asm volatile(
                "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                    smem_u32(hv + c0)),
                "l"(sl.vecs() + c0), "r"(bytes), "r"(smem_u32(&sh.full[k]))
                : "memory");
        }
        if (!ok) break;
        k = 0;
        // slot it & 1 was last read for row it - 2, before any chunk of row it - 1 was free
        sh.token[it & 1] = token_in(a, x, r);
        mbar_arrive(&sh.info);
      }
    }
    __syncwarp();
  } else {
    // this thread's part of chunk k of the it-th row of this CTA
    auto sum_chunk = [&](Soft &st, int held, int k, int it) {
      const int c0 = chunk(held, k), c1 = chunk(held, k + 1);
      if (ok) ok = mbar_wait_bounded(&sh.full[k], it & 1, a.max_polls);
      if (ok)
        add_range<T, false, NT, false>(st, hv + c0, c1 - c0, a.c, tid);
      else
        sh.dead = 1;
    };
    auto sum_rest = [&](Soft &st, const Slice<T> &sl, int held) {
      add_range<T, false, NT, true>(st, sl.vecs() + held, sl.hi - held, a.c, tid);
      const int e = sl.edge(tid);
      if (e >= 0) add<false>(st, Elem<T>::to_f32(sl.x[e]), a.c);
    };
    int64_t pos = blockIdx.x, r = a.order[pos];
    Soft st;
    if (pos < active) {
      const Slice<T> sl(logits + rows.offset(r), a.vocab, 0, 1);
      const int held = min(sl.hi, a.hold);
      sum_rest(st, sl, held);
      for (k = 0; k < K; ++k) sum_chunk(st, held, k, 0);
    }
    for (; pos < active; pos += gridDim.x, ++it) {
      const bool more = pos + gridDim.x < active;
      const int64_t next = more ? a.order[pos + gridDim.x] : r;
      // the row's sums, joined over the block
      warp_join<false>(st, a.c);
      if (lane == 0) sh.part[warp] = make_float2(st.m, st.s);
      bar_sync<NT>();
      if (warp == 0) {
        st = Soft();
        if (lane < NT / 32) {
          st.m = sh.part[lane].x;
          st.s = sh.part[lane].y;
        }
        warp_join<false>(st, a.c);
        if (ok) ok = mbar_wait_bounded(&sh.info, it & 1, a.max_polls);
        if (!ok) sh.dead = 1;
        __syncwarp();
        if (lane == 0) {
          sh.stop = sh.dead;
          if (!sh.stop) sh.result = kept_result(a, sh.token[it & 1], st, r, sums);
        }
        __syncwarp();
      }
      bar_sync<NT>();
      if (sh.stop) break;
      const Slope g{sh.result.m, a.c, sh.result.k, 0.f, sh.result.slope, sh.result.tok};
      const Slice<T> sl(logits + rows.offset(r), a.vocab, 0, 1), sn(logits + rows.offset(next), a.vocab, 0, 1);
      const int held = min(sl.hi, a.hold), held_n = min(sn.hi, a.hold);
      T *out = grad + r * (int64_t)a.vocab;
      st = Soft();
      // what is not held first: it is the longest since it was read, and the chunks' refills are then in flight
      // until the end
      grad_range<T, false, NT>(sl, g, out, sl.vecs() + held, held, sl.hi, tid);
      for (k = 0; k < K; ++k) {
        const int c0 = chunk(held, k), c1 = chunk(held, k + 1);
        grad_range<T, false, NT>(sl, g, out, hv + c0, c0, c1, tid);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[k]);
        if (more && k > 0) sum_chunk(st, held_n, k - 1, it + 1);
      }
      grad_edge<T, false>(sl, g, out, tid);
      if (more) {
        sum_rest(st, sn, held_n);
        sum_chunk(st, held_n, K - 1, it + 1);
      }
      r = next;
    }
    for (; pos < active; pos += gridDim.x) {  // (only after a wait that ran out)
      r = a.order[pos];
      if (tid == 0) {
        grad[r * (int64_t)a.vocab] = from_f32<T>(NAN);
        a.logp[r] = NAN;
        a.slopes[r] = make_float4(NAN, NAN, NAN, __int_as_float(-1));
      }
    }
    for (; pos < n; pos += gridDim.x) zero_row<T, NT>(a, grad, a.order[pos], tid);
  }
  if (!ok) flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
  if (__syncthreads_or(!ok)) {
    sums.loss = sums.kl = sums.clipped = NAN;
    // copies in flight land before the shared memory goes away: the chunks before k for row it, the others for the last
    if (tid == NT && it + k > 0)
      for (int j = 0; j < K; ++j)
        if (!mbar_wait_bounded(&sh.full[j], (j < k ? it : it - 1) & 1, a.max_polls)) break;
  }
  finish<NT + 32>(a, sums, blockIdx.x, gridDim.x);
}

// The gradient again, for an upstream u other than 1, from what the loss kept of
// each row: u enters the fp32 slope, so an element is rounded once, where the
// stored gradient times u would have been rounded twice, and an fp16 element below
// the type's smallest step would have been lost before a loss scale could lift it.
// Nothing to do where u is 1, or in a row whose gradient is zero (no weight, or
// clipped): policy_loss wrote that. NT threads per row, or per share of one (ctas of
// them, of 64 KB and less); a persistent grid, since a launch for u = 1 should cost
// no more than a launch (1.6 us). Bound by HBM: 2752 of 4096 rows of 151,936 bf16
// take 292 us, 5.7 TB/s of what is read and written.
template <typename T, int NT>
__global__ void __launch_bounds__(kThreads, 4)
policy_grad_scaled_kernel(const T *logits, Rows rows, T *grad, const float4 *slopes, const int32_t *order,
                          const int32_t *counts, const float *upstream, int32_t vocab, int32_t ctas, float c) {
  const float u = *upstream;
  if (u == 1.f) return;
  const int64_t items = (int64_t)counts[0] * ctas, step = gridDim.x * (int64_t)(kThreads / NT);
  const int tid = threadIdx.x % NT;
  for (int64_t at = blockIdx.x * (int64_t)(kThreads / NT) + threadIdx.x / NT; at < items; at += step) {
    const int64_t r = order[at / ctas];
    const float4 st = slopes[r];
    if (st.y == 0.f && st.z == 0.f) continue;
    const Slice<T> sl(logits + rows.offset(r), vocab, (int)(at % ctas), ctas);
    const Slope g{st.x, c, st.y * u, 0.f, st.z * u, __float_as_int(st.w)};
    T *out = grad + r * (int64_t)vocab;
    grad_range<T, false, NT>(sl, g, out, sl.vecs() + sl.lo, sl.lo, sl.hi, tid);
    grad_edge<T, false>(sl, g, out, tid);
  }
}

// grad *= *upstream, nothing where it is 1
template <typename T>
__global__ void __launch_bounds__(kThreads) scale_grad_kernel(T *grad, int64_t n, const float *upstream) {
  const float u = *upstream;
  if (u == 1.f) return;
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < n; i += gridDim.x * (int64_t)kThreads)
    grad[i] = from_f32<T>(Elem<T>::to_f32(grad[i]) * u);
}

// CTAs that share a row: as many as leave each at most `most` bytes of it, and
// more, while that leaves each 4 KB, where the rows alone do not fill the
// machine (148 SMs with two CTAs each).
int row_ctas(int64_t rows, int64_t row_bytes, int64_t most) {
  int ctas = 1;
  while (ctas < kMaxCluster && (row_bytes > most * ctas ||
                                (rows * ctas < 2 * 148 && row_bytes >= 2 * 4096 * (int64_t)ctas)))
    ctas *= 2;
  return ctas;
}

// Rows of up to 16 KB go to a warp each where that gives every SM eight of them.
bool warp_rows(int64_t rows, int64_t row_bytes) { return row_bytes <= 16 * 1024 && rows >= 8 * 148; }

template <typename K, typename... Args>
int launch_rows(const char *what, K kern, int64_t rows, int ctas, void *stream, Args... args) {
  if (rows * ctas > INT32_MAX) {
    set_error_detail("%s: %lld rows are too many for one call", what, (long long)rows);
    return PKV_ERR_UNSUPPORTED;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  (void)cudaLaunchKernelEx(&cfg, kern, args...);
  return check_launch(what);
}

template <typename T, int NT, int NV, int W, int PerSm>
int launch_row(const T *logits, Rows rows, T *grad, const PolicyArgs &a, void *stream) {
  static_assert(148 * PerSm <= kMaxBlocks, "blocks with sums");
  const unsigned blocks = (unsigned)std::min<int64_t>(((int64_t)a.batch * a.length - 1) / W + 1, 148 * PerSm);
  policy_row_kernel<T, NT, NV, W, PerSm>
      <<<blocks, NT * W, 0, reinterpret_cast<cudaStream_t>(stream)>>>(logits, rows, grad, a);
  return check_launch("pkv_policy_loss");
}

template <typename T, int NT, int K, int PerSm>
int launch_held(const T *logits, Rows rows, T *grad, PolicyArgs a, void *stream) {
  a.hold = K * NT * kUnroll;
  const int smem = a.hold * 16;
  auto kern = policy_grad_kernel<T, NT, K, PerSm>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_launch("cudaFuncSetAttribute(policy_grad)");
  const unsigned blocks = (unsigned)std::min<int64_t>((int64_t)a.batch * a.length, 148 * PerSm);
  kern<<<blocks, NT + 32, smem, reinterpret_cast<cudaStream_t>(stream)>>>(logits, rows, grad, a);
  return check_launch("pkv_policy_loss");
}

// By what holds a row: a warp's registers, a small or a larger block's, or shared memory.
template <typename T>
int launch_grad(const T *logits, Rows rows, T *grad, const PolicyArgs &a, void *stream) {
  const int64_t bytes = (int64_t)a.vocab * sizeof(T);
  if (bytes <= 32 * 16 * 16) return launch_row<T, 32, 16, 4, 4>(logits, rows, grad, a, stream);
  if (bytes <= 128 * 16 * 16) return launch_row<T, 128, 16, 1, 4>(logits, rows, grad, a, stream);
  if (bytes <= 256 * 16 * 16) return launch_row<T, 256, 16, 1, 2>(logits, rows, grad, a, stream);
  // Two blocks on an SM, 96 KB of a row each, or one with 168 KB: rows of 100 KB take 176 us for 4096 in two and 254
  // in one, of 200 KB 167 us for 2048 in two and 175 in one, of 304 KB 568 us for 4096 in two and 481 in one.
  if (bytes <= 200 * 1024) return launch_held<T, 384, 4, 2>(logits, rows, grad, a, stream);
  return launch_held<T, 896, 3, 1>(logits, rows, grad, a, stream);
}

// The parts of a policy loss's workspace: the blocks' sums, two counters, what a
// scaled gradient takes of a row, an index per token, a count per sequence.
struct PolicyWorkspace {
  size_t counts, slopes, order, before, bytes;
};
PolicyWorkspace policy_workspace(int32_t batch, int32_t length) {
  const size_t rows = (size_t)batch * length;
  PolicyWorkspace w;
  w.counts = kMaxBlocks * 24;
  w.slopes = w.counts + 16;
  w.order = w.slopes + rows * sizeof(float4);
  w.before = w.order + rows * 4;
  w.bytes = w.before + ((size_t)batch + 1) * 4;
  return w;
}

bool bad_logits(const char *fn, const void *logits, int32_t dtype, int64_t rows, int32_t vocab, int32_t inner,
                float temperature) {
  if (rows >= 0 && rows <= INT32_MAX && vocab > 0 && inner > 0 && temperature > 0.f && (logits || rows == 0) &&
      aligned_to(logits, dtype_size(dtype)))
    return false;
  set_error_detail("%s: rows %lld, vocab %d, inner %d, temperature %g, logits %p", fn, (long long)rows, vocab, inner,
                   (double)temperature, logits);
  return true;
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_token_logprobs(const void *logits, int32_t dtype, const int64_t *tokens, int64_t rows,
                                  int32_t vocab, int32_t inner, int64_t outer_stride, int64_t row_stride,
                                  float temperature, float *logprobs, float *entropy, float *stats, int32_t *status,
                                  void *stream) {
  if (dtype_size(dtype) == 0) return PKV_ERR_UNSUPPORTED;
  if (bad_logits("pkv_token_logprobs", logits, dtype, rows, vocab, inner, temperature)) return PKV_ERR_INVALID_ARG;
  if (rows == 0) return PKV_OK;
  if (!tokens || !logprobs || !all_aligned(8, {tokens, stats}) || !all_aligned(4, {logprobs, entropy, status})) {
    set_error_detail("pkv_token_logprobs: NULL or misaligned pointer");
    return PKV_ERR_INVALID_ARG;
  }
  const Rows rw{outer_stride, row_stride, inner};
  const int64_t bytes = (int64_t)vocab * dtype_size(dtype);
  LogprobArgs p{tokens, logprobs, entropy, reinterpret_cast<float2 *>(stats), status, rows, vocab,
                row_ctas(rows, bytes, INT64_MAX / kMaxCluster), 1.f / temperature, (float)(kLog2e / temperature)};
  if (warp_rows(rows, bytes)) {
    PKV_BY_DTYPE(dtype, return launch_rows("pkv_token_logprobs",
                                           entropy ? logprob_warp_kernel<T, true> : logprob_warp_kernel<T, false>,
                                           (rows - 1) / kWarps + 1, 1, stream, (const T *)logits, rw, p))
  } else {
    PKV_BY_DTYPE(dtype, return launch_rows("pkv_token_logprobs",
                                           entropy ? logprob_kernel<T, true> : logprob_kernel<T, false>, rows, p.ctas,
                                           stream, (const T *)logits, rw, p))
  }
  return PKV_ERR_UNSUPPORTED;
}

extern "C" int pkv_token_logprobs_grad(const void *logits, int32_t dtype, const int64_t *tokens, int64_t rows,
                                       int32_t vocab, int32_t inner, int64_t outer_stride, int64_t row_stride,
                                       float temperature, const float *stats, const float *entropy,
                                       const float *d_logprobs, const float *d_entropy, void *d_logits,
                                       void *stream) {
  if (dtype_size(dtype) == 0) return PKV_ERR_UNSUPPORTED;
  if (bad_logits("pkv_token_logprobs_grad", logits, dtype, rows, vocab, inner, temperature))
    return PKV_ERR_INVALID_ARG;
  if (rows == 0) return PKV_OK;
  if (!tokens || !stats || !d_logits || (d_entropy && !entropy) || !aligned_to(d_logits, dtype_size(dtype)) ||
      !all_aligned(8, {tokens, stats}) || !all_aligned(4, {entropy, d_logprobs, d_entropy})) {
    set_error_detail("pkv_token_logprobs_grad: NULL or misaligned pointer");
    return PKV_ERR_INVALID_ARG;
  }
  const Rows rw{outer_stride, row_stride, inner};
  const int64_t bytes = (int64_t)vocab * dtype_size(dtype);
  LogprobArgs p{tokens, nullptr, const_cast<float *>(entropy), reinterpret_cast<float2 *>(const_cast<float *>(stats)),
                nullptr, rows, vocab, 1, 1.f / temperature, (float)(kLog2e / temperature)};
  if (warp_rows(rows, bytes)) {
    PKV_BY_DTYPE(dtype, return launch_rows("pkv_token_logprobs_grad",
                                           d_entropy ? logprob_grad_kernel<T, true, 32>
                                                     : logprob_grad_kernel<T, false, 32>,
                                           (rows - 1) / kWarps + 1, 1, stream, (const T *)logits, rw, p, d_logprobs,
                                           d_entropy, (T *)d_logits))
  } else {
    // shares of 64 KB, and of as little as 4 KB where the rows are few; they do not talk to each other
    p.ctas = row_ctas(rows, bytes, 64 * 1024);
    PKV_BY_DTYPE(dtype, return launch_rows("pkv_token_logprobs_grad",
                                           d_entropy ? logprob_grad_kernel<T, true, kThreads>
                                                     : logprob_grad_kernel<T, false, kThreads>,
                                           rows * p.ctas, 1, stream, (const T *)logits, rw, p, d_logprobs, d_entropy,
                                           (T *)d_logits))
  }
  return PKV_ERR_UNSUPPORTED;
}

extern "C" size_t pkv_policy_loss_workspace_size(int32_t batch, int32_t length) {
  if (batch < 0 || length < 0 || (int64_t)batch * length > INT32_MAX) return 0;
  return policy_workspace(batch, length).bytes;
}

extern "C" int pkv_policy_loss(const void *logits, int32_t dtype, const int64_t *tokens, const float *old_logprobs,
                               const float *ref_logprobs, const float *advantages, int64_t adv_stride_b,
                               int64_t adv_stride_t, const uint8_t *mask, int32_t batch, int32_t length,
                               int32_t vocab, int64_t batch_stride, int64_t row_stride, float temperature,
                               float clip_low, float clip_high, float kl_coef, int32_t reduction, float *out,
                               float *logprobs, void *d_logits, void *workspace, size_t workspace_bytes,
                               int32_t *status, void *stream) {
  if (dtype_size(dtype) == 0) return PKV_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)batch * length;
  const bool test_timeout = (reduction & PKV_POLICY_TEST_WAIT_TIMEOUT) != 0;
  reduction &= ~PKV_POLICY_TEST_WAIT_TIMEOUT;
  if (batch < 0 || length < 0 ||
      bad_logits("pkv_policy_loss", logits, dtype, rows, vocab, std::max(1, length), temperature))
    return PKV_ERR_INVALID_ARG;
  if (rows == 0) {  // nothing to add up
    if (out && cudaMemsetAsync(out, 0, 3 * sizeof(float), reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess)
      return PKV_OK;
    return out ? check_launch("pkv_policy_loss") : PKV_ERR_INVALID_ARG;
  }
  if (!tokens || !old_logprobs || !advantages || !out || !logprobs || !aligned_to(d_logits, dtype_size(dtype)) ||
      !aligned_to(tokens, 8) || !all_aligned(4, {old_logprobs, ref_logprobs, advantages, out, logprobs, status}) ||
      !(clip_low >= 0.f) || !(clip_high >= 0.f) || reduction < PKV_REDUCE_TOKEN || reduction > PKV_REDUCE_SUM) {
    set_error_detail("pkv_policy_loss: NULL or misaligned pointer, clip range %g / %g or reduction %d",
                     (double)clip_low, (double)clip_high, reduction);
    return PKV_ERR_INVALID_ARG;
  }
  if (!workspace || workspace_bytes < pkv_policy_loss_workspace_size(batch, length) || !aligned_to(workspace, 16))
    return PKV_ERR_WORKSPACE;
  PolicyArgs a{};
  a.max_polls = test_timeout ? 4096 : kMaxPolls;
  a.withhold = test_timeout;
  a.tokens = tokens;
  a.old_logp = old_logprobs;
  a.ref_logp = ref_logprobs;
  a.adv = advantages;
  a.mask = mask;
  a.out = out;
  a.logp = logprobs;
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  const PolicyWorkspace w = policy_workspace(batch, length);
  a.partial = reinterpret_cast<double *>(ws);
  a.counts = reinterpret_cast<int32_t *>(ws + w.counts);
  a.slopes = reinterpret_cast<float4 *>(ws + w.slopes);
  a.order = reinterpret_cast<int32_t *>(ws + w.order);
  a.before = reinterpret_cast<int32_t *>(ws + w.before);
  a.status = status;
  a.adv_b = adv_stride_b;
  a.adv_t = adv_stride_t;
  a.batch = batch;
  a.length = length;
  a.vocab = vocab;
  a.reduction = reduction;
  a.inv_t = 1.f / temperature;
  a.c = (float)(kLog2e / temperature);
  a.clip_low = clip_low;
  a.clip_high = clip_high;
  a.kl_coef = kl_coef;
  const Rows rw{batch_stride, row_stride, length};
  const int64_t row_bytes = (int64_t)vocab * dtype_size(dtype);
  a.ctas = row_ctas(rows, row_bytes, INT64_MAX / kMaxCluster);
  policy_prep_kernel<<<(unsigned)((rows - 1) / kPrepThreads + 1), kPrepThreads, 0,
                       reinterpret_cast<cudaStream_t>(stream)>>>(a);
  const int rc = check_launch("policy_prep_kernel");
  if (rc) return rc;
  if (d_logits) {
    PKV_BY_DTYPE(dtype, return launch_grad((const T *)logits, rw, (T *)d_logits, a, stream))
  } else {
    PKV_BY_DTYPE(dtype, return launch_rows("pkv_policy_loss", policy_kernel<T>,
                                           std::min<int64_t>(rows, kMaxBlocks), a.ctas, stream, (const T *)logits, rw,
                                           a))
  }
  return PKV_ERR_UNSUPPORTED;
}

extern "C" int pkv_policy_loss_grad(const void *logits, int32_t dtype, int32_t batch, int32_t length, int32_t vocab,
                                    int64_t batch_stride, int64_t row_stride, float temperature,
                                    const void *workspace, size_t workspace_bytes, const float *upstream,
                                    void *d_logits, void *stream) {
  if (dtype_size(dtype) == 0) return PKV_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)batch * length;
  if (batch < 0 || length < 0 ||
      bad_logits("pkv_policy_loss_grad", logits, dtype, rows, vocab, std::max(1, length), temperature))
    return PKV_ERR_INVALID_ARG;
  if (rows == 0) return PKV_OK;
  if (!upstream || !d_logits || !aligned_to(upstream, 4) || !aligned_to(d_logits, dtype_size(dtype))) {
    set_error_detail("pkv_policy_loss_grad: NULL or misaligned pointer");
    return PKV_ERR_INVALID_ARG;
  }
  const PolicyWorkspace w = policy_workspace(batch, length);
  if (!workspace || workspace_bytes < w.bytes || !aligned_to(workspace, 16)) return PKV_ERR_WORKSPACE;
  const uint8_t *ws = static_cast<const uint8_t *>(workspace);
  const auto *counts = reinterpret_cast<const int32_t *>(ws + w.counts);
  const auto *slopes = reinterpret_cast<const float4 *>(ws + w.slopes);
  const auto *order = reinterpret_cast<const int32_t *>(ws + w.order);
  const Rows rw{batch_stride, row_stride, length};
  const int64_t bytes = (int64_t)vocab * dtype_size(dtype);
  const bool warps = warp_rows(rows, bytes);
  const int ctas = warps ? 1 : row_ctas(rows, bytes, 64 * 1024);
  const unsigned blocks =
      (unsigned)std::min<int64_t>(warps ? (rows - 1) / kWarps + 1 : rows * ctas, 148 * 4);
  const float c = (float)(kLog2e / temperature);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PKV_BY_DTYPE(dtype, {
    auto k = warps ? policy_grad_scaled_kernel<T, 32> : policy_grad_scaled_kernel<T, kThreads>;
    k<<<blocks, kThreads, 0, st>>>((const T *)logits, rw, (T *)d_logits, slopes, order, counts, upstream, vocab, ctas,
                                   c);
  })
  return check_launch("pkv_policy_loss_grad");
}

extern "C" int pkv_scale_grad(void *grad, int64_t n, int32_t dtype, const float *upstream, void *stream) {
  if (dtype_size(dtype) == 0) return PKV_ERR_UNSUPPORTED;
  if (n < 0 || (n > 0 && (!grad || !upstream)) || !aligned_to(grad, dtype_size(dtype)) || !aligned_to(upstream, 4)) {
    set_error_detail("pkv_scale_grad: n %lld, NULL or misaligned pointer", (long long)n);
    return PKV_ERR_INVALID_ARG;
  }
  if (n == 0) return PKV_OK;
  const unsigned blocks = (unsigned)std::min<int64_t>((n + kThreads - 1) / kThreads, 148 * 8);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PKV_BY_DTYPE(dtype, (scale_grad_kernel<T><<<blocks, kThreads, 0, st>>>((T *)grad, n, upstream)))
  return check_launch("pkv_scale_grad");
}
