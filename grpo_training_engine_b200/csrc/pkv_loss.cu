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
constexpr int64_t kHoldTarget = 40 * 1024;  // bytes of a row per CTA that leave room for five CTAs on an SM
constexpr int64_t kHoldMost = 200 * 1024;   // of a longer share, what is kept in shared memory

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
  // The head or tail element that this thread has, or -1.
  __device__ __forceinline__ int edge() const {
    const int t = threadIdx.x;
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

// A vector: its exponentials are added to each other before they are added to
// the running sum, which keeps what is small beside a dominant entry.
template <typename T, bool Entropy>
__device__ __forceinline__ void add_vec(Soft &a, uint4 v, float c) {
  constexpr int P = Vec<T>::kPairs;
  const float vm = Vec<T>::max(v);
  if (!(vm <= a.m)) rescale<Entropy>(a, max_nan(a.m, vm), c);
  float2 f[P], s = make_float2(0.f, 0.f), w = s;
  Vec<T>::unpack(v, f);
  const float2 nm = make_float2(-a.m, -a.m), cc = make_float2(c, c);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float2 t = mul2(add2(f[i], nm), cc), e = make_float2(fast_exp2(t.x), fast_exp2(t.y));
    s = i == 0 ? e : add2(s, e);
    if (Entropy) w = fma2(e, make_float2(fmaxf(t.x, -1e4f), fmaxf(t.y, -1e4f)), w);
  }
  a.s += s.x + s.y;
  if (Entropy) a.w += w.x + w.y;
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

struct Joint {
  Soft warp[kWarps];
  Soft cta[kMaxCluster];  // written by the CTAs of the cluster
};

// Joined over the block and over the CTAs that share the row (the caller has
// arrived at the cluster barrier once); every thread returns the same values.
template <bool Entropy>
__device__ __forceinline__ Soft row_join(Soft a, float c, Joint &red, int rank, int ctas) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Soft b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.w = Entropy ? __shfl_xor_sync(0xffffffffu, a.w, o) : 0.f;
    join<Entropy>(a, b, c);
  }
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

// This thread's part of a slice, streamed from global memory from vector `lo` on.
template <typename T, bool Entropy>
__device__ __forceinline__ void add_stream(Soft &a, const Slice<T> &sl, int lo, float c) {
  const uint4 *p = sl.vecs();
  int i = lo + (int)threadIdx.x;
  for (; i + (kUnroll - 1) * kThreads < sl.hi; i += kUnroll * kThreads) {
    uint4 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = __ldg(p + i + u * kThreads);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) add_vec<T, Entropy>(a, v[u], c);
  }
  for (; i < sl.hi; i += kThreads) add_vec<T, Entropy>(a, __ldg(p + i), c);
}

// ---------------------------------------------------------------------------
// token log-probabilities
// ---------------------------------------------------------------------------
template <typename T, bool Entropy>
__global__ void __launch_bounds__(kThreads)
logprob_kernel(const T *logits, Rows rows, const int64_t *tokens, int vocab, int ctas, float inv_t, float c,
               float *logp, float *entropy, float2 *stats, int32_t *status) {
  __shared__ Joint red;
  if (ctas > 1) cluster_arrive();
  const int64_t r = blockIdx.x / ctas;
  const int rank = blockIdx.x % ctas;
  const T *x = logits + rows.offset(r);
  const Slice<T> sl(x, vocab, rank, ctas);
  Soft a;
  add_stream<T, Entropy>(a, sl, sl.lo, c);
  const int e = sl.edge();
  if (e >= 0) add<Entropy>(a, Elem<T>::to_f32(x[e]), c);
  a = row_join<Entropy>(a, c, red, rank, ctas);
  if (rank == 0 && threadIdx.x == 0) {
    const int64_t tok = tokens[r];
    const bool in = tok >= 0 && tok < vocab;
    const float lns = logf(a.s);
    if (!in) flag_status(status, PKV_DEV_TOKEN_OUT_OF_RANGE);
    logp[r] = in ? (Elem<T>::to_f32(x[tok]) - a.m) * inv_t - lns : NAN;
    if (Entropy) entropy[r] = lns - kLn2 * (a.w / a.s);
    if (stats != nullptr) stats[r] = make_float2(a.m, a.s);
  }
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

// v0: the vector's first element
template <typename T, bool Entropy>
__device__ __forceinline__ uint4 grad_vec(const Slope &g, uint4 v, int v0) {
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
  const int64_t k = g.tok - v0;
  if (k >= 0 && k < 2 * P) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (k == 2 * i) f[i].x += g.hot;
      if (k == 2 * i + 1) f[i].y += g.hot;
    }
  }
  return Vec<T>::pack(f);
}

// The gradient of this CTA's slice: from shared memory up to vector `held`,
// from global memory (the second read: L2) beyond. `out` is the row's gradient;
// where its vectors do not begin where the logits' do, elements go one by one.
template <typename T, bool Entropy>
__device__ __forceinline__ void grad_slice(const Slice<T> &sl, const Slope &g, T *out, const uint4 *held_v, int held) {
  if ((reinterpret_cast<uintptr_t>(out + sl.head) & 15) == 0) {
    uint4 *o = reinterpret_cast<uint4 *>(out + sl.head);
    for (int i = sl.lo + (int)threadIdx.x; i < held; i += kThreads)
      __stcs(o + i, grad_vec<T, Entropy>(g, held_v[i - sl.lo], sl.at(i)));
    int i = held + (int)threadIdx.x;
    for (; i + (kUnroll - 1) * kThreads < sl.hi; i += kUnroll * kThreads) {
      uint4 v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) v[u] = __ldg(sl.vecs() + i + u * kThreads);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        __stcs(o + i + u * kThreads, grad_vec<T, Entropy>(g, v[u], sl.at(i + u * kThreads)));
    }
    for (; i < sl.hi; i += kThreads) __stcs(o + i, grad_vec<T, Entropy>(g, __ldg(sl.vecs() + i), sl.at(i)));
  } else {
    const T *h = reinterpret_cast<const T *>(held_v);
    for (int v = sl.at(sl.lo) + (int)threadIdx.x; v < sl.at(held); v += kThreads)
      out[v] = from_f32<T>(grad_of<Entropy>(g, Elem<T>::to_f32(h[v - sl.at(sl.lo)]), v));
    for (int v = sl.at(held) + (int)threadIdx.x; v < sl.at(sl.hi); v += kThreads)
      out[v] = from_f32<T>(grad_of<Entropy>(g, Elem<T>::to_f32(sl.x[v]), v));
  }
  const int e = sl.edge();
  if (e >= 0) out[e] = from_f32<T>(grad_of<Entropy>(g, Elem<T>::to_f32(sl.x[e]), e));
}

template <typename T, bool Entropy>
__global__ void __launch_bounds__(kThreads)
logprob_grad_kernel(const T *logits, Rows rows, const int64_t *tokens, int vocab, int ctas, float inv_t, float c,
                    const float2 *stats, const float *entropy, const float *d_logp, const float *d_entropy, T *grad) {
  const int64_t r = blockIdx.x / ctas;
  const Slice<T> sl(logits + rows.offset(r), vocab, blockIdx.x % ctas, ctas);
  const float2 st = stats[r];
  const float g = d_logp != nullptr ? d_logp[r] : 0.f, h = Entropy ? d_entropy[r] : 0.f, k = inv_t / st.y;
  // -p (g + h (log p + H)) / T with log p = t ln2 - ln s
  Slope sp{st.x, c, Entropy ? -k * (g + h * (entropy[r] - logf(st.y))) : -k * g, -h * kLn2 * k, g * inv_t, tokens[r]};
  grad_slice<T, Entropy>(sl, sp, grad + r * (int64_t)vocab, nullptr, sl.lo);
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
  float4 *terms;           // workspace [batch * length]: w l, kl, clipped
  float *weight;           // workspace [batch * length]
  int32_t *order;          // workspace [batch * length]: tokens with a weight first
  int32_t *before;         // workspace [batch + 1]: such tokens before each sequence
  int32_t *counts;         // workspace: [0] tokens with a weight, [1] rows done
  int32_t *status;
  int64_t adv_b, adv_t;
  int32_t batch, length, vocab, reduction, ctas, hold;  // hold: vectors of a slice kept in shared memory
  float inv_t, c, clip_low, clip_high, kl_coef;
};

constexpr int kPrepThreads = 1024;

// One block: the tokens with a weight in front, each one's weight, counters.
// A running count over the tokens, kept at each sequence's start, gives the
// sequences' lengths.
__global__ void __launch_bounds__(kPrepThreads) policy_prep_kernel(PolicyArgs a) {
  __shared__ int warp_sum[kPrepThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t n = (int64_t)a.batch * a.length;
  int mine = 0;
  const int64_t per = (n + kPrepThreads - 1) / kPrepThreads, lo = min(n, tid * per), hi = min(n, lo + per);
  for (int64_t i = lo; i < hi; ++i) mine += a.mask == nullptr || a.mask[i] != 0;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int total = 0, start = incl - mine;
  for (int i = 0; i < kPrepThreads / 32; ++i) {
    if (i < warp) start += warp_sum[i];
    total += warp_sum[i];
  }
  if (tid == 0) {
    a.before[a.batch] = total;
    a.counts[0] = total;
    a.counts[1] = 0;
  }
  int active = start, idle = total + (int)lo - start;
  for (int64_t i = lo; i < hi; ++i) {
    if (i % a.length == 0) a.before[i / a.length] = active;
    const bool on = a.mask == nullptr || a.mask[i] != 0;
    a.order[on ? active++ : idle++] = (int32_t)i;
  }
  __syncthreads();
  for (int64_t i = tid; i < n; i += kPrepThreads) {
    const int64_t b = i / a.length;
    const int len = a.before[b + 1] - a.before[b];
    a.weight[i] = a.reduction == PKV_REDUCE_TOKEN      ? 1.f / (float)max(1, total)
                  : a.reduction == PKV_REDUCE_SEQUENCE ? 1.f / ((float)max(1, len) * (float)a.batch)
                                                       : 1.f;
  }
}

constexpr int kChunks = 4;  // bulk copies of a slice: the first is worked on while the last arrive

// One cluster per row. With a gradient the row is read once into the shared
// memory of the cluster's CTAs by bulk copies, summed from there, and its
// gradient written from there.
template <typename T, bool Grad>
__global__ void __launch_bounds__(kThreads)
policy_kernel(const T *logits, Rows rows, T *grad, PolicyArgs a) {
  extern __shared__ __align__(16) uint8_t held_raw[];
  __shared__ Joint red;
  __shared__ uint64_t bars[kChunks];
  __shared__ float slope_s;
  __shared__ int last_s;
  if (a.ctas > 1) cluster_arrive();
  const int64_t pos = blockIdx.x / a.ctas, r = a.order[pos];
  const int rank = blockIdx.x % a.ctas, tid = threadIdx.x;
  T *out = grad + r * (int64_t)a.vocab;
  if (pos >= a.counts[0]) {
    if (a.ctas > 1) cluster_wait();
    if (Grad) {
      const Slice<T> sl(out, a.vocab, rank, a.ctas);
      uint4 *o = reinterpret_cast<uint4 *>(out + sl.head);
      for (int i = sl.lo + tid; i < sl.hi; i += kThreads) __stcs(o + i, make_uint4(0, 0, 0, 0));
      const int e = sl.edge();
      if (e >= 0) out[e] = from_f32<T>(0.f);
    }
    if (rank == 0 && tid == 0) {
      a.logp[r] = 0.f;
      a.terms[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
    const T *x = logits + rows.offset(r);
    const Slice<T> sl(x, a.vocab, rank, a.ctas);
    const uint4 *hv = reinterpret_cast<const uint4 *>(held_raw);
    const int held = Grad ? min(sl.hi, sl.lo + a.hold) : sl.lo, n_held = held - sl.lo;
    if (Grad) {
      if (tid == 0) {
        for (int k = 0; k < kChunks; ++k) mbar_init(&bars[k], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        for (int k = 0; k < kChunks; ++k) {
          const int c0 = (int)((int64_t)n_held * k / kChunks), c1 = (int)((int64_t)n_held * (k + 1) / kChunks);
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&bars[k])),
                       "r"((c1 - c0) * 16)
                       : "memory");
          if (c1 > c0)
            asm volatile(
                "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                    smem_u32(hv + c0)),
                "l"(sl.vecs() + sl.lo + c0), "r"((c1 - c0) * 16), "r"(smem_u32(&bars[k]))
                : "memory");
        }
      }
      __syncthreads();
    }
    Soft st;
    const int e = sl.edge();
    if (e >= 0) add<false>(st, Elem<T>::to_f32(x[e]), a.c);
    bool ok = true;
    if (Grad) {
      for (int k = 0; k < kChunks; ++k) {
        const int c0 = (int)((int64_t)n_held * k / kChunks), c1 = (int)((int64_t)n_held * (k + 1) / kChunks);
        ok = mbar_wait_bounded(&bars[k], 0) && ok;
        for (int i = c0 + tid; i < c1; i += kThreads) add_vec<T, false>(st, hv[i], a.c);
      }
      if (!ok) flag_status(a.status, PKV_DEV_WAIT_TIMEOUT);
    }
    add_stream<T, false>(st, sl, held, a.c);
    st = row_join<false>(st, a.c, red, rank, a.ctas);
    const int64_t tok = a.tokens[r];
    if (tid == 0) {
      const float w = a.weight[r];
      const bool in = tok >= 0 && tok < a.vocab;
      const float lp = in ? (Elem<T>::to_f32(x[tok]) - st.m) * a.inv_t - logf(st.s) : NAN;
      const float adv = a.adv[(r / a.length) * a.adv_b + (r % a.length) * a.adv_t];
      const float ratio = expf(lp - a.old_logp[r]);
      const float free = ratio * adv, clip = fminf(fmaxf(ratio, 1.f - a.clip_low), 1.f + a.clip_high) * adv;
      const bool clipped = clip < free;
      float l = clipped ? -clip : -free, slope = clipped ? 0.f : -free, kl = 0.f;
      if (a.ref_logp != nullptr) {
        const float d = a.ref_logp[r] - lp, em = expm1f(d);
        kl = em - d;
        l += a.kl_coef * kl;
        slope -= a.kl_coef * em;
      }
      slope_s = slope * w * a.inv_t;
      if (rank == 0) {
        if (!in) flag_status(a.status, PKV_DEV_TOKEN_OUT_OF_RANGE);
        a.logp[r] = lp;
        a.terms[r] = make_float4(w * l, kl, clipped ? 1.f : 0.f, 0.f);
      }
    }
    __syncthreads();
    if (Grad) grad_slice<T, false>(sl, Slope{st.m, a.c, -slope_s / st.s, 0.f, slope_s, tok}, out, hv, held);
  }
  if (rank != 0) return;
  // the last row's CTA adds the rows' terms in row order, in 64 bits
  const int64_t n = (int64_t)a.batch * a.length;
  if (tid == 0) {
    __threadfence();
    last_s = atomicAdd(&a.counts[1], 1) == (int)n - 1;
  }
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  __shared__ double sums[3][kThreads];
  double l = 0, kl = 0, cl = 0;
  for (int64_t i = tid; i < n; i += kThreads) {
    const float4 t = __ldcg(a.terms + i);
    l += t.x;
    kl += t.y;
    cl += t.z;
  }
  sums[0][tid] = l;
  sums[1][tid] = kl;
  sums[2][tid] = cl;
  for (int o = kThreads / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (tid < o)
      for (int j = 0; j < 3; ++j) sums[j][tid] += sums[j][tid + o];
  }
  if (tid == 0) {
    const double count = max(1, a.counts[0]);
    a.out[0] = (float)sums[0][0];
    a.out[1] = (float)(sums[1][0] / count);
    a.out[2] = (float)(sums[2][0] / count);
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

template <typename K, typename... Args>
int launch_rows(const char *what, K kern, int64_t rows, int ctas, size_t smem, void *stream, Args... args) {
  if (rows * ctas > INT32_MAX) {
    set_error_detail("%s: %lld rows are too many for one call", what, (long long)rows);
    return PKV_ERR_UNSUPPORTED;
  }
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return check_launch(what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
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
  if (!tokens || !logprobs) {
    set_error_detail("pkv_token_logprobs: NULL pointer");
    return PKV_ERR_INVALID_ARG;
  }
  const Rows rw{outer_stride, row_stride, inner};
  const int ctas = row_ctas(rows, (int64_t)vocab * dtype_size(dtype), INT64_MAX / kMaxCluster);
  const float inv_t = 1.f / temperature, c = (float)(kLog2e / temperature);
  float2 *s2 = reinterpret_cast<float2 *>(stats);
  PKV_BY_DTYPE(dtype, return launch_rows("pkv_token_logprobs",
                                         entropy ? logprob_kernel<T, true> : logprob_kernel<T, false>, rows, ctas, 0,
                                         stream, (const T *)logits, rw, tokens, vocab, ctas, inv_t, c, logprobs,
                                         entropy, s2, status))
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
  if (!tokens || !stats || !d_logits || (d_entropy && !entropy) || !aligned_to(d_logits, dtype_size(dtype))) {
    set_error_detail("pkv_token_logprobs_grad: NULL or misaligned pointer");
    return PKV_ERR_INVALID_ARG;
  }
  const Rows rw{outer_stride, row_stride, inner};
  const int ctas = row_ctas(rows, (int64_t)vocab * dtype_size(dtype), 64 * 1024);
  const float inv_t = 1.f / temperature, c = (float)(kLog2e / temperature);
  const float2 *s2 = reinterpret_cast<const float2 *>(stats);
  PKV_BY_DTYPE(dtype, return launch_rows("pkv_token_logprobs_grad",
                                         d_entropy ? logprob_grad_kernel<T, true> : logprob_grad_kernel<T, false>, rows,
                                         ctas, 0, stream, (const T *)logits, rw, tokens, vocab, ctas, inv_t, c, s2,
                                         entropy, d_logprobs, d_entropy, (T *)d_logits))
  return PKV_ERR_UNSUPPORTED;
}

extern "C" size_t pkv_policy_loss_workspace_size(int32_t batch, int32_t length) {
  if (batch < 0 || length < 0 || (int64_t)batch * length > INT32_MAX) return 0;
  // terms (16 bytes), weight, order (4 each) per token; two counters; a count per sequence
  return 16 + (size_t)batch * length * 24 + ((size_t)batch + 1) * 4;
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
  if (batch < 0 || length < 0 ||
      bad_logits("pkv_policy_loss", logits, dtype, rows, vocab, std::max(1, length), temperature))
    return PKV_ERR_INVALID_ARG;
  if (rows == 0) {  // nothing to add up
    if (out && cudaMemsetAsync(out, 0, 3 * sizeof(float), reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess)
      return PKV_OK;
    return out ? check_launch("pkv_policy_loss") : PKV_ERR_INVALID_ARG;
  }
  if (!tokens || !old_logprobs || !advantages || !out || !logprobs || !aligned_to(d_logits, dtype_size(dtype)) ||
      !(clip_low >= 0.f) || !(clip_high >= 0.f) || reduction < PKV_REDUCE_TOKEN || reduction > PKV_REDUCE_SUM) {
    set_error_detail("pkv_policy_loss: NULL pointer, clip range %g / %g or reduction %d", (double)clip_low,
                     (double)clip_high, reduction);
    return PKV_ERR_INVALID_ARG;
  }
  if (!workspace || workspace_bytes < pkv_policy_loss_workspace_size(batch, length) || !aligned_to(workspace, 16))
    return PKV_ERR_WORKSPACE;
  PolicyArgs a{};
  a.tokens = tokens;
  a.old_logp = old_logprobs;
  a.ref_logp = ref_logprobs;
  a.adv = advantages;
  a.mask = mask;
  a.out = out;
  a.logp = logprobs;
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  a.counts = reinterpret_cast<int32_t *>(ws);
  a.terms = reinterpret_cast<float4 *>(ws + 16);
  a.weight = reinterpret_cast<float *>(ws + 16 + 16 * rows);
  a.order = reinterpret_cast<int32_t *>(ws + 16 + 20 * rows);
  a.before = reinterpret_cast<int32_t *>(ws + 16 + 24 * rows);
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
  a.ctas = row_ctas(rows, row_bytes, d_logits ? kHoldTarget : INT64_MAX / kMaxCluster);
  // a slice has at most one vector more than its even share
  const int64_t share = row_bytes / 16 / a.ctas + 1;
  a.hold = d_logits ? (int)std::min<int64_t>(share, kHoldMost / 16) : 0;
  policy_prep_kernel<<<1, kPrepThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
  const int rc = check_launch("policy_prep_kernel");
  if (rc) return rc;
  PKV_BY_DTYPE(dtype, return launch_rows("pkv_policy_loss", d_logits ? policy_kernel<T, true> : policy_kernel<T, false>,
                                         rows, a.ctas, (size_t)a.hold * 16, stream, (const T *)logits, rw,
                                         (T *)d_logits, a))
  return PKV_ERR_UNSUPPORTED;
}

extern "C" int pkv_scale_grad(void *grad, int64_t n, int32_t dtype, const float *upstream, void *stream) {
  if (dtype_size(dtype) == 0) return PKV_ERR_UNSUPPORTED;
  if (n < 0 || (n > 0 && (!grad || !upstream))) {
    set_error_detail("pkv_scale_grad: n %lld or NULL pointer", (long long)n);
    return PKV_ERR_INVALID_ARG;
  }
  if (n == 0) return PKV_OK;
  const unsigned blocks = (unsigned)std::min<int64_t>((n + kThreads - 1) / kThreads, 148 * 8);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PKV_BY_DTYPE(dtype, (scale_grad_kernel<T><<<blocks, kThreads, 0, st>>>((T *)grad, n, upstream)))
  return check_launch("pkv_scale_grad");
}
