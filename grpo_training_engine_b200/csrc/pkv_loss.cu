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

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kRowThreads = 512;

// Where row r of the logits begins: rows are (outer, inner) pairs.
struct Rows {
  int64_t outer_stride, row_stride;
  int32_t inner;
  __device__ __forceinline__ int64_t offset(int64_t r) const {
    return (r / inner) * outer_stride + (r % inner) * row_stride;
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

// Joined over the block; every thread returns the same values.
template <bool Entropy>
__device__ __forceinline__ Soft block_join(Soft a, float c, Soft *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Soft b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.w = Entropy ? __shfl_xor_sync(0xffffffffu, a.w, o) : 0.f;
    join<Entropy>(a, b, c);
  }
  const int warp = threadIdx.x >> 5;
  __syncthreads();  // the last row's values have been read
  if ((threadIdx.x & 31) == 0) red[warp] = a;
  __syncthreads();
  a = red[0];
  for (int i = 1; i < kRowThreads / 32; ++i) join<Entropy>(a, red[i], c);
  return a;
}

template <typename T, bool Entropy>
__device__ __forceinline__ Soft row_soft(const T *x, int vocab, float c, Soft *red) {
  Soft a;
  for (int v = threadIdx.x; v < vocab; v += kRowThreads) add<Entropy>(a, Elem<T>::to_f32(x[v]), c);
  return block_join<Entropy>(a, c, red);
}

// ---------------------------------------------------------------------------
// token log-probabilities
// ---------------------------------------------------------------------------
template <typename T, bool Entropy>
__global__ void __launch_bounds__(kRowThreads)
logprob_kernel(const T *logits, Rows rows, const int64_t *tokens, int vocab, float inv_t, float *logp, float *entropy,
               float2 *stats, int32_t *status) {
  __shared__ Soft red[kRowThreads / 32];
  const int64_t r = blockIdx.x;
  const T *x = logits + rows.offset(r);
  const Soft a = row_soft<T, Entropy>(x, vocab, kLog2e * inv_t, red);
  if (threadIdx.x == 0) {
    const int64_t tok = tokens[r];
    const float lns = logf(a.s);
    if (tok < 0 || tok >= vocab) flag_status(status, PKV_DEV_TOKEN_OUT_OF_RANGE);
    logp[r] = tok < 0 || tok >= vocab ? NAN : (Elem<T>::to_f32(x[tok]) - a.m) * inv_t - lns;
    if (Entropy) entropy[r] = lns - kLn2 * (a.w / a.s);
    if (stats != nullptr) stats[r] = make_float2(a.m, a.s);
  }
}

template <typename T, bool Entropy>
__global__ void __launch_bounds__(kRowThreads)
logprob_grad_kernel(const T *logits, Rows rows, const int64_t *tokens, int vocab, float inv_t, const float2 *stats,
                    const float *entropy, const float *d_logp, const float *d_entropy, T *grad) {
  const int64_t r = blockIdx.x;
  const T *x = logits + rows.offset(r);
  T *out = grad + r * (int64_t)vocab;
  const float2 st = stats[r];
  const float c = kLog2e * inv_t, g = d_logp != nullptr ? d_logp[r] : 0.f, h = Entropy ? d_entropy[r] : 0.f;
  const float k = inv_t / st.y;
  // -p (g + h (log p + H)) / T = e (a + b t)
  const float b = -h * kLn2 * k, a = Entropy ? -k * (g + h * (entropy[r] - logf(st.y))) : -k * g;
  const int64_t tok = tokens[r];
  for (int v = threadIdx.x; v < vocab; v += kRowThreads) {
    const float t = (Elem<T>::to_f32(x[v]) - st.x) * c, e = fast_exp2(t);
    float d = Entropy ? e * (a + b * fmaxf(t, -1e4f)) : e * a;
    if (v == tok) d += g * inv_t;
    out[v] = from_f32<T>(d);
  }
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
  float *weight;           // workspace [batch * length]
  float4 *terms;           // workspace [batch * length]: w l, kl, clipped
  int32_t *order;          // workspace: active rows first
  int32_t *counts;         // workspace: [0] rows with a weight, [1] blocks done
  int32_t *status;
  int64_t adv_b, adv_t;
  int32_t batch, length, vocab, reduction;
  float inv_t, clip_low, clip_high, kl_coef;
};

constexpr int kPrepThreads = 1024;

// One block: the weight of every token, the tokens with one in front, counters.
__global__ void __launch_bounds__(kPrepThreads) policy_prep_kernel(PolicyArgs a) {
  __shared__ int warp_sum[kPrepThreads / 32];
  __shared__ int total_s;
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
  if (tid == 0) {
    int run = 0;
    for (int i = 0; i < kPrepThreads / 32; ++i) {
      const int v = warp_sum[i];
      warp_sum[i] = run;
      run += v;
    }
    total_s = run;
    a.counts[0] = run;
    a.counts[1] = 0;
  }
  __syncthreads();
  const int total = total_s;
  int active = warp_sum[warp] + incl - mine;  // active tokens before this thread's
  int idle = total + (int)lo - active;
  for (int64_t i = lo; i < hi; ++i) {
    const bool on = a.mask == nullptr || a.mask[i] != 0;
    a.order[on ? active++ : idle++] = (int32_t)i;
    float w = 0.f;
    if (on) {
      w = 1.f;
      if (a.reduction == PKV_REDUCE_TOKEN) w = 1.f / (float)total;
      if (a.reduction == PKV_REDUCE_SEQUENCE) {
        const int64_t b = i / a.length;
        int len = 0;
        for (int t = 0; t < a.length; ++t) len += a.mask == nullptr || a.mask[b * a.length + t] != 0;
        w = 1.f / ((float)len * (float)a.batch);
      }
    }
    a.weight[i] = w;
  }
}

template <typename T, bool Grad>
__global__ void __launch_bounds__(kRowThreads)
policy_kernel(const T *logits, Rows rows, T *grad, PolicyArgs a) {
  __shared__ Soft red[kRowThreads / 32];
  __shared__ float slope_s;
  __shared__ int last_s;
  const int64_t r = a.order[blockIdx.x];
  const float w = a.weight[r];
  T *out = grad + r * (int64_t)a.vocab;
  if (blockIdx.x >= a.counts[0]) {
    if (Grad)
      for (int v = threadIdx.x; v < a.vocab; v += kRowThreads) out[v] = from_f32<T>(0.f);
    if (threadIdx.x == 0) {
      a.logp[r] = 0.f;
      a.terms[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
    const T *x = logits + rows.offset(r);
    const float c = kLog2e * a.inv_t;
    const Soft st = row_soft<T, false>(x, a.vocab, c, red);
    const int64_t tok = a.tokens[r];
    if (threadIdx.x == 0) {
      const bool in = tok >= 0 && tok < a.vocab;
      if (!in) flag_status(a.status, PKV_DEV_TOKEN_OUT_OF_RANGE);
      const float lp = in ? (Elem<T>::to_f32(x[tok]) - st.m) * a.inv_t - logf(st.s) : NAN;
      const float adv = a.adv[(r / a.length) * a.adv_b + (r % a.length) * a.adv_t];
      const float ratio = expf(lp - a.old_logp[r]);
      const float free = ratio * adv, held = fminf(fmaxf(ratio, 1.f - a.clip_low), 1.f + a.clip_high) * adv;
      const bool clipped = held < free;
      float l = clipped ? -held : -free, slope = clipped ? 0.f : -free, kl = 0.f;
      if (a.ref_logp != nullptr) {
        const float d = a.ref_logp[r] - lp, em = expm1f(d);
        kl = em - d;
        l += a.kl_coef * kl;
        slope -= a.kl_coef * em;
      }
      a.logp[r] = lp;
      a.terms[r] = make_float4(w * l, kl, clipped ? 1.f : 0.f, 0.f);
      slope_s = slope * w * a.inv_t;
    }
    __syncthreads();
    if (Grad) {
      const float slope = slope_s, k = -slope / st.s;
      for (int v = threadIdx.x; v < a.vocab; v += kRowThreads) {
        float d = fast_exp2((Elem<T>::to_f32(x[v]) - st.m) * c) * k;
        if (v == tok) d += slope;
        out[v] = from_f32<T>(d);
      }
    }
  }
  // the last block adds the rows' terms in row order, in 64 bits
  if (threadIdx.x == 0) {
    __threadfence();
    last_s = atomicAdd(&a.counts[1], 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  __shared__ double sums[3][kRowThreads];
  double l = 0, kl = 0, cl = 0;
  for (int64_t i = threadIdx.x; i < (int64_t)a.batch * a.length; i += kRowThreads) {
    const float4 t = a.terms[i];
    l += t.x;
    kl += t.y;
    cl += t.z;
  }
  sums[0][threadIdx.x] = l;
  sums[1][threadIdx.x] = kl;
  sums[2][threadIdx.x] = cl;
  for (int o = kRowThreads / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (threadIdx.x < o)
      for (int j = 0; j < 3; ++j) sums[j][threadIdx.x] += sums[j][threadIdx.x + o];
  }
  if (threadIdx.x == 0) {
    const double n = max(1, a.counts[0]);
    a.out[0] = (float)sums[0][0];
    a.out[1] = (float)(sums[1][0] / n);
    a.out[2] = (float)(sums[2][0] / n);
  }
}

// grad *= *upstream, nothing where it is 1
template <typename T>
__global__ void __launch_bounds__(256) scale_grad_kernel(T *grad, int64_t n, const float *upstream) {
  const float u = *upstream;
  if (u == 1.f) return;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll)
    grad[i] = from_f32<T>(Elem<T>::to_f32(grad[i]) * u);
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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const float inv_t = 1.f / temperature;
  float2 *s2 = reinterpret_cast<float2 *>(stats);
  PKV_BY_DTYPE(dtype, {
    if (entropy)
      logprob_kernel<T, true><<<(unsigned)rows, kRowThreads, 0, st>>>((const T *)logits, rw, tokens, vocab, inv_t,
                                                                      logprobs, entropy, s2, status);
    else
      logprob_kernel<T, false><<<(unsigned)rows, kRowThreads, 0, st>>>((const T *)logits, rw, tokens, vocab, inv_t,
                                                                       logprobs, entropy, s2, status);
  })
  return check_launch("pkv_token_logprobs");
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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const float inv_t = 1.f / temperature;
  const float2 *s2 = reinterpret_cast<const float2 *>(stats);
  PKV_BY_DTYPE(dtype, {
    if (d_entropy)
      logprob_grad_kernel<T, true><<<(unsigned)rows, kRowThreads, 0, st>>>(
          (const T *)logits, rw, tokens, vocab, inv_t, s2, entropy, d_logprobs, d_entropy, (T *)d_logits);
    else
      logprob_grad_kernel<T, false><<<(unsigned)rows, kRowThreads, 0, st>>>(
          (const T *)logits, rw, tokens, vocab, inv_t, s2, entropy, d_logprobs, d_entropy, (T *)d_logits);
  })
  return check_launch("pkv_token_logprobs_grad");
}

extern "C" size_t pkv_policy_loss_workspace_size(int32_t batch, int32_t length) {
  if (batch < 0 || length < 0 || (int64_t)batch * length > INT32_MAX) return 0;
  // terms (16 bytes), weight, order (4 each) per token; two counters
  return 16 + (size_t)batch * length * 24;
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
  a.status = status;
  a.adv_b = adv_stride_b;
  a.adv_t = adv_stride_t;
  a.batch = batch;
  a.length = length;
  a.vocab = vocab;
  a.reduction = reduction;
  a.inv_t = 1.f / temperature;
  a.clip_low = clip_low;
  a.clip_high = clip_high;
  a.kl_coef = kl_coef;
  const Rows rw{batch_stride, row_stride, length};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  policy_prep_kernel<<<1, kPrepThreads, 0, st>>>(a);
  PKV_BY_DTYPE(dtype, {
    if (d_logits)
      policy_kernel<T, true><<<(unsigned)rows, kRowThreads, 0, st>>>((const T *)logits, rw, (T *)d_logits, a);
    else
      policy_kernel<T, false><<<(unsigned)rows, kRowThreads, 0, st>>>((const T *)logits, rw, (T *)d_logits, a);
  })
  return check_launch("pkv_policy_loss");
}

extern "C" int pkv_scale_grad(void *grad, int64_t n, int32_t dtype, const float *upstream, void *stream) {
  if (dtype_size(dtype) == 0) return PKV_ERR_UNSUPPORTED;
  if (n < 0 || (n > 0 && (!grad || !upstream))) {
    set_error_detail("pkv_scale_grad: n %lld or NULL pointer", (long long)n);
    return PKV_ERR_INVALID_ARG;
  }
  if (n == 0) return PKV_OK;
  const unsigned blocks = (unsigned)std::min<int64_t>((n + 255) / 256, 148 * 8);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PKV_BY_DTYPE(dtype, (scale_grad_kernel<T><<<blocks, 256, 0, st>>>((T *)grad, n, upstream)))
  return check_launch("pkv_scale_grad");
}
