// losses.cu -- losses over vocabulary logits z [n, V], forward and backward: token log-probabilities,
// the clipped policy loss with a KL term, the paired preference loss and the distillation loss from a
// teacher's top logits.
//
// With x = z / T, a row's softmax q_j = e^{x_j} / sum_i e^{x_i} is held as two numbers, the row's largest
// logit m (exact: it is one of the row's elements) and s = sum_j e^{(z_j - m) / T} in fp32, so that
//   log q_j = (z_j - m) / T - log s     and     q_j = e^{(z_j - m) / T} / s
// lose nothing to a large m.  Exponentials are taken to base 2: e^{(z - m)/T} = 2^{(z - m) k}, k = log2(e) / T,
// with ex2.approx (2 ulp).  The difference is formed before the product: a fused z k - m k would leave the
// rounding of m k at z = m (a lone entry's log-probability would not be 0) and overflow at the type's lowest
// value.  Where every logit of a row is
// -inf (or one is NaN or +inf) the row's results are NaN, as the formula gives.
//
// One CTA per row, two passes over it: the row's statistics, then (where a gradient is asked for) the
// gradient.
#include <math.h>

#include "kdn_common.cuh"
#include "kdn_internal.h"

namespace kdn {

__device__ int g_loss_error;

namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kThreads = 256;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ int64_t ld_index(const void* p, int index_dtype, int64_t i) {
  return index_dtype == KDN_INDEX_I64 ? static_cast<const int64_t*>(p)[i]
                                      : int64_t(static_cast<const int32_t*>(p)[i]);
}

__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < int(blockDim.x >> 5); ++w) v = fmaxf(v, red[w]);
  return v;
}

__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < int(blockDim.x >> 5); ++w) v += red[w];
  return v;
}

__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < int(blockDim.x >> 5); ++w) v += red[w];
  return v;
}

// the label of a row, or -1 for a row that counts for nothing (its label is ignore_index; a label outside
// the vocabulary is recorded and treated the same way)
__device__ __forceinline__ int64_t row_label(const LossRows& a, int64_t r) {
  const int64_t y = ld_index(a.labels, a.index_dtype, r);
  if (y == a.ignore_index) return -1;
  if (y < 0 || y >= a.V) {
    if (threadIdx.x == 0) record_device_error(&g_loss_error, kErrSlotOutOfRange);
    return -1;
  }
  return y;
}

struct PolicyRow {
  float w, loss, dlogp;  // weight, weight x loss, d(weight x loss) / d logp
};

// The clipped policy loss of one token: r = e^(logp - old),
//   l = -min(r A, clip(r, 1 - lo, 1 + hi) A) + c_kl (e^g - 1 - g) - c_H H,   g = ref - logp,
// where e^g - 1 - g >= 0 estimates KL(policy || reference) from the policy's own sample.  The gradient of the
// first term is -r A where the unclipped product is the smaller (or the two are equal), else zero.
__device__ __forceinline__ PolicyRow policy_row(const PolicyTerms& t, int64_t r, float logp, float H) {
  PolicyRow p;
  p.w = t.weights ? t.weights[r] : *t.scale;
  const float adv = t.advantages[r], ratio = expf(logp - t.old_logps[r]);
  const float free = ratio * adv, clipped = fminf(fmaxf(ratio, 1.f - t.clip_low), 1.f + t.clip_high) * adv;
  float l = free <= clipped ? -free : -clipped;
  float d = free <= clipped ? -free : 0.f;
  if (t.ref_logps) {
    const float g = t.ref_logps[r] - logp, em = expm1f(g);
    l = fmaf(t.kl_coef, em - g, l);
    d = fmaf(-t.kl_coef, em, d);
  }
  l = fmaf(-t.entropy_coef, H, l);
  p.loss = p.w == 0.f ? 0.f : p.w * l;  // a row of weight zero counts for nothing, whatever it holds
  p.dlogp = p.w * d;
  return p;
}

template <typename T>
__device__ __forceinline__ void zero_row(T* out, int V) {
  for (int j = threadIdx.x; j < V; j += kThreads) from_f32(out + j, 0.f);
}

// -------------------------------------------------------------------- token log-probabilities, policy loss
template <typename T>
__global__ void __launch_bounds__(kThreads) logp_kernel(LossRows a, PolicyTerms t) {
  __shared__ float red[kThreads / 32];
  const int64_t r = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + r * a.ld;
  T* dz = a.dlogits ? static_cast<T*>(a.dlogits) + r * a.ld_d : nullptr;
  const int V = int(a.V);
  const int64_t y = row_label(a, r);
  if (y < 0) {
    if (threadIdx.x == 0) {
      a.logps[r] = 0.f;
      if (a.stats) a.stats[2 * r] = 0.f, a.stats[2 * r + 1] = 1.f;
      if (a.coef_zero) a.coef_zero[r] = 0.f;
      if (t.entropy) t.entropy[r] = 0.f;
      if (t.row_loss) t.row_loss[r] = 0.f;
    }
    if (dz) zero_row(dz, V);
    return;
  }
  float mx = -INFINITY;
  for (int j = threadIdx.x; j < V; j += kThreads) mx = fmaxf(mx, to_f32(z[j]));
  mx = block_max(mx, red);
  float s = 0.f, u = 0.f;
  for (int j = threadIdx.x; j < V; j += kThreads) {
    const float d = (to_f32(z[j]) - mx) * a.k;
    const float e = ex2(d);
    s += e;
    u = fmaf(e, fmaxf(d, -1000.f), u);
  }
  s = block_sum(s, red);
  u = block_sum(u, red);
  const float l2s = log2f(s);
  const float logp = kLn2 * ((to_f32(z[y]) - mx) * a.k - l2s);
  if (threadIdx.x == 0) {
    a.logps[r] = logp;
    if (a.stats) a.stats[2 * r] = mx, a.stats[2 * r + 1] = s;
    if (a.coef_zero) a.coef_zero[r] = 0.f;
  }
  if (!t.row_loss) return;
  const float H = kLn2 * (l2s - u / s);
  const PolicyRow p = policy_row(t, r, logp, H);
  if (threadIdx.x == 0) {
    t.row_loss[r] = p.loss;
    if (t.entropy) t.entropy[r] = H;
  }
  if (!dz) return;
  if (p.w == 0.f) {
    zero_row(dz, V);
    return;
  }
  const float c = p.dlogp * a.inv_t, h = p.w * t.entropy_coef * a.inv_t;
  const float A = (h * (H - kLn2 * l2s) - c) / s, B = h * kLn2 / s;
  for (int j = threadIdx.x; j < V; j += kThreads) {
    const float d = (to_f32(z[j]) - mx) * a.k;
    float g = ex2(d) * fmaf(B, fmaxf(d, -1000.f), A);
    if (j == y) g += c;
    from_f32(dz + j, g);
  }
}

// d/dz of sum_t dlogps_t logp_t from the saved statistics
template <typename T>
__global__ void __launch_bounds__(kThreads) logp_backward_kernel(LossRows a, const float* __restrict__ dlogps) {
  const int64_t r = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + r * a.ld;
  T* dz = static_cast<T*>(a.dlogits) + r * a.ld_d;
  const int V = int(a.V);
  const int64_t y = row_label(a, r);
  const float c = y < 0 ? 0.f : dlogps[r] * a.inv_t;
  if (c == 0.f) {
    zero_row(dz, V);
    return;
  }
  const float mx = a.stats[2 * r], A = -c / a.stats[2 * r + 1];
  for (int j = threadIdx.x; j < V; j += kThreads) {
    float g = ex2((to_f32(z[j]) - mx) * a.k) * A;
    if (j == y) g += c;
    from_f32(dz + j, g);
  }
}

// ------------------------------------------------------------------------------------------- distillation
template <typename T>
__global__ void __launch_bounds__(kThreads) distill_kernel(LossRows a, DistillTerms t) {
  extern __shared__ float sm[];
  __shared__ float red[kThreads / 32];
  float* tp = sm;                                 // [K] teacher probabilities
  int* tid = reinterpret_cast<int*>(sm + t.K);    // [K] ids, -1 where there is none
  const int64_t r = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + r * a.ld;
  T* dz = a.dlogits ? static_cast<T*>(a.dlogits) + r * a.ld_d : nullptr;
  const int V = int(a.V), K = t.K;
  const float w = t.weights ? t.weights[r] : *t.scale;
  // teacher: log p_k = t_k / T - its log-sum-exp (given, or over the entries of the row)
  float tm = -INFINITY, valid = 0.f;
  for (int k = threadIdx.x; k < K; k += kThreads) {
    const int64_t id = ld_index(t.ids, a.index_dtype, r * K + k);
    const bool ok = id >= 0 && id < V;
    if (id >= V) record_device_error(&g_loss_error, kErrSlotOutOfRange);
    tid[k] = ok ? int(id) : -1;
    tp[k] = ok ? ld_as_f32(t.logits, t.dtype, r * K + k) : -INFINITY;
    tm = fmaxf(tm, tp[k]);
    valid += ok ? 1.f : 0.f;
  }
  tm = block_max(tm, red);
  if (block_sum(valid, red) == 0.f || ld_index(t.ids, a.index_dtype, r * K) < 0) {  // the row counts for nothing
    if (threadIdx.x == 0) t.divergence[r] = 0.f, t.row_loss[r] = 0.f;
    if (dz) zero_row(dz, V);
    return;
  }
  float tl = 0.f;  // log of the sum of the teacher's exponentials below its largest entry
  if (!t.lse) {
    for (int k = threadIdx.x; k < K; k += kThreads) tl += ex2((tp[k] - tm) * a.k);
    tl = logf(block_sum(tl, red));
  }
  // student
  float mx = -INFINITY;
  for (int j = threadIdx.x; j < V; j += kThreads) mx = fmaxf(mx, to_f32(z[j]));
  mx = block_max(mx, red);
  float s = 0.f, rest = 0.f;  // all of the row, and what lies outside the teacher's ids
  for (int j = threadIdx.x; j < V; j += kThreads) {
    const float e = ex2((to_f32(z[j]) - mx) * a.k);
    s += e;
    if (t.lse) {
      bool in = false;
      for (int k = 0; k < K; ++k) in |= tid[k] == j;
      if (!in) rest += e;
    }
  }
  s = block_sum(s, red);
  rest = block_sum(rest, red);
  const float l2s = log2f(s);
  float kl = 0.f, ps = 0.f;
  for (int k = threadIdx.x; k < K; k += kThreads) {
    if (tid[k] < 0) {
      tp[k] = 0.f;
      continue;
    }
    const float lp = t.lse ? fmaf(tp[k], a.inv_t, -t.lse[r]) : fmaf(tp[k] - tm, a.inv_t, -tl);
    const float p = expf(lp);
    tp[k] = p;
    ps += p;
    if (p > 0.f) kl = fmaf(p, lp - kLn2 * ((to_f32(z[tid[k]]) - mx) * a.k - l2s), kl);
  }
  kl = block_sum(kl, red);
  ps = block_sum(ps, red);
  float A = ps, R = 0.f;
  if (t.lse) {
    const float pr = fmaxf(1.f - ps, 0.f), qr = rest / s;
    if (pr > 0.f) kl += pr * (logf(pr) - logf(qr));
    A = ps + pr;
    R = pr > 0.f ? pr / qr : 0.f;
  }
  if (threadIdx.x == 0) {
    t.divergence[r] = kl;
    t.row_loss[r] = w == 0.f ? 0.f : w * t.t2 * kl;
  }
  if (!dz) return;
  if (w == 0.f) {
    zero_row(dz, V);
    return;
  }
  const float c = w * t.temperature;
  for (int j = threadIdx.x; j < V; j += kThreads) {
    float P = 0.f;
    bool in = false;
    for (int k = 0; k < K; ++k)
      if (tid[k] == j) P += tp[k], in = true;
    const float q = ex2((to_f32(z[j]) - mx) * a.k) / s;
    from_f32(dz + j, c * (in ? fmaf(q, A, -P) : q * (A - R)));
  }
}

// -------------------------------------------------------------------------------------------- small kernels
// scale = 1 / (rows that count): rows whose label is not ignore_index, or (K > 0) whose first id is >= 0
__global__ void __launch_bounds__(1024) live_scale_kernel(const void* __restrict__ labels, int index_dtype, int64_t n,
                                                          int64_t stride, bool by_sign, int64_t ignore_index,
                                                          float* __restrict__ scale) {
  __shared__ double red[32];
  int64_t c = 0;
  for (int64_t r = threadIdx.x; r < n; r += 1024) {
    const int64_t y = ld_index(labels, index_dtype, r * stride);
    c += by_sign ? y >= 0 : y != ignore_index;
  }
  const double live = block_sum_f64(double(c), red);
  if (threadIdx.x == 0) *scale = live > 0.0 ? float(1.0 / live) : 0.f;
}

// loss = factor * sum_r part[r], in a fixed order (one CTA)
__global__ void __launch_bounds__(1024) loss_sum_kernel(const float* __restrict__ part, int64_t n, double factor,
                                                        float* __restrict__ loss) {
  __shared__ double red[32];
  double v = 0.0;
  for (int64_t r = threadIdx.x; r < n; r += 1024) v += double(part[r]);
  v = block_sum_f64(v, red);
  if (threadIdx.x == 0) *loss = float(v * factor);
}

// One CTA per pair (sequences 2p chosen, 2p + 1 rejected): the log ratios of both, the pair's loss, and
// d loss / d logp of their tokens.
__global__ void __launch_bounds__(kThreads) pair_kernel(PairTerms t) {
  __shared__ double red[kThreads / 32];
  const int64_t p = blockIdx.x;
  int64_t lo[2], hi[2];
  double sum[2], cnt[2];
  for (int i = 0; i < 2; ++i) {
    lo[i] = t.cu[2 * p + i];
    hi[i] = t.cu[2 * p + i + 1];
    if (lo[i] < 0 || hi[i] > t.n || hi[i] < lo[i]) {  // offsets out of range: the sequence counts as empty
      if (threadIdx.x == 0) record_device_error(&g_loss_error, kErrSlotOutOfRange);
      lo[i] = hi[i] = 0;
    }
    double v = 0.0, c = 0.0;
    for (int64_t r = lo[i] + threadIdx.x; r < hi[i]; r += kThreads) {
      if (ld_index(t.labels, t.index_dtype, r) == t.ignore_index) continue;
      v += double(t.logps[r]) - (t.ref ? double(t.ref[r]) : 0.0);
      c += 1.0;
    }
    sum[i] = block_sum_f64(v, red);
    cnt[i] = t.normalise ? fmax(block_sum_f64(c, red), 1.0) : 1.0;
    sum[i] /= cnt[i];
  }
  const double h = double(t.beta) * (sum[0] - sum[1]);
  // log sigmoid(h) = min(h, 0) - log1p(e^-|h|)
  const double l1p = log1p(exp(-fabs(h)));
  const double eps = double(t.smoothing);
  const double dh = 1.0 / (1.0 + exp(-h)) - (1.0 - eps);
  if (threadIdx.x == 0) {
    t.log_ratios[2 * p] = float(sum[0]);
    t.log_ratios[2 * p + 1] = float(sum[1]);
    t.pair_loss[p] = float(-((1.0 - eps) * (fmin(h, 0.0) - l1p) + eps * (fmin(-h, 0.0) - l1p)));
  }
  for (int i = 0; i < 2; ++i) {
    const float c = float((i == 0 ? dh : -dh) * double(t.beta) / (double(t.pairs) * cnt[i]));
    for (int64_t r = lo[i] + threadIdx.x; r < hi[i]; r += kThreads) t.coef[r] = c;
  }
}

// x *= *scale, row by row; nothing is read or written where the scale is one
template <typename T>
__global__ void __launch_bounds__(kThreads) scale_kernel(T* __restrict__ x, int64_t ld, int64_t n, int64_t V,
                                                         const float* __restrict__ scale) {
  const float f = *scale;
  if (f == 1.f) return;
  for (int64_t r = blockIdx.x; r < n; r += gridDim.x)
    for (int64_t j = threadIdx.x; j < V; j += kThreads) from_f32(x + r * ld + j, to_f32(x[r * ld + j]) * f);
}

cudaError_t launch_logp(const LossRows& a, const PolicyTerms& t, cudaStream_t stream) {
  if (a.dtype == KDN_DTYPE_BF16)
    logp_kernel<__nv_bfloat16><<<unsigned(a.n), kThreads, 0, stream>>>(a, t);
  else
    logp_kernel<float><<<unsigned(a.n), kThreads, 0, stream>>>(a, t);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_token_logprobs(const LossRows& a, cudaStream_t stream) {
  return launch_logp(a, PolicyTerms{}, stream);
}

cudaError_t launch_token_logprobs_backward(const LossRows& a, const float* dlogps, cudaStream_t stream) {
  if (a.dtype == KDN_DTYPE_BF16)
    logp_backward_kernel<__nv_bfloat16><<<unsigned(a.n), kThreads, 0, stream>>>(a, dlogps);
  else
    logp_backward_kernel<float><<<unsigned(a.n), kThreads, 0, stream>>>(a, dlogps);
  return cudaGetLastError();
}

cudaError_t launch_policy_loss(const LossRows& a, const PolicyTerms& t, float* loss, cudaStream_t stream) {
  if (!t.weights) {
    live_scale_kernel<<<1, 1024, 0, stream>>>(a.labels, a.index_dtype, a.n, 1, false, a.ignore_index,
                                              const_cast<float*>(t.scale));
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  if (cudaError_t e = launch_logp(a, t, stream); e != cudaSuccess) return e;
  loss_sum_kernel<<<1, 1024, 0, stream>>>(t.row_loss, a.n, 1.0, loss);
  return cudaGetLastError();
}

cudaError_t launch_preference_loss(const LossRows& a, const PairTerms& t, float* loss, cudaStream_t stream) {
  if (a.n > 0) {
    LossRows f = a;  // forward: log-probabilities and statistics only
    f.dlogits = nullptr;
    f.coef_zero = t.coef;
    if (cudaError_t e = launch_logp(f, PolicyTerms{}, stream); e != cudaSuccess) return e;
  }
  pair_kernel<<<unsigned(t.pairs), kThreads, 0, stream>>>(t);
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  loss_sum_kernel<<<1, 1024, 0, stream>>>(t.pair_loss, t.pairs, 1.0 / double(t.pairs), loss);
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  return a.dlogits && a.n > 0 ? launch_token_logprobs_backward(a, t.coef, stream) : cudaSuccess;
}

cudaError_t launch_distillation_loss(const LossRows& a, const DistillTerms& t, float* loss, cudaStream_t stream) {
  if (!t.weights) {
    live_scale_kernel<<<1, 1024, 0, stream>>>(t.ids, a.index_dtype, a.n, t.K, true, 0, const_cast<float*>(t.scale));
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  const size_t smem = size_t(t.K) * 8;
  if (a.dtype == KDN_DTYPE_BF16)
    distill_kernel<__nv_bfloat16><<<unsigned(a.n), kThreads, smem, stream>>>(a, t);
  else
    distill_kernel<float><<<unsigned(a.n), kThreads, smem, stream>>>(a, t);
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  loss_sum_kernel<<<1, 1024, 0, stream>>>(t.row_loss, a.n, 1.0, loss);
  return cudaGetLastError();
}

cudaError_t launch_scale_rows(void* x, int dtype, int64_t ld, int64_t n, int64_t V, const float* scale,
                              cudaStream_t stream) {
  const unsigned grid = unsigned(n < 148 * 8 ? n : 148 * 8);
  if (dtype == KDN_DTYPE_BF16)
    scale_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(static_cast<__nv_bfloat16*>(x), ld, n, V, scale);
  else
    scale_kernel<float><<<grid, kThreads, 0, stream>>>(static_cast<float*>(x), ld, n, V, scale);
  return cudaGetLastError();
}

cudaError_t loss_read_error(cudaStream_t stream, int* code) {
  int h = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&h, g_loss_error, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
  if (e != cudaSuccess) return e;
  if ((e = cudaStreamSynchronize(stream)) != cudaSuccess) return e;
  if (h != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_loss_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream);
    if (e != cudaSuccess) return e;
    if ((e = cudaStreamSynchronize(stream)) != cudaSuccess) return e;
  }
  *code = h;
  return cudaSuccess;
}

}  // namespace kdn
