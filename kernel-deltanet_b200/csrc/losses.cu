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
// value.  Where every logit of a row is -inf (or one is NaN or +inf) the row's results are NaN, as the formula gives.
//
// Two kinds of kernels.  In the first a row belongs to a warp, a CTA or a cluster of up to 8 CTAs, each with a
// contiguous share of the row's 16-byte vectors.  A share of up to 8 vectors a thread stays in registers between the
// two passes over it (statistics, then gradient), so the logits are read from memory once and the gradient is written
// once; the row's statistics are merged through warp shuffles, one barrier, and (in a cluster) one exchange through
// distributed shared memory.  Longer shares are taken in rounds and read again for the gradient.  The second, for the
// losses of a policy or a teacher over many long rows, streams them through a ring in shared memory:
// loss_stream_kernel.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kdn_common.cuh"
#include "kdn_internal.h"
#include "loss_plan.h"
#include "tc_prims.cuh"

namespace kdn {

__device__ int g_loss_error;

namespace {

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two fp32 operations in one instruction
__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tsub.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
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
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// First thing in the kernels of a call that makes several launches: the next kernel of the same call may be launched
// (it waits in turn, its launch overlaps this one's end), and the previous one's results are awaited (at once where it
// was launched without overlap).  Worth 1 to 2 us a launch.
__device__ __forceinline__ void await_previous() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ int64_t ld_index(const void* p, int index_dtype, int64_t i) {
  return index_dtype == KDN_INDEX_I64 ? static_cast<const int64_t*>(p)[i]
                                      : int64_t(static_cast<const int32_t*>(p)[i]);
}

// ------------------------------------------------------------------------------------- 16-byte vectors of a row
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int E = 4;
  static constexpr uint32_t kFill = 0xff800000u;  // -inf
  static __device__ __forceinline__ float2 pair(const uint4& v, int i) {
    return i == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                  : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ float2 minus(const uint4& v, int i, float m) {
    return sub2(pair(v, i), make_float2(m, m));
  }
  template <int N>
  static __device__ __forceinline__ float largest(const uint4* v) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[i].x), __uint_as_float(v[i].y)),
                         fmaxf(__uint_as_float(v[i].z), __uint_as_float(v[i].w))));
    return m;
  }
  static __device__ __forceinline__ uint4 pack(const float2* f) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x),
                      __float_as_uint(f[1].y));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int E = 8;
  static constexpr uint32_t kFill = 0xff80ff80u;
  static __device__ __forceinline__ uint32_t word(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
  }
  static __device__ __forceinline__ float2 pair(const uint4& v, int i) {
    const uint32_t w = word(v, i);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  // elements 2i, 2i + 1 as fp32 less m: a subtraction takes a bf16 operand as it is
  static __device__ __forceinline__ float2 minus(const uint4& v, int i, float m) {
    float2 r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tsub.rn.f32.bf16 %0, l, %3;\n\tsub.rn.f32.bf16 %1, h, %3;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "r"(word(v, i)), "f"(m));
    return r;
  }
  template <int N>
  static __device__ __forceinline__ float largest(const uint4* v) {
    auto h = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    __nv_bfloat162 m = __hmax2(__hmax2(h(v[0].x), h(v[0].y)), __hmax2(h(v[0].z), h(v[0].w)));
#pragma unroll
    for (int i = 1; i < N; ++i)
      m = __hmax2(m, __hmax2(__hmax2(h(v[i].x), h(v[i].y)), __hmax2(h(v[i].z), h(v[i].w))));
    return fmaxf(fmaxf(__low2float(m), __high2float(m)), -INFINITY);  // NaN only where every one is: -inf
  }
  static __device__ __forceinline__ uint4 pack(const float2* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 t = __float22bfloat162_rn(f[i]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// the vector that starts at element j0 of a row of V (one that reaches over an end of the row); elements outside
// the row are -inf
template <typename T>
__device__ __noinline__ uint4 load_edge(const T* z, int j0, int V) {
  uint32_t w[4] = {Vec<T>::kFill, Vec<T>::kFill, Vec<T>::kFill, Vec<T>::kFill};
#pragma unroll
  for (int e = 0; e < Vec<T>::E; ++e) {
    const int j = j0 + e;
    if (j < 0 || j >= V) continue;
    if constexpr (sizeof(T) == 4) {
      w[e] = __float_as_uint(z[j]);
    } else {
      const uint32_t b = reinterpret_cast<const uint16_t*>(z)[j];
      w[e / 2] = (e & 1) ? ((w[e / 2] & 0xffffu) | (b << 16)) : ((w[e / 2] & 0xffff0000u) | b);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// such a vector read whole: what lies outside the row becomes -inf / is not stored
template <typename T>
__device__ __noinline__ uint4 mask_edge(uint4 v, int j0, int V) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < Vec<T>::E; ++e) {
    if (j0 + e >= 0 && j0 + e < V) continue;
    if constexpr (sizeof(T) == 4)
      w[e] = Vec<T>::kFill;
    else
      w[e / 2] = (e & 1) ? ((w[e / 2] & 0xffffu) | 0xff800000u) : ((w[e / 2] & 0xffff0000u) | 0xff80u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// a vector whose elements of a set bit become -inf
template <typename T>
__device__ __forceinline__ uint4 mask_bits(uint4 v, uint32_t bits) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = sizeof(T) == 4 ? 0u - (bits >> i & 1u)
                                      : (bits >> 2 * i & 1u) * 0xffffu + (bits >> (2 * i + 1) & 1u) * 0xffff0000u;
    w[i] = (w[i] & ~m) | (Vec<T>::kFill & m);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __noinline__ void store_edge(T* dz, uint4 v, int j0, int V) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < Vec<T>::E; ++e) {
    const int j = j0 + e;
    if (j < 0 || j >= V) continue;
    if constexpr (sizeof(T) == 4)
      dz[j] = __uint_as_float(w[e]);
    else
      reinterpret_cast<uint16_t*>(dz)[j] = uint16_t((e & 1) ? w[e / 2] >> 16 : w[e / 2]);
  }
}

// A CTA's share of a row: vector vi holds the row's elements [vi E - off, vi E - off + E), off the row's start
// within its first 16 bytes; vectors [v0, v1) are the share.
template <typename T>
struct Share {
  static constexpr int E = Vec<T>::E;
  const T* z;
  T* dz;
  int off, V, v0, v1;
  bool same;  // the gradient's row starts at the same place within 16 bytes

  __device__ __forceinline__ Share(const LossRows& a, int64_t r, int rank, int parts) {
    z = static_cast<const T*>(a.logits) + r * a.ld;
    dz = a.dlogits ? static_cast<T*>(a.dlogits) + r * a.ld_d : nullptr;
    V = int(a.V);
    const uint32_t at = uint32_t(reinterpret_cast<uintptr_t>(z)) & 15u;
    off = int(at / sizeof(T));
    same = (uint32_t(reinterpret_cast<uintptr_t>(dz)) & 15u) == at;
    const int nvec = (off + V + E - 1) / E, per = (nvec + parts - 1) / parts;
    v0 = min(rank * per, nvec);
    v1 = min(v0 + per, nvec);
  }
  __device__ __forceinline__ bool whole(int vi) const { return vi * E >= off && (vi + 1) * E - off <= V; }
  __device__ __forceinline__ uint4 load(int vi) const {
    if (whole(vi)) return ld_stream(z + (vi * E - off));
    return load_edge(z, vi * E - off, V);
  }
  __device__ __forceinline__ void store(int vi, const float2* g) const {
    if (same && whole(vi)) {
      __stcs(reinterpret_cast<uint4*>(dz + (vi * E - off)), Vec<T>::pack(g));  // not read again here
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = vi * E - off + e;
      if (j >= 0 && j < V) from_f32(dz + j, (e & 1) ? g[e / 2].y : g[e / 2].x);
    }
  }
  template <int NT>
  __device__ __forceinline__ void zero(int tid) const {
    const float2 g[4] = {};
    for (int vi = v0 + tid; vi < v1; vi += NT) store(vi, g);
  }
};

// The CTAs of the kernels that keep a row in registers: NT threads a row (32: four rows to a CTA).
template <int NT>
struct Cta {
  static constexpr int kThreads = NT < 128 ? 128 : NT, kRows = kThreads / NT;
  static __device__ __forceinline__ int64_t row(int parts) {
    return int64_t(blockIdx.x / unsigned(parts)) * kRows + threadIdx.x / NT;
  }
};

// x / T + c in fp32, rounded once: the quotient's two halves (see LossRows; not through log2(e) / T or one rounded
// 1 / T, whose error would show in a log-probability)
__device__ __forceinline__ float over_t(const LossRows& a, float x, float c) {
  return fmaf(x, a.inv_hi, fmaf(x, a.inv_lo, c));
}
// ... where x / T and c nearly cancel: what is rounded on the way is of the size of the result, not of c (whose unit in
// the last place the product with the lower half is below)
__device__ __forceinline__ float over_t_less(const LossRows& a, float x, float c) {
  return fmaf(x, a.inv_lo, fmaf(x, a.inv_hi, c));
}

// Largest logit m of a part of a row, the sum s of exponentials below it and (kMoment) u = sum e^d d (base 2), which a
// change of m shifts.
template <bool kMoment>
struct Stats {
  float m = -INFINITY, s = 0.f;
};
template <>
struct Stats<true> {
  float m = -INFINITY, s = 0.f, u = 0.f;
};
using Sum = Stats<false>;

// The distillation loss: the logits outside the teacher's ids and those at them, each below its own largest.  A
// student's mass outside the ids may lie so far below the row's largest logit that every exponential relative to that is
// zero, while its logarithm and an entry's share of it are ordinary numbers.
struct Apart {
  Sum out, in;
};

// Statistics relative to another largest logit.  A part without a finite logit has m = -inf and sums of zero (or NaN)
// and is left as it is.  (The factor is expf's, which errs to both sides; ex2.approx truncates, and a sum is rescaled
// several times.)
__device__ __forceinline__ void rescale(Stats<true>& a, float m, const LossRows& r) {
  if (a.m == m) return;
  const float d = (a.m - m) * r.k, f = expf(over_t(r, a.m - m, 0.f));
  a.u = f == 0.f ? 0.f : f * fmaf(a.s, d, a.u);
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ void rescale(Sum& a, float m, const LossRows& r) {
  if (a.m == m) return;
  a.s *= expf(over_t(r, a.m - m, 0.f));
  a.m = m;
}

// a and b together
template <bool kMoment>
__device__ __forceinline__ void add(Stats<kMoment>& a, Stats<kMoment> b, const LossRows& r) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m, r);
  rescale(b, m, r);
  a.s += b.s;
  if constexpr (kMoment) a.u += b.u;
}
__device__ __forceinline__ void add(Apart& a, const Apart& b, const LossRows& r) {
  add(a.out, b.out, r);
  add(a.in, b.in, r);
}

__device__ __forceinline__ float4 pack(const Stats<true>& a) { return make_float4(a.m, a.s, a.u, 0.f); }
__device__ __forceinline__ float4 pack(const Sum& a) { return make_float4(a.m, a.s, 0.f, 0.f); }
__device__ __forceinline__ float4 pack(const Apart& a) { return make_float4(a.out.m, a.out.s, a.in.m, a.in.s); }
__device__ __forceinline__ void unpack(const float4& t, Stats<true>& a) { a.m = t.x, a.s = t.y, a.u = t.z; }
__device__ __forceinline__ void unpack(const float4& t, Sum& a) { a.m = t.x, a.s = t.y; }
__device__ __forceinline__ void unpack(const float4& t, Apart& a) {
  a.out.m = t.x, a.out.s = t.y, a.in.m = t.z, a.in.s = t.w;
}

// the largest of a warp's values (none is NaN), in the order of their bits as integers
__device__ __forceinline__ float warp_max(float x) {
  const int i = __float_as_int(x);
  const int m = __reduce_max_sync(0xffffffffu, i ^ ((i >> 31) & 0x7fffffff));
  return __int_as_float(m ^ ((m >> 31) & 0x7fffffff));
}

// the statistics of a warp's lanes together; kLeft > 1: of lanes of equal index modulo kLeft, about the warp's maximum
template <int kLeft = 1, bool kMoment>
__device__ __forceinline__ Stats<kMoment> merge_warp(Stats<kMoment> a, const LossRows& r) {
  rescale(a, warp_max(a.m), r);
#pragma unroll
  for (int o = 16; o >= kLeft; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    if constexpr (kMoment) a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
  }
  return a;
}
__device__ __forceinline__ Apart merge_warp(Apart a, const LossRows& r) {
  const float out = warp_max(a.out.m), in = warp_max(a.in.m);
  rescale(a.out, out, r);
  rescale(a.in, in, r);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.out.s += __shfl_xor_sync(0xffffffffu, a.out.s, o);
    a.in.s += __shfl_xor_sync(0xffffffffu, a.in.s, o);
  }
  return a;
}

// ... of `count` parts in shared memory, by every warp that asks
template <typename S>
__device__ __forceinline__ S merge_parts(const float4* p, int count, const LossRows& r) {
  const int lane = threadIdx.x & 31;
  S a, b;
  if (lane < count) unpack(p[lane], a);
  for (int i = lane + 32; i < count; i += 32) {
    unpack(p[i], b);
    add(a, b, r);
  }
  return merge_warp(a, r);
}

// ... of all threads of the row's cluster
template <int NT, typename S>
__device__ __forceinline__ S merge_rows(S a, const LossRows& r, int rank, int parts) {
  a = merge_warp(a, r);
  if constexpr (NT == 32) return a;
  __shared__ float4 part[NT / 32];
  __shared__ float4 remote[kMaxCluster];
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = pack(a);
  __syncthreads();
  a = merge_parts<S>(part, NT / 32, r);
  if (parts > 1) {
    if (threadIdx.x < unsigned(parts)) {
      const float4 t = pack(a);
      tc::st_cluster_v4(tc::mapa(tc::smem_u32(&remote[rank]), threadIdx.x), t.x, t.y, t.z, t.w);
    }
    tc::cluster_arrive();
    tc::cluster_wait();
    a = merge_parts<S>(remote, parts, r);
  }
  return a;
}

// a row counts when its label is not ignore_index and lies in the vocabulary
__device__ __forceinline__ bool counts(int64_t y, int64_t ignore_index, int64_t V) {
  return y != ignore_index && y >= 0 && y < V;
}

// the label of a row, or -1 for a row that counts for nothing (its label is ignore_index; a label outside
// the vocabulary is recorded and treated the same way)
__device__ __forceinline__ int64_t row_label(const LossRows& a, int64_t r, bool record) {
  const int64_t y = ld_index(a.labels, a.index_dtype, r);
  if (y == a.ignore_index) return -1;
  if (y < 0 || y >= a.V) {
    if (record) record_device_error(&g_loss_error, kErrSlotOutOfRange);
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
// first term is -r A where the unclipped product is the smaller (or the two are equal), else zero.  A NaN in either
// product is NaN in the loss and in the gradient (so no fminf or fmaxf here: they return their other argument).
struct PolicyIn {
  float w, adv, old, ref;
};
// (kCounted: the weight stands in memory; else, without weights and scale, the caller counts the rows)
template <bool kCounted>
__device__ __forceinline__ PolicyIn policy_inputs(const PolicyTerms& t, int64_t r) {
  if (!kCounted && !t.row_loss) return PolicyIn{};
  return PolicyIn{t.weights ? t.weights[r] : kCounted || t.scale ? *t.scale : 0.f, t.advantages[r], t.old_logps[r],
                  t.ref_logps ? t.ref_logps[r] : 0.f};
}
__device__ __forceinline__ PolicyRow policy_row(const PolicyTerms& t, const PolicyIn& in, float logp, float H) {
  PolicyRow p;
  p.w = in.w;
  const float adv = in.adv, ratio = expf(logp - in.old);
  const float lo = 1.f - t.clip_low, hi = 1.f + t.clip_high;
  const float clipped = (ratio < lo ? lo : ratio > hi ? hi : ratio) * adv;
  const float free = adv == 0.f ? clipped : ratio * adv;  // zero, too, where the ratio has overflowed
  float l = free > clipped ? -clipped : -free;
  float d = free > clipped ? 0.f : -free;
  if (t.ref_logps) {
    const float g = in.ref - logp, em = expm1f(g);
    l = fmaf(t.kl_coef, em - g, l);
    d = fmaf(-t.kl_coef, em, d);
  }
  l = fmaf(-t.entropy_coef, H, l);
  p.loss = p.w == 0.f ? 0.f : p.w * l;  // a row of weight zero counts for nothing, whatever it holds
  p.dlogp = p.w * d;
  return p;
}

// 1 / (rows that count) for a few rows, by every warp that asks: by their labels, or (ids) those whose first id is not
// negative.
__device__ __forceinline__ float mean_of_few(const LossRows& a, const void* ids, int K) {
  int live = 0;
  for (int64_t r = threadIdx.x & 31; r < a.n; r += 32)
    live += ids ? ld_index(ids, a.index_dtype, r * K) >= 0
                : counts(ld_index(a.labels, a.index_dtype, r), a.ignore_index, a.V);
  live = __reduce_add_sync(0xffffffffu, live);
  return live > 0 ? 1.f / float(live) : 0.f;
}

// before the pairs are formed: no coefficient yet, no pair done
__device__ __forceinline__ void zero_coef(const LossRows& a, int64_t r) {
  a.coef_zero[r] = 0.f;
  if (r == 0) *a.pairs_done = 0u;
}

// What the gradient of a row needs: dz_j = 2^d (A + B d) with d = (z_j - m) k, and dz_y; for the distillation loss the
// entries at the teacher's ids are c (total q - p), q = 2^((z_j - top) k) / sum.
struct RowCoef {
  float m, A, B, at_label;
  int y;  // -1: the gradient is zero
  float c, total, top, sum;
};

// From a row's statistics: the coefficients of its gradient (to `ready` as soon as they are known), then its outputs
// (written where `write` is set).
//   log q_j = ln 2 d_j - log s,   entropy H = -sum q log q = log s - ln 2 (sum e d) / s,
//   dz_j = (w / T) (dl/dlogp (1[j = y] - q_j) + c_H q_j (log q_j + H)).
template <bool kEntropy, int kGrad, typename F>
__device__ __forceinline__ RowCoef finish_row(const LossRows& a, const PolicyTerms& t, const PolicyIn& in, int64_t r,
                                              int y, float zy, const Stats<kEntropy>& st, bool write, F ready) {
  // products rounded on their own, so that calls with and without a gradient give the same bits
  const float dy = __fmul_rn(zy - st.m, a.k), ls = logf(st.s);
  const float logp = over_t(a, zy - st.m, -ls);
  RowCoef o{st.m, 0.f, 0.f, 0.f, -1, 0.f, 0.f, 0.f, 0.f};
  float H = 0.f;
  if constexpr (kEntropy) H = fmaf(-kLn2, st.u / st.s, ls);
  const PolicyRow p = t.row_loss ? policy_row(t, in, logp, H) : PolicyRow{};
  if (kGrad != 0 && p.w != 0.f) {
    const float c = p.dlogp * a.inv_t, h = kGrad == 2 ? p.w * t.entropy_coef * a.inv_t : 0.f;
    o.y = y;
    o.A = kGrad == 2 ? (h * (H - ls) - c) / st.s : -c / st.s;
    o.B = h * kLn2 / st.s;
    o.at_label = fmaf(ex2(dy), kGrad == 2 ? fmaf(o.B, fmaxf(dy, -1000.f), o.A) : o.A, c);
  }
  ready(o);
  if (write) {
    a.logps[r] = logp;
    if (a.stats) a.stats[2 * r] = st.m, a.stats[2 * r + 1] = st.s;
    if (a.coef_zero) zero_coef(a, r);
    if (t.row_loss) t.row_loss[r] = p.loss;
    if (t.entropy) t.entropy[r] = H;
  }
  return o;
}

// the outputs of a row that counts for nothing
__device__ __forceinline__ void finish_dead_row(const LossRows& a, const PolicyTerms& t, int64_t r) {
  a.logps[r] = 0.f;
  if (a.stats) a.stats[2 * r] = 0.f, a.stats[2 * r + 1] = 1.f;
  if (a.coef_zero) zero_coef(a, r);
  if (t.entropy) t.entropy[r] = 0.f;
  if (t.row_loss) t.row_loss[r] = 0.f;
}

__device__ __forceinline__ void finish_dead_row(const LossRows&, const DistillTerms& t, int64_t r) {
  t.divergence[r] = 0.f;
  t.row_loss[r] = 0.f;
}

// p (log p - log q) of one teacher entry, added to kl; an entry of probability zero adds nothing
__device__ __forceinline__ float distill_term(const LossRows& a, float kl, float lp, float z, float m, float ls) {
  const float p = expf(lp);
  return p != 0.f ? fmaf(p, lp - over_t(a, z - m, -ls), kl) : kl;
}

// the teacher's probability at an id that is given more than once
__device__ __forceinline__ float mass_at(const int* ids, const float* lp, int K, int id) {
  float p = 0.f;
  for (int k = 0; k < K; ++k)
    if (ids[k] == id) p += expf(lp[k]);
  return p;
}

// the first entry of the same id as entry k
__device__ __noinline__ int first_of(const int* ids, int k) {
  int i = 0;
  while (ids[i] != ids[k]) ++i;
  return i;
}

// The row's softmax from the student's sums outside the ids and at them, and what is left of the teacher: p_r = 1 - P,
// P = sum p, where the rest is a class of its own (else zero).  Where the student has nothing left, or less than an fp32
// number of the row's own scale could hold (q_r < 2^-126), a p_r of the size of P's rounding is none: times log q_r it
// would be any number.
struct Rest {
  float m, sum;  // the row's largest logit, its sum of exponentials below that
  float f;       // e^((largest outside - m) / T)
  float p;
};
__device__ __forceinline__ Rest rest_of(const LossRows& a, bool tail, float mass, const Apart& st) {
  Rest o;
  o.m = fmaxf(st.out.m, st.in.m);
  o.f = expf(over_t(a, st.out.m - o.m, 0.f));
  o.sum = fmaf(st.out.s, o.f, st.in.s * expf(over_t(a, st.in.m - o.m, 0.f)));
  o.p = tail ? fmaxf(1.f - mass, 0.f) : 0.f;
  if (o.p > 0.f && o.p < 0x1p-20f && st.out.s * o.f < 0x1p-126f * o.sum) o.p = 0.f;
  return o;
}
// The coefficients of the row's gradient (mass < 0: the teacher has no id),
//   dz_j = w T ((P + p_r) q_j - p_j) at an id,   w T ((P + p_r) q_j - p_r q_j / q_r) elsewhere,
// where q_j / q_r is taken below the largest logit outside the ids.  (No logit there: the gradient there is zero.)
__device__ __forceinline__ RowCoef distill_coef(const LossRows& a, float mass, float weight, const Rest& rest,
                                                const Apart& st) {
  RowCoef o{st.out.s == 0.f ? rest.m : st.out.m, 0.f, 0.f, 0.f, -1, 0.f, 0.f, rest.m, rest.sum};
  if (mass < 0.f || weight == 0.f) return o;
  o.y = 0;
  o.c = weight * float(a.temperature);
  o.total = mass + rest.p;
  o.A = o.c * (o.total * rest.f / rest.sum - (rest.p > 0.f && st.out.s != 0.f ? rest.p / st.out.s : 0.f));
  return o;
}
// ... and, with the divergence over the ids, its outputs (ls: the log of the row's sum)
__device__ __forceinline__ void write_distill_row(const LossRows& a, const DistillTerms& t, int64_t r, float mass,
                                                  float weight, float kl, const Rest& rest, const Apart& st, float ls) {
  if (rest.p > 0.f) kl += rest.p * (logf(rest.p) - over_t(a, st.out.m - rest.m, logf(st.out.s) - ls));
  t.divergence[r] = mass < 0.f ? 0.f : kl;
  t.row_loss[r] = mass < 0.f || weight == 0.f ? 0.f : weight * t.t2 * kl;
}

// One warp: a row's teacher entries (K <= 32 N), lane + 32 i a lane: ids (-1: none) and log-probabilities; returns the
// sum of the probabilities, -1 without an id.
template <int N>
__device__ __forceinline__ float teacher_probabilities(const LossRows& a, const DistillTerms& t, int64_t r, bool record,
                                                       int (&id)[N], float (&lp)[N]) {
  const int lane = threadIdx.x & 31;
  float m = -INFINITY, s = 0.f, mass = 0.f;
  bool any = false;
  int64_t j[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {  // all loads before the first use
    const int k = lane + 32 * i;
    j[i] = k < t.K ? ld_index(t.ids, a.index_dtype, r * t.K + k) : -1;
    lp[i] = k < t.K ? ld_as_f32(t.logits, t.dtype, r * t.K + k) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (j[i] >= a.V) {
      if (record) record_device_error(&g_loss_error, kErrSlotOutOfRange);
      j[i] = -1;
    }
    id[i] = j[i] < 0 ? -1 : int(j[i]);
    if (id[i] < 0) lp[i] = -INFINITY;
    any |= id[i] >= 0;
    m = fmaxf(m, lp[i]);
  }
  const float lse = t.lse ? t.lse[r] : 0.f;
  m = warp_max(m);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (id[i] >= 0) s += ex2((lp[i] - m) * a.k);
  s = logf(warp_sum(s));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (id[i] < 0) continue;
    lp[i] = t.lse ? over_t_less(a, lp[i], -lse) : over_t(a, lp[i] - m, -s);
    mass += expf(lp[i]);
  }
  mass = warp_sum(mass);
  return __any_sync(0xffffffffu, any) ? mass : -1.f;
}

// the gradient of one vector of logits (but for the label's own term)
template <typename T, int kGrad>
__device__ __forceinline__ void vector_grad(const uint4& v, float m, float k, float A, float B, float2* g) {
#pragma unroll
  for (int j = 0; j < Vec<T>::E / 2; ++j) {
    const float2 d = mul2(Vec<T>::minus(v, j, m), make_float2(k, k));
    const float2 e = make_float2(ex2(d.x), ex2(d.y));
    if constexpr (kGrad == 2)
      g[j] = mul2(e, fma2(make_float2(B, B), make_float2(fmaxf(d.x, -1000.f), fmaxf(d.y, -1000.f)),
                          make_float2(A, A)));
    else
      g[j] = mul2(e, make_float2(A, A));
  }
}

// g[e] += c for an e that is not known at compile time
template <typename T>
__device__ __forceinline__ void add_at(float2* g, int e, float c) {
#pragma unroll
  for (int j = 0; j < Vec<T>::E / 2; ++j) {
    if (e == 2 * j) g[j].x += c;
    if (e == 2 * j + 1) g[j].y += c;
  }
}

// log2(e) / T in two halves: with one, its rounding (up to 6e-8) moves every exponent of a part of a row the same way,
// and the log of the row's sum by its distance from the part's largest logits, 1e-7 and more.  (A gradient's exponentials
// and the few at the teacher's ids take the rounded factor: it moves a term at e^-7 by 4e-7 of itself, far below a bf16
// gradient's rounding and a few units of the last place of an fp32 one.)
struct Log2Scale {
  float hi, lo;
};

// The statistics of N vectors: s = sum 2^d and (kMoment) u = sum 2^d d with d = (z - base) k.
template <typename T, int N, bool kMoment>
__device__ __forceinline__ void accumulate(const uint4* v, float base, Log2Scale k, float& s_out, float& u_out) {
  float2 s = make_float2(0.f, 0.f), u = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < Vec<T>::E / 2; ++j) {
      const float2 z = Vec<T>::minus(v[i], j, base);
      const float2 d = fma2(z, make_float2(k.hi, k.hi), mul2(z, make_float2(k.lo, k.lo)));
      const float2 e = make_float2(ex2(d.x), ex2(d.y));
      s = add2(s, e);
      if constexpr (kMoment)  // a logit of -inf adds 0 x -1000, not 0 x -inf
        u = fma2(e, make_float2(fmaxf(d.x, -1000.f), fmaxf(d.y, -1000.f)), u);
    }
  s_out = s.x + s.y;
  u_out = u.x + u.y;
}

// `st` with N more vectors
template <typename T, int N, bool kMoment>
__device__ __forceinline__ void add_vectors(Stats<kMoment>& st, const uint4* v, const LossRows& a) {
  const float m = fmaxf(st.m, Vec<T>::template largest<N>(v));
  rescale(st, m, a);
  float s, u;
  const float base = m == -INFINITY ? 0.f : m;  // without a finite logit: 2^-inf each
  accumulate<T, N, kMoment>(v, base, Log2Scale{a.k_hi, a.k_lo}, s, u);
  st.s += s;
  if constexpr (kMoment) st.u += u;
}

// -------------------------------------------------------------------- token log-probabilities, policy loss
// kEntropy: the row's entropy is formed; kGrad: the gradient is (kGrad == 2: with the entropy's term).
// Without a gradient the memory bounds it: bf16 8192 x 32000, 7168 rows that count, 459 MB read in 81 us, 86 % of the
// measured copy rate (CTAs of 128 threads at different places of their rows; what is missing is the last round of
// them).  With one, a CTA that keeps its row in registers loads, computes and stores by turns, and the SM's few CTAs
// run in step: 600 x 32000 26 us, 45 % of the rate of one read and one write; many long rows are the streaming
// kernel's.
template <typename T, int NT, bool kEntropy, int kGrad>
__global__ void __launch_bounds__(Cta<NT>::kThreads, 1024 / Cta<NT>::kThreads)
    logp_kernel(LossRows a, PolicyTerms t, int parts) {
  await_previous();
  const int64_t r = Cta<NT>::row(parts);
  if (r >= a.n) return;
  const int rank = int(blockIdx.x % unsigned(parts));
  const Share<T> w(a, r, rank, parts);
  const int tid = int(threadIdx.x) % NT;
  const bool first = rank == 0 && tid == 0;
  const int64_t y = row_label(a, r, first);
  if (y < 0) {  // the same for every CTA of the cluster
    if (first) finish_dead_row(a, t, r);
    if (kGrad) w.template zero<NT>(tid);
    return;
  }
  if (parts > 1) tc::cluster_arrive();
  const float zy = to_f32(w.z[y]);
  PolicyIn in = policy_inputs<false>(t, r);
  uint4 v[kNV];
  auto load = [&](int at) {
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int vi = at + tid + i * NT;
      v[i] = vi < w.v1 ? w.load(vi) : make_uint4(Vec<T>::kFill, Vec<T>::kFill, Vec<T>::kFill, Vec<T>::kFill);
    }
  };
  const int rounds = max(1, (w.v1 - w.v0 + NT * kNV - 1) / (NT * kNV));
  Stats<kEntropy> st;
  for (int q = 0; q < rounds; ++q) {
    load(w.v0 + q * NT * kNV);
    add_vectors<T, kNV>(st, v, a);
  }
  if (t.row_loss && !t.weights && !t.scale) in.w = mean_of_few(a, nullptr, 0);
  if (parts > 1) tc::cluster_wait();  // every CTA of the cluster runs: their shared memory may be written
  st = merge_rows<NT>(st, a, rank, parts);
  const RowCoef o = finish_row<kEntropy, kGrad>(a, t, in, r, int(y), zy, st, first, [](const RowCoef&) {});
  if constexpr (kGrad != 0) {
    if (o.y < 0) {
      w.template zero<NT>(tid);
      return;
    }
    const int vy = (int(y) + w.off) / Vec<T>::E;
    for (int q = rounds - 1; q >= 0; --q) {
      if (q < rounds - 1) load(w.v0 + q * NT * kNV);
#pragma unroll
      for (int i = 0; i < kNV; ++i) {
        const int vi = w.v0 + q * NT * kNV + tid + i * NT;
        if (vi >= w.v1) break;
        float2 g[Vec<T>::E / 2];
        vector_grad<T, kGrad>(v[i], o.m, a.k, o.A, o.B, g);
        w.store(vi, g);
        if (vi == vy) from_f32(w.dz + y, o.at_label);  // after this thread's own store of the vector
      }
    }
  }
}

// d/dz of sum_t dlogps_t logp_t from the saved statistics: one read, one write, nothing to reduce.  Bound by memory:
// 8192 x 32000 bf16 in 165 us, 97 % of the measured copy rate.  (Loading a row before the coefficients are awaited made
// a call of 8192 x 32000 slower, 239 us against 221: every CTA then waits for its coefficient behind its loads.)
template <typename T, int NT>
__global__ void __launch_bounds__(Cta<NT>::kThreads, 1024 / Cta<NT>::kThreads)
    logp_backward_kernel(LossRows a, const float* dlogps, int parts) {
  await_previous();
  const int64_t r = a.n - 1 - Cta<NT>::row(parts);  // what the forward pass read last may still be in L2
  if (r < 0) return;
  const int tid = int(threadIdx.x) % NT;
  const Share<T> w(a, r, int(blockIdx.x % unsigned(parts)), parts);
  const int64_t y = row_label(a, r, tid == 0);
  const float c = y < 0 ? 0.f : dlogps[r] * a.inv_t;
  if (c == 0.f) {
    w.template zero<NT>(tid);
    return;
  }
  const float m = a.stats[2 * r], A = -c / a.stats[2 * r + 1];
  const int vy = (int(y) + w.off) / Vec<T>::E, ey = (int(y) + w.off) % Vec<T>::E;
  for (int at = w.v0 + tid; at < w.v1; at += NT * kNV) {
    uint4 v[kNV];
#pragma unroll
    for (int i = 0; i < kNV; ++i)
      if (at + i * NT < w.v1) v[i] = w.load(at + i * NT);
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int vi = at + i * NT;
      if (vi >= w.v1) break;
      float2 g[Vec<T>::E / 2];
      vector_grad<T, 1>(v[i], m, a.k, A, 0.f, g);
      if (vi == vy) add_at<T>(g, ey, c);
      w.store(vi, g);
    }
  }
}

// ------------------------------------------------------------------------- many rows: the streaming kernel
// One resident CTA (or cluster) an SM takes rows as they come, and its warps have roles, so that reading, arithmetic
// and writing of different rows overlap (with a CTA per row, the CTAs of an SM load together and compute together: a
// 32000-entry bf16 row takes about 2100 cycles of ex2 for its statistics, 2100 for its gradient, and 5600 of memory
// time at the measured copy rate):
//   producer   takes the next group of rows (the grid has a cluster for each; a resident one cancels the launch of
//              one that has not started and does its work instead, so SMs that met many ignored rows take more),
//              reads their labels, queues them for the other roles, and copies the share of those that count into a
//              ring of 16 KiB chunks in shared memory;
//   teacher    (distillation only) forms the teacher's probabilities of a row;
//   marker     (distillation only) adds up the exponentials at the teacher's ids in every chunk that arrives and puts
//              -inf in their place, so that what the statistics role sums is the student's mass outside the ids (one
//              minus the mass inside would lose it when that is near one);
//   statistics (8 warps) maximum and sums of every chunk as it arrives, then a warp's partial results: 8 for the policy
//              loss, whose control warps have the time to add them up, else one; in a cluster, one to the shared memory
//              of every CTA of it;
//   control    (2 warps, row about) merges a row's partials, publishes the coefficients of its gradient, and then
//              computes and writes the row's outputs;
//   gradient   (8 warps) reads the row's chunks once more from shared memory, writes the gradient, frees them;
//   patcher    (distillation only) writes the gradient's entries at the ids once the row's gradient is written.
// A slot's, a row's and a buffer's barriers are waited for by each role at every use and in order: a wait by parity
// cannot tell a use from the one two before.  Every wait is bounded; after one that gave up a role ends,
// kErrLossWaitTimeout is recorded, and the CTA returns when its copies have landed.
//
// What bounds it: bf16 rows of 32000, 3.4 us a row and SM for the policy loss against 2.9 us of memory (7168 of 8192
// rows of 131072, two CTAs a row: 742 us, 83 % of the measured copy rate of one read and one write; fp32 32000 with a
// teacher's 64 entries: 5.9 us a row, 98 %).  The statistics warps are busy for 5600 of a row's 6900 cycles; a row
// stays in the ring until its gradient is written, and the ring holds three of 64 KB, so the time from a row's last
// chunk to its coefficients counts in full.  Other shapes of the ring and the roles, the same policy loss: 256 threads
// x 4 vectors 748 us (kept); x 3 828, x 2 867, x 5 810, x 6 817; 320 threads x 3 813, 384 x 3 833, 384 x 2 815.
constexpr int kBuf = 8;                // rows between a partial result and its use, see Exchange
constexpr int kQueue = 32;             // rows between the producer and the last of the other roles
constexpr int kRoleWarps = kRoleThreads / 32;
constexpr int kControlWarps = 2;
constexpr int kMaxTop = 128;           // teacher entries of a row that the streaming kernel takes
constexpr int kTeachers = 6;           // rows between the teacher and the patcher (even: control takes rows in turn)
constexpr uint32_t kLossWaitLimit = 1u << 20;

constexpr int kSlots = 13;             // chunks of the ring
constexpr size_t kRingBytes = size_t(kSlots) * kChunk * 16;

// What the kinds of losses differ in: their roles.
template <typename Terms>
struct Streaming {
  static constexpr bool kDistill = std::is_same_v<Terms, DistillTerms>;
  static constexpr int kMarkers = kDistill ? 1 : 0;
  static constexpr int kPartLanes = kDistill ? 1 : 8;  // partial results of a statistics warp (1 in a cluster)
  static constexpr int kThreads = 2 * kRoleThreads + 32 * (kControlWarps + 1 + (kDistill ? 3 : 0));
};

struct __align__(16) QueuedRow {
  int64_t row;  // -1: no more rows
  int label;    // -1: the row counts for nothing (-2: its label lies outside the vocabulary)
  int pad;
};

// A row's teacher: log-probabilities at its ids (-1: none).
struct Teacher {
  float lp[kMaxTop];
  int id[kMaxTop];
};

// What the roles pass on.  Rows that count use the 8 buffers for partial results and coefficients in turn.  They are
// free when they are written.  With a gradient, a row leaves the ring when its coefficients have been used, and when
// the last chunk of a row is there the ring holds nothing older than the 6 rows before it (a share is 2 chunks or
// more), in a cluster than the 2 rows before it (more than 4 chunks), where another CTA's control is then at most 6
// rows behind.  Without one, statistics (and the marker) wait for the control warps to be at most half of the buffers
// behind.  The teachers' buffers are handed back by a barrier.
template <bool kDistill>
struct Exchange {
  uint4 response;                                                  // of a request for more rows
  // packed sums of the statistics warps (kPartLanes of each, or one for each of every CTA of a cluster) and the marker
  float4 part[kBuf * kMaxCluster * (kRoleWarps + kDistill)];
  QueuedRow queue[kQueue];
  RowCoef coef[kBuf];
  Teacher teacher[kDistill ? kTeachers : 1];
  float mass[kTeachers];  // the sum of a teacher's probabilities, -1 without an id
  int twice[kTeachers];   // an id was given twice
  int ticket[2];          // the cluster's next group of rows, -1: none
  uint32_t sink[2 * kRoleWarps];  // see free_chunk
  uint32_t spare[32];
  uint64_t full[kSlots], empty[kSlots], marked[kSlots];
  uint64_t part_full[kBuf], coef_full[kBuf];
  uint64_t teacher_full[kTeachers], teacher_free[kTeachers];
  uint64_t row_done[kTeachers];  // the gradient is written and the row's ids are known to be given once or more
  uint64_t queue_full[kQueue], queue_empty[kQueue];
  uint64_t response_full, ticket_full[2], ticket_free[2];
};

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ void sts16(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// arrive on the barrier at the same address of CTA `rank` of the cluster / wait for arrivals of other CTAs
__device__ __forceinline__ void arrive_cluster(uint64_t* bar, uint32_t rank) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(tc::mapa(tc::smem_u32(bar), rank))
               : "memory");
}
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity) {
  bool done = false;
  for (uint32_t i = 0; i < kLossWaitLimit && !done; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(tc::smem_u32(bar)), "r"(parity)
        : "memory");
    done = ok != 0;
  }
  return __all_sync(0xffffffffu, done);
}
// a warp's bounded wait, the same answer in every lane
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, tc::mbar_wait_bounded(bar, parity, kLossWaitLimit));
}

// 16 bytes to the same place of CTA `rank` of the cluster, counted by the barrier of that CTA
__device__ __forceinline__ void st_async(float4* p, uint64_t* bar, uint32_t rank, const float4& t) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                   tc::mapa(tc::smem_u32(p), rank)),
               "f"(t.x), "f"(t.y), "f"(t.z), "f"(t.w), "r"(tc::mapa(tc::smem_u32(bar), rank))
               : "memory");
}

// Asks for the launch of a cluster that has not started to be cancelled; the answer (16 bytes) completes `bar`.
__device__ __forceinline__ void request_rows(uint4* response, uint64_t* bar) {
  tc::mbar_arrive_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   tc::smem_u32(response)),
               "r"(tc::smem_u32(bar))
               : "memory");
}
// the first CTA of the cluster that was cancelled, or -1 when there was none left
__device__ __forceinline__ int64_t requested_cta(const uint4* response) {
  uint32_t got, x;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\tld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(tc::smem_u32(response))
      : "memory");
  return got ? int64_t(x) : -1;
}

// A place in a circular buffer: its index and the parity of its current use.
struct Place {
  int size, i = 0;
  uint32_t parity = 0;
  bool wrapped = false;
  __device__ __forceinline__ explicit Place(int n) : size(n) {}
  __device__ __forceinline__ void next() {
    if (++i == size) i = 0, parity ^= 1u, wrapped = true;
  }
};

// a share of `per` vectors for every row, whatever its start within 16 bytes
template <typename T>
struct RowShare {
  static constexpr int E = Vec<T>::E;
  int off, v0, count;  // as Share; vectors of the share
  bool ragged;         // an end of the row lies inside one of them
  __device__ __forceinline__ RowShare(const T* z, int V, int per, int rank) {
    off = int((uint32_t(reinterpret_cast<uintptr_t>(z)) & 15u) / sizeof(T));
    const int nvec = (off + V + E - 1) / E;
    v0 = rank * per;
    count = max(0, min(per, nvec - v0));
    ragged = (v0 == 0 && off > 0) || (v0 + count == nvec && (off + V) % E != 0);
  }
};

// Hands a chunk back once the warp's loads of it have returned.  An arrival does not wait for loads still under way
// (it overtook them: the next copy was then read in their place); the store of a word that needs all of them does.
template <int N>
__device__ __forceinline__ void free_chunk(uint64_t* bar, const uint4 (&v)[N], uint32_t* sink) {
  uint32_t all = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) all ^= v[i].x;
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(tc::smem_u32(sink)), "r"(all) : "memory");
    tc::mbar_arrive(bar);
  }
}

// The next row of a role's walk through the queue.
struct QueueReader {
  Place at{kQueue};
  template <typename X>
  __device__ __forceinline__ bool next(X& x, QueuedRow& row) {
    const bool ok = warp_wait(&x.queue_full[at.i], at.parity);
    if (ok) row = x.queue[at.i];
    // through a shuffle: it needs the loaded values, and the slot is handed back after it
    row.row = __shfl_sync(0xffffffffu, row.row, 0);
    row.label = __shfl_sync(0xffffffffu, row.label, 0);
    if ((threadIdx.x & 31) == 0) tc::mbar_arrive(&x.queue_empty[at.i]);
    at.next();
    return ok;
  }
};

// Sets an element of a chunk in shared memory / reads it.
template <typename T>
__device__ __forceinline__ void put_bits(uint32_t a, uint32_t bits) {
  if constexpr (sizeof(T) == 4)
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(bits) : "memory");
  else
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(uint16_t(bits)) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t get_bits(uint32_t a) {
  if constexpr (sizeof(T) == 4) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
  } else {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
    return v;
  }
}
template <typename T>
__device__ __forceinline__ float bits_to_f32(uint32_t bits) {
  return __uint_as_float(sizeof(T) == 4 ? bits : bits << 16);
}

template <typename T, typename Terms, int kGrad>
__global__ void __launch_bounds__(Streaming<Terms>::kThreads, 1)
    loss_stream_kernel(LossRows a, Terms t, int group_rows, int per, int parts) {
  extern __shared__ __align__(128) uint8_t ring_mem[];
  constexpr bool kDistill = Streaming<Terms>::kDistill;
  constexpr int E = Vec<T>::E, kMarkers = Streaming<Terms>::kMarkers;
  constexpr int kPartLanes = Streaming<Terms>::kPartLanes;
  // warps: statistics, gradient, control, producer, teacher, marker, patcher
  constexpr int kGradWarp = kRoleWarps, kControlWarp = 2 * kRoleWarps, kProducerWarp = kControlWarp + kControlWarps;
  constexpr int kTeacherWarp = kProducerWarp + 1, kMarkerWarp = kProducerWarp + 2;
  __shared__ Exchange<kDistill> x;
  const int tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int rank = int(blockIdx.x % unsigned(parts)), V = int(a.V);
  const uint32_t ring = tc::smem_u32(ring_mem);
  const T* logits = static_cast<const T*>(a.logits);
  const int row_parts = parts == 1 ? kRoleWarps * kPartLanes + kMarkers : parts * (kRoleWarps + kMarkers);
  const uint32_t part_bytes = uint32_t(row_parts) * 16u;
  if (tid < 64) {  // a few barriers a thread
    if (tid < kSlots) {
      tc::mbar_init(&x.full[tid], 1);
      tc::mbar_init(&x.empty[tid], kRoleWarps);
      tc::mbar_init(&x.marked[tid], 1);
    }
    if (tid < kBuf) {
      tc::mbar_init(&x.part_full[tid], parts == 1 ? kRoleWarps + kMarkers : 1);
      if (parts > 1) tc::mbar_arrive_expect_tx(&x.part_full[tid], part_bytes);
      tc::mbar_init(&x.coef_full[tid], 1);
    }
    if (tid >= 16 && tid < 16 + kTeachers) {
      tc::mbar_init(&x.teacher_full[tid - 16], 1);
      tc::mbar_init(&x.teacher_free[tid - 16], kGrad ? 2 : 1);  // control and patcher
      tc::mbar_init(&x.row_done[tid - 16], kRoleWarps + 1);
    }
    if (tid >= 32) {
      tc::mbar_init(&x.queue_full[tid - 32], 1);
      tc::mbar_init(&x.queue_empty[tid - 32], (kGrad ? 2 : 1) * (kRoleWarps + kDistill) + kControlWarps + kDistill);
    }
    if (tid == 24) tc::mbar_init(&x.response_full, 1);
    if (tid == 25 || tid == 26) {
      tc::mbar_init(&x.ticket_full[tid - 25], 1);
      tc::mbar_init(&x.ticket_free[tid - 25], uint32_t(parts));
    }
    tc::fence_mbar_init();
  }
  await_previous();
  __syncthreads();
  if (parts > 1) {  // the barriers of every CTA of the cluster are set before one of them is arrived on
    tc::cluster_arrive();
    tc::cluster_wait();
  }
  bool ok = true;
  QueueReader reader;
  QueuedRow row;
  Place buf(kBuf), slot(kSlots), teach(kTeachers);
  Place read(buf.size);  // half of the buffers behind buf
  int ahead = 0;
  // a warp's partial results of the row (statistics warps, then the marker): lanes [0, lanes), or the warp's one to
  // every CTA of the cluster
  const auto publish = [&](const float4& sums, int index, int lanes) {
    if (kGrad == 0 && ++ahead > buf.size / 2) {
      ok = ok && warp_wait(&x.coef_full[read.i], read.parity);
      read.next();
    }
    if (parts == 1) {
      if (ok && lane < lanes) x.part[buf.i * row_parts + index + lane] = sums;
      __syncwarp();
      if (ok && lane == 0) tc::mbar_arrive(&x.part_full[buf.i]);
    } else if (ok && lane < parts) {
      st_async(&x.part[buf.i * row_parts + rank * (kRoleWarps + kMarkers) + index], &x.part_full[buf.i], uint32_t(lane),
               sums);
    }
    buf.next();
  };

  if (warp < kGradWarp) {
    // ------------------------------------------------------------------------------------------- statistics
    while ((ok = ok && reader.next(x, row)) && row.row >= 0) {
      if (row.label < 0) continue;
      const RowShare<T> sh(logits + row.row * a.ld, V, per, rank);
      Stats<!kDistill> st;
      for (int at = 0; at < sh.count && ok; at += kChunk, slot.next()) {
        ok = warp_wait(kDistill ? &x.marked[slot.i] : &x.full[slot.i], slot.parity);
        const uint32_t src = ring + uint32_t(slot.i * kChunk + tid) * 16u;
        const int left = sh.count - at - tid;
        uint4 v[kPer];
        if (sh.count - at >= kChunk) {
#pragma unroll
          for (int i = 0; i < kPer; ++i) v[i] = lds16(src + i * kRoleThreads * 16);
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            v[i] = make_uint4(Vec<T>::kFill, Vec<T>::kFill, Vec<T>::kFill, Vec<T>::kFill);
            if (i * kRoleThreads < left) v[i] = lds16(src + i * kRoleThreads * 16);
          }
        }
        if (sh.ragged) {  // what lies outside the row becomes -inf
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int j0 = (sh.v0 + at + tid + i * kRoleThreads) * E - sh.off;
            if (i * kRoleThreads < left && (j0 < 0 || j0 + E > V)) v[i] = mask_edge<T>(v[i], j0, V);
          }
        }
        if (kGrad == 0) free_chunk(&x.empty[slot.i], v, &x.sink[warp]);  // nobody else reads the chunk
        add_vectors<T, kPer>(st, v, a);
      }
      const auto sums = [](const Stats<!kDistill>& t) {
        if constexpr (kDistill)
          return pack(Apart{t, Sum{}});
        else
          return pack(t);
      };
      if (parts == 1)
        publish(sums(merge_warp<kPartLanes>(st, a)), warp * kPartLanes, kPartLanes);
      else
        publish(sums(merge_warp(st, a)), warp, 1);
    }
  } else if (warp < kControlWarp) {
    // --------------------------------------------------------------------------------------------- gradient
    // (without one its warps leave at once)
    const int tg = tid - kRoleThreads;
    const bool same = ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.dlogits)) & 15) == 0 &&
                      ((a.ld - a.ld_d) * int64_t(sizeof(T)) & 15) == 0;
    while (kGrad != 0 && (ok = ok && reader.next(x, row)) && row.row >= 0) {
      const RowShare<T> sh(logits + row.row * a.ld, V, per, rank);
      T* dz = static_cast<T*>(a.dlogits) + row.row * a.ld_d;
      const bool live = row.label >= 0, plain = same && !sh.ragged;
      RowCoef o;
      o.y = -1;
      if (live) {
        ok = warp_wait(&x.coef_full[buf.i], buf.parity);
        o = x.coef[buf.i];
        buf.next();
      }
      const int label = kDistill || o.y < 0 ? -1 : (o.y + sh.off) / E - sh.v0;  // its vector of the share
      for (int at = 0; at < sh.count && ok; at += kChunk) {
        uint4 v[kPer];
        if (live) {
          ok = warp_wait(&x.full[slot.i], slot.parity);  // at once: the statistics role has read the chunk
          const uint32_t src = ring + uint32_t(slot.i * kChunk + tg) * 16u;
#pragma unroll
          for (int i = 0; i < kPer; ++i) v[i] = lds16(src + i * kRoleThreads * 16);
          free_chunk(&x.empty[slot.i], v, &x.sink[warp]);
          slot.next();
        }
        const int left = sh.count - at - tg, j0 = (sh.v0 + at + tg) * E - sh.off;
        if (plain && o.y >= 0) {
          uint4* dst = reinterpret_cast<uint4*>(dz + j0);
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            float2 g[E / 2];
            vector_grad<T, kGrad>(v[i], o.m, a.k, o.A, o.B, g);
            if (i * kRoleThreads < left) dst[i * kRoleThreads] = Vec<T>::pack(g);
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < kPer; ++i) {
            if (i * kRoleThreads >= left) break;
            const int ji = j0 + i * kRoleThreads * E;
            float2 g[E / 2] = {};
            const uint4 vi = i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3];
            if (o.y >= 0) vector_grad<T, kGrad>(vi, o.m, a.k, o.A, o.B, g);
            if (same && ji >= 0 && ji + E <= V)
              *reinterpret_cast<uint4*>(dz + ji) = Vec<T>::pack(g);
            else
              store_edge<T>(dz, Vec<T>::pack(g), ji, V);
          }
        }
        // the label's own entry, after its thread's store of the vector
        if (label >= at && label < at + kChunk && label < sh.count && (label & (kRoleThreads - 1)) == tg)
          from_f32(dz + o.y, o.at_label);
      }
      if (kDistill && live) {
        __syncwarp();
        if (lane == 0 && ok) tc::mbar_arrive(&x.row_done[teach.i]);
        teach.next();
      }
    }
  } else if (warp < kProducerWarp) {
    // ---------------------------------------------------------------------------------------------- control
    const bool write = rank == 0 && lane == 0;
    // The rows that count are taken in turn (so that one's buffer was last used by a row that this warp, too, has seen
    // done), and so are the others.
    int turn = warp - kControlWarp, dead_turn = turn;
    while ((ok = ok && reader.next(x, row)) && row.row >= 0) {
      int& next = row.label < 0 ? dead_turn : turn;
      const bool mine = next == 0;
      next = next == 0 ? kControlWarps - 1 : next - 1;
      if (row.label < 0) {
        if (!mine) continue;
        if (lane == 0 && row.label == -2) record_device_error(&g_loss_error, kErrSlotOutOfRange);
        if (write) finish_dead_row(a, t, row.row);
        continue;
      }
      if (mine) {
        const auto ready = [&](const RowCoef& o) {
          if (lane != 0) return;
          if (parts > 1) tc::mbar_arrive_expect_tx(&x.part_full[buf.i], part_bytes);  // for its next use
          x.coef[buf.i] = o;
          tc::mbar_arrive(&x.coef_full[buf.i]);
        };
        if constexpr (!kDistill) {
          // asked for while the row's statistics are still being formed
          const float zy = to_f32((logits + row.row * a.ld)[row.label]);
          const PolicyIn in = policy_inputs<true>(t, row.row);
          ok = wait_cluster(&x.part_full[buf.i], buf.parity);
          if (!ok) break;
          const auto st = merge_parts<Stats<true>>(x.part + buf.i * row_parts, row_parts, a);
          finish_row<true, kGrad>(a, t, in, row.row, row.label, zy, st, write, ready);
        } else {
          ok = warp_wait(&x.teacher_full[teach.i], teach.parity);
          if (!ok) break;
          const Teacher& te = x.teacher[teach.i];
          const float mass = x.mass[teach.i], wt = t.weights ? t.weights[row.row] : *t.scale;
          float zk[kMaxTop / 32];  // the student's logits at the ids
#pragma unroll
          for (int i = 0; i < kMaxTop / 32; ++i) {
            const int k = lane + 32 * i;
            zk[i] = k < t.K && te.id[k] >= 0 ? to_f32((logits + row.row * a.ld)[te.id[k]]) : 0.f;
          }
          ok = wait_cluster(&x.part_full[buf.i], buf.parity);
          if (!ok) break;
          const Apart st = merge_parts<Apart>(x.part + buf.i * row_parts, row_parts, a);
          const Rest rest = rest_of(a, t.lse != nullptr, mass, st);
          ready(distill_coef(a, mass, wt, rest, st));
          float kl = 0.f;
          const float ls = logf(rest.sum);
#pragma unroll
          for (int i = 0; i < kMaxTop / 32; ++i) {
            const int k = lane + 32 * i;
            if (k >= t.K || te.id[k] < 0) continue;
            kl = distill_term(a, kl, te.lp[k], zk[i], rest.m, ls);
          }
          kl = warp_sum(kl);  // needs every lane's entries: the teacher's buffer is handed back after it
          if (lane == 0) tc::mbar_arrive(&x.teacher_free[teach.i]);
          if (write) write_distill_row(a, t, row.row, mass, wt, kl, rest, st, ls);
        }
      }
      buf.next();
      teach.next();
    }
  } else if (warp == kProducerWarp) {
    // --------------------------------------------------------------------------------------------- producer
    Place q(kQueue), tk(2);
    uint32_t response_parity = 0;
    const auto push = [&](int64_t r, int label) {
      if (q.wrapped) ok = ok && warp_wait(&x.queue_empty[q.i], q.parity ^ 1u);
      if (lane == 0) {
        x.queue[q.i] = QueuedRow{r, label, 0};
        tc::mbar_arrive(&x.queue_full[q.i]);
      }
      q.next();
    };
    // Group k's rows are copied while the answer about group k + 2 is on its way: group k + 1's is read, and passed on
    // to the cluster, before group k is begun.
    int group = int(blockIdx.x) / parts, next = -1;
    bool asked = rank == 0;  // an answer is on its way
    if (asked && lane == 0) request_rows(&x.response, &x.response_full);
    while (ok && group >= 0) {
      const int64_t first = int64_t(group) * group_rows;
      const int rows = int(min(int64_t(group_rows), a.n - first));
      int mine = -1;
      if (lane < rows) {
        if constexpr (kDistill) {
          mine = ld_index(t.ids, a.index_dtype, (first + lane) * t.K) < 0 ? -1 : 0;
        } else {
          const int64_t y = ld_index(a.labels, a.index_dtype, first + lane);
          mine = y == a.ignore_index ? -1 : (y < 0 || y >= V) ? -2 : int(y);
        }
      }
      if (rank == 0) {
        const bool answered = warp_wait(&x.response_full, response_parity);
        const int64_t cta = answered ? requested_cta(&x.response) : -1;
        next = __shfl_sync(0xffffffffu, cta < 0 ? -1 : int(cta / parts), 0);
        ok = ok && answered;
        if (answered) {
          asked = next >= 0;
          response_parity ^= 1u;
          tc::fence_proxy_async_smem();  // read before the next answer is written there
          __syncwarp();
          if (asked && lane == 0) request_rows(&x.response, &x.response_full);
        }
        if (parts > 1) {
          if (tk.wrapped) ok = wait_cluster(&x.ticket_free[tk.i], tk.parity ^ 1u) && ok;
          if (lane < parts) {
            const uint32_t to = tc::mapa(tc::smem_u32(&x.ticket[tk.i]), uint32_t(lane));
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(next) : "memory");
            arrive_cluster(&x.ticket_full[tk.i], uint32_t(lane));
          }
        }
      }
      for (int i = 0; i < rows && ok; ++i) {
        const int64_t r = first + i;
        const int label = __shfl_sync(0xffffffffu, mine, i);
        push(r, label);
        if (label < 0) continue;
        const T* z = logits + r * a.ld;
        const RowShare<T> sh(z, V, per, rank);
        // a vector that reaches over an end of the row is copied whole, unless that end is the tensor's
        const bool head = r == 0 && sh.v0 == 0 && sh.off > 0;
        const bool tail = r == a.n - 1 && (sh.v0 + sh.count) * E - sh.off > V;
        for (int at = 0; at < sh.count && ok; at += kChunk, slot.next()) {
          if (slot.wrapped) ok = warp_wait(&x.empty[slot.i], slot.parity ^ 1u);
          if (lane != 0 || !ok) continue;
          if (kDistill) tc::fence_proxy_async_smem();  // the marker has written to the slot: the copy comes after
          const uint32_t dst = ring + uint32_t(slot.i * kChunk) * 16u;
          int lo = at, hi = min(at + kChunk, sh.count);
          const int count = hi - lo;
          if (head && lo == 0) {
            sts16(dst, load_edge(z, -sh.off, V));
            ++lo;
          }
          if (tail && hi == sh.count && hi > lo) {
            --hi;
            sts16(dst + (hi - at) * 16, load_edge(z, (sh.v0 + hi) * E - sh.off, V));
          }
          if (hi - lo < count) tc::fence_proxy_async_smem();  // these stores before the slot's next copy
          const uint32_t bytes = uint32_t(hi - lo) * 16u;
          if (bytes) {
            tc::mbar_arrive_expect_tx(&x.full[slot.i], bytes);
            tc::bulk_load(dst + (lo - at) * 16, z + ((sh.v0 + lo) * E - sh.off), bytes, &x.full[slot.i]);
          } else {
            tc::mbar_arrive(&x.full[slot.i]);
          }
        }
      }
      if (parts > 1) {
        ok = wait_cluster(&x.ticket_full[tk.i], tk.parity) && ok;
        next = __shfl_sync(0xffffffffu, x.ticket[tk.i], 0);
        if (lane == 0) arrive_cluster(&x.ticket_free[tk.i], 0);
        tk.next();
      }
      group = next;
    }
    if (!ok && asked)  // the answer lands before the CTA leaves
      tc::mbar_wait_bounded(&x.response_full, response_parity, 1u << 16);
    push(-1, -1);
    if (!ok)  // copies in flight land before the CTA leaves: wait for every slot's last use
      for (int i = 0; i < kSlots; ++i)
        if (slot.wrapped || i < slot.i)
          tc::mbar_wait_bounded(&x.full[i], i < slot.i ? slot.parity : slot.parity ^ 1u, 1u << 16);
  } else if constexpr (kDistill) {
    if (warp == kTeacherWarp) {
      // -------------------------------------------------------------------------------------------- teacher
      while ((ok = ok && reader.next(x, row)) && row.row >= 0) {
        if (row.label < 0) continue;
        int id[kMaxTop / 32];
        float lp[kMaxTop / 32];
        const float mass = teacher_probabilities(a, t, row.row, rank == 0, id, lp);
        if (teach.wrapped) ok = warp_wait(&x.teacher_free[teach.i], teach.parity ^ 1u);
        if (!ok) break;
        Teacher& te = x.teacher[teach.i];
#pragma unroll
        for (int i = 0; i < kMaxTop / 32; ++i) {
          te.id[lane + 32 * i] = id[i];
          te.lp[lane + 32 * i] = lp[i];
        }
        if (lane == 0) x.mass[teach.i] = mass;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&x.teacher_full[teach.i]);
        teach.next();
      }
    } else if (warp == kMarkerWarp) {
      // --------------------------------------------------------------------------------------------- marker
      while ((ok = ok && reader.next(x, row)) && row.row >= 0) {
        if (row.label < 0) continue;
        ok = warp_wait(&x.teacher_full[teach.i], teach.parity);
        if (!ok) break;
        int id[kMaxTop / 32];
#pragma unroll
        for (int i = 0; i < kMaxTop / 32; ++i) id[i] = x.teacher[teach.i].id[lane + 32 * i];
        const RowShare<T> sh(logits + row.row * a.ld, V, per, rank);
        Sum st;
        bool again = false;
        for (int at = 0; at < sh.count && ok; at += kChunk, slot.next()) {
          ok = warp_wait(&x.full[slot.i], slot.parity);
          const int lo = (sh.v0 + at) * E - sh.off, hi = (sh.v0 + min(at + kChunk, sh.count)) * E - sh.off;
          const uint32_t base = ring + uint32_t(slot.i * kChunk) * 16u;
          uint32_t place[kMaxTop / 32];  // an entry's element in the chunk; a word of the lane's own where it has none
          bool here[kMaxTop / 32], any = false;
#pragma unroll
          for (int i = 0; i < kMaxTop / 32; ++i) {
            here[i] = id[i] >= 0 && id[i] >= lo && id[i] < hi;
            place[i] = here[i] ? base + uint32_t(id[i] - lo) * uint32_t(sizeof(T)) : tc::smem_u32(&x.spare[lane]);
            any |= here[i];
          }
          if (__any_sync(0xffffffffu, any)) {
            // every entry leaves its number; where another one's is found there, the same id was given again
            uint32_t bits[kMaxTop / 32], found[kMaxTop / 32];
#pragma unroll
            for (int i = 0; i < kMaxTop / 32; ++i) bits[i] = get_bits<T>(place[i]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kMaxTop / 32; ++i) put_bits<T>(place[i], uint32_t(lane + 32 * i));
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kMaxTop / 32; ++i) found[i] = get_bits<T>(place[i]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kMaxTop / 32; ++i) put_bits<T>(place[i], Vec<T>::kFill);
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&x.marked[slot.i]);
            uint32_t differ = 0u;
#pragma unroll
            for (int i = 0; i < kMaxTop / 32; ++i) differ |= here[i] ? found[i] ^ uint32_t(lane + 32 * i) : 0u;
            if (__any_sync(0xffffffffu, differ)) {  // the first entry of an id counts, whichever store came last
              again = true;
#pragma unroll
              for (int i = 0; i < kMaxTop / 32; ++i)
                if (here[i]) here[i] = first_of(x.teacher[teach.i].id, lane + 32 * i) == lane + 32 * i;
            }
            float m = st.m;
#pragma unroll
            for (int i = 0; i < kMaxTop / 32; ++i) {
              here[i] = here[i] && bits_to_f32<T>(bits[i]) != -INFINITY;
              if (here[i]) m = fmaxf(m, bits_to_f32<T>(bits[i]));
            }
            rescale(st, m, a);
#pragma unroll
            for (int i = 0; i < kMaxTop / 32; ++i)
              if (here[i]) st.s += ex2((bits_to_f32<T>(bits[i]) - m) * a.k);
          } else if (lane == 0) {
            tc::mbar_arrive(&x.marked[slot.i]);
          }
        }
        if (lane == 0 && kGrad != 0) {
          x.twice[teach.i] = again;
          tc::mbar_arrive(&x.row_done[teach.i]);
        }
        publish(pack(Apart{Sum{}, merge_warp(st, a)}), parts == 1 ? kRoleWarps * kPartLanes : kRoleWarps, 1);
        teach.next();
      }
    } else if (kGrad != 0) {
      // -------------------------------------------------------------------------------------------- patcher
      while ((ok = ok && reader.next(x, row)) && row.row >= 0) {
        if (row.label < 0) continue;
        ok = warp_wait(&x.coef_full[buf.i], buf.parity);
        if (!ok) break;
        const RowCoef o = x.coef[buf.i];
        const T* z = logits + row.row * a.ld;
        const RowShare<T> sh(z, V, per, rank);
        const Teacher& te = x.teacher[teach.i];
        int id[kMaxTop / 32];  // the ids of this share
        float zk[kMaxTop / 32];
#pragma unroll
        for (int i = 0; i < kMaxTop / 32; ++i) {
          id[i] = o.y >= 0 ? te.id[lane + 32 * i] : -1;
          const int vi = (id[i] + sh.off) / E - sh.v0;
          if (vi < 0 || vi >= sh.count) id[i] = -1;
          zk[i] = id[i] >= 0 ? to_f32(z[id[i]]) : 0.f;  // asked for while the gradient is being written
        }
        ok = warp_wait(&x.row_done[teach.i], teach.parity);
        if (!ok) break;
        const bool twice = x.twice[teach.i] != 0;
#pragma unroll
        for (int i = 0; i < kMaxTop / 32; ++i) {
          if (id[i] < 0) continue;
          const float p = twice ? mass_at(te.id, te.lp, t.K, id[i]) : expf(te.lp[lane + 32 * i]);
          const float q = ex2((zk[i] - o.top) * a.k) / o.sum;
          from_f32(static_cast<T*>(a.dlogits) + row.row * a.ld_d + id[i], o.c * fmaf(q, o.total, -p));
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&x.teacher_free[teach.i]);
        buf.next();
        teach.next();
      }
    }
  }
  if (!ok && lane == 0) record_device_error(&g_loss_error, kErrLossWaitTimeout);
  if (parts > 1) {  // no CTA leaves while another may still write to its shared memory
    tc::cluster_arrive();
    tc::cluster_wait();
  }
}

// ------------------------------------------------------------------------------------------- distillation
// Teacher entries are held in shared memory; a bit per element of the share marks the teacher's ids, so that the
// student's mass outside them is a sum of its own (one minus the mass inside would lose what is left when that is
// near one).  The gradient is written densely, then the entries at the ids are written over.  For few rows, short rows
// and more than 128 entries: 16 x 32000 bf16 with 32 entries 10 us with the sum of the losses, the latency of one row
// (teacher, statistics, merge, gradient one after another).  4096 x 32000: 64 entries 175 us, where the streaming kernel
// takes 118; 200 entries 259 us, with a rest class 206.
template <typename T, int NT, bool kTail, bool kGrad>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_kernel(LossRows a, DistillTerms t, int parts) {
  extern __shared__ float sm[];
  await_previous();
  const int K = t.K;
  float* tp = sm;                                // [K] teacher logits, then probabilities
  int* id = reinterpret_cast<int*>(sm + K);      // [K] ids, -1 where there is none
  __shared__ uint32_t mark[NT * kNV / 4];        // a byte per vector of a round, a bit per element
  __shared__ float mass;                         // the sum of p
  __shared__ int twice;                          // an id was given twice
  const int64_t r = blockIdx.x / unsigned(parts);
  const int rank = int(blockIdx.x % unsigned(parts));
  const Share<T> w(a, r, rank, parts);
  const int tid = int(threadIdx.x), lane = tid & 31;
  const bool first = rank == 0 && tid == 0;
  if (ld_index(t.ids, a.index_dtype, r * K) < 0) {  // the row counts for nothing (the same for the cluster)
    if (first) t.divergence[r] = 0.f, t.row_loss[r] = 0.f;
    if (kGrad) w.template zero<NT>(tid);
    return;
  }
  if (parts > 1) tc::cluster_arrive();
  uint4 v[kNV];
  auto load = [&](int at) {
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int vi = at + tid + i * NT;
      v[i] = vi < w.v1 ? w.load(vi) : make_uint4(Vec<T>::kFill, Vec<T>::kFill, Vec<T>::kFill, Vec<T>::kFill);
    }
  };
  load(w.v0);
  if (tid == 0) twice = 0;
  int valid = 0;
  for (int k = tid; k < K; k += NT) {
    const int64_t i = ld_index(t.ids, a.index_dtype, r * K + k);
    const bool ok = i >= 0 && i < w.V;
    if (i >= w.V) record_device_error(&g_loss_error, kErrSlotOutOfRange);
    id[k] = ok ? int(i) : -1;
    tp[k] = ok ? ld_as_f32(t.logits, t.dtype, r * K + k) : -INFINITY;
    valid |= ok;
  }
  const bool any = __syncthreads_or(valid) != 0;
  if (tid < 32) {  // the teacher's probabilities, by one warp while the others go on
    float tm = -INFINITY, sum = 0.f, ps = 0.f;
    if (!t.lse) {
      for (int k = lane; k < K; k += 32) tm = fmaxf(tm, tp[k]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, o));
      for (int k = lane; k < K; k += 32)
        if (id[k] >= 0) sum += ex2((tp[k] - tm) * a.k);
      sum = logf(warp_sum(sum));
    }
    for (int k = lane; k < K; k += 32) {
      const float lp = t.lse ? over_t_less(a, tp[k], -t.lse[r]) : over_t(a, tp[k] - tm, -sum);
      tp[k] = id[k] < 0 ? -INFINITY : lp;
      if (id[k] >= 0) ps += expf(lp);
    }
    ps = warp_sum(ps);
    if (lane == 0) mass = ps;
  }
  const int rounds = max(1, (w.v1 - w.v0 + NT * kNV - 1) / (NT * kNV));
  Apart st;  // without kTail: all of the row outside
  for (int q = 0; q < rounds; ++q) {
    const int at = w.v0 + q * NT * kNV;
    if (q > 0) {
      __syncthreads();
      load(at);
    }
#pragma unroll
    for (int i = 0; i < kNV / 4; ++i) mark[tid + i * NT] = 0u;
    __syncthreads();
    for (int k = tid; k < K; k += NT) {
      if (id[k] < 0) continue;
      const int vi = (id[k] + w.off) / Vec<T>::E - at;
      if (vi < 0 || vi >= NT * kNV || vi + at >= w.v1) continue;
      const uint32_t bit = 1u << (8 * (vi & 3) + (id[k] + w.off) % Vec<T>::E);
      if (atomicOr(&mark[vi >> 2], bit) & bit) twice = 1;
    }
    __syncthreads();
    if constexpr (kTail) {
      for (int k = tid; k < K; k += NT) {
        const int vi = (id[k] + w.off) / Vec<T>::E - at;
        if (id[k] < 0 || vi < 0 || vi >= NT * kNV || vi + at >= w.v1) continue;
        if (twice && first_of(id, k) != k) continue;  // by its place, not by which thread came first
        const float zk = to_f32(w.z[id[k]]), m = fmaxf(st.in.m, zk);
        rescale(st.in, m, a);
        st.in.s += zk == -INFINITY ? 0.f : ex2((zk - m) * a.k);
      }
      // the vectors without the ids' logits (their entries of the gradient are written over in any case)
#pragma unroll
      for (int i = 0; i < kNV; ++i) {
        const uint32_t bits = reinterpret_cast<const uint8_t*>(mark)[tid + i * NT];
        if (bits != 0) v[i] = mask_bits<T>(v[i], bits);
      }
    }
    add_vectors<T, kNV>(st.out, v, a);
  }
  if (parts > 1) tc::cluster_wait();
  st = merge_rows<NT>(st, a, rank, parts);
  const float ps = any ? mass : -1.f;
  const Rest rest = rest_of(a, kTail, ps, st);
  const float wt = t.weights ? t.weights[r] : t.scale ? *t.scale : mean_of_few(a, t.ids, K);
  if (rank == 0 && tid < 32) {
    float kl = 0.f;
    const float ls = logf(rest.sum);
    for (int k = lane; k < K; k += 32) {
      if (id[k] >= 0) kl = distill_term(a, kl, tp[k], to_f32(w.z[id[k]]), rest.m, ls);
    }
    kl = warp_sum(kl);
    if (lane == 0) write_distill_row(a, t, r, ps, wt, kl, rest, st, ls);
  }
  if constexpr (kGrad) {
    const RowCoef o = distill_coef(a, ps, wt, rest, st);
    if (o.y < 0) {
      w.template zero<NT>(tid);
      return;
    }
    for (int q = rounds - 1; q >= 0; --q) {
      if (q < rounds - 1) load(w.v0 + q * NT * kNV);
#pragma unroll
      for (int i = 0; i < kNV; ++i) {
        const int vi = w.v0 + q * NT * kNV + tid + i * NT;
        if (vi >= w.v1) break;
        float2 g[Vec<T>::E / 2];
        vector_grad<T, 1>(v[i], o.m, a.k, o.A, 0.f, g);
        w.store(vi, g);
      }
    }
    __syncthreads();  // the dense gradient is written: the ids' entries go over it
    for (int k = tid; k < K; k += NT) {
      if (id[k] < 0) continue;
      const int vi = (id[k] + w.off) / Vec<T>::E;
      if (vi < w.v0 || vi >= w.v1) continue;
      float P = expf(tp[k]);
      if (twice) {  // every one of them writes the sum
        P = 0.f;
        for (int i = 0; i < K; ++i)
          if (id[i] == id[k]) P += expf(tp[i]);
      }
      const float qk = ex2((to_f32(w.z[id[k]]) - o.top) * a.k) / o.sum;
      from_f32(w.dz + id[k], o.c * fmaf(qk, o.total, -P));
    }
  }
}

// -------------------------------------------------------------------------------------------- small kernels
constexpr int kSmall = 256;

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

// The two sums over rows, one CTA each (a fixed order): latency, 2 to 3 us after the kernel before them.
// scale = 1 / (rows that count): by their labels, or (by_sign) those whose first id is not negative
__global__ void __launch_bounds__(1024) live_scale_kernel(const void* __restrict__ labels, int index_dtype, int64_t n,
                                                          int64_t stride, bool by_sign, int64_t ignore_index, int64_t V,
                                                          float* __restrict__ scale) {
  await_previous();
  __shared__ double red[32];
  int64_t c = 0;
  for (int64_t r = threadIdx.x; r < n; r += 1024) {
    const int64_t y = ld_index(labels, index_dtype, r * stride);
    c += by_sign ? y >= 0 : counts(y, ignore_index, V);
  }
  const double live = block_sum_f64(double(c), red);
  if (threadIdx.x == 0) *scale = live > 0.0 ? float(1.0 / live) : 0.f;
}

// loss = factor * sum_r part[r], in a fixed order (one CTA)
__global__ void __launch_bounds__(1024) loss_sum_kernel(const float* part, int64_t n, double factor,
                                                        float* __restrict__ loss) {
  await_previous();
  __shared__ double red[32];
  double v = 0.0;
  for (int64_t r = threadIdx.x; r < n; r += 1024) v += double(part[r]);
  v = block_sum_f64(v, red);
  if (threadIdx.x == 0) *loss = float(v * factor);
}

// One CTA per pair (sequences 2p chosen, 2p + 1 rejected; half of the threads each): the log ratios of both, the pair's
// loss, and d loss / d logp of their tokens.  The CTA that is done last adds the pairs' losses, in the pairs' order.
// What bounds it is one chain of loads: offsets, labels, logits.  None of them is of the forward kernel's making, so a
// thread's first kAhead tokens are looked up while that one still runs, and only the statistics are waited for.
constexpr int kPairThreads = 512, kAhead = 4;
__global__ void __launch_bounds__(kPairThreads) pair_kernel(LossRows a, PairTerms t) {
  constexpr int kHalf = kPairThreads / 2, kHalfWarps = kHalf / 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ double red[kPairThreads / 32];
  __shared__ int live[kPairThreads / 32];
  const int64_t p = blockIdx.x;
  const int side = int(threadIdx.x) / kHalf, tid = int(threadIdx.x) % kHalf;
  int64_t lo = t.cu[2 * p + side], hi = t.cu[2 * p + side + 1];
  const bool outside = lo < 0 || hi > a.n || hi < lo;  // offsets out of range: the sequence counts as empty
  if (outside) lo = hi = 0;
  const double inv_t = 1.0 / a.temperature;
  // a token: whether it counts, and its logit less the reference's log-probability
  int count = 0;
  struct Token {
    double z, ref;
    bool use;
  };
  const auto token = [&](int64_t r) {
    Token k{0.0, 0.0, false};
    const int64_t y = ld_index(a.labels, a.index_dtype, r);
    if (!counts(y, a.ignore_index, a.V)) return k;  // (one outside the vocabulary is recorded by the forward kernel)
    ++count;
    k.use = true;
    k.z = double(ld_as_f32(a.logits, a.dtype, r * a.ld + y));
    k.ref = t.ref ? double(t.ref[r]) : 0.0;
    return k;
  };
  // from the row's statistics, and not from its log-probability in fp32: a log ratio is a sum of differences of near
  // values
  const auto ratio = [&](const Token& k, int64_t r) {
    return (k.z - double(a.stats[2 * r])) * inv_t - log(double(a.stats[2 * r + 1])) - k.ref;
  };
  Token ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int64_t r = lo + tid + i * kHalf;
    ahead[i] = r < hi ? token(r) : Token{0.0, 0.0, false};
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (outside && tid == 0) record_device_error(&g_loss_error, kErrSlotOutOfRange);
  double v = 0.0;
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (ahead[i].use) v += ratio(ahead[i], lo + tid + i * kHalf);
  for (int64_t r = lo + tid + kAhead * kHalf; r < hi; r += kHalf) {
    const Token k = token(r);
    if (k.use) v += ratio(k, r);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  count = __reduce_add_sync(0xffffffffu, count);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v, live[threadIdx.x >> 5] = count;
  __syncthreads();
  double sum[2], cnt[2];
  for (int i = 0; i < 2; ++i) {
    double sv = 0.0;
    int sc = 0;
    for (int w = 0; w < kHalfWarps; ++w) sv += red[i * kHalfWarps + w], sc += live[i * kHalfWarps + w];
    cnt[i] = t.normalise ? fmax(double(sc), 1.0) : 1.0;
    sum[i] = sv / cnt[i];
  }
  const double h = double(t.beta) * (sum[0] - sum[1]), eps = double(t.smoothing);
  const double e = exp(-fabs(h));  // sigmoid(h) = 1 / (1 + e^-h), without an overflow
  const double dh = (h < 0.0 ? e : 1.0) / (1.0 + e) - (1.0 - eps);
  const float c = float((side == 0 ? dh : -dh) * double(t.beta) / (double(t.pairs) * cnt[side]));
  for (int64_t r = lo + tid; r < hi; r += kHalf) t.coef[r] = c;
  if (threadIdx.x == 0) {
    const double l1p = log1p(e);  // log sigmoid(h) = min(h, 0) - log1p(e^-|h|)
    t.log_ratios[2 * p] = float(sum[0]);
    t.log_ratios[2 * p + 1] = float(sum[1]);
    t.pair_loss[p] = float(-((1.0 - eps) * (fmin(h, 0.0) - l1p) + eps * (fmin(-h, 0.0) - l1p)));
  }
  __shared__ bool last;
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(t.pairs_done, 1u) == unsigned(t.pairs - 1);
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  v = 0.0;
  for (int64_t q = threadIdx.x; q < t.pairs; q += kPairThreads) v += double(__ldcg(t.pair_loss + q));
  v = block_sum_f64(v, red);
  if (threadIdx.x == 0) *t.loss = float(v / double(t.pairs));
}

// x *= *scale; nothing is read or written where the scale is one, which is the common case (so the grid is small, and
// its CTAs take share after share of a row: a warp 256 vectors, or 256 threads 2048).  One read, one write, bound by
// memory: 8192 x 32000 bf16 in 165 us, 97 % of the measured copy rate.  A bf16 gradient is rounded a second time
// here (the upstream gradient is not known when it is formed): within 2^-7 of itself instead of 2^-8 where the scale is no
// power of two.
template <typename T, int NT>
__global__ void __launch_bounds__(kSmall) scale_kernel(LossRows a, const float* __restrict__ scale, int parts) {
  constexpr int kUnits = kSmall / NT;  // shares of a CTA
  const float f = *scale;
  if (f == 1.f) return;
  const int tid = int(threadIdx.x) % NT;
  for (int64_t u = int64_t(blockIdx.x) * kUnits + threadIdx.x / NT; u < a.n * parts; u += int64_t(gridDim.x) * kUnits) {
    const Share<T> w(a, u / parts, int(u % parts), parts);
    for (int at = w.v0 + tid; at < w.v1; at += NT * kNV) {
      uint4 v[kNV];
#pragma unroll
      for (int i = 0; i < kNV; ++i)
        if (const int vi = at + i * NT; vi < w.v1)  // (not through the read-only path: it is written here)
          v[i] = w.whole(vi) ? *reinterpret_cast<const uint4*>(w.dz + (vi * w.E - w.off))
                             : load_edge(w.z, vi * w.E - w.off, w.V);
#pragma unroll
      for (int i = 0; i < kNV; ++i) {
        if (at + i * NT >= w.v1) break;
        float2 g[Vec<T>::E / 2];
#pragma unroll
        for (int j = 0; j < Vec<T>::E / 2; ++j) g[j] = mul2(Vec<T>::minus(v[i], j, 0.f), make_float2(f, f));
        w.store(at + i * NT, g);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------- launches
// the most 16-byte vectors that a row reaches into
int64_t row_vectors(const LossRows& a) {
  const int64_t E = a.dtype == KDN_DTYPE_BF16 ? 8 : 4;
  const bool aligned = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && (a.ld % E == 0 || a.n == 1);
  return aligned ? (a.V + E - 1) / E : (a.V + 2 * E - 2) / E;
}
LossShape shape_of(const LossRows& a) { return {a.n, row_vectors(a), current_sm_count()}; }

// One launch.  `after`: the previous one on the stream is of the same call, and this one's start may overlap its end.
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), int64_t grid, int threads, int cluster, size_t smem, bool after,
                   cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2] = {};
  cfg.attrs = attrs;
  if (after) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attrs[cfg.numAttrs].val.clusterDim.x = unsigned(cluster);
    attrs[cfg.numAttrs].val.clusterDim.y = attrs[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ... of a kernel with `parts` CTAs a row as its last argument
template <typename K, typename... Args>
cudaError_t launch_rows(K kernel, int64_t rows, Split s, bool cluster, size_t smem, bool after, cudaStream_t stream,
                        Args... args) {
  if (s.threads == 32) rows = (rows + 3) / 4, s.threads = 128;
  return launch(kernel, rows * s.parts, s.threads, cluster ? s.parts : 1, smem, after, stream, args..., s.parts);
}

// f(T of the logits, threads) as types
template <typename F>
cudaError_t dispatch(const LossRows& a, Split s, F f) {
  using std::integral_constant;
  if (a.dtype == KDN_DTYPE_BF16) {
    if (s.threads == 32) return f(__nv_bfloat16{}, integral_constant<int, 32>{});
    if (s.threads == 128) return f(__nv_bfloat16{}, integral_constant<int, 128>{});
    if (s.threads == 256) return f(__nv_bfloat16{}, integral_constant<int, 256>{});
    return f(__nv_bfloat16{}, integral_constant<int, 512>{});
  }
  if (s.threads == 32) return f(float{}, integral_constant<int, 32>{});
  if (s.threads == 128) return f(float{}, integral_constant<int, 128>{});
  if (s.threads == 256) return f(float{}, integral_constant<int, 256>{});
  return f(float{}, integral_constant<int, 512>{});
}

template <typename Terms, typename K>
cudaError_t launch_stream(K kernel, const LossRows& a, const Terms& t, Stream s, bool after, cudaStream_t stream) {
  using S = Streaming<Terms>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kRingBytes));
      e != cudaSuccess)
    return e;
  const int64_t group = group_rows(shape_of(a), s);
  return launch_rows(kernel, (a.n + group - 1) / group, Split{S::kThreads, s.parts}, true, kRingBytes, after,
                     stream, a, t, int(group), s.per);
}

cudaError_t launch_logp(const LossRows& a, const PolicyTerms& t, Stream st, bool after, cudaStream_t stream) {
  if (st.parts > 0) {
    const auto go = [&](auto z) {
      using T = decltype(z);
      if (!a.dlogits) return launch_stream(loss_stream_kernel<T, PolicyTerms, 0>, a, t, st, after, stream);
      return t.entropy_coef != 0.f ? launch_stream(loss_stream_kernel<T, PolicyTerms, 2>, a, t, st, after, stream)
                                   : launch_stream(loss_stream_kernel<T, PolicyTerms, 1>, a, t, st, after, stream);
    };
    return a.dtype == KDN_DTYPE_BF16 ? go(__nv_bfloat16{}) : go(float{});
  }
  const Split s = t.row_loss ? choose_split(shape_of(a)) : choose_scan_split(shape_of(a));
  return dispatch(a, s, [&](auto z, auto nt) {
    using T = decltype(z);
    constexpr int NT = decltype(nt)::value;
    const auto go = [&](auto kernel) { return launch_rows(kernel, a.n, s, true, 0, after, stream, a, t); };
    if (!t.row_loss) return go(logp_kernel<T, NT, false, 0>);
    if (!a.dlogits) return go(logp_kernel<T, NT, true, 0>);
    return t.entropy_coef != 0.f ? go(logp_kernel<T, NT, true, 2>) : go(logp_kernel<T, NT, true, 1>);
  });
}

cudaError_t launch_distill(const LossRows& a, const DistillTerms& t, Stream st, bool after, cudaStream_t stream) {
  if (st.parts > 0) {
    const auto go = [&](auto z) {
      using T = decltype(z);
      return a.dlogits ? launch_stream(loss_stream_kernel<T, DistillTerms, 1>, a, t, st, after, stream)
                       : launch_stream(loss_stream_kernel<T, DistillTerms, 0>, a, t, st, after, stream);
    };
    return a.dtype == KDN_DTYPE_BF16 ? go(__nv_bfloat16{}) : go(float{});
  }
  Split s = choose_split(shape_of(a));
  s.threads = std::max(s.threads, 128);
  return dispatch(a, s, [&](auto z, auto nt) {
    using T = decltype(z);
    constexpr int NT = decltype(nt)::value < 128 ? 128 : decltype(nt)::value;
    const auto go = [&](auto kernel) {
      return launch_rows(kernel, a.n, s, true, size_t(t.K) * 8, after, stream, a, t);
    };
    if (t.lse) return a.dlogits ? go(distill_kernel<T, NT, true, true>) : go(distill_kernel<T, NT, true, false>);
    return a.dlogits ? go(distill_kernel<T, NT, false, true>) : go(distill_kernel<T, NT, false, false>);
  });
}

}  // namespace

cudaError_t launch_token_logprobs(const LossRows& a, cudaStream_t stream) {
  return launch_logp(a, PolicyTerms{}, Stream{0, 0}, false, stream);
}

cudaError_t launch_token_logprobs_backward(const LossRows& a, const float* dlogps, bool after, cudaStream_t stream) {
  // Nothing ties a row's CTAs together: at most two rounds of 256 threads each.  B200, bf16, 8192 x 32000: 165 us with
  // 256 threads and one CTA a row, 180 with two CTAs, 173 with four of 128 threads, 190 with 512 threads and 4 vectors.
  const int64_t vecs = row_vectors(a);
  Split s{vecs <= 512 ? 32 : vecs <= 128 * kNV ? 128 : 256, 1};
  while (vecs > 4096 * int64_t(s.parts)) s.parts *= 2;
  return dispatch(a, s, [&](auto z, auto nt) {
    return launch_rows(logp_backward_kernel<decltype(z), decltype(nt)::value>, a.n, s, false, 0, after, stream, a,
                       dlogps);
  });
}

cudaError_t launch_policy_loss(const LossRows& a, PolicyTerms t, float* loss, cudaStream_t stream) {
  const Stream st = choose_stream(shape_of(a));
  const bool mean = !t.weights && !counts_rows_itself(shape_of(a), st);
  if (!mean) t.scale = nullptr;
  if (mean) {
    const cudaError_t e = launch(live_scale_kernel, 1, 1024, 1, 0, false, stream, a.labels, a.index_dtype, a.n, 1,
                                 false, a.ignore_index, a.V, const_cast<float*>(t.scale));
    if (e != cudaSuccess) return e;
  }
  if (cudaError_t e = launch_logp(a, t, st, mean, stream); e != cudaSuccess) return e;
  return launch(loss_sum_kernel, 1, 1024, 1, 0, true, stream, t.row_loss, a.n, 1.0, loss);
}

cudaError_t launch_preference_loss(const LossRows& a, const PairTerms& t, cudaStream_t stream) {
  LossRows f = a;  // forward: log-probabilities and statistics only
  f.dlogits = nullptr;
  f.coef_zero = t.coef;
  f.pairs_done = t.pairs_done;
  cudaError_t e = a.n > 0 ? launch_logp(f, PolicyTerms{}, Stream{0, 0}, false, stream)
                          : cudaMemsetAsync(t.pairs_done, 0, sizeof(unsigned), stream);
  if (e != cudaSuccess) return e;
  e = launch(pair_kernel, t.pairs, kPairThreads, 1, 0, a.n > 0, stream, a, t);
  if (e != cudaSuccess || !a.dlogits || a.n == 0) return e;
  return launch_token_logprobs_backward(a, t.coef, true, stream);
}

cudaError_t launch_distillation_loss(const LossRows& a, DistillTerms t, float* loss, cudaStream_t stream) {
  const Stream st = t.K <= kMaxTop ? choose_stream(shape_of(a)) : Stream{0, 0};
  const bool mean = !t.weights && !counts_rows_itself(shape_of(a), st);
  if (!mean) t.scale = nullptr;
  if (mean) {
    const cudaError_t e = launch(live_scale_kernel, 1, 1024, 1, 0, false, stream, t.ids, a.index_dtype, a.n, t.K, true,
                                 0, a.V, const_cast<float*>(t.scale));
    if (e != cudaSuccess) return e;
  }
  if (cudaError_t e = launch_distill(a, t, st, mean, stream); e != cudaSuccess) return e;
  return launch(loss_sum_kernel, 1, 1024, 1, 0, true, stream, t.row_loss, a.n, 1.0, loss);
}

cudaError_t launch_scale_rows(void* x, int dtype, int64_t ld, int64_t n, int64_t V, const float* scale,
                              cudaStream_t stream) {
  LossRows a = {};
  a.logits = a.dlogits = x;
  a.dtype = dtype;
  a.ld = a.ld_d = ld;
  a.n = n;
  a.V = V;
  // a warp a share for short rows: 16384 x 1000 bf16 10 us, 35 with 256 threads
  const int64_t vecs = row_vectors(a), threads = vecs <= 512 ? 32 : kSmall;
  const int parts = int((vecs + threads * kNV - 1) / (threads * kNV));
  const int64_t units = kSmall / threads;
  const int64_t grid = std::min<int64_t>((n * parts + units - 1) / units, 8 * current_sm_count());
  const auto go = [&](auto kernel) { return launch(kernel, grid, kSmall, 1, 0, false, stream, a, scale, parts); };
  if (dtype == KDN_DTYPE_BF16)
    return threads == 32 ? go(scale_kernel<__nv_bfloat16, 32>) : go(scale_kernel<__nv_bfloat16, kSmall>);
  return threads == 32 ? go(scale_kernel<float, 32>) : go(scale_kernel<float, kSmall>);
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
