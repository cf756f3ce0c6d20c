// token_loss.cu -- losses over LM-head logits other than cross-entropy: token log probabilities and
// their gradient, the preference loss on pairs of answers, and the clipped policy loss.
//
// For a row x of V logits with target t:  m = max x,  s = sum exp(x - m),  logp = (x_t - m) - log s,
// d logp / d x_c = [c = t] - exp(x_c - m) / s.  The pair (m, s) is what the backward gets: beside a
// logit of the type's lowest value a log-sum-exp could not hold log s.  A target outside [0, V) marks
// a row without a token: logp 0, gradient 0.  Logits of -inf have probability 0; a row of nothing but
// -inf has m = logp = -inf, s = 0 and gradient 0.  NaN and +inf propagate within their row, unless the row's weight (or upstream
// gradient) is 0: such a row's gradient is 0 whatever it holds.
//
// Sums are fp32 with a running maximum, the final logarithm and all per-row scalars fp64 (a few
// operations per row), so that logp carries one rounding.
//
// Bound: DRAM.  One block per row.
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>

#include "mt_api.h"
#include "vec_io.cuh"

namespace mt {
namespace {

constexpr int kThreads = 512;

// Running maximum and sum of exponentials relative to it.  m = -inf only while nothing above -inf
// was seen; a NaN leaves m alone and turns s into NaN.
struct Stat {
  float m, s;
};

__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ Stat merge(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m), z = finite_or_zero(m);
  return {m, a.s * __expf(a.m - z) + b.s * __expf(b.m - z)};
}

template <class T>
__device__ __forceinline__ Stat row_stat(const T* __restrict__ x, int V) {
  Stat st{-INFINITY, 0.f};
  const int nvec = V / 8;
  for (int c = threadIdx.x; c < nvec; c += kThreads) {
    float f[8];
    load8(x + c * 8, f);
    float m = f[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, f[j]);
    m = isnan(m) ? -INFINITY : m;  // all eight NaN
    const float z = finite_or_zero(m);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += __expf(f[j] - z);
    st = merge(st, {m, s});
  }
  for (int c = nvec * 8 + threadIdx.x; c < V; c += kThreads) {
    const float f = to_f32(x[c]);
    st = merge(st, {isnan(f) ? -INFINITY : f, isnan(f) ? f : (f == -INFINITY ? 0.f : __expf(f - f))});
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st = merge(st, {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o)});
  __shared__ Stat warp_stat[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) warp_stat[warp] = st;
  __syncthreads();
  st = lane < kThreads / 32 ? warp_stat[lane] : Stat{-INFINITY, 0.f};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st = merge(st, {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o)});
  return st;
}

__device__ __forceinline__ bool is_empty(Stat st) { return st.m == -INFINITY && st.s == 0.f; }

template <class T>
__device__ __forceinline__ double logp_of(const T* x, int64_t t, int V, Stat st) {
  if (t < 0 || t >= V) return 0.0;
  if (is_empty(st)) return -INFINITY;
  return ((double)to_f32(x[t]) - (double)st.m) - log((double)st.s);
}

// out = coef ([c = t] - exp(x_c - m) / s); with coef 0 or an empty row, zeros.
template <class T>
__device__ __forceinline__ void row_grad(const T* x, T* out, int V, int t, float coef, Stat st) {
  const bool zero = coef == 0.f || is_empty(st);
  const float shift = finite_or_zero(st.m), scale = 1.0f / st.s;
  const int nvec = V / 8;
  for (int c = threadIdx.x; c < nvec; c += kThreads) {
    float f[8];
    load8(x + c * 8, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float p = __expf(f[j] - shift) * scale;
      f[j] = zero ? 0.f : ((c * 8 + j == t ? 1.f : 0.f) - p) * coef;
    }
    store8(out + c * 8, f);
  }
  for (int c = nvec * 8 + threadIdx.x; c < V; c += kThreads) {
    const float p = __expf(to_f32(x[c]) - shift) * scale;
    out[c] = from_f32<T>(zero ? 0.f : ((c == t ? 1.f : 0.f) - p) * coef);
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
    logprobs_kernel(const T* __restrict__ logits, long ld, const int64_t* __restrict__ targets,
                    float* __restrict__ logps, float2* __restrict__ stats, int V) {
  const long row = blockIdx.x;
  const T* x = logits + row * ld;
  const Stat st = row_stat(x, V);
  if (threadIdx.x == 0) {
    stats[row] = make_float2(st.m, st.s);
    logps[row] = (float)logp_of(x, targets[row], V, st);
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
    logprobs_bwd_kernel(const T* logits, long ld, const int64_t* __restrict__ targets, const float2* __restrict__ stats,
                        const float* __restrict__ dlogps, T* out, long ldo, int V) {
  const long row = blockIdx.x;
  const int64_t t = targets[row];
  const float2 st = stats[row];
  const bool valid = t >= 0 && t < V;
  row_grad(logits + row * ld, out + row * ldo, V, (int)t, valid ? dlogps[row] : 0.f, Stat{st.x, st.y});
}

// Loss and d loss / d logp of one token.
__device__ __forceinline__ void policy_terms(const PolicyArgs& a, long row, double logp, bool valid, float* loss,
                                             float* coef) {
  const float w = a.weights ? a.weights[row] : 1.f;
  if (!valid || w == 0.f) {
    *loss = *coef = 0.f;
    return;
  }
  const double adv = a.advantages[row];
  const double ratio = exp(logp - (double)a.old_logps[row]);
  const double free_ = -adv * ratio;
  const double bound = -adv * fmin(fmax(ratio, 1.0 - a.clip_low), 1.0 + a.clip_high);
  double l = fmax(free_, bound), d = free_ >= bound ? free_ : 0.0;
  if (isnan(free_)) l = d = free_;
  if (a.ref_logps) {
    const double back = (double)a.ref_logps[row] - logp, e = expm1(back);
    l += a.kl_coef * (e - back);
    d -= a.kl_coef * e;
  }
  *loss = (float)(w * l);
  *coef = (float)((double)w * d * a.grad_scale);
}

template <class T>
__global__ void __launch_bounds__(kThreads) policy_kernel(PolicyArgs a) {
  __shared__ float sh_coef;
  const long row = blockIdx.x;
  const T* x = (const T*)a.logits + row * a.ld;
  const int64_t t = a.targets[row];
  const bool valid = t >= 0 && t < a.V;
  const Stat st = row_stat(x, a.V);
  if (threadIdx.x == 0) {
    const double logp = logp_of(x, t, a.V, st);
    a.logps[row] = (float)logp;
    float loss, coef;
    policy_terms(a, row, logp, valid, &loss, &coef);
    a.losses[row] = loss;
    sh_coef = coef;
  }
  __syncthreads();
  row_grad(x, (T*)a.out + row * a.ldo, a.V, (int)t, sh_coef, st);
}

// One block per pair (rows 2i: preferred, 2i + 1: rejected).
constexpr int kPairThreads = 256;

__device__ __forceinline__ double block_sum(double v, double* slots) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < kPairThreads / 32; ++w) s += slots[w];
  return s;
}

__global__ void __launch_bounds__(kPairThreads) preference_kernel(PreferenceArgs a) {
  __shared__ double slots[kPairThreads / 32];
  double r[2], count[2];
  for (int k = 0; k < 2; ++k) {
    const long base = ((long)blockIdx.x * 2 + k) * a.S;
    double s = 0.0, n = 0.0;
    for (int i = threadIdx.x; i < a.S; i += kPairThreads)
      if (a.mask[base + i]) {
        s += (double)a.logps[base + i] - (double)a.ref_logps[base + i];
        n += 1.0;
      }
    r[k] = block_sum(s, slots);
    count[k] = fmax(block_sum(n, slots), 1.0);
  }
  const double beta = a.beta, eps = a.label_smoothing;
  double loss, up[2];
  if (a.squared) {
    const double gap = r[0] / count[0] - r[1] / count[1] - 0.5 / beta;
    loss = gap * gap;
    up[0] = 2.0 * gap / count[0];
    up[1] = -2.0 * gap / count[1];
  } else {
    const double h = beta * (r[0] - r[1]);
    const double tail = log1p(exp(-fabs(h)));
    loss = (1.0 - eps) * (tail + fmax(-h, 0.0)) + eps * (tail + fmax(h, 0.0));
    up[0] = beta * (eps - 1.0 / (1.0 + exp(h)));
    up[1] = -up[0];
  }
  if (threadIdx.x == 0) {
    a.losses[blockIdx.x] = (float)loss;
    a.rewards[blockIdx.x * 2] = (float)(beta * r[0]);
    a.rewards[blockIdx.x * 2 + 1] = (float)(beta * r[1]);
  }
  for (int k = 0; k < 2; ++k) {
    const long base = ((long)blockIdx.x * 2 + k) * a.S;
    const float g = (float)(up[k] * a.grad_scale);
    for (int i = threadIdx.x; i < a.S; i += kPairThreads) a.dlogps[base + i] = a.mask[base + i] ? g : 0.f;
  }
}

}  // namespace

int token_logprobs(const void* logits, long ld, int dtype, const int64_t* targets, float* logps, float* stats, int rows,
                   int V, cudaStream_t s) {
  if (ld % 8) return -1;
  if (rows == 0) return 0;
  return with_dtype(dtype, [&](auto v) {
    using T = decltype(v);
    logprobs_kernel<<<rows, kThreads, 0, s>>>((const T*)logits, ld, targets, logps, (float2*)stats, V);
    return (int)cudaGetLastError();
  });
}

int token_logprobs_bwd(const void* logits, long ld, int dtype, const int64_t* targets, const float* stats,
                       const float* dlogps, void* out, long ldo, int rows, int V, cudaStream_t s) {
  if (ld % 8 || ldo % 8) return -1;
  if (rows == 0) return 0;
  return with_dtype(dtype, [&](auto v) {
    using T = decltype(v);
    logprobs_bwd_kernel<<<rows, kThreads, 0, s>>>((const T*)logits, ld, targets, (const float2*)stats, dlogps, (T*)out, ldo, V);
    return (int)cudaGetLastError();
  });
}

int policy_loss(const PolicyArgs& a, cudaStream_t s) {
  if (a.ld % 8 || a.ldo % 8) return -1;
  if (a.rows == 0) return 0;
  return with_dtype(a.dtype, [&](auto v) {
    policy_kernel<decltype(v)><<<a.rows, kThreads, 0, s>>>(a);
    return (int)cudaGetLastError();
  });
}

int preference_loss(const PreferenceArgs& a, cudaStream_t s) {
  if (a.pairs == 0) return 0;
  preference_kernel<<<a.pairs, kPairThreads, 0, s>>>(a);
  return (int)cudaGetLastError();
}

}  // namespace mt
