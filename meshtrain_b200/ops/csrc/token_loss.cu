// token_loss.cu -- losses over LM-head logits other than cross-entropy: token log probabilities and
// their gradient, the preference loss on pairs of answers, and the clipped policy loss.
//
// For a row x of V logits with target t:  m = max x,  s = sum exp(x - m),  logp = (x_t - m) - log s,
// d logp / d x_c = [c = t] - exp(x_c - m) / s.  The pair (m, s) is what the backward gets: beside a
// logit of the type's lowest value a log-sum-exp could not hold log s.  A target outside [0, V) marks
// a row without a token: logp 0, gradient 0.  Logits of -inf have probability 0; a row of nothing but
// -inf has m = logp = -inf, s = 0 and gradient 0.  NaN and +inf propagate within their row, unless the
// row's weight (or upstream gradient) is 0: such a row's gradient is 0 whatever it holds.  An infinite
// coefficient makes every entry ([c = t] - p_c) times that infinity.
//
// Sums are fp32; logp is formed in fp64 from the fp32 maximum and sum, so that it carries one rounding.
// Exponentials are ex2 of (x - m) log2(e) with the constant in two parts: with one fp32 constant every
// term is off by 1.3e-8 |x - m| to the same side, and ex2.approx's own results are low by 5e-8 on
// average; both would add up over the tokens of an answer (see kEx2Low).
//
// Bound: DRAM, one read of the logits and (for a gradient) one write.  Three layouts, by width and rows:
//   row_kernel: a team of threads (a warp, 4 warps, 16 warps, or a cluster of 2, 4 or 8 blocks of 16
//     warps) holds a row in registers, 32 logits per thread.  Narrow rows, and few rows of any width,
//     which a cluster splits.
//   stream_logprobs_kernel: many wide rows, statistics only.  4096 x 50257 bf16: 72 us, 5.7 TB/s (87% of
//     the copy rate); 4096 x 128256: 166 us, 6.3 TB/s.
//   stream_policy_kernel: many wide rows, statistics and gradient from one reading.  8192 x 50257 bf16:
//     304 us, 5.4 TB/s (83%); 4096 x 128256: 413 us, 5.1 TB/s (78%; a tenth of such a row is read again,
//     from L2).  It computes two exponentials per logit, on a unit that does 16 per SM and clock, for
//     60% of its time, and waits twice per row for the row's statistic.
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mt_api.h"
#include "vec_io.cuh"

namespace mt {
namespace {

// Maximum and sum of exponentials relative to it.  m = -inf only while nothing above -inf was seen; a
// NaN leaves m alone and turns s into NaN.
struct Stat {
  float m, s;
};

__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ bool is_empty(Stat st) { return st.m == -INFINITY && st.s == 0.f; }

// ex2.approx.ftz averages 5.05e-8 below 2^t for t in [-20, -1] and 2.9e-8 in [-1, 0] (measured on B200 at
// random arguments).  log2(1 + 4.1e-8), added to the argument ahead of its last rounding, takes that out:
// sums of 1024 to 128256 terms are within 1e-8 on average with it, up to 1.3e-7 low without.
constexpr float kEx2Low = 5.9e-8f;
constexpr float kLog2eHi = 1.44269502162933349609375f, kLog2eLo = 1.92596303e-8f;  // their sum is log2(e) to 2^-49

// The two parts as packed pairs, held in registers: as literals they would be moved there again
// before every packed instruction.
struct Log2e {
  uint64_t hi, lo, low;
  __device__ __forceinline__ Log2e() {
    asm volatile("mov.b64 %0, {%1, %1};" : "=l"(low) : "f"(kEx2Low));
    asm volatile("mov.b64 %0, {%1, %1};" : "=l"(hi) : "f"(kLog2eHi));
    asm volatile("mov.b64 %0, {%1, %1};" : "=l"(lo) : "f"(kLog2eLo));
  }
};

// The eight x - m of a vector; the 16-bit types' subtraction reads them in place (one instruction for
// the conversion and the difference).
__device__ __forceinline__ void diffs(const Raw8<float>& r, float m, float* d) {
  unpack8(r, d);
#pragma unroll
  for (int j = 0; j < 8; ++j) d[j] -= m;
}
__device__ __forceinline__ void diffs(const Raw8<__nv_bfloat16>& r, float m, float* d) {
  const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tsub.f32.bf16 %0, a, %3;\n\tsub.f32.bf16 %1, b, %3;\n\t}"
        : "=f"(d[2 * j]), "=f"(d[2 * j + 1])
        : "r"(w[j]), "f"(m));
}
__device__ __forceinline__ void diffs(const Raw8<__half>& r, float m, float* d) {
  const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tsub.f32.f16 %0, a, %3;\n\tsub.f32.f16 %1, b, %3;\n\t}"
        : "=f"(d[2 * j]), "=f"(d[2 * j + 1])
        : "r"(w[j]), "f"(m));
}

// e^d for two values (0 for results below 2^-126).
__device__ __forceinline__ void exp2_of(const Log2e& l, float d0, float d1, float* e) {
  const uint64_t d = f2pack(d0, d1);
  const uint64_t t = fma_f32x2(d, l.hi, fma_f32x2(d, l.lo, l.low));
  float t0, t1;
  f2unpack(t, t0, t1);
  e[0] = ex2_approx(t0);
  e[1] = ex2_approx(t1);
}
__device__ __forceinline__ float exp_diff(float x, float m) {
  const float d = x - m;
  return ex2_approx(fmaf(d, kLog2eHi, fmaf(d, kLog2eLo, kEx2Low)));
}

__device__ __forceinline__ float warp_max(float v) {  // NaN is ignored
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// log s in fp64 from an fp32 logarithm of the part in [0.75, 1.5), whose error is below 3e-8.
__device__ __forceinline__ double log_f64(float s) {
  if (!(s > 0.f && s < INFINITY)) return log((double)s);
  const int k = (__float_as_int(s) - 0x3f400000) >> 23;
  const float f = __int_as_float(__float_as_int(s) - (k << 23));
  return (double)k * 0.69314718055994530942 + (double)logf(f);
}

// Log probability of a target whose logit is xt; `valid`: the target is one.
__device__ __forceinline__ double logp_of(float xt, bool valid, Stat st) {
  if (!valid) return 0.0;
  if (is_empty(st)) return -INFINITY;
  return ((double)xt - (double)st.m) - log_f64(st.s);
}

// What a row's loss needs besides its logits, loaded ahead.
struct RowInputs {
  int64_t t;
  float xt, w, adv, old, ref;
};

// Loss and d loss / d logp of one token.  The exponentials of the ratio and of the KL term are fp32
// (1e-7 of their value); their arguments are differences taken in fp64.  Of what overflows, A rho is 0 where
// A is, and exp(d) - d - 1 is infinite.
__device__ __forceinline__ void policy_terms(const PolicyArgs& a, const RowInputs& in, double logp, bool valid,
                                             float* loss, float* coef) {
  *loss = *coef = 0.f;
  if (!valid || in.w == 0.f) return;
  const float ratio = expf((float)(logp - (double)in.old));
  const float lo = (float)(1.0 - a.clip_low), hi = (float)(1.0 + a.clip_high);
  const float free_ = in.adv == 0.f && ratio == INFINITY ? 0.f : -in.adv * ratio;
  const float bound = -in.adv * fminf(fmaxf(ratio, lo), hi);
  float l = fmaxf(free_, bound), d = free_ >= bound ? free_ : 0.f;
  if (isnan(free_)) l = d = free_;
  if (a.ref_logps) {
    const float back = (float)((double)in.ref - logp), e = expm1f(back), kl = (float)a.kl_coef;
    l += kl * (e == INFINITY ? e : e - back);
    d -= kl * e;
  }
  *loss = in.w * l;
  *coef = (float)((double)(in.w * d) * a.grad_scale);
}

struct RowArgs {
  PolicyArgs p;   // logits, targets, per-row inputs and outputs
  float2* stats;  // log probabilities only: (m, s)
  int rows;
  int slice;  // columns of one block of a cluster, a multiple of 8
};

template <class T, bool POLICY>
__device__ __forceinline__ RowInputs row_inputs(const RowArgs& a, long row) {
  RowInputs in{};
  in.t = a.p.targets[row];
  if (in.t >= 0 && in.t < a.p.V) in.xt = to_f32(((const T*)a.p.logits)[row * a.p.ld + in.t]);
  if (POLICY) {
    in.w = a.p.weights ? a.p.weights[row] : 1.f;
    in.adv = a.p.advantages[row];
    in.old = a.p.old_logps[row];
    if (a.p.ref_logps) in.ref = a.p.ref_logps[row];
  }
  return in;
}

// Writes a row's per-row outputs and returns the coefficient of its gradient.
template <bool POLICY>
__device__ __forceinline__ float finish_row(const RowArgs& a, long row, const RowInputs& in, Stat st, bool writer) {
  const bool valid = in.t >= 0 && in.t < a.p.V;
  const double logp = logp_of(in.xt, valid, st);
  float loss = 0.f, coef = 0.f;
  if (POLICY) policy_terms(a.p, in, logp, valid, &loss, &coef);
  if (writer) {
    a.p.logps[row] = (float)logp;
    if (POLICY)
      a.p.losses[row] = loss;
    else
      a.stats[row] = make_float2(st.m, st.s);
  }
  return is_empty(st) ? 0.f : coef;
}

constexpr int kVecs = 4;  // vectors of 8 logits per thread

// Asynchronous copy of `bytes` (0 .. 16) of global memory into 16 bytes of shared memory, the rest zero.
__device__ __forceinline__ void copy_async16(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Largest of N vectors' values; NaN is ignored (-inf or NaN if there is nothing else).
template <int N>
__device__ __forceinline__ float max_of(const Raw8<float>* r) {
  float m = -INFINITY;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float f[8];
    unpack8(r[u], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, f[j]);
  }
  return m;
}
template <int N, class H2>
__device__ __forceinline__ H2 max_of_pairs(const H2* h) {
  H2 m = h[0];
#pragma unroll
  for (int i = 1; i < 4 * N; ++i) m = __hmax2(m, h[i]);
  return m;
}
template <int N>
__device__ __forceinline__ float max_of(const Raw8<__nv_bfloat16>* r) {
  const float2 f = __bfloat1622float2(max_of_pairs<N>(reinterpret_cast<const __nv_bfloat162*>(r)));
  return fmaxf(f.x, f.y);
}
template <int N>
__device__ __forceinline__ float max_of(const Raw8<__half>* r) {
  const float2 f = __half22float2(max_of_pairs<N>(reinterpret_cast<const __half2*>(r)));
  return fmaxf(f.x, f.y);
}

// Adds N vectors to a running statistic.
template <int N, class T>
__device__ __forceinline__ void add_vectors(const Log2e& l, Stat& st, const Raw8<T>* raw) {
  const float m = fmaxf(st.m, max_of<N>(raw));
  const float z = finite_or_zero(m);
  uint64_t sum = 0;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float d[8];
    diffs(raw[u], z, d);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float e[2];
      exp2_of(l, d[j], d[j + 1], e);
      sum = add_f32x2(sum, f2pack(e[0], e[1]));
    }
  }
  float s0, s1;
  f2unpack(sum, s0, s1);
  st = {m, st.s * expf(st.m - z) + (s0 + s1)};
}

// What a row's gradient needs: coef ([c = target] - e^(x - m) / s) = e^(x - m) f + [c = target] coef.
struct RowGrad {
  float z, f, coef;
  int target;
  __device__ __forceinline__ RowGrad(Stat st, float c, int t)
      : z(finite_or_zero(st.m)), f(-c / st.s), coef(c), target(t) {}

  // The target's own entry; s is the row's sum.  Beside an infinite coefficient (a ratio past the type's range, a
  // KL term at probability 0) the two parts would be infinities of either sign, so it is multiplied out there.
  __device__ __forceinline__ float at_target(float x, float s) const {
    const float e = exp_diff(x, z);
    return isinf(coef) ? coef * (1.f - e / s) : fmaf(e, f, coef);
  }
  __device__ __forceinline__ float elsewhere(float x) const { return coef == 0.f ? 0.f : exp_diff(x, z) * f; }
  // The gradient of a vector that does not hold the target.  16-bit results are rounded to 11 bits or
  // fewer, so the low part of log2(e), which changes 1e-8 |x - m| of them, is left out there.
  template <class T>
  __device__ __forceinline__ void plain(const Log2e& l, Raw8<T>& r) const {
    float g[8];
    diffs(r, z, g);
    const uint64_t f2 = f2pack(f, f);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float e[2];
      if constexpr (sizeof(T) == 2) {
        f2unpack(mul_f32x2(f2pack(g[j], g[j + 1]), l.hi), e[0], e[1]);
        e[0] = ex2_approx(e[0]);
        e[1] = ex2_approx(e[1]);
      } else {
        exp2_of(l, g[j], g[j + 1], e);
      }
      f2unpack(mul_f32x2(f2pack(e[0], e[1]), f2), g[j], g[j + 1]);
    }
    pack8(g, r);
  }
  // The gradient of any vector, at column c, with the target's entry given; zeros in a masked row, whatever it holds.
  template <class T>
  __device__ __forceinline__ void vector(const Log2e& l, Raw8<T>& r, int c, float entry) const {
    if (coef == 0.f) {
#pragma unroll
      for (int q = 0; q < (int)sizeof(Raw8<T>) / 16; ++q) r.q[q] = make_uint4(0, 0, 0, 0);
    } else if ((unsigned)(target - c) < 8u) {
      float g[8];
      unpack8(r, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = c + j == target ? entry : elsewhere(g[j]);
      pack8(g, r);
    } else {
      plain(l, r);
    }
  }
};

// WARPS per block and team (1: every warp of a 256-thread block is a team of its own), CL blocks of a
// cluster per row.  Dynamic shared memory: kVecs vectors per thread.
template <class T, int WARPS, int CL, bool POLICY>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : WARPS * 32, WARPS == 1 ? 4 : 32 / WARPS) row_kernel(RowArgs a) {
  constexpr int TEAM = WARPS * 32;
  constexpr int BLOCK = WARPS == 1 ? 256 : TEAM;
  extern __shared__ uint4 stage_mem[];
  __shared__ float2 pairs[2][WARPS * CL];  // of all the cluster's warps, for even and odd turns
  __shared__ float sh_coef, sh_entry;
  __shared__ int sh_target;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tid = WARPS == 1 ? lane : threadIdx.x;  // within the block's share of the team
  const int rank = CL > 1 ? (int)cluster_ctarank() : 0;
  const int c0 = rank * a.slice;
  const int cols = min(a.slice, a.p.V - c0);  // may be <= 0 in the last blocks of a cluster
  const int step = WARPS == 1 ? gridDim.x * (BLOCK / 32) : gridDim.x / CL;
  long row = WARPS == 1 ? (long)blockIdx.x * (BLOCK / 32) + warp : blockIdx.x / CL;
  // this thread's slot of vector k: [k][half][thread], so that a warp's accesses are contiguous
  constexpr int Q = sizeof(Raw8<T>) / 16;
  uint4* slot = stage_mem + threadIdx.x;

  auto fetch = [&](long r) {
    const T* x = (const T*)a.p.logits + r * a.p.ld + c0;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int c = (k * TEAM + tid) * 8;
      if (c < cols) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const int have = min(16, max(0, (cols - c) * (int)sizeof(T) - 16 * q));
          copy_async16(slot + (k * Q + q) * BLOCK, (const char*)(x + c) + (have ? 16 * q : 0), have);
        }
      }
    }
  };

  if (CL > 1) cluster_sync();  // every block of the cluster runs before its shared memory is written
  const Log2e log2e;
  RowInputs in{};
  const bool scalar = WARPS == 1 || warp == 0;  // warps that form the row's scalars
  if (row < a.rows) {
    fetch(row);
    if (scalar) in = row_inputs<T, POLICY>(a, row);
  }
  for (int turn = 0; row < a.rows; row += step, turn ^= 1) {
    copy_async_wait();
    Raw8<T> raw[kVecs];
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int c = (k * TEAM + tid) * 8;
      if (c < cols) {
#pragma unroll
        for (int q = 0; q < Q; ++q) raw[k].q[q] = slot[(k * Q + q) * BLOCK];
        if (c + 8 > cols) {
          T* v = reinterpret_cast<T*>(&raw[k]);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (c + j >= cols) v[j] = from_f32<T>(-INFINITY);
        }
        top = fmaxf(top, max_of<1>(&raw[k]));
      }
    }
    top = warp_max(top);
    // every value of the stage has been used: the next row may arrive in it
    const long next = row + step;
    RowInputs next_in{};
    if (next < a.rows) {
      fetch(next);
      if (scalar) next_in = row_inputs<T, POLICY>(a, next);
    }
    const float z = finite_or_zero(top);
    uint64_t sum2 = 0;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      if ((k * TEAM + tid) * 8 < cols) {
        float d[8];
        diffs(raw[k], z, d);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float e[2];
          exp2_of(log2e, d[j], d[j + 1], e);
          sum2 = add_f32x2(sum2, f2pack(e[0], e[1]));
        }
      }
    }
    float s0, s1;
    f2unpack(sum2, s0, s1);
    float sum = s0 + s1;
    sum = warp_sum(sum);
    Stat st{top, sum};
    float coef;
    if (WARPS == 1) {
      coef = finish_row<POLICY>(a, row, in, st, lane == 0);
    } else {
      if (CL == 1) {
        if (lane == 0) pairs[turn][warp] = make_float2(top, sum);
        __syncthreads();
      } else {
        // one store per block of the cluster, then one barrier.  Slots alternate between turns: a
        // block that is a turn ahead has passed this turn's barrier, after everyone read the last turn's.
        if (lane < CL) {
          const uint32_t dst = cluster_addr(&pairs[turn][rank * WARPS + warp], lane);
          asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(top), "f"(sum) : "memory");
        }
        __syncwarp();
        cluster_sync();
      }
      float2 p[(WARPS * CL + 31) / 32];
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < (WARPS * CL + 31) / 32; ++i) {
        const int w = i * 32 + lane;
        p[i] = w < WARPS * CL ? pairs[turn][w] : make_float2(-INFINITY, 0.f);
        m = fmaxf(m, p[i].x);
      }
      m = warp_max(m);
      const float mz = finite_or_zero(m);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < (WARPS * CL + 31) / 32; ++i) s += p[i].y * expf(p[i].x - mz);
      st = {m, warp_sum(s)};
      if (warp == 0) {
        const float c = finish_row<POLICY>(a, row, in, st, rank == 0 && lane == 0);
        if (lane == 0) {
          sh_coef = c;
          sh_target = (int)in.t;  // only looked at when it is one: otherwise the coefficient is 0
          if (POLICY) sh_entry = RowGrad(st, c, sh_target).at_target(in.xt, st.s);
        }
      }
      if (POLICY) {
        __syncthreads();
        coef = sh_coef;
      }
    }
    if (POLICY) {
      const RowGrad grad(st, coef, (WARPS == 1 ? (int)in.t : sh_target) - c0);
      const float entry = WARPS == 1 ? grad.at_target(in.xt, st.s) : sh_entry;
      T* out = (T*)a.p.out + row * a.p.ldo + c0;
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        const int c = (k * TEAM + tid) * 8;
        if (c < cols) {
          grad.vector(log2e, raw[k], c, entry);
          if (c + 8 <= cols) {
            straw8(out + c, raw[k]);
          } else {
            const T* g = reinterpret_cast<const T*>(&raw[k]);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (c + j < cols) out[c + j] = g[j];
          }
        }
      }
    }
    in = next_in;
  }
}

// Wide rows, many of them: a block of NT threads per row at a time, each thread with a running
// (maximum, sum) over batches of kVecs vectors.
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Adds the vectors [v0, full) of a row, every NT-th of them from v0 + tid on, read with plain loads;
// those of the last batch, which may be partial, are in flight together too.
template <int NT, class T>
__device__ __forceinline__ void add_span(const Log2e& l, Stat& st, const T* x, int v0, int full, int tid) {
  constexpr int N = sizeof(T) == 2 ? 4 : 2;
  Raw8<T> raw[N];
  for (; v0 + N * NT <= full; v0 += N * NT) {
    const T* xv = x + (long)(v0 + tid) * 8;
#pragma unroll
    for (int u = 0; u < N; ++u) raw[u] = ldraw8(xv + u * NT * 8);
    add_vectors<N>(l, st, raw);
  }
  const int left = full - v0 - tid;
  const T* xv = x + (long)(v0 + tid) * 8;
#pragma unroll
  for (int u = 0; u < N; ++u)
    if (u * NT < left) raw[u] = ldraw8(xv + u * NT * 8);
#pragma unroll
  for (int u = 0; u < N; ++u)
    if (u * NT < left) add_vectors<1>(l, st, raw + u);
}

__device__ __forceinline__ void add_one(Stat& st, float x) {
  const float m = fmaxf(st.m, x), z = finite_or_zero(m);
  st = {m, st.s * expf(st.m - z) + exp_diff(x, z)};
}

// A warp's statistic, and that of W pairs: the maxima first, then the sums relative to them.
__device__ __forceinline__ Stat warp_stat(Stat st) {
  const float m = warp_max(st.m);
  return {m, warp_sum(st.s * expf(st.m - finite_or_zero(m)))};
}

// Log probabilities.  A block's last warp forms the rows' results from the others' pairs; the others
// go on to the next row at once, up to kAhead rows ahead, so that their loads never stop.
constexpr int kAhead = 4;

template <class T, int NT>
__global__ void __launch_bounds__(NT + 32, 1024 / NT) stream_logprobs_kernel(RowArgs a) {
  constexpr int W = NT / 32;
  __shared__ float2 pairs[kAhead][W];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int V = a.p.V, full = V / 8;
  if (warp == W) {
    RowInputs in = row_inputs<T, false>(a, blockIdx.x);
    int slot = 0;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
      const long next = row + gridDim.x;
      RowInputs next_in{};
      if (next < a.rows) next_in = row_inputs<T, false>(a, next);
      bar_sync(1 + slot, NT + 32);  // the pairs are there
      const float2 p = lane < W ? pairs[slot][lane] : make_float2(-INFINITY, 0.f);
      const Stat st = warp_stat(Stat{p.x, p.y});
      if (row + (long)kAhead * gridDim.x < a.rows) bar_arrive(1 + kAhead + slot, NT + 32);  // and free again
      finish_row<false>(a, row, in, st, lane == 0);
      in = next_in;
      slot = slot + 1 == kAhead ? 0 : slot + 1;
    }
    return;
  }
  const Log2e log2e;
  const int tail = full * 8 + tid;  // the row's last V % 8 columns, one each for the first threads
  int slot = 0;
  bool again = false;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.p.logits + row * a.p.ld;
    Stat st{-INFINITY, 0.f};
    add_span<NT>(log2e, st, x, 0, full, tid);
    if (tail < V) add_one(st, to_f32(x[tail]));
    __syncwarp();
    st = warp_stat(st);
    if (again) bar_sync(1 + kAhead + slot, NT + 32);
    if (lane == 0) pairs[slot][warp] = make_float2(st.m, st.s);
    __syncwarp();
    bar_arrive(1 + slot, NT + 32);
    if (++slot == kAhead) {
      slot = 0;
      again = true;
    }
  }
}

// Policy loss.  The first `cached` vectors of a row live in shared memory from their arrival until the
// row's gradient is written.  One loop does both ends: a round's slots are turned into gradient and
// stored, asynchronous copies bring the next row's vectors into them, and the vectors that were asked for
// kLag rounds ago join the next row's statistic.  Each thread only ever touches its own slots, so the
// loop has no barrier; reads and writes of DRAM run side by side.  Columns that do not fit are read by
// a pass of their own before the row's statistic is complete, and right after it again, from L2.
constexpr int kLag = 2;

// The same with 32-bit shared addresses, which the compiler offsets by literals.
__device__ __forceinline__ uint4 shared_load16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int PENDING>
__device__ __forceinline__ void copy_async_wait_for() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_async_small(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}

// Blocks of the policy kernel per SM: 768 threads (640 in one), so that each has 85 registers or more.  With 1024
// threads of 64, V = 50257 (8192 rows) took 327 us instead of 305.
constexpr int policy_blocks(int NT) { return NT > 400 ? 1 : NT > 256 ? 2 : NT > 128 ? 3 : 6; }

template <class T, int NT>
__global__ void __launch_bounds__(NT, policy_blocks(NT)) stream_policy_kernel(RowArgs a, int cached) {
  extern __shared__ uint4 cache[];  // [part of a vector][cached]
  constexpr int W = NT / 32, NV = sizeof(T) == 2 ? 2 : 1, ROUND = NV * NT, Q = sizeof(Raw8<T>) / 16;
  __shared__ float2 pairs[2][W];
  __shared__ RowInputs coming;  // of the next row, by asynchronous copies (but for the target's logit)
  __shared__ float sh_coef, sh_entry;
  __shared__ int sh_target;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int V = a.p.V, full = V / 8;
  const int tail = full * 8 + tid;  // the row's last V % 8 columns, one each for the first threads
  const int whole = cached / ROUND;                // rounds that every thread takes part in fully
  const int left = cached - whole * ROUND - tid;   // of the last, partial one: vector u if u NT < left
  const Log2e log2e;
  const uint32_t mine = smem_u32(cache + tid);     // this thread's slots: every NT-th
  const uint32_t part = cached * 16;               // bytes between the parts of a vector

  auto load_slot = [&](uint32_t at) {
    Raw8<T> r;
#pragma unroll
    for (int q = 0; q < Q; ++q) r.q[q] = shared_load16(at + q * part);
    return r;
  };
  auto fetch_slot = [&](uint32_t at, const T* x) {
#pragma unroll
    for (int q = 0; q < Q; ++q) copy_async16(at + q * part, (const char*)x + 16 * q);
  };
  auto add_round = [&](Stat& st, uint32_t at) {
    Raw8<T> raw[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) raw[u] = load_slot(at + u * NT * 16);
    add_vectors<NV>(log2e, st, raw);
  };
  auto add_partial = [&](Stat& st) {
#pragma unroll
    for (int u = 0; u < NV; ++u)
      if (u * NT < left) {
        const Raw8<T> raw = load_slot(mine + (whole * ROUND + u * NT) * 16);
        add_vectors<1>(log2e, st, &raw);
      }
  };
  auto fetch_inputs = [&](long row) {  // by one thread
    copy_async_small<8>(&coming.t, a.p.targets + row);
    if (a.p.weights) copy_async_small<4>(&coming.w, a.p.weights + row);
    copy_async_small<4>(&coming.adv, a.p.advantages + row);
    copy_async_small<4>(&coming.old, a.p.old_logps + row);
    if (a.p.ref_logps) copy_async_small<4>(&coming.ref, a.p.ref_logps + row);
  };

  const long ld = a.p.ld;
  Stat st{-INFINITY, 0.f};  // of the cached part of the coming row
  {
    const T* xr = (const T*)a.p.logits + blockIdx.x * ld;
    if (tid == 0) fetch_inputs(blockIdx.x);
    for (int v = tid; v < cached; v += NT) fetch_slot(mine + (v - tid) * 16, xr + (long)v * 8);
    copy_async_wait();
    for (int r = 0; r < whole; ++r) add_round(st, mine + r * ROUND * 16);
    add_partial(st);
  }
  int turn = 0;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x, ++turn) {
    const long next = row + gridDim.x;
    const T* x = (const T*)a.p.logits + row * ld;
    T* out = (T*)a.p.out + row * a.p.ldo;
    const float xtail = tail < V ? to_f32(x[tail]) : -INFINITY;
    add_span<NT>(log2e, st, x, cached, full, tid);
    if (tail < V) add_one(st, xtail);
    __syncwarp();
    st = warp_stat(st);
    if (lane == 0) pairs[turn & 1][warp] = make_float2(st.m, st.s);
    __syncthreads();
    const float2 p = lane < W ? pairs[turn & 1][lane] : make_float2(-INFINITY, 0.f);
    st = warp_stat(Stat{p.x, p.y});
    if (warp == 0) {
      RowInputs in = coming;
      if (!a.p.weights) in.w = 1.f;
      if (in.t >= 0 && in.t < V) {
        const int tv = (int)in.t >> 3;
        if (tv < cached) {
          constexpr int per = 16 / sizeof(T);  // columns of one part of a vector
          const int q = ((int)in.t & 7) / per;
          in.xt = to_f32(reinterpret_cast<const T*>(cache + q * cached + tv)[(int)in.t & (per - 1)]);
        } else {
          in.xt = to_f32(x[in.t]);
        }
      }
      const float c = finish_row<true>(a, row, in, st, lane == 0);
      if (lane == 0) {
        sh_coef = c;
        sh_target = (int)in.t;  // only looked at when it is one: otherwise the coefficient is 0
        sh_entry = RowGrad(st, c, sh_target).at_target(in.xt, st.s);
      }
    }
    __syncthreads();
    const RowGrad grad(st, sh_coef, sh_target);
    const float entry = sh_entry;
    const bool more = next < a.rows;
    if (more && tid == 0) fetch_inputs(next);
    const T* xn = (const T*)a.p.logits + next * ld + tid * 8;
    st = {-INFINITY, 0.f};

    // a row's gradient pass, for masked rows (zeros, whatever they hold) and others
    auto pass = [&](auto masked) {
      auto turned = [&](Raw8<T> r) {
        if constexpr (decltype(masked)::value) {
#pragma unroll
          for (int q = 0; q < Q; ++q) r.q[q] = make_uint4(0, 0, 0, 0);
        } else {
          grad.plain(log2e, r);
        }
        return r;
      };
      for (int v0 = cached; v0 < full; v0 += 2 * ROUND) {
        const long at = (long)(v0 + tid) * 8;
        const int rest = full - v0 - tid;
        Raw8<T> raw[2 * NV];
#pragma unroll
        for (int u = 0; u < 2 * NV; ++u)
          if (u * NT < rest) raw[u] = ldraw8(x + at + u * NT * 8);
#pragma unroll
        for (int u = 0; u < 2 * NV; ++u)
          if (u * NT < rest) straw8(out + at + u * NT * 8, turned(raw[u]));
      }
      uint32_t at = mine;
      T* o = out + tid * 8;
      const T* xf = xn;
      for (int r = 0; r < whole; ++r) {
#pragma unroll
        for (int u = 0; u < NV; ++u) straw8(o + u * NT * 8, turned(load_slot(at + u * NT * 16)));
        if (more) {
          __syncwarp();
#pragma unroll
          for (int u = 0; u < NV; ++u) fetch_slot(at + u * NT * 16, xf + u * NT * 8);
          copy_async_commit();
          if (r >= kLag) {
            copy_async_wait_for<kLag>();
            add_round(st, at - kLag * ROUND * 16);
          }
        }
        at += ROUND * 16;
        o += ROUND * 8;
        xf += ROUND * 8;
      }
#pragma unroll
      for (int u = 0; u < NV; ++u)
        if (u * NT < left) {
          straw8(o + u * NT * 8, turned(load_slot(at + u * NT * 16)));
          if (more) fetch_slot(at + u * NT * 16, xf + u * NT * 8);
        }
    };
    if (grad.coef == 0.f) {
      pass(std::true_type{});
    } else {
      pass(std::false_type{});
      // the target's own entry, by the thread that wrote its vector
      const int tv = grad.target >> 3;
      if (tv < full && tid == (tv < cached ? tv % NT : (tv - cached) % NT))
        out[grad.target] = from_f32<T>(entry);
    }
    if (tail < V) out[tail] = from_f32<T>(tail == grad.target && grad.coef != 0.f ? entry : grad.elsewhere(xtail));
    copy_async_wait();
    if (more) {
      for (int r = max(0, whole - kLag); r < whole; ++r) add_round(st, mine + r * ROUND * 16);
      add_partial(st);
    }
  }
}

// Gradient of the logits from stored statistics: a block takes kGradVecs vectors per thread of one row,
// rows from the last to the first, since the last rows are what the forward left in L2.
constexpr int kGradThreads = 256, kGradVecs = 4;

template <class T>
__global__ void __launch_bounds__(kGradThreads)
    logprobs_bwd_kernel(const T* logits, long ld, const int64_t* __restrict__ targets,
                        const float2* __restrict__ stats, const float* __restrict__ dlogps, T* out, long ldo, int rows,
                        int V, int threads_per_row, int blocks_per_row) {
  // narrow rows share a block: threads_per_row threads each
  const int sub = threadIdx.x / threads_per_row, tid = threadIdx.x - sub * threads_per_row;
  const int group = blockIdx.x / blocks_per_row, part = blockIdx.x - group * blocks_per_row;
  const long row = rows - 1 - ((long)group * (kGradThreads / threads_per_row) + sub);
  if (row < 0) return;
  const int full = V / 8;
  const int v0 = part * (kGradThreads * kGradVecs) + tid;
  const int left = full - v0;  // vector k of this thread is one of the row's if k threads_per_row < left
  const T* x = logits + row * ld;
  T* o = out + row * ldo;
  const int64_t t64 = targets[row];
  const float2 s2 = stats[row];
  const float up = dlogps[row];
  const Stat st{s2.x, s2.y};
  const bool valid = t64 >= 0 && t64 < V;
  const RowGrad grad(st, valid && !is_empty(st) ? up : 0.f, (int)t64);
  if (grad.coef == 0.f) {  // a masked row: zeros, whatever it holds
    Raw8<T> none;
#pragma unroll
    for (int q = 0; q < (int)sizeof(Raw8<T>) / 16; ++q) none.q[q] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k)
      if (k * threads_per_row < left) straw8(o + (long)(v0 + k * threads_per_row) * 8, none);
  } else {
    const Log2e log2e;
    Raw8<T> raw[kGradVecs];
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k)
      if (k * threads_per_row < left) raw[k] = ldraw8(x + (long)(v0 + k * threads_per_row) * 8);
    // the thread that writes the target's vector writes the target's own entry after it
    const int from = (grad.target >> 3) - v0;
    const bool owner = grad.target < full * 8 && from >= 0 && from < kGradVecs * threads_per_row &&
                       from % threads_per_row == 0;
    const float entry = owner ? grad.at_target(to_f32(x[grad.target]), st.s) : 0.f;
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k)
      if (k * threads_per_row < left) {
        grad.plain(log2e, raw[k]);
        straw8(o + (long)(v0 + k * threads_per_row) * 8, raw[k]);
      }
    if (owner) o[grad.target] = from_f32<T>(entry);
  }
  if (part == blocks_per_row - 1)
    for (int c = full * 8 + tid; c < V; c += threads_per_row) {
      const float xc = to_f32(x[c]);
      o[c] = from_f32<T>(c == grad.target && grad.coef != 0.f ? grad.at_target(xc, st.s) : grad.elsewhere(xc));
    }
}

// A pair of answers (rows 2i: preferred, 2i + 1: rejected) per block, or per cluster of CL blocks that
// share its tokens.  Sums are fp64, in a fixed order.
template <int CL, int NT>
__global__ void __launch_bounds__(NT) preference_kernel(PreferenceArgs a) {
  constexpr int W = NT / 32;
  __shared__ double warp_part[4][W];       // sum and count of either row, per warp
  __shared__ double block_part[CL][4];     // and per block of the cluster
  const int rank = CL > 1 ? (int)cluster_ctarank() : 0, pair = blockIdx.x / CL;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = (a.S + CL - 1) / CL, i0 = rank * slice, i1 = min(a.S, i0 + slice);
  if (CL > 1) cluster_sync();  // every block of the cluster runs before its shared memory is written
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long base = ((long)pair * 2 + k) * a.S;
    double s = 0.0;
    int n = 0;
#pragma unroll 4
    for (int i = i0 + (int)threadIdx.x; i < i1; i += NT) {
      // masked tokens are loaded too, ahead of knowing their mask, and left out
      const float lp = a.logps[base + i], ref = a.ref_logps[base + i];
      if (a.mask[base + i]) {
        s += (double)lp - (double)ref;
        ++n;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      n += __shfl_xor_sync(0xffffffffu, n, o);
    }
    if (lane == 0) {
      warp_part[2 * k][warp] = s;
      warp_part[2 * k + 1][warp] = (double)n;
    }
  }
  __syncthreads();
  if (threadIdx.x < 4 * CL) {  // thread 4 r + q brings value q to block r
    const int q = threadIdx.x & 3, to = threadIdx.x >> 2;
    double v = 0.0;
#pragma unroll
    for (int w = 0; w < W; ++w) v += warp_part[q][w];
    if (CL == 1) {
      block_part[0][q] = v;
    } else {
      const uint32_t dst = cluster_addr(&block_part[rank][q], to);
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(dst), "d"(v) : "memory");
    }
  }
  __syncwarp();
  if (CL > 1) cluster_sync();
  else __syncthreads();
  double total[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int r = 0; r < CL; ++r)
#pragma unroll
    for (int q = 0; q < 4; ++q) total[q] += block_part[r][q];
  const double r[2] = {total[0], total[2]}, count[2] = {fmax(total[1], 1.0), fmax(total[3], 1.0)};
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
    // a side of weight 0 is left out: it may be infinite.  A margin that is no number stays one.
    loss = (eps < 1.0 ? (1.0 - eps) * (tail + fmax(-h, 0.0)) : 0.0) + (eps > 0.0 ? eps * (tail + fmax(h, 0.0)) : 0.0);
    up[0] = beta * (eps - 1.0 / (1.0 + exp(h)));
    up[1] = -up[0];
  }
  if (rank == 0 && threadIdx.x == 0) {
    a.losses[pair] = (float)loss;
    a.rewards[pair * 2] = (float)(beta * r[0]);
    a.rewards[pair * 2 + 1] = (float)(beta * r[1]);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long base = ((long)pair * 2 + k) * a.S;
    const float g = (float)(up[k] * a.grad_scale);
#pragma unroll 4
    for (int i = i0 + (int)threadIdx.x; i < i1; i += NT) a.dlogps[base + i] = a.mask[base + i] ? g : 0.f;
  }
}

}  // namespace

namespace {

// Launches row_kernel with as many teams as fit on the GPU at once (or as there are rows).
template <class T, int WARPS, int CL, bool POLICY>
int launch_rows(RowArgs a, cudaStream_t s) {
  constexpr int BLOCK = WARPS == 1 ? 256 : WARPS * 32;
  constexpr int smem = BLOCK * kVecs * (int)sizeof(Raw8<T>);
  auto kern = row_kernel<T, WARPS, CL, POLICY>;
  int dev = 0;
  cudaGetDevice(&dev);
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(BLOCK);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CL;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = CL > 1 ? 1 : 0;
  static std::atomic<int> resident[64];  // teams (clusters or blocks) that run at once, per device
  int fit = resident[dev & 63].load();
  if (fit == 0) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    if (CL > 1) {
      cfg.gridDim = dim3(CL);
      e = cudaOccupancyMaxActiveClusters(&fit, kern, &cfg);
    } else {
      int sms = 148;
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, BLOCK, smem);
      fit *= sms;
    }
    if (e != cudaSuccess) return (int)e;
    if (fit < 1) return -2;
    resident[dev & 63].store(fit);
  }
  a.slice = ((a.p.V + CL - 1) / CL + 7) / 8 * 8;
  const int teams = WARPS == 1 ? (a.rows + BLOCK / 32 - 1) / (BLOCK / 32) : a.rows;
  cfg.gridDim = dim3((unsigned)std::min(teams, fit) * CL);
  return (int)cudaLaunchKernelEx(&cfg, kern, a);
}

int sm_count(int* sms) {
  static std::atomic<int> known[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  *sms = known[dev & 63].load();
  if (*sms == 0) {
    e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return (int)e;
    known[dev & 63].store(*sms);
  }
  return 0;
}

// A block's share of the SM's shared memory when 1024 / NT blocks run on it.
constexpr int cache_bytes(int NT) { return ((224 << 10) / policy_blocks(NT) - 1024 - 256) / 64 * 64; }

template <class T, bool POLICY, int NT>
int launch_stream(const RowArgs& a, int sms, cudaStream_t s) {
  const int blocks = (int)std::min<long>(a.rows, (long)sms * (POLICY ? policy_blocks(NT) : 1024 / NT));
  if constexpr (POLICY) {
    constexpr int most = cache_bytes(NT) / (int)sizeof(Raw8<T>);
    auto kern = stream_policy_kernel<T, NT>;
    int dev = 0;
    cudaGetDevice(&dev);
    static std::atomic<bool> ready[64];
    if (!ready[dev & 63].load()) {
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           most * (int)sizeof(Raw8<T>));
      if (e != cudaSuccess) return (int)e;
      ready[dev & 63].store(true);
    }
    const int cached = std::min(most, a.p.V / 8);
    kern<<<blocks, NT, cached * sizeof(Raw8<T>), s>>>(a, cached);
  } else {
    stream_logprobs_kernel<T, NT><<<blocks, NT + 32, 0, s>>>(a);
  }
  return (int)cudaGetLastError();
}

template <class T, bool POLICY>
int dispatch_rows(const RowArgs& a, cudaStream_t s) {
  constexpr int per_thread = kVecs * 8;
  const int V = a.p.V;
  int sms = 0;
  if (int e = sm_count(&sms)) return e;
  if (V <= 32 * per_thread) return launch_rows<T, 1, 1, POLICY>(a, s);
  // V = 4096, 16384 rows: 35 us (the stream kernel 41) for log probabilities, 67 (71) for the policy loss
  if (V <= 128 * per_thread && a.rows > sms) return launch_rows<T, 4, 1, POLICY>(a, s);
  // blocks per row that hold it in registers, and more of them while the rows leave half of the GPU
  // idle and every block keeps 2048 columns
  int need = 1;
  while (need <= 8 && V > need * 512 * per_thread) need *= 2;
  if (a.rows > sms || need > 8) {
    if constexpr (!POLICY) {
      // 128 / 256 / 512 threads: V = 50257 (8192 rows) 184 / 141 / 159 us, 128256 (4096 rows) 224 / 171 / 171
      return launch_stream<T, POLICY, 256>(a, sms, s);
    } else {
      // Small blocks for narrow rows: more rows are under way at once, which covers the barriers, until
      // much of a row has to be read twice.  B200, bf16, us with 128 / 256 / 384 / 640 threads:
      //   V = 16384 (16384 rows) 183 / 228 / 286 / 455
      //   V = 32000 (8192 rows)  211 / 194 / 212 / 310
      //   V = 50257 (8192 rows)  397 / 310 / 304 / 406
      //   V = 100000 (4096 rows) 468 / 398 / 342 / 329
      //   V = 128256 (4096 rows) 612 / 527 / 448 / 414
      // fp32 rows take 384 threads at most: 393 us at V = 50257 (4096 rows), 443 with 640.
      const long bytes = (long)V * sizeof(T);
      if (bytes <= cache_bytes(128) * 5L / 4) return launch_stream<T, POLICY, 128>(a, sms, s);
      if (bytes <= cache_bytes(256) * 5L / 4) return launch_stream<T, POLICY, 256>(a, sms, s);
      if (sizeof(T) == 4 || bytes <= cache_bytes(384) * 3L / 2) return launch_stream<T, POLICY, 384>(a, sms, s);
      return launch_stream<T, POLICY, 640>(a, sms, s);
    }
  }
  while (need < 8 && (long)a.rows * need <= sms && V / (2 * need) >= 2048) need *= 2;
  switch (need) {
    case 1: return launch_rows<T, 16, 1, POLICY>(a, s);
    case 2: return launch_rows<T, 16, 2, POLICY>(a, s);
    case 4: return launch_rows<T, 16, 4, POLICY>(a, s);
    default: return launch_rows<T, 16, 8, POLICY>(a, s);
  }
}

}  // namespace

int token_logprobs(const void* logits, long ld, int dtype, const int64_t* targets, float* logps, float* stats, int rows,
                   int V, cudaStream_t s) {
  if (ld % 8) return -1;
  if (rows == 0) return 0;
  RowArgs a{};
  a.p.logits = logits;
  a.p.ld = ld;
  a.p.targets = targets;
  a.p.logps = logps;
  a.p.V = V;
  a.stats = (float2*)stats;
  a.rows = rows;
  return with_dtype(dtype, [&](auto v) { return dispatch_rows<decltype(v), false>(a, s); });
}

int token_logprobs_bwd(const void* logits, long ld, int dtype, const int64_t* targets, const float* stats,
                       const float* dlogps, void* out, long ldo, int rows, int V, cudaStream_t s) {
  if (ld % 8 || ldo % 8) return -1;
  if (rows == 0) return 0;
  // threads of a row: a power of two that covers it with kGradVecs vectors each, at most the block's
  const int vecs = (V + 7) / 8;
  int per_row = 1;
  while (per_row < kGradThreads && per_row * kGradVecs < vecs) per_row *= 2;
  const int rows_per_block = kGradThreads / per_row;
  const int blocks_per_row = std::max(1, (V / 8 + per_row * kGradVecs - 1) / (per_row * kGradVecs));
  const long blocks = ((long)rows + rows_per_block - 1) / rows_per_block * blocks_per_row;
  if (blocks > INT32_MAX) return -1;
  return with_dtype(dtype, [&](auto v) {
    using T = decltype(v);
    logprobs_bwd_kernel<<<(unsigned)blocks, kGradThreads, 0, s>>>(
        (const T*)logits, ld, targets, (const float2*)stats, dlogps, (T*)out, ldo, rows, V, per_row, blocks_per_row);
    return (int)cudaGetLastError();
  });
}

int policy_loss(const PolicyArgs& p, cudaStream_t s) {
  if (p.ld % 8 || p.ldo % 8) return -1;
  if (p.rows == 0) return 0;
  RowArgs a{};
  a.p = p;
  a.rows = p.rows;
  return with_dtype(p.dtype, [&](auto v) { return dispatch_rows<decltype(v), true>(a, s); });
}

int preference_loss(const PreferenceArgs& a, cudaStream_t s) {
  if (a.pairs == 0) return 0;
  // One block per pair, or 8 for long answers: 4.3 / 3.9 us at 2048 tokens (64 pairs: 4.5 / 5.4), 6.4 / 5.1 at
  // 4096 (6.6 / 6.6), 18 / 7.4 at 16384.  Few pairs of very long answers take blocks of 1024 threads: 38 -> 14 us
  // at 131072 tokens (64 pairs of 16384: 9.4 -> 30).
  if (a.S < 4096) {
    preference_kernel<1, 256><<<a.pairs, 256, 0, s>>>(a);
    return (int)cudaGetLastError();
  }
  if (a.pairs > INT32_MAX / 8) return -1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)a.pairs * 8);
  const bool wide = a.S >= 16384 && a.pairs <= 8;
  cfg.blockDim = dim3(wide ? 1024 : 256);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 8;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, wide ? preference_kernel<8, 1024> : preference_kernel<8, 256>, a);
}

}  // namespace mt
