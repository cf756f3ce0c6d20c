// qk_norm_rope.cu -- RMS norm of every query and key head and its rotation, in one pass, and its backward.
//
// Head x (n values) of a row at position p = row mod S, gain g, half = n/2:
//   r = (mean(x^2) + eps)^(-1/2)      u = x r g      angle_i = p theta^(-2i/n)
//   y_i = u_i cos_i - u_{i+half} sin_i               y_{i+half} = u_{i+half} cos_i + u_i sin_i
// and backward from dy (r is formed again from x, which has to be read anyway):
//   du = the inverse rotation of dy   dg += sum over rows and heads of du x r
//   w = du g                          dx = r (w - x r mean(w x r))
// Sums, r and the rotation are fp32, each output is rounded once.  Angles are formed in fp64 and
// reduced to a fraction of a turn before the fp32 sine: at position 10^5 an fp32 angle is off by up
// to 4e-3 rad, more than a bf16 rounding.
//
// Bound: DRAM (forward reads and writes each head once, backward reads two and writes one).  A head
// is spread over G lanes, each holding 8 adjacent values of either half, so that the rotation's pairs
// meet in one thread, every access is a 16-byte vector and a norm is log2(G) shuffles.  A warp takes
// one row (or a share of its heads when there are few rows) and computes the row's sines once for
// all heads.  In the backward what a thread will read is on its way three turns ahead, by asynchronous
// copies into slots of shared memory that no other thread touches: with plain loads, registers limited
// what was in flight (115 us instead of 89 below).  In the forward four heads' plain loads per turn do
// as well (61 us; the queue 64).
//
// B200, 16384 rows of 32 + 8 heads of 128, bf16: forward 61 us (5.5 TB/s, 84% of the copy rate),
// backward 89 us (5.7 TB/s, 87%), the gains' sum included.
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mt_api.h"
#include "vec_io.cuh"

namespace mt {
namespace {

constexpr int kWarps = 8;
constexpr int kPerSm = 2;  // resident blocks: the kernels hold a head pair's values in about 128 registers
constexpr int kMaxHalf = 128;

// theta^(-2i/n) / (2 pi) as a product of the powers 2^k of the ratio theta^(-2/n): the host forms
// eight powers in fp64, a thread multiplies those of i's bits.
struct Turns {
  double unit;      // 1 / (2 pi)
  double ratio[7];  // theta^(-2/n * 2^k)
};

__device__ __forceinline__ double turns_per_position(const Turns& t, int i) {
  double f = t.unit;
#pragma unroll
  for (int k = 0; k < 7; ++k)
    if (i >> k & 1) f *= t.ratio[k];
  return f;
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The (cos, sin) of a row's position for all pairs, into this warp's shared rows.
__device__ __forceinline__ void row_turns(const double* freq, float* cs, float* sn, int half, int pos, int lane) {
  __syncwarp();
  for (int i = lane; i < half; i += 32) {
    double t = (double)pos * freq[i];
    t -= rint(t);
    sincospif(2.0f * (float)t, &sn[i], &cs[i]);
  }
  __syncwarp();
}

__device__ __forceinline__ void copy_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// What a thread reads in its coming turns: the two vectors of a head of x and of dy each, DEPTH turns
// ahead.  A row is turns_q turns over the query heads, then turns_k over the key heads, `slots` heads a
// turn.  Slots are [turn][vector part][thread]; fetch() is called once per turn and asks for the next one.
template <class T, int DEPTH>
struct HeadQueue {
  static constexpr int Q = sizeof(Raw8<T>) / 16, PARTS = 4 * Q;
  uint4* mem;
  const T* base[2];
  long ld[2];
  long row, rows, row_step;
  int turn, turns_q, turns_k, slot, slots, H, HK, half, hd, stage;
  bool on;

  __device__ __forceinline__ void fetch() {
    if (row < rows) {
      const bool key = turn >= turns_q;
      const int h = (key ? turn - turns_q : turn) * slots + slot;
      if (on && h < (key ? HK : H)) {
        uint4* c = mem + stage * PARTS * kWarps * 32;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const T* p = base[m] + row * ld[m] + (long)(h + (key ? H : 0)) * hd;
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            copy_async16(c + (m * 2 * Q + q) * kWarps * 32, (const char*)p + 16 * q);
            copy_async16(c + (m * 2 * Q + Q + q) * kWarps * 32, (const char*)(p + half) + 16 * q);
          }
        }
      }
      if (++turn == turns_q + turns_k) {
        turn = 0;
        row += row_step;
      }
    }
    copy_async_commit();
    stage = stage + 1 == DEPTH ? 0 : stage + 1;
  }
  // The oldest turn's vectors; its slots are the next fetch()'s.
  __device__ __forceinline__ void read(int m, Raw8<T>& a, Raw8<T>& b) const {
    const uint4* c = mem + (stage * PARTS + m * 2 * Q) * kWarps * 32;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      a.q[q] = c[q * kWarps * 32];
      b.q[q] = c[(Q + q) * kWarps * 32];
    }
  }
};

// U heads per turn, their loads in flight together.
template <class T, int G, int U>
__global__ void __launch_bounds__(kWarps * 32, kPerSm)
    qk_norm_rope_fwd_kernel(const T* __restrict__ x, long ldx, const T* __restrict__ gq, const T* __restrict__ gk,
                            T* __restrict__ y, long ldy, int rows, int S, int H, int HK, int hd, float eps,
                            int warps_per_row, Turns turns) {
  __shared__ double freq[kMaxHalf];
  __shared__ float cs_all[kWarps][kMaxHalf], sn_all[kWarps][kMaxHalf];
  const int half = hd >> 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < half; i += blockDim.x) freq[i] = turns_per_position(turns, i);
  __syncthreads();
  const int d = (lane % G) * 8;  // this lane's values: d .. d+7 and half+d .. half+d+7
  const bool on = d < half;
  const int slots = (32 / G) * warps_per_row;
  const int slot = (warp % warps_per_row) * (32 / G) + lane / G;
  const int rows_per_block = kWarps / warps_per_row;
  const float inv_n = 1.0f / (float)hd;
  for (long row = (long)blockIdx.x * rows_per_block + warp / warps_per_row; row < rows;
       row += (long)gridDim.x * rows_per_block) {
    row_turns(freq, cs_all[warp], sn_all[warp], half, (int)(row % S), lane);
    float cs[8], sn[8];
    if (on) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cs[j] = cs_all[warp][d + j];
        sn[j] = sn_all[warp][d + j];
      }
    }
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
      const int n = part ? HK : H;
      const T* gain = part ? gk : gq;
      const T* xr = x + row * ldx + (part ? (long)H * hd : 0) + d;
      T* yr = y + row * ldy + (part ? (long)H * hd : 0) + d;
      float ga[8], gb[8];
      if (on) {
        load8(gain + d, ga);
        load8(gain + half + d, gb);
      }
      // every lane runs the same number of turns: the shuffles need the whole warp
      for (int h0 = 0; h0 < n; h0 += slots * U) {
        Raw8<T> ra[U], rb[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * slots + slot;
          if (on && h < n) {
            ra[u] = ldraw8(xr + (long)h * hd);
            rb[u] = ldraw8(xr + (long)h * hd + half);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * slots + slot;
          const bool mine = on && h < n;
          float a[8], b[8], ss = 0.f;
          if (mine) {
            unpack8(ra[u], a);
            unpack8(rb[u], b);
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += a[j] * a[j] + b[j] * b[j];
          }
          const float r = rsqrtf(group_sum<G>(ss) * inv_n + eps);
          if (mine) {
            float o1[8], o2[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float ua = a[j] * r * ga[j], ub = b[j] * r * gb[j];
              o1[j] = ua * cs[j] - ub * sn[j];
              o2[j] = ub * cs[j] + ua * sn[j];
            }
            store8(yr + (long)h * hd, o1);
            store8(yr + (long)h * hd + half, o2);
          }
        }
      }
    }
  }
}

// The gain gradients of a block go to its row of `partial` [blocks][2][hd]; gain_sum_kernel adds the
// rows in a fixed order, so that equal inputs give equal bits.
template <class T, int G, int DEPTH>
__global__ void __launch_bounds__(kWarps * 32, kPerSm)
    qk_norm_rope_bwd_kernel(const T* dy, long lddy, const T* __restrict__ x, long ldx, const T* __restrict__ gq,
                            const T* __restrict__ gk, T* dx, long lddx, float* __restrict__ partial, int rows, int S,
                            int H, int HK, int hd, float eps, int warps_per_row, Turns turns) {
  extern __shared__ uint4 ring[];
  __shared__ double freq[kMaxHalf];
  __shared__ float cs_all[kWarps][kMaxHalf], sn_all[kWarps][kMaxHalf];
  __shared__ float red[kWarps][2 * kMaxHalf];
  __shared__ float4 key_acc_all[4 * kWarps * 32];  // the key gain's gradient; the query gain's is in registers
  const int half = hd >> 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int d = (lane % G) * 8;
  const bool on = d < half;
  const int slots = (32 / G) * warps_per_row;
  const int slot = (warp % warps_per_row) * (32 / G) + lane / G;
  const int rows_per_block = kWarps / warps_per_row;
  const long row0 = (long)blockIdx.x * rows_per_block + warp / warps_per_row, row_step = (long)gridDim.x * rows_per_block;
  const float inv_n = 1.0f / (float)hd;
  HeadQueue<T, DEPTH> queue{ring + threadIdx.x, {x + d, dy + d}, {ldx, lddy}, row0, rows, row_step, 0,
                            (H + slots - 1) / slots, (HK + slots - 1) / slots, slot, slots, H, HK, half, hd, 0, on};
#pragma unroll
  for (int k = 0; k < DEPTH; ++k) queue.fetch();
  for (int i = threadIdx.x; i < half; i += blockDim.x) freq[i] = turns_per_position(turns, i);
  __syncthreads();
  float acc[16];
  float4* const key_acc = key_acc_all + threadIdx.x;  // 4 of them, kWarps * 32 apart
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) key_acc[j * kWarps * 32] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (long row = row0; row < rows; row += row_step) {
    row_turns(freq, cs_all[warp], sn_all[warp], half, (int)(row % S), lane);
    float cs[8], sn[8];
    if (on) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cs[j] = cs_all[warp][d + j];
        sn[j] = sn_all[warp][d + j];
      }
    }
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
      const int n = part ? HK : H;
      T* dxr = dx + row * lddx + (part ? (long)H * hd : 0) + d;
      float ga[8], gb[8];
      if (on) {
        load8((part ? gk : gq) + d, ga);
        load8((part ? gk : gq) + half + d, gb);
      }
      for (int h = slot; h - slot < n; h += slots) {
        copy_async_wait<DEPTH - 1>();
        const bool mine = on && h < n;
        float a[8], b[8], va[8], vb[8], ss = 0.f, dot = 0.f;
        if (mine) {
          Raw8<T> xa, xb, ya, yb;
          float ea[8], eb[8];
          queue.read(0, xa, xb);
          queue.read(1, ya, yb);
          unpack8(xa, a);
          unpack8(xb, b);
          unpack8(ya, ea);
          unpack8(yb, eb);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            va[j] = ea[j] * cs[j] + eb[j] * sn[j];
            vb[j] = eb[j] * cs[j] - ea[j] * sn[j];
            ss += a[j] * a[j] + b[j] * b[j];
            dot += va[j] * ga[j] * a[j] + vb[j] * gb[j] * b[j];
          }
        }
        const float r = rsqrtf(group_sum<G>(ss) * inv_n + eps);
        const float m = group_sum<G>(dot) * inv_n * r * r;  // mean(w x r) r
        __syncwarp();
        queue.fetch();
        if (mine) {
          float o1[8], o2[8], g1[8], g2[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float wa = va[j] * r, wb = vb[j] * r;
            g1[j] = wa * a[j];
            g2[j] = wb * b[j];
            o1[j] = wa * ga[j] - a[j] * (m * r);
            o2[j] = wb * gb[j] - b[j] * (m * r);
          }
          store8(dxr + (long)h * hd, o1);
          store8(dxr + (long)h * hd + half, o2);
          if (part == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              acc[j] += g1[j];
              acc[8 + j] += g2[j];
            }
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float* g = j < 2 ? g1 + 4 * j : g2 + 4 * (j - 2);
              float4 v = key_acc[j * kWarps * 32];
              v.x += g[0];
              v.y += g[1];
              v.z += g[2];
              v.w += g[3];
              key_acc[j * kWarps * 32] = v;
            }
          }
        }
      }
    }
  }
  copy_async_wait<0>();
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    if (part) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 v = key_acc[j * kWarps * 32];
        acc[4 * j] = v.x;
        acc[4 * j + 1] = v.y;
        acc[4 * j + 2] = v.z;
        acc[4 * j + 3] = v.w;
      }
    }
    // lanes that hold the same columns, then the block's warps, in a fixed order
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float v = acc[j];
#pragma unroll
      for (int o = 16; o >= G; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane < G && on) red[warp][(j < 8 ? 0 : half) + d + (j & 7)] = v;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < hd; c += blockDim.x) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) s += red[w][c];
      partial[((long)blockIdx.x * 2 + part) * hd + c] = s;
    }
    __syncthreads();
  }
}

// Sum of the blocks' partial gain gradients: 8 columns and 128 groups of rows per block, each thread's
// few loads in flight together.
constexpr int kSumCols = 8, kSumGroups = 128;

__global__ void __launch_bounds__(kSumCols * kSumGroups)
    gain_sum_kernel(const float* __restrict__ partial, int blocks, int hd, float* __restrict__ dgq,
                    float* __restrict__ dgk) {
  __shared__ float part[kSumCols * kSumGroups / 32][kSumCols];
  const int c = threadIdx.x % kSumCols, g = threadIdx.x / kSumCols, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.x * kSumCols + c;  // of 2 hd, a multiple of kSumCols
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched ahead of the backward kernel's end
  float s = 0.f;
#pragma unroll 4
  for (int b = g; b < blocks; b += kSumGroups) s += partial[(long)b * 2 * hd + col];
  s += __shfl_xor_sync(0xffffffffu, s, 8);
  s += __shfl_xor_sync(0xffffffffu, s, 16);
  if (lane < kSumCols) part[warp][c] = s;
  __syncthreads();
  if (threadIdx.x < kSumCols) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kSumCols * kSumGroups / 32; ++w) t += part[w][c];
    float* out = col < hd ? dgq + col : dgk + (col - hd);
    *out += t;
  }
}

Turns turns_of(int hd, double theta) {
  Turns t;
  t.unit = 0.15915494309189533577;  // 1 / (2 pi)
  double r = pow(theta, -2.0 / (double)hd);
  for (int k = 0; k < 7; ++k, r *= r) t.ratio[k] = r;
  return t;
}

// Warps that share a row's heads: one (a row's sines are computed by each), unless the rows fill less than
// half of the GPU's warps with one each.  1000 rows of 32 + 8 heads of 128, forward / backward: 6.9 / 13.0 us
// with this limit of 8 warps per SM, 7.5 / 15.8 with 16, 10.3 / 19.1 with 32.
int warps_per_row_of(int rows, int heads, int slots, int sms) {
  int w = 1;
  while (w < kWarps && (long)rows * w < 8L * sms && w * slots < heads) w *= 2;
  return w;
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Calls fn(lanes per head) with the smallest power of two that covers half / 8.
template <class F>
int with_lanes(int hd, F&& fn) {
  const int need = hd / 16;
  if (need <= 1) return fn(std::integral_constant<int, 1>{});
  if (need <= 2) return fn(std::integral_constant<int, 2>{});
  if (need <= 4) return fn(std::integral_constant<int, 4>{});
  if (need <= 8) return fn(std::integral_constant<int, 8>{});
  return fn(std::integral_constant<int, 16>{});
}

int grid_of(int rows, int rows_per_block, int sms) {
  return (int)std::min<long>(((long)rows + rows_per_block - 1) / rows_per_block, (long)kPerSm * sms);
}

// Launch with `smem` bytes of dynamic shared memory, which is opted into once per kernel and device.
template <class K, class... A>
int launch(K kern, std::atomic<bool>* ready, int blocks, int smem, cudaStream_t s, A... args) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (!ready[dev & 63].load()) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    ready[dev & 63].store(true);
  }
  kern<<<blocks, kWarps * 32, smem, s>>>(args...);
  return (int)cudaGetLastError();
}

}  // namespace

int qk_norm_rope_blocks(int rows, int heads, int hd) {
  int lanes = 1;
  while (lanes * 16 < hd) lanes *= 2;
  const int sms = sm_count();
  return grid_of(rows, kWarps / warps_per_row_of(rows, heads, 32 / lanes, sms), sms);
}

int qk_norm_rope_fwd(const QkNormRopeArgs& a, cudaStream_t s) {
  if (a.hd % 16 || a.hd < 16 || a.hd > 2 * kMaxHalf || a.S < 1) return -1;
  if (a.rows == 0 || a.H + a.HK == 0) return 0;
  const int sms = sm_count();
  return with_dtype(a.dtype, [&](auto v) {
    using T = decltype(v);
    return with_lanes(a.hd, [&](auto lanes) {
      constexpr int G = decltype(lanes)::value, U = sizeof(T) == 2 ? 4 : 2;  // 16 lines of 128 bytes per warp in flight
      const int w = warps_per_row_of(a.rows, a.H + a.HK, 32 / G, sms);
      auto kern = w > 1 ? qk_norm_rope_fwd_kernel<T, G, 1> : qk_norm_rope_fwd_kernel<T, G, U>;
      kern<<<grid_of(a.rows, kWarps / w, sms), kWarps * 32, 0, s>>>(
          (const T*)a.x, a.ldx, (const T*)a.gq, (const T*)a.gk, (T*)a.out, a.ldo, a.rows, a.S, a.H, a.HK, a.hd, a.eps,
          w, turns_of(a.hd, a.theta));
      return (int)cudaGetLastError();
    });
  });
}

int qk_norm_rope_bwd(const QkNormRopeArgs& a, const void* dy, long lddy, float* partial, float* dgq, float* dgk,
                     cudaStream_t s) {
  if (a.hd % 16 || a.hd < 16 || a.hd > 2 * kMaxHalf || a.S < 1) return -1;
  if (a.rows == 0 || a.H + a.HK == 0) return 0;
  const int sms = sm_count();
  return with_dtype(a.dtype, [&](auto v) {
    using T = decltype(v);
    return with_lanes(a.hd, [&](auto lanes) {
      constexpr int G = decltype(lanes)::value, DEPTH = sizeof(T) == 2 ? 3 : 2;
      static std::atomic<bool> ready[64];
      const int w = warps_per_row_of(a.rows, a.H + a.HK, 32 / G, sms);
      const int blocks = grid_of(a.rows, kWarps / w, sms);
      const int rc = launch(qk_norm_rope_bwd_kernel<T, G, DEPTH>, ready, blocks,
                            DEPTH * 4 * kWarps * 32 * (int)sizeof(Raw8<T>), s, (const T*)dy, lddy, (const T*)a.x, a.ldx,
                            (const T*)a.gq, (const T*)a.gk, (T*)a.out, a.ldo, partial, a.rows, a.S, a.H, a.HK, a.hd,
                            a.eps, w, turns_of(a.hd, a.theta));
      if (rc) return rc;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(2 * a.hd / kSumCols);
      cfg.blockDim = dim3(kSumCols * kSumGroups);
      cfg.stream = s;
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr.val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      return (int)cudaLaunchKernelEx(&cfg, gain_sum_kernel, (const float*)partial, blocks, a.hd, dgq, dgk);
    });
  });
}

}  // namespace mt
