// dropout.cu -- dropout whose mask is a function of (seed, offset, element) and is never stored.
//
// Element j keeps its value if the j-th 16-bit word of the random stream is at least
// cut = round(65536 p); kept values are scaled by 65536 / (65536 - cut), the inverse of the exact
// keep probability.  Words come from Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011): one evaluation at counter (j / 8, offset)
// under the key `seed` gives the 128 bits of eight adjacent elements.  The backward is the same call
// on the gradient, and a recomputed forward sees the same mask, whatever the launch shape.
//
//   y = residual + keep x scale      (one rounding; a dropped element adds exactly 0)
//
// Bound: DRAM (two or three accesses per element).  16384 x 4096 bf16, forward with residual and
// gradient: 106 us together, 6.3 TB/s (96% of the copy rate).  Eight elements' random words are ten rounds
// of two 32-bit products and four exclusive-ors; four groups' loads per thread are in flight meanwhile.
#include <cuda_runtime.h>

#include "mt_api.h"
#include "vec_io.cuh"

namespace mt {
namespace {

constexpr int kThreads = 256;

// The ten rounds' keys, formed on the host: as kernel parameters they are operands of the rounds'
// exclusive-ors, where key additions in the kernel were a sixth of its instructions.
struct RoundKeys {
  uint2 k[10];
};

__device__ __forceinline__ uint4 philox4x32(uint4 c, const RoundKeys& keys) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ keys.k[i].x, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ keys.k[i].y,
                   (uint32_t)a);
  }
  return c;
}

// N groups of eight elements per thread, kThreads groups apart; all loads are issued ahead of the
// random words, which are most of a group's instructions.
template <class T, bool RESIDUAL, int N>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T* x, const T* residual, T* y, long n, uint32_t cut, float scale, uint64_t offset,
                   const int64_t* __restrict__ offset_ptr, RoundKeys keys) {
  const long full = n / 8;
  const long g0 = (long)blockIdx.x * (kThreads * N) + threadIdx.x;
  Raw8<T> xr[N], rr[N];
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const long g = g0 + u * kThreads;
    if (g < full) {
      xr[u] = ldraw8(x + g * 8);
      if (RESIDUAL) rr[u] = ldraw8(residual + g * 8);
    }
  }
  if (offset_ptr) offset += (uint64_t)*offset_ptr;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const long g = g0 + u * kThreads;
    if (g * 8 >= n) break;
    const uint4 bits = philox4x32(make_uint4((uint32_t)g, (uint32_t)(g >> 32), (uint32_t)offset,
                                             (uint32_t)(offset >> 32)), keys);
    const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
    if (g < full) {
      float v[8], r[8];
      unpack8(xr[u], v);
      if (RESIDUAL) unpack8(rr[u], r);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // the upper half is compared in place: w >= cut << 16 as the lower half cannot tip it
        const bool keep = j & 1 ? w[j >> 1] >= cut << 16 : (w[j >> 1] & 0xffffu) >= cut;
        v[j] = keep ? v[j] * scale : 0.f;
        if (RESIDUAL) v[j] += r[j];
      }
      store8(y + g * 8, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (g * 8 + j < n) {
          const uint32_t bit16 = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
          float v = bit16 >= cut ? to_f32(x[g * 8 + j]) * scale : 0.f;
          if (RESIDUAL) v += to_f32(residual[g * 8 + j]);
          y[g * 8 + j] = from_f32<T>(v);
        }
      }
    }
  }
}

template <class T, int N>
int launch(const DropoutArgs& a, const RoundKeys& keys, cudaStream_t s) {
  const long groups = (a.n + 7) / 8, blocks = (groups + kThreads * N - 1) / (kThreads * N);
  if (blocks > INT32_MAX) return -1;
  const float scale = 65536.0f / (float)(65536u - a.cut);
  auto kern = a.residual ? dropout_kernel<T, true, N> : dropout_kernel<T, false, N>;
  kern<<<(unsigned)blocks, kThreads, 0, s>>>((const T*)a.x, (const T*)a.residual, (T*)a.out, a.n, a.cut, scale,
                                             a.offset, a.offset_ptr, keys);
  return (int)cudaGetLastError();
}

}  // namespace

int dropout_apply(const DropoutArgs& a, cudaStream_t s) {
  if (a.n == 0) return 0;
  RoundKeys keys;
  for (uint32_t i = 0; i < 10; ++i)
    keys.k[i] = make_uint2((uint32_t)a.seed + i * 0x9E3779B9u, (uint32_t)(a.seed >> 32) + i * 0xBB67AE85u);
  return with_dtype(a.dtype, [&](auto v) {
    using T = decltype(v);
    constexpr int N = sizeof(T) == 2 ? 4 : 2;
    // few elements (under four blocks per SM): one group per thread spreads them over more SMs
    return a.n <= (long)kThreads * 8 * 148 * 4 ? launch<T, 1>(a, keys, s) : launch<T, N>(a, keys, s);
  });
}

}  // namespace mt
