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
// Bound: DRAM (two or three accesses per element).
#include <cuda_runtime.h>

#include <algorithm>

#include "mt_api.h"
#include "vec_io.cuh"

namespace mt {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint4 philox4x32(uint4 c, uint2 k) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k.x, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k.y, (uint32_t)a);
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
}

template <class T, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T* x, const T* residual, T* y, long n, uint32_t cut, float scale, uint2 seed, uint64_t offset,
                   const int64_t* __restrict__ offset_ptr) {
  if (offset_ptr) offset += (uint64_t)*offset_ptr;
  const long groups = (n + 7) / 8;
  for (long g = (long)blockIdx.x * kThreads + threadIdx.x; g < groups; g += (long)gridDim.x * kThreads) {
    const uint4 bits = philox4x32(make_uint4((uint32_t)g, (uint32_t)(g >> 32), (uint32_t)offset,
                                             (uint32_t)(offset >> 32)), seed);
    const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
    const long j0 = g * 8;
    if (j0 + 8 <= n) {
      float v[8], r[8];
      load8(x + j0, v);
      if (RESIDUAL) load8(residual + j0, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t u = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
        v[j] = u >= cut ? v[j] * scale : 0.f;
        if (RESIDUAL) v[j] += r[j];
      }
      store8(y + j0, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j0 + j < n) {
          const uint32_t u = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
          float v = u >= cut ? to_f32(x[j0 + j]) * scale : 0.f;
          if (RESIDUAL) v += to_f32(residual[j0 + j]);
          y[j0 + j] = from_f32<T>(v);
        }
      }
    }
  }
}

}  // namespace

int dropout_apply(const DropoutArgs& a, cudaStream_t s) {
  if (a.n == 0) return 0;
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const long blocks = std::min<long>(((a.n + 7) / 8 + kThreads - 1) / kThreads, 8L * sms);
  const float scale = 65536.0f / (float)(65536u - a.cut);
  const uint2 seed = make_uint2((uint32_t)a.seed, (uint32_t)(a.seed >> 32));
  return with_dtype(a.dtype, [&](auto v) {
    using T = decltype(v);
    auto kern = a.residual ? dropout_kernel<T, true> : dropout_kernel<T, false>;
    kern<<<(unsigned)blocks, kThreads, 0, s>>>((const T*)a.x, (const T*)a.residual, (T*)a.out, a.n, a.cut, scale, seed,
                                               a.offset, a.offset_ptr);
    return (int)cudaGetLastError();
  });
}

}  // namespace mt
