// vec_io.cuh -- eight-element loads and stores of bf16 / fp16 / fp32 with fp32 values.
//
// Eight 16-bit elements are one 16-byte access, eight fp32 elements two.  Pointers
// are 16-byte aligned.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "sm100.cuh"

namespace mt {

// Raw registers of eight elements, so that loads can be issued ahead of their conversion.
template <class T>
struct Raw8 {
  uint4 q[sizeof(T) * 8 / 16];
};

template <class T>
__device__ __forceinline__ Raw8<T> ldraw8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) * 8 / 16); ++i) r.q[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <class T>
__device__ __forceinline__ void straw8(T* p, const Raw8<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) * 8 / 16); ++i) reinterpret_cast<uint4*>(p)[i] = r.q[i];
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16>& r, float* f) {
  const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 t = unpack_bf16x2(w[j]);
    f[2 * j] = t.x;
    f[2 * j + 1] = t.y;
  }
}
__device__ __forceinline__ void unpack8(const Raw8<__half>& r, float* f) {
  const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
    f[2 * j] = t.x;
    f[2 * j + 1] = t.y;
  }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[4 * i] = __uint_as_float(r.q[i].x);
    f[4 * i + 1] = __uint_as_float(r.q[i].y);
    f[4 * i + 2] = __uint_as_float(r.q[i].z);
    f[4 * i + 3] = __uint_as_float(r.q[i].w);
  }
}

__device__ __forceinline__ void pack8(const float* f, Raw8<__nv_bfloat16>& r) {
  r.q[0] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void pack8(const float* f, Raw8<__half>& r) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
    w[j] = *reinterpret_cast<const uint32_t*>(&h);
  }
  r.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack8(const float* f, Raw8<float>& r) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    r.q[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                        __float_as_uint(f[4 * i + 3]));
}

template <class T>
__device__ __forceinline__ void load8(const T* p, float* f) {
  unpack8(ldraw8(p), f);
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float* f) {
  Raw8<T> r;
  pack8(f, r);
  straw8(p, r);
}

// Calls fn with a value of the element type that `dtype` (mt::DType) names.
template <class F>
int with_dtype(int dtype, F&& fn) {
  switch (dtype) {
    case 0: return fn(__nv_bfloat16{});
    case 1: return fn(__half{});
    case 2: return fn(float{});
  }
  return -1;
}

}  // namespace mt
