// kvcache.cuh -- layout and decoding of the paged 4-bit key/value cache, shared
// by its kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"

namespace wh {

struct KvCacheDev {
  int blocks, page, kv_heads, head_dim;
  int shared;  // the values are the keys
  int page_shift;  // log2(page), -1 where page is no power of two
  uint8_t *keys, *key_scales, *values, *value_scales;
  long long block_stride, scale_block_stride;  // bytes
};

// Which of a request's blocks holds row i.
__device__ __forceinline__ int kv_page_of(const KvCacheDev& c, int i) {
  return c.page_shift >= 0 ? i >> c.page_shift : i / c.page;
}

constexpr uint32_t kKvScaleNan = 253;  // scale bytes from here on: the block is not finite

// The scale a byte stands for, NaN from kKvScaleNan on.
__device__ __forceinline__ float kv_scale(uint32_t b) {
  return b >= kKvScaleNan ? __uint_as_float(0x7fc00000u) : decode_ue8m0(b);
}
// One byte of codes -> the two OCP E2M1 values, low nibble first.
__device__ __forceinline__ float2 e2m1x2_to_f2(uint32_t byte) {
  uint32_t h;
  asm("{ .reg .b8 t; cvt.u8.u32 t, %1; cvt.rn.f16x2.e2m1x2 %0, t; }" : "=r"(h) : "r"(byte));
  return h2_to_f2(h);
}
// 8 codes of one block of 32 (code i in bits 4i..4i+3) -> values
__device__ __forceinline__ void kv_decode8(uint32_t w, uint32_t scale_byte, float (&v)[8]) {
  const float s = kv_scale(scale_byte);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = e2m1x2_to_f2((w >> (8 * j)) & 0xFFu);
    v[2 * j] = __fmul_rn(f.x, s);
    v[2 * j + 1] = __fmul_rn(f.y, s);
  }
}

// 8 consecutive elements, 16-byte aligned, as they lie in memory
template <class T>
struct KvRaw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void widen(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (std::is_same<T, float>::value) {
          v[(4 * i + j) & 7] = __uint_as_float(x[j]);
        } else if (std::is_same<T, __nv_bfloat16>::value) {
          v[2 * j] = __uint_as_float(x[j] << 16);
          v[2 * j + 1] = __uint_as_float(x[j] & 0xFFFF0000u);
        } else {
          const float2 f = h2_to_f2(x[j]);
          v[2 * j] = f.x;
          v[2 * j + 1] = f.y;
        }
      }
    }
  }
};
template <class T>
__device__ __forceinline__ void kv_load8(const T* p, float (&v)[8]) {
  KvRaw8<T> r;
  r.load(p);
  r.widen(v);
}
__device__ __forceinline__ void kv_store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void kv_store8(__nv_bfloat16* p, const float (&v)[8]) {
  union { uint4 u; __nv_bfloat162 h[4]; } o;
#pragma unroll
  for (int j = 0; j < 4; ++j) o.h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<uint4*>(p) = o.u;
}
__device__ __forceinline__ void kv_store8(__half* p, const float (&v)[8]) {
  union { uint4 u; __half2 h[4]; } o;
#pragma unroll
  for (int j = 0; j < 4; ++j) o.h[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<uint4*>(p) = o.u;
}
// 4 consecutive elements of x * by, aligned to their size
__device__ __forceinline__ void kv_store4(float* p, const float4& x, float by) {
  *reinterpret_cast<float4*>(p) = make_float4(x.x * by, x.y * by, x.z * by, x.w * by);
}
__device__ __forceinline__ void kv_store4(__nv_bfloat16* p, const float4& x, float by) {
  union { uint2 u; __nv_bfloat162 h[2]; } o;
  o.h[0] = __floats2bfloat162_rn(x.x * by, x.y * by);
  o.h[1] = __floats2bfloat162_rn(x.z * by, x.w * by);
  *reinterpret_cast<uint2*>(p) = o.u;
}
__device__ __forceinline__ void kv_store4(__half* p, const float4& x, float by) {
  union { uint2 u; __half2 h[2]; } o;
  o.h[0] = __floats2half2_rn(x.x * by, x.y * by);
  o.h[1] = __floats2half2_rn(x.z * by, x.w * by);
  *reinterpret_cast<uint2*>(p) = o.u;
}

}  // namespace wh
