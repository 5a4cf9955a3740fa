// The 8-bit form of an activation: 32 consecutive elements of a row share a power of two 2^e, and each is kept as e4m3(x / 2^e).
//
// e is the smallest integer >= -126 for which the largest finite |x| of the block is at most 448 * 2^e, the largest e4m3 number.  With
// |x| = m 2^k, 1 <= m < 2, that is k - 8 for m <= 1.75 and k - 7 above, which the exponent field of |x| + 2^(k-2) gives: adding a quarter
// of 2^k carries into the exponent from m = 1.75 on, so one unit in the last place is taken off first.  Scaling by 2^-e is exact, so a
// value is rounded once, by at most half a step (2^-4 of it, or 2^-10 * 2^e in the subnormal range); what a checkpoint stands for does not depend on
// who computes it.  The scale is one byte, e + 127.  Infinities and NaN are kept as NaN (e4m3 has no infinity): they show in the
// backward pass instead of becoming 448 * 2^e.
#pragma once
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "attn_util.cuh"

namespace tmpi {
namespace act8 {

constexpr int BLOCK = 32;

// the bits of |x|, 0 for what is not finite: the largest of a block decides about its scale (as integers they compare like the values)
__device__ __forceinline__ uint32_t magnitude(float x) {
  const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
  return a < 0x7f800000u ? a : 0u;
}
// e + 127 of the block with the largest magnitude `a`
__device__ __forceinline__ uint32_t scale_byte(uint32_t a) {
  const int k = (int)((a + 0x1fffffu) >> 23);            // biased exponent, one more for m > 1.75
  return (uint32_t)max(k - 8, 1);
}
// 2^-e and 2^e; e + 127 is 1 to 247
__device__ __forceinline__ float inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float value(uint32_t byte) { return __uint_as_float(byte << 23); }

// two elements, `inv` = 2^-e
__device__ __forceinline__ uint32_t pack2(float x0, float x1, float inv) {
  const float nan = __uint_as_float(0x7fffffffu);
  float2 v;
  v.x = fabsf(x0) < __uint_as_float(0x7f800000u) ? x0 * inv : nan;
  v.y = fabsf(x1) < __uint_as_float(0x7f800000u) ? x1 * inv : nan;
  return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ void unpack2(uint32_t q, float scale, float* x0, float* x1) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(q & 0xffffu), __NV_E4M3);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  *x0 = f.x * scale;
  *x1 = f.y * scale;
}

// A whole block by one thread; returns its scale byte.  Where none is infinite, which the maximum tells, the elements need no look of their own (a NaN
// converts to NaN; a maximum leaves it out as long as there is a number).
__device__ __forceinline__ uint32_t pack_block(const float (&x)[32], uint32_t (&q)[8]) {
  float m[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = fmaxf(fmaxf(fabsf(x[8 * j]), fabsf(x[8 * j + 1])), fabsf(x[8 * j + 2]));
    m[j] = fmaxf(fmaxf(m[j], fabsf(x[8 * j + 3])), fabsf(x[8 * j + 4]));
    m[j] = fmaxf(fmaxf(m[j], fabsf(x[8 * j + 5])), fabsf(x[8 * j + 6]));
    m[j] = fmaxf(m[j], fabsf(x[8 * j + 7]));
  }
  uint32_t top = __float_as_uint(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
  const bool finite = top < 0x7f800000u;
  if (!finite) {
    top = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) top = max(top, magnitude(x[j]));
  }
  const uint32_t byte = scale_byte(top);
  const float inv = inverse(byte);
  if (finite) {
    const unsigned long long inv2 = attn_util::pack2(__float_as_uint(inv), __float_as_uint(inv));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t h[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float2 v;
        attn_util::unpack2(attn_util::mul2(attn_util::pack2(__float_as_uint(x[4 * j + 2 * i]), __float_as_uint(x[4 * j + 2 * i + 1])), inv2), v.x, v.y);
        h[i] = __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
      }
      q[j] = h[0] | h[1] << 16;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = pack2(x[4 * j], x[4 * j + 1], inv) | pack2(x[4 * j + 2], x[4 * j + 3], inv) << 16;
  }
  return byte;
}

// 8 elements of a checkpoint
__device__ __forceinline__ void unpack8(uint2 q, float scale, float (&x)[8]) {
  unpack2(q.x, scale, &x[0], &x[1]);
  unpack2(q.x >> 16, scale, &x[2], &x[3]);
  unpack2(q.y, scale, &x[4], &x[5]);
  unpack2(q.y >> 16, scale, &x[6], &x[7]);
}
__device__ __forceinline__ uint2 pack8(const float (&x)[8], float inv) {
  return make_uint2(pack2(x[0], x[1], inv) | pack2(x[2], x[3], inv) << 16, pack2(x[4], x[5], inv) | pack2(x[6], x[7], inv) << 16);
}

// the same where all are finite
__device__ __forceinline__ uint2 pack8_finite(const float (&x)[8], float inv) {
  const unsigned long long inv2 = attn_util::pack2(__float_as_uint(inv), __float_as_uint(inv));
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 v;
    attn_util::unpack2(attn_util::mul2(attn_util::pack2(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1])), inv2), v.x, v.y);
    h[i] = __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

}  // namespace act8
}  // namespace tmpi
