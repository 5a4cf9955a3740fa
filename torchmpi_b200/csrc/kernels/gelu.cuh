// GELU (erf form) and its derivative, shared by the elementwise passes (bias_grad.cu) and the GEMM epilogue.
#pragma once
#include <cuda_runtime.h>
#include "attn_util.cuh"

namespace tmpi {

// gelu(z) = z * Phi(z);  d/dz [z * Phi(z)] = Phi(z) + z * phi(z).  Phi through the rational erf approximation of Abramowitz and
// Stegun 7.1.26 (absolute error 1.5e-7), which shares its exp(-z^2 / 2) with phi: one ex2, one rcp and a
// dozen multiply-adds per element where erff() is a few dozen.  Two elements at a time: the multiply-adds are packed
// fp32 pairs, which halves their issue slots (those bound the GEMM epilogue and the elementwise passes alike), and ex2 and
// rcp flush subnormals (an exponential below 2^-126 adds nothing to either result): the GELU backward with the bias
// gradient, 8192 x 4096 bf16, 44 -> 37 us.
__device__ __forceinline__ void normal_parts2(unsigned long long z, unsigned long long* cdf, unsigned long long* e) {
  using namespace attn_util;
  auto both = [](float v) { return pack2(__float_as_uint(v), __float_as_uint(v)); };
  float z0, z1, x0, x1;
  unpack2(z, z0, z1);
  unpack2(mul2(mul2(both(-0.5f * 1.4426950408889634f), z), z), x0, x1);
  *e = pack2(__float_as_uint(ex2(x0)), __float_as_uint(ex2(x1)));
  unpack2(fma2(both(0.3275911f * 0.70710678118654752f), pack2(__float_as_uint(fabsf(z0)), __float_as_uint(fabsf(z1))), both(1.f)), x0, x1);
  const unsigned long long t = pack2(__float_as_uint(rcp(x0)), __float_as_uint(rcp(x1)));
  unsigned long long poly = fma2(both(1.061405429f), t, both(-1.453152027f));
  poly = fma2(poly, t, both(1.421413741f));
  poly = fma2(poly, t, both(-0.284496736f));
  poly = fma2(poly, t, both(0.254829592f));
  const unsigned long long q = mul2(mul2(mul2(both(0.5f), poly), t), *e);                 // 1 - Phi(|z|)
  float q0, q1, p0, p1;
  unpack2(q, q0, q1);
  unpack2(fma2(q, both(-1.f), both(1.f)), p0, p1);
  *cdf = pack2(__float_as_uint(z0 >= 0.f ? p0 : q0), __float_as_uint(z1 >= 0.f ? p1 : q1));
}

__device__ __forceinline__ void gelu_grad2(float z0, float z1, float* g0, float* g1) {
  using namespace attn_util;
  const unsigned long long z = pack2(__float_as_uint(z0), __float_as_uint(z1));
  const unsigned long long c = pack2(__float_as_uint(0.3989422804014327f), __float_as_uint(0.3989422804014327f));
  unsigned long long cdf, e;
  normal_parts2(z, &cdf, &e);
  unpack2(fma2(mul2(z, c), e, cdf), *g0, *g1);
}

__device__ __forceinline__ void gelu_value2(float z0, float z1, float* y0, float* y1) {
  using namespace attn_util;
  const unsigned long long z = pack2(__float_as_uint(z0), __float_as_uint(z1));
  unsigned long long cdf, e;
  normal_parts2(z, &cdf, &e);
  unpack2(mul2(z, cdf), *y0, *y1);
}

// both, from one pass over the normal distribution's parts
__device__ __forceinline__ void gelu_both2(float z0, float z1, float* y0, float* y1, float* g0, float* g1) {
  using namespace attn_util;
  const unsigned long long z = pack2(__float_as_uint(z0), __float_as_uint(z1));
  const unsigned long long c = pack2(__float_as_uint(0.3989422804014327f), __float_as_uint(0.3989422804014327f));
  unsigned long long cdf, e;
  normal_parts2(z, &cdf, &e);
  unpack2(mul2(z, cdf), *y0, *y1);
  unpack2(fma2(mul2(z, c), e, cdf), *g0, *g1);
}

// The same for results that are rounded to 16 bits, in fewer instructions: Phi(z) = 1 / (1 + 2^x) with x = -log2(Phi / (1 - Phi)), an odd and smooth function
// of z, as z times a polynomial of degree 6 in z^2 (least squares made equal-ripple on |z| <= 5; beyond it grows like z^13, so that Phi goes to 0 or
// 1).  No absolute value, no choice between two tails, one exponential: 10 packed operations and 4 of the special-function unit for two elements,
// where the rational form above takes 12, 6 and 4.  Absolute errors in fp32: Phi and slope 1.4e-6, gelu 1.1e-6.
// That is at most a third of a half step of bf16 for gelu down to z = -5 (below it, where gelu is under 2e-6 in magnitude, more), and up to 2.3 half steps of fp16 (at
// -3.6); of the slope, more next to its root at -0.75 alone.
__device__ __forceinline__ unsigned long long quick_cdf2(unsigned long long z, unsigned long long t) {      // t = z^2
  using namespace attn_util;
  auto both = [](float v) { return attn_util::pack2(__float_as_uint(v), __float_as_uint(v)); };
  unsigned long long p = fma2(both(-3.29422556e-09f), t, both(2.84630659e-07f));
  p = fma2(p, t, both(-9.59334011e-06f));
  p = fma2(p, t, both(0.00014446408f));
  p = fma2(p, t, both(0.000148453692f));
  p = fma2(p, t, both(-0.104912885f));
  p = mul2(fma2(p, t, both(-2.30217791f)), z);
  float x0, x1;
  unpack2(p, x0, x1);
  unpack2(add2(pack2(__float_as_uint(ex2(x0)), __float_as_uint(ex2(x1))), both(1.f)), x0, x1);
  return pack2(__float_as_uint(rcp(x0)), __float_as_uint(rcp(x1)));
}
__device__ __forceinline__ unsigned long long quick_gelu2(unsigned long long z) { return attn_util::mul2(z, quick_cdf2(z, attn_util::mul2(z, z))); }
__device__ __forceinline__ void quick_gelu_both2(unsigned long long z, unsigned long long* y, unsigned long long* slope) {
  using namespace attn_util;
  auto both = [](float v) { return attn_util::pack2(__float_as_uint(v), __float_as_uint(v)); };
  const unsigned long long t = mul2(z, z), cdf = quick_cdf2(z, t);
  float x0, x1;
  unpack2(mul2(t, both(-0.5f * 1.4426950408889634f)), x0, x1);
  *y = mul2(z, cdf);
  *slope = fma2(mul2(z, both(0.3989422804014327f)), pack2(__float_as_uint(ex2(x0)), __float_as_uint(ex2(x1))), cdf);
}

}  // namespace tmpi
