// The arithmetic of an AdamW step on one element, and the 8-bit form of its moments, for host and device.
#pragma once

#ifdef __CUDACC__
#include <cuda_runtime.h>
#endif

#include <cmath>
#include <cstdint>
#include <cstring>

#include "adamw.h"

#ifdef __CUDACC__
#define BAGUA_HD __host__ __device__ __forceinline__
#else
#define BAGUA_HD inline
#endif

namespace bagua {
namespace adamw {

BAGUA_HD uint32_t float_bits(float x) {
#ifdef __CUDA_ARCH__
  return __float_as_uint(x);
#else
  uint32_t u;
  std::memcpy(&u, &x, 4);
  return u;
#endif
}
BAGUA_HD float bits_float(uint32_t u) {
#ifdef __CUDA_ARCH__
  return __uint_as_float(u);
#else
  float x;
  std::memcpy(&x, &u, 4);
  return x;
#endif
}

// A bijection of 32 bits, shifts and odd multipliers in turn, whose every output bit depends on every input bit: the published hash
// lowbias32, whose constants C. Wellons found by a search for the least bias (2018, in the public domain).
BAGUA_HD uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}
// What the tensors of a step take their keys from, and the key of the k-th.
BAGUA_HD uint32_t step_random(uint64_t seed, int64_t step) {
  uint32_t x = mix((uint32_t)seed);
  if (seed >> 32) x = mix(x ^ (uint32_t)(seed >> 32));
  return mix(x + (uint32_t)step);
}
BAGUA_HD uint32_t segment_key(uint32_t random, uint32_t k) { return mix(random + k); }
// 32 random bits of element i of a tensor: the low half rounds the first moment, the high half the second.
constexpr uint32_t kStride = 0x9e3779b9u;  // between the numbers that neighbouring elements' bits are made from
BAGUA_HD uint32_t random_base(uint32_t key, int64_t i) { return (uint32_t)i * kStride + key + (uint32_t)((uint64_t)i >> 32) * 0x85ebca77u; }
BAGUA_HD uint32_t random_bits(uint32_t key, int64_t i) { return mix(random_base(key, i)); }

// A code's 7 or 8 bits, moved to where fp32 has its fraction and the low end of its exponent, are the code's value times 2^-120:
// codes with exponent 0 become fp32's own subnormal numbers.  The way back is a shift too, and adding random bits below the cut
// before it is the stochastic rounding, for codes of every exponent alike.
constexpr float kUp = 0x1p120f, kDown = 0x1p-120f, kLargest1 = 480.f, kLargest2 = 496.f, kSmallestScale = 0x1p-126f;
// Scales below this can be multiplied by 2^120, their reciprocals by 2^-120, without leaving fp32's range: the products with a block's
// elements then take one factor instead of two.
constexpr float kPlainScale = 64.f;

// A code's bits, to be multiplied by 2^120 and its block's scale.
BAGUA_HD float code1_bits(uint32_t code) { return bits_float(((code & 0x7fu) << 20) | ((code & 0x80u) << 24)); }
BAGUA_HD float code2_bits(uint32_t code) { return bits_float(code << 19); }
BAGUA_HD float decode1(uint32_t code, float scale) { return code1_bits(code) * kUp * scale; }
BAGUA_HD float decode2(uint32_t code, float scale) { return code2_bits(code) * kUp * scale; }

// The scale of a block whose largest value is `top`, as bits of a number that is not negative; its reciprocal in `per`.
BAGUA_HD float block_scale(uint32_t top, float largest, float* per) {
  if (top >= 0x7f800000u) {
    *per = 0.f;
    return bits_float(0x7fc00000u);
  }
  float s = bits_float(top) * (1.f / largest);
  s = s < kSmallestScale ? kSmallestScale : s;
  *per = 1.f / s;
  return top ? s : 0.f;
}
// y = x / scale times 2^-120, at most the largest value but for a rounding.
BAGUA_HD float scaled(float x, float per, bool plain) { return plain ? x * (per * kDown) : x * per * kDown; }
BAGUA_HD uint32_t sum_up_to(uint32_t a, uint32_t b, uint32_t most) {
#ifdef __CUDA_ARCH__
  return __viaddmin_u32(a, b, most);
#else
  return a + b < most ? a + b : most;
#endif
}
// y, at least 0, with random bits added.  Neither sum leaves 32 bits, for a y that is not finite either.
constexpr uint32_t kLastBits = 0x07ffffffu;  // those of both largest codes, and of what is cut off
BAGUA_HD uint32_t sum1(float y, uint32_t random) { return sum_up_to(float_bits(y), (random << 4 & 0xffff0u) | 8u, kLastBits); }
BAGUA_HD uint32_t sum2(float y, uint32_t random) { return sum_up_to(float_bits(y), (random >> 13 & 0x7fff8u) | 4u, kLastBits); }
// The codes, of a moment x with the sign (first) or above 0 (second).
BAGUA_HD uint32_t cut1(uint32_t sum, float x) { return sum >> 20 | (float_bits(x) >> 24 & 0x80u); }
BAGUA_HD uint32_t cut2(uint32_t sum, float x) {
  const uint32_t c = sum >> 19, least = float_bits(x) < 1u ? float_bits(x) : 1u;  // 1 unless x is 0
  return c > least ? c : least;
}
// How far a sum lies above the last border but kSlack, all bits of what is cut off at the top: less than kNear1 or kNear2 if the border
// is nearer than kSlack steps of fp32.  y is off by 15 half steps at most: the moments' 5 (a first moment without cancellation), the
// scale's 6 (their largest's 4, the factor, the product) with its own two in the definition, its reciprocal and the product with it.
constexpr uint32_t kSlack = 16, kNear1 = 2 * kSlack << 12, kNear2 = 2 * kSlack << 13;
BAGUA_HD uint32_t above1(uint32_t sum) { return (sum << 12) + (kSlack << 12); }
BAGUA_HD uint32_t above2(uint32_t sum) { return (sum << 13) + (kSlack << 13); }

BAGUA_HD Hyper make_hyper(const GroupValues& g, int64_t step, uint64_t seed) {
  Hyper h;
  // (the first one nearer to 0, so that both have the sign of their sum: an infinite parameter, as a mask may be, stays so)
  const double keep = 1.0 - g.lr * g.weight_decay;
  h.keep = (float)keep;
  if (fabs((double)h.keep) >= fabs(keep) && h.keep != 0) h.keep = bits_float(float_bits(h.keep) - 1);
  h.rest = (float)(keep - h.keep);
  h.rate = (float)(g.lr / (1.0 - pow(g.b1, (double)step)));
  h.root = (float)(1.0 / sqrt(1.0 - pow(g.b2, (double)step)));
  h.eps = (float)g.eps;
  h.b1 = (float)g.b1;
  h.c1 = (float)(1.0 - g.b1);
  h.b2 = (float)g.b2;
  h.c2 = (float)(1.0 - g.b2);
  h.random = step_random(seed, step);
  h.beta1 = g.b1;
  h.beta2 = g.b2;
  return h;
}

// Products and multiply-adds spelled out: which of two products is rounded is not left to the compiler.
BAGUA_HD float product(float a, float b) {
#ifdef __CUDA_ARCH__
  return __fmul_rn(a, b);
#else
  return a * b;
#endif
}
BAGUA_HD float multiply_add(float a, float b, float c) {
#ifdef __CUDA_ARCH__
  return __fmaf_rn(a, b, c);
#else
  return __builtin_fmaf(a, b, c);
#endif
}
// The new moments, from the old ones times their betas.
BAGUA_HD void moments(const Hyper& h, float g, float b1_m, float b2_v, float& m, float& v) {
  m = multiply_add(h.c1, g, b1_m);
  v = multiply_add(product(h.c2, g), g, b2_v);
}
// The same of codes in 64 bits, the scale of a block's largest (rounded to fp32 before the product, as the definition has it), and a
// code (of `fraction` bits behind the exponent) with 16 random bits.
BAGUA_HD double product64(double a, double b) {
#ifdef __CUDA_ARCH__
  return __dmul_rn(a, b);
#else
  return a * b;
#endif
}
BAGUA_HD double multiply_add64(double a, double b, double c) {
#ifdef __CUDA_ARCH__
  return __fma_rn(a, b, c);
#else
  return __builtin_fma(a, b, c);
#endif
}
BAGUA_HD double first64(const Hyper& h, float g, uint32_t code, float scale) {
  return multiply_add64(1.0 - h.beta1, g, product64(product64(code1_bits(code) * kUp, scale), h.beta1));
}
BAGUA_HD double second64(const Hyper& h, float g, uint32_t code, float scale) {
  return multiply_add64(1.0 - h.beta2, product64(g, g), product64(product64(code2_bits(code) * kUp, scale), h.beta2));
}
BAGUA_HD float scale64(float top, float largest, double* per) {
  float s = top * (1.f / largest);
  s = s < kSmallestScale ? kSmallestScale : s;
  *per = 1.0 / s;
  return top > 0 ? s : 0.f;
}
BAGUA_HD double power_of_two(int e) {
#ifdef __CUDA_ARCH__
  return __hiloint2double((1023 + e) << 20, 0);
#else
  return std::ldexp(1.0, e);
#endif
}
BAGUA_HD uint32_t code64(double y, int fraction, uint32_t random) {
  uint64_t bits;
#ifdef __CUDA_ARCH__
  bits = (uint64_t)__double_as_longlong(y);
#else
  std::memcpy(&bits, &y, 8);
#endif
  int e = (int)(bits >> 52) - 1023;
  e = e < -6 ? -6 : e;
  const uint32_t q = (uint32_t)multiply_add64(y, power_of_two(fraction - e), (random + 0.5) * 0x1p-16);
  const uint32_t code = ((uint32_t)(e + 6) << fraction) + q, last = (16u << fraction) - 1;
  return code < last ? code : last;
}
BAGUA_HD uint32_t first_code64(double m, double per, uint32_t random) {
  return code64(m < 0 ? -m * per : m * per, 3, random & 0xffffu) | (m < 0 ? 0x80u : 0u);
}
BAGUA_HD uint32_t second_code64(double v, double per, uint32_t random) {
  const uint32_t c = code64(v * per, 4, random >> 16);
  return c == 0 && (float)v > 0 ? 1 : c;
}
// The new parameter.
BAGUA_HD float parameter(const Hyper& h, float p, float m, float v) {
#ifdef __CUDA_ARCH__
  const float d = __fmaf_rn(__fsqrt_rn(v), h.root, h.eps);
  const float u = __fmul_rn(h.rate, __fdiv_rn(m, d));
#else
  const float d = __builtin_fmaf(__builtin_sqrtf(v), h.root, h.eps);
  const float u = h.rate * (m / d);
#endif
  return multiply_add(p, h.keep, multiply_add(p, h.rest, -u));
}
BAGUA_HD void update(const Hyper& h, float& p, float g, float& m, float& v) {
  moments(h, g, product(h.b1, m), product(h.b2, v), m, v);
  p = parameter(h, p, m, v);
}

}  // namespace adamw
}  // namespace bagua
