// The arithmetic of an AdamW step on one element, and the 8-bit form of its moments, for host and device.
#pragma once

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

// A bijection of 32 bits, shifts and odd multipliers in turn, whose every output bit depends on every input bit.
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
BAGUA_HD uint32_t random_bits(uint32_t key, int64_t i) {
  return mix((uint32_t)i * 0x9e3779b9u + key + (uint32_t)((uint64_t)i >> 32) * 0x85ebca77u);
}

// A code's 7 or 8 bits, moved to where fp32 has its fraction and the low end of its exponent, are the code's value times 2^-120:
// codes with exponent 0 become fp32's own subnormal numbers.  The way back is a shift too, and adding random bits below the cut
// before it is the stochastic rounding, for codes of every exponent alike.
constexpr float kUp = 0x1p120f, kDown = 0x1p-120f, kLargest1 = 480.f, kLargest2 = 496.f, kSmallestScale = 0x1p-126f;

BAGUA_HD float decode1(uint32_t code, float scale) {  // scale: the block's
  return bits_float(((code & 0x7fu) << 20) | ((code & 0x80u) << 24)) * kUp * scale;
}
BAGUA_HD float decode2(uint32_t code, float scale) { return bits_float(code << 19) * kUp * scale; }

// The scale of a block whose largest value is `top`, as bits of a number that is not negative; its reciprocal in `per`.
BAGUA_HD float block_scale(uint32_t top, float largest, float* per) {
  if (top >= 0x7f800000u) {
    *per = 0.f;
    return bits_float(0x7fc00000u);
  }
  float s = bits_float(top) / largest;
  s = s < kSmallestScale ? kSmallestScale : s;
  *per = 1.f / s;
  return top ? s : 0.f;
}
// y = x / scale, at most the largest value but for a rounding.
BAGUA_HD uint32_t encode1(float x, float per, uint32_t random) {
  const uint32_t b = float_bits(x * per * kDown);
  uint32_t c = ((b & 0x7fffffffu) + ((random & 0xffffu) << 4) + 8u) >> 20;
  c = c > 0x7fu ? 0x7fu : c;
  return c | (b >> 31 << 7);
}
BAGUA_HD uint32_t encode2(float x, float per, uint32_t random) {
  uint32_t c = (float_bits(x * per * kDown) + ((random >> 16) << 3) + 4u) >> 19;
  c = c > 0xffu ? 0xffu : c;
  return c == 0u && x > 0.f ? 1u : c;
}

BAGUA_HD Hyper make_hyper(const GroupValues& g, int64_t step, uint64_t seed) {
  Hyper h;
  h.keep = (float)(1.0 - g.lr * g.weight_decay);
  h.rate = (float)(g.lr / (1.0 - pow(g.b1, (double)step)));
  h.root = (float)(1.0 / sqrt(1.0 - pow(g.b2, (double)step)));
  h.eps = (float)g.eps;
  h.b1 = (float)g.b1;
  h.c1 = (float)(1.0 - g.b1);
  h.b2 = (float)g.b2;
  h.c2 = (float)(1.0 - g.b2);
  h.random = step_random(seed, step);
  return h;
}

// Both moments' new values and the parameter's.
BAGUA_HD void update(const Hyper& h, float& p, float g, float& m, float& v) {
#ifdef __CUDA_ARCH__
  // multiply-adds spelled out: which of two products is rounded is not left to the compiler
  m = __fmaf_rn(h.c1, g, __fmul_rn(h.b1, m));
  v = __fmaf_rn(__fmul_rn(h.c2, g), g, __fmul_rn(h.b2, v));
  const float d = __fmaf_rn(__fsqrt_rn(v), h.root, h.eps);
  p = __fmaf_rn(p, h.keep, -__fmul_rn(h.rate, __fdiv_rn(m, d)));
#else
  m = __builtin_fmaf(h.c1, g, h.b1 * m);
  v = __builtin_fmaf(h.c2 * g, g, h.b2 * v);
  const float d = __builtin_fmaf(__builtin_sqrtf(v), h.root, h.eps);
  p = __builtin_fmaf(p, h.keep, -(h.rate * (m / d)));
#endif
}

}  // namespace adamw
}  // namespace bagua
