// Floating-point elements of host memory: widened to fp32 when loaded, rounded once when stored.
#pragma once

#include <cstdint>
#include <cstring>
#include <string>

#include "../common.h"

namespace bagua {
namespace kernels {

inline float bf16_to_float(uint16_t v) {
  uint32_t u = (uint32_t)v << 16;
  float f;
  std::memcpy(&f, &u, 4);
  return f;
}
inline uint16_t float_to_bf16(float f) {
  uint32_t u;
  std::memcpy(&u, &f, 4);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40);  // NaN
  uint32_t rounding = 0x7fffu + ((u >> 16) & 1u);
  return (uint16_t)((u + rounding) >> 16);
}

template <DType D>
struct Elem;
template <>
struct Elem<DType::F32> {
  using T = float;
  static float ld(const T* p) { return *p; }
  static void st(T* p, float v) { *p = v; }
};
template <>
struct Elem<DType::F16> {
  using T = _Float16;
  static float ld(const T* p) { return (float)*p; }
  static void st(T* p, float v) { *p = (_Float16)v; }
};
template <>
struct Elem<DType::BF16> {
  using T = uint16_t;
  static float ld(const T* p) { return bf16_to_float(*p); }
  static void st(T* p, float v) { *p = float_to_bf16(v); }
};

template <typename F>
void dispatch_float(DType dt, F&& f) {
  switch (dt) {
    case DType::F32: f(Elem<DType::F32>{}); return;
    case DType::F16: f(Elem<DType::F16>{}); return;
    case DType::BF16: f(Elem<DType::BF16>{}); return;
    default:
      throw BaguaError(ErrorKind::Tensor, std::string("kernel does not support dtype ") + dtype_name(dt));
  }
}

}  // namespace kernels
}  // namespace bagua
