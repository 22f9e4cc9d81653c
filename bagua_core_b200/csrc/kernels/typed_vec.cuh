// Floating-point elements in registers as fp32: eight neighbours loaded and stored 16 bytes at a time, pairs computed together.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace bagua {
namespace kernels {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Two fp32 values that are added or multiplied by one instruction, each rounded as alone.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ float2 halves(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Pair add(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The elements as they lie in memory.
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* at) {
  Raw8<T> r;
#pragma unroll
  for (int k = 0; k < (int)sizeof(T) / 2; ++k) r.v[k] = reinterpret_cast<const uint4*>(at)[k];
  return r;
}
template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float (&f)[8]) {
  const T* x = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = to_float(x[k]);
}
template <typename T>
__device__ __forceinline__ Raw8<T> narrow8(const float (&f)[8]) {
  Raw8<T> r;
  T* x = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = from_float<T>(f[k]);
  return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* at, const Raw8<T>& r) {
#pragma unroll
  for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(at)[k] = r.v[k];
}

}  // namespace kernels
}  // namespace bagua
