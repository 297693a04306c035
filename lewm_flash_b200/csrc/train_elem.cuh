// Element types and packed float32 pairs of the training operators.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace lewm {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Two float32 values in a register pair; the packed instructions of sm_100 do both at once, each
// rounded like the single one.
struct F2 {
  unsigned long long u;
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.u) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ F2 f2(float v) { return f2(v, v); }
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.u));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(a.u), "l"(b.u), "l"(c.u));
  return r;
}
__device__ __forceinline__ float both(F2 a) {
  const float2 v = split(a);
  return v.x + v.y;
}

// A pair of consecutive elements from and to 32 or 64 bits.
__device__ __forceinline__ F2 unpack(const float* q) { return f2(q[0], q[1]); }
__device__ __forceinline__ F2 unpack(const __nv_bfloat16* q) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(q);
  return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ F2 unpack(const __half* q) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(q));
  return f2(v.x, v.y);
}
__device__ __forceinline__ void pack(float* q, F2 a) {
  const float2 v = split(a);
  q[0] = v.x, q[1] = v.y;
}
__device__ __forceinline__ void pack(__nv_bfloat16* q, F2 a) {
  const float2 v = split(a);
  *reinterpret_cast<__nv_bfloat162*>(q) = __floats2bfloat162_rn(v.x, v.y);
}
__device__ __forceinline__ void pack(__half* q, F2 a) {
  const float2 v = split(a);
  *reinterpret_cast<__half2*>(q) = __floats2half2_rn(v.x, v.y);
}

// E consecutive elements moved as one access.
template <typename T, int E>
struct alignas(sizeof(T) * E) Vec {
  T v[E];
};

}  // namespace lewm
