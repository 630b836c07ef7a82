// Two f32 an instruction, which sm_100a has for sums and products, and what else goes with it.
#pragma once
#include <cuda_runtime.h>

namespace omni {

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\nfma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// The largest of three; a NaN among them stays.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x on the pipe that multiplies, to 1.02e-4 of the value: x = n + f with n whole and |f| <= 1/2, and 2^f from the cubic with value 1
// at 0 whose largest relative error there is smallest. 0 from -127 down; x below 128. A NaN comes out as a number.
__device__ __forceinline__ float2 exp2_cubic(float2 x) {
  const float kWhole = 12582912.f;  // 1.5 * 2^23: a sum with it has n in its low bits
  const float2 y = make_float2(fmaxf(x.x, -127.f), fmaxf(x.y, -127.f));
  const float2 t = add2(y, both(kWhole)), f = fma2(add2(t, both(-kWhole)), both(-1.f), y);
  float2 p = fma2(f, both(0.05500905960798264f), both(0.2422109693288803f));
  p = fma2(p, f, both(0.6932829022407532f));
  p = fma2(p, f, both(1.f));
  return make_float2(__int_as_float((__float_as_int(t.x) << 23) + __float_as_int(p.x)), __int_as_float((__float_as_int(t.y) << 23) + __float_as_int(p.y)));
}

}  // namespace omni
