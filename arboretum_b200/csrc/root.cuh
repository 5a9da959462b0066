// Pairs of floats in one instruction, and the square root of a pair.
#pragma once
#include <cuda_runtime.h>

namespace arb {

// two float operations in one instruction, each rounded like the single one
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{.reg .b64 x, y, z, w; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 w, x, y, z; "
      "mov.b64 {%0, %1}, w;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
// a + b as a * one + b: of a packed product and a packed sum the assembler makes one operation with one
// rounding, whatever it is told; `one` is 1 that it does not know of
__device__ __forceinline__ float2 add2(float2 a, float2 b, float one) { return fma2(a, make_float2(one, one), b); }
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// Root of v >= 0, rounded to the nearest like sqrtf: the hardware's reciprocal root q gives s = v q, and
// the residual v - s^2, exact in a fused multiply-add, corrects it by half of itself times q (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", IBM J. Res. Develop. 34,
// 1990).  A third of sqrtf's instructions.  Equal to sqrtf on all of
// [2^-100, 2^126], every float of it; the others take sqrtf.
__device__ __forceinline__ float2 root_of(float2 v) {
  float2 q;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(q.x) : "f"(v.x));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(q.y) : "f"(v.y));
  const float2 s = mul2(v, q);
  return fma2(fma2(mul2(s, both(-1.0f)), s, v), mul2(q, both(0.5f)), s);
}
// bits of the largest and of the smallest value
__device__ __forceinline__ bool root_is_plain(unsigned largest, unsigned smallest) {
  return largest <= 0x7E800000u && smallest >= 0x0D800000u;  // 2^126, 2^-100
}

}  // namespace arb
