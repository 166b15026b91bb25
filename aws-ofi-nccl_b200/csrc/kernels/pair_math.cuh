// Pairs of floats, on which one instruction of the float units works, and quotients and roots of them from the units' approximations.
#pragma once
#include <cuda_runtime.h>
#include <math.h>

namespace b200 {

// Two floats in a register pair: an instruction of the float units works on both, each rounded as by itself.
struct Pair {
  unsigned long long bits;
  Pair() = default;
  __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void to(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(bits)); }
};
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return r;
}
__device__ __forceinline__ Pair both(float a) { return Pair(a, a); }
__device__ __forceinline__ Pair both(float2 a) { return Pair(a.x, a.y); }

// The largest of three magnitudes, a NaN if there is one
__device__ __forceinline__ float largest(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}
__device__ __forceinline__ float reciprocal_root(float v) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(v));
  return y;
}
__device__ __forceinline__ float reciprocal(float v) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(v));
  return y;
}
// 1 / v for 2^-110 < v < 2^120, rounded as IEEE's: one Newton step from the unit's reciprocal (as minus_roots; of all floats of that range none
// differs: csrc/tests/gpu_pair_math.cu looks at each)
__device__ __forceinline__ float inverse(float v) {
  const float y = reciprocal(v);
  return fmaf(fmaf(-v, y, 1.f), y, y);
}

// The negative roots of pairs of numbers, given as -v: one Newton step from the unit's reciprocal root y, v y + (v - (v y)^2) y / 2, whose residual a fused
// multiply-add has exactly (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990), with the sign of v
// so that nothing has to be negated. What is left of y's error is its square, 2^-44 of the root: of all floats from 2^-100 on none differs from IEEE's
// root (gpu_pair_math.cu). Below, 2^-126 counts beside them: the root of 2^-115 is off by an ulp, that of 2^-126 by an eighth.
__device__ __forceinline__ Pair minus_roots(Pair minus_v) {
  float a, b;   // zero gets a reciprocal root that is finite
  fma2(minus_v, both(1.f), both(-0x1p-126f)).to(a, b);
  const Pair y(reciprocal_root(fabsf(a)), reciprocal_root(fabsf(b))), g = minus_v * y;
  return fma2(fma2(g, g, minus_v), y * both(0.5f), g);
}
// The same for any number: small ones are scaled by 2^100.
__device__ __forceinline__ Pair any_minus_roots(Pair minus_v, Pair plain) {
  float a, b, lo, hi, x, y;
  minus_v.to(a, b);
  plain.to(x, y);
  (minus_roots(minus_v * both(0x1p100f)) * both(0x1p-50f)).to(lo, hi);
  x = a == -INFINITY ? -INFINITY : a > -0x1p-100f ? lo : x;
  y = b == -INFINITY ? -INFINITY : b > -0x1p-100f ? hi : y;
  return Pair(x, y);
}

}  // namespace b200
