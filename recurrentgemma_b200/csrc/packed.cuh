// float32 arithmetic on pairs, and the hardware exponential, for the kernels of the state space layer.
#pragma once

#include <stdint.h>

namespace rgk {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two float32 operations in one instruction, on pairs as they lie in memory: half the issue slots of the same work
// (the multiply-add pipe itself takes as long for a pair as for two).
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 split(Pair v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of a pair on the multiply-add pipe: x = n + f with n from the low bits of a sum with 1.5 2^23 (+ 126, so that they
// are the exponent of 2^(n-1)), times 2^(f+1) as a polynomial of degree 5 with constant term 2, fitted on [-1/2, 1/2] for the
// smallest largest relative error (9.1e-8; 1.6e-7 in float32 arithmetic, and on average none near 0, where the hardware's
// exponential is 2e-8 too small).  Infinite from 2^128, zero below 2^-125.5; a NaN stays one.
__device__ __forceinline__ float exponent_range(float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(-126.0f));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(r) : "f"(128.0f));
  return r;
}
__device__ __forceinline__ Pair exp2_poly(Pair x) {
  constexpr float kMagic = 12583038.0f;
  const float2 v = split(x);
  x = pair(exponent_range(v.x), exponent_range(v.y));
  const Pair r = add2(x, pair(kMagic, kMagic));
  const Pair f = add2(x, fma2(r, pair(-1.0f, -1.0f), pair(kMagic, kMagic)));
  Pair q = pair(0.002652945462614298f, 0.002652945462614298f);
  q = fma2(q, f, pair(0.019343025982379913f, 0.019343025982379913f));
  q = fma2(q, f, pair(0.11101467162370682f, 0.11101467162370682f));
  q = fma2(q, f, pair(0.48044484853744507f, 0.48044484853744507f));
  q = fma2(q, f, pair(1.3862940073013306f, 1.3862940073013306f));
  q = fma2(q, f, pair(2.0f, 2.0f));
  const float2 n = split(r);
  return mul2(q, pair(__uint_as_float(__float_as_uint(n.x) << 23), __uint_as_float(__float_as_uint(n.y) << 23)));
}
__device__ __forceinline__ Pair exp2_pair(Pair x) {
  const float2 v = split(x);
  return pair(exp2_fast(v.x), exp2_fast(v.y));
}

__device__ __forceinline__ float2 silu_fast(float v0, float v1) {
  const float2 arg = split(mul2(pair(v0, v1), pair(-kLog2e, -kLog2e)));
  float r0, r1;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(1.0f + exp2_fast(arg.x)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(1.0f + exp2_fast(arg.y)));
  return split(mul2(pair(v0, v1), pair(r0, r1)));
}

}  // namespace rgk
