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
// 2^(n+f) of a pair, r = 1.5 2^23 + 126 + n (so that its low bits are the exponent of 2^(n-1)): 2^(n-1) times 2^(f+1) as a
// polynomial of degree 6 with constant term 2, fitted on [-1/2, 1/2] for the smallest largest relative error (2.0e-9; in
// float32 arithmetic 7.7e-8, 2.7e-8 rms and 1e-9 on average, where degree 5 has 1.7e-7, 6.6e-8 rms and -2e-8, and the
// hardware's exponential is 2e-8 too small near 0).
constexpr float kExponent = 12583038.0f;
__device__ __forceinline__ Pair exp2_parts(Pair f, Pair r) {
  Pair q = pair(0.0003070672391913831f, 0.0003070672391913831f);
  q = fma2(q, f, pair(0.0026797750033438206f, 0.0026797750033438206f));
  q = fma2(q, f, pair(0.01923687383532524f, 0.01923687383532524f));
  q = fma2(q, f, pair(0.11100664734840393f, 0.11100664734840393f));
  q = fma2(q, f, pair(0.4804529547691345f, 0.4804529547691345f));
  q = fma2(q, f, pair(1.3862943649291992f, 1.3862943649291992f));
  q = fma2(q, f, pair(2.0f, 2.0f));
  const float2 n = split(r);
  return mul2(q, pair(__uint_as_float(__float_as_uint(n.x) << 23), __uint_as_float(__float_as_uint(n.y) << 23)));
}
__device__ __forceinline__ float clamp_nan(float v, float lo, float hi) {       // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(lo));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(r) : "f"(hi));
  return r;
}
// 2^x on the multiply-add pipe.  Infinite from 2^128, zero below 2^-125.5.
__device__ __forceinline__ Pair exp2_poly(Pair x) {
  const float2 v = split(x);
  x = pair(clamp_nan(v.x, -126.0f, 128.0f), clamp_nan(v.y, -126.0f, 128.0f));
  const Pair r = add2(x, pair(kExponent, kExponent));
  return exp2_parts(add2(x, fma2(r, pair(-1.0f, -1.0f), pair(kExponent, kExponent))), r);
}
// e^v of v up to 89: log2(e) in two terms, so that the rounding of a large argument does not become one of the result
// (1e-7 of e^-7 with one).
__device__ __forceinline__ Pair exp_poly(float v0, float v1) {
  constexpr float kLog2eLow = 1.92596303e-8f;                    // log2(e) - kLog2e
  const Pair v = pair(clamp_nan(v0, -87.33655f, 89.0f), clamp_nan(v1, -87.33655f, 89.0f));
  const Pair r = fma2(v, pair(kLog2e, kLog2e), pair(kExponent, kExponent));
  const Pair n = fma2(r, pair(-1.0f, -1.0f), pair(kExponent, kExponent));       // -n
  return exp2_parts(fma2(v, pair(kLog2eLow, kLog2eLow), fma2(v, pair(kLog2e, kLog2e), n)), r);
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
