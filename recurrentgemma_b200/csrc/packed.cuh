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
__device__ __forceinline__ Pair exp2_pair(Pair x) {
  const float2 v = split(x);
  return pair(exp2_fast(v.x), exp2_fast(v.y));
}
// 2^x of a pair for what is multiplied up over many steps: for |x| <= 1/2 a polynomial of degree 6 with constant term 1,
// fitted for the smallest largest relative error (2.0e-9; in float32 arithmetic 7.7e-8, 2.7e-8 rms and none on average, where
// the hardware's exponential is 2e-8 too small near 0); beyond that, where half of what there was is gone after a step
// or two, the hardware's.
__device__ __forceinline__ Pair exp2_exact(Pair x) {
  Pair q = pair(0.00015353361959569156f, 0.00015353361959569156f);
  q = fma2(q, x, pair(0.0013398875016719103f, 0.0013398875016719103f));
  q = fma2(q, x, pair(0.00961843691766262f, 0.00961843691766262f));
  q = fma2(q, x, pair(0.055503323674201965f, 0.055503323674201965f));
  q = fma2(q, x, pair(0.24022647738456726f, 0.24022647738456726f));
  q = fma2(q, x, pair(0.6931471824645996f, 0.6931471824645996f));
  q = fma2(q, x, pair(1.0f, 1.0f));
  const float2 v = split(x), near = split(q), far = split(exp2_pair(x));
  return pair(fabsf(v.x) <= 0.5f ? near.x : far.x, fabsf(v.y) <= 0.5f ? near.y : far.y);
}
// e^v by the hardware's exponential, with what rounding v log2(e) has left out put back (1e-7 of e^-7 without).  Zero below
// -104, and as of 88 above it.
constexpr float kLog2eLow = 1.92596299e-8f, kLn2 = 0.69314718056f;              // log2(e) - kLog2e
__device__ __forceinline__ float exp_bounded(float v) {          // (no differences of infinities; a NaN stays one)
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(-104.0f));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(88.0f));
  return v;
}
__device__ __forceinline__ float exp_exact(float v) {
  v = exp_bounded(v);
  const float arg = v * kLog2e, r = exp2_fast(arg);
  return fmaf(r, kLn2 * fmaf(v, kLog2eLow, fmaf(v, kLog2e, -arg)), r);
}
__device__ __forceinline__ Pair exp_exact(float v0, float v1) {
  const Pair v = pair(exp_bounded(v0), exp_bounded(v1)), log2e = pair(kLog2e, kLog2e);
  const Pair arg = mul2(v, log2e), r = exp2_pair(arg);
  const Pair low = fma2(v, pair(kLog2eLow, kLog2eLow), fma2(v, log2e, mul2(arg, pair(-1.0f, -1.0f))));
  return fma2(r, mul2(low, pair(kLn2, kLn2)), r);
}

__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// silu by the hardware's exponential and reciprocal, of a pair or of one; kExact: with exp_exact, 1.1 units of 2^-24 off on
// average whatever the size of v (without, 1.1 for v of N(0, 1) and 3.8 for v of up to 20).
template <bool kExact = false> __device__ __forceinline__ float2 silu_fast(float v0, float v1) {
  const Pair e = kExact ? exp_exact(-v0, -v1) : exp2_pair(mul2(pair(v0, v1), pair(-kLog2e, -kLog2e)));
  const float2 below = split(add2(e, pair(1.0f, 1.0f)));
  return split(mul2(pair(v0, v1), pair(rcp_fast(below.x), rcp_fast(below.y))));
}
template <bool kExact> __device__ __forceinline__ float silu_fast(float v) {
  return v * rcp_fast(1.0f + (kExact ? exp_exact(-v) : exp2_fast(v * -kLog2e)));
}

}  // namespace rgk
