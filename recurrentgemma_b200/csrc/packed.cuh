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
