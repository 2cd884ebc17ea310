// The selective state space recurrence: N float32 states a channel, each with a decay of its own,
//   D_t = softplus(dt_t + dt_bias),  h_t[n] = exp(D_t a[n]) h_{t-1}[n] + D_t x_t b_t[n],
//   y_t = (sum_n h_t[n] c_t[n] + d x_t) silu(z_t),
// where a document start drops h_{t-1}.  b and c are shared by the channels of a group.
//
// Bound: the special functions.  An (element, state) takes one exponential and four multiply-adds' worth of
// float32 work, and an SM has 16 special-function results a clock but 128 multiply-adds: for 16 states (and
// two functions each for softplus and silu) 168 M elements take 0.75 ms where their bytes take 0.21.
//
// The recurrence runs in time order in registers: L neighbouring lanes share a channel, each with S of its
// states, and time is not split - the lanes are, which leaves no work to do twice.  A CTA walks over tiles of
// 32 time steps: (1) the raw tile, brought in by cp.async while the one before is worked on, becomes D and
// D x in float32 (the softplus once an element, shared by all threads), b and c are widened; (2) the recurrence,
// which reads those as broadcasts and leaves sums over its S states, joined over the L lanes by exchanging
// halves of four time steps (three shuffles for four steps and the first four lanes, not eight); (3) d x, the gate
// and the store, again by element.
#include "rgk_common.cuh"
#include "rgk_internal.h"

namespace rgk {
namespace {

constexpr int kThreads = 128;
constexpr int kTile = 32;                                        // time steps; one bit each in a warp's vote
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// softplus(v) = max(v, 0) + log1p(e), e = exp(-|v|) in (0, 1]: log1p(e) / e by a polynomial fitted for the
// smallest largest relative error on [0, 1] (5e-9; 1.8e-7 in float32 arithmetic).  Steps of 1e-3 come out with their relative
// precision, which the hardware logarithm of 1 + e would lose.
__device__ __forceinline__ float softplus_step(float v) {
  const float e = exp2_fast(-fabsf(v) * kLog2e);
  float p = -0.0032440212089568377f;
  p = fmaf(p, e, 0.01985144428908825f);
  p = fmaf(p, e, -0.056959498673677444f);
  p = fmaf(p, e, 0.10603651404380798f);
  p = fmaf(p, e, -0.15305590629577637f);
  p = fmaf(p, e, 0.1967593878507614f);
  p = fmaf(p, e, -0.24954134225845337f);
  p = fmaf(p, e, 0.3332996368408203f);
  p = fmaf(p, e, -0.4999990165233612f);
  p = fmaf(p, e, 1.0f);
  return fmaf(p, e, v > 0.0f ? v : 0.0f);                        // (a NaN stays one: e is)
}

__device__ __forceinline__ float silu_fast(float v) { return __fdividef(v, 1.0f + exp2_fast(-v * kLog2e)); }

template <typename T> __device__ __forceinline__ float widen1(T v) { return static_cast<float>(v); }
// four consecutive elements, at an address aligned to four of them
__device__ __forceinline__ void widen4(const __nv_bfloat16* p, float* f) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x); f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
}
__device__ __forceinline__ void widen4(const float* p, float* f) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
}

// Asynchronous copy of kBytes (4, 8 or 16), or zeros where there is nothing to copy.
template <int kBytes>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool there) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  const int n = there ? kBytes : 0;
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(d), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" :: "r"(d), "l"(src), "n"(kBytes), "r"(n) : "memory");
}

// kTile rows of `width` elements (a multiple of the copies' size) into rows of `pitch`; rows from `rows` on and
// elements from `there` on become zero.  kBytes: of one copy; sizeof(T) < 4: plain loads.
template <typename T, int kBytes>
__device__ __forceinline__ void fetch(T* dst, int pitch, const T* src, int64_t stride, int rows, int width, int there) {
  constexpr int kPer = kBytes / (int)sizeof(T);
  const int per_row = width / kPer;
  for (int i = threadIdx.x; i < kTile * per_row; i += kThreads) {
    const int r = i / per_row, e = (i - r * per_row) * kPer;
    const bool in = r < rows && e < there;
    const T* s = in ? src + r * stride + e : src;
    if constexpr (kBytes >= 4) copy_async<kBytes>(dst + r * pitch + e, s, in);
    else dst[r * pitch + e] = in ? *s : T(0.0f);
  }
}
template <typename T>
__device__ __forceinline__ void fetch_rows(int bytes, T* dst, int pitch, const T* src, int64_t stride, int rows,
                                           int width, int there) {
  if (bytes == 16) fetch<T, 16>(dst, pitch, src, stride, rows, width, there);
  else if (bytes == 8) fetch<T, 8>(dst, pitch, src, stride, rows, width, there);
  else if (bytes == 4) fetch<T, 4>(dst, pitch, src, stride, rows, width, there);
  else fetch<T, sizeof(T) == 4 ? 4 : 2>(dst, pitch, src, stride, rows, width, there);
}

// Shared memory: two stages of raw x, dt, z, b, c; then D and D x, y, b and c in float32.
template <typename T, int S, int L> struct Smem {
  static constexpr int kChan = kThreads / L;                     // channels of a CTA
  static constexpr int kPad = S * L;                             // states, rounded up
  static constexpr int kPitchY = kChan + 8;                      // the four rows that a warp writes at once on banks of their own
  static constexpr int kRow = kTile * kChan * (int)sizeof(T);
  static constexpr int kRowN = kTile * kPad * (int)sizeof(T);
  static constexpr int kStage = 3 * kRow + 2 * kRowN;
  static constexpr int kOffStep = 2 * kStage;
  static constexpr int kOffY = kOffStep + kTile * kChan * 8;
  static constexpr int kOffB = kOffY + kTile * kPitchY * 4;
  static constexpr int kOffC = kOffB + kTile * kPad * 4;
  static constexpr int kBytes = kOffC + kTile * kPad * 4;
};

template <typename T, int S, int L>
__global__ void __launch_bounds__(kThreads)
selective_scan_kernel(const SelectiveArgs p) {
  using Sm = Smem<T, S, L>;
  constexpr int kChan = Sm::kChan, kPad = Sm::kPad;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t b = blockIdx.y;
  const int blocks = (p.per_group + kChan - 1) / kChan;          // of a group
  const int g = blockIdx.x / blocks, e0 = (blockIdx.x - g * blocks) * kChan;
  const int there = min(kChan, p.per_group - e0);                // channels that exist
  const int64_t first = (int64_t)g * p.per_group + e0;           // the CTA's first channel

  const T* x = static_cast<const T*>(p.x) + b * p.x_batch + first;
  const T* dt = static_cast<const T*>(p.dt) + b * p.dt_batch + first;
  const T* z = p.z == nullptr ? nullptr : static_cast<const T*>(p.z) + b * p.z_batch + first;
  const T* bb = static_cast<const T*>(p.b) + b * p.b_batch + (int64_t)g * p.N;
  const T* cc = static_cast<const T*>(p.c) + b * p.c_batch + (int64_t)g * p.N;
  auto raw = [&](int stage, int which) { return reinterpret_cast<T*>(smem + stage * Sm::kStage + which * Sm::kRow); };
  auto raw_n = [&](int stage, int which) {
    return reinterpret_cast<T*>(smem + stage * Sm::kStage + 3 * Sm::kRow + which * Sm::kRowN);
  };
  float2* s_step = reinterpret_cast<float2*>(smem + Sm::kOffStep);
  float* s_y = reinterpret_cast<float*>(smem + Sm::kOffY);
  float* s_b = reinterpret_cast<float*>(smem + Sm::kOffB);
  float* s_c = reinterpret_cast<float*>(smem + Sm::kOffC);

  // the places of states that do not exist are never copied to: zero once
  if (p.N < kPad) {
    for (int i = tid; i < 2 * kTile * kPad; i += kThreads) {
      raw_n(0, 0)[i] = T(0.0f);
      raw_n(1, 0)[i] = T(0.0f);
    }
    __syncthreads();
  }
  auto ask = [&](int64_t t0, int stage) {
    const int rows = (int)min((int64_t)kTile, p.T - t0);
    fetch_rows<T>(p.copy_x, raw(stage, 0), kChan, x + t0 * p.x_token, p.x_token, rows, kChan, there);
    fetch_rows<T>(p.copy_x, raw(stage, 1), kChan, dt + t0 * p.dt_token, p.dt_token, rows, kChan, there);
    if (z != nullptr) fetch_rows<T>(p.copy_x, raw(stage, 2), kChan, z + t0 * p.z_token, p.z_token, rows, kChan, there);
    fetch_rows<T>(p.copy_n, raw_n(stage, 0), kPad, bb + t0 * p.b_token, p.b_token, rows, p.N, p.N);
    fetch_rows<T>(p.copy_n, raw_n(stage, 1), kPad, cc + t0 * p.c_token, p.c_token, rows, p.N, p.N);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // a thread's states: n = q * 4 L + l * 4 + i for its values 4 q + i (S = 4 Q; S < 4: n = l * S + i)
  const int l = tid & (L - 1), ch = tid / L;
  constexpr int kVec = S < 4 ? S : 4;
  auto state_of = [&](int s) { return (s / kVec) * kVec * L + l * kVec + s % kVec; };
  float h[S], a2[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int n = state_of(s);
    const bool in = ch < there && n < p.N;
    a2[s] = in ? p.a[(first + ch) * p.N + n] * kLog2e : 0.0f;
    h[s] = in && p.state_in != nullptr ? p.state_in[(b * p.E + first + ch) * p.N + n] : 0.0f;
  }

  const int tiles = (int)((p.T + kTile - 1) / kTile);
  if (tiles > 0) ask(0, 0);
  for (int tile = 0; tile < tiles; ++tile) {
    const int64_t t0 = (int64_t)tile * kTile;
    const int stage = tile & 1, rows = (int)min((int64_t)kTile, p.T - t0);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                             // the tile is here; the one before is done with
    if (tile + 1 < tiles) ask(t0 + kTile, stage ^ 1);
    uint32_t starts = 0;
    if (p.pos != nullptr)
      starts = __ballot_sync(0xffffffffu, lane < rows && pos_is_zero(p.pos, p.pos64, b * p.T + t0 + lane));

    for (int i = tid; i < kTile * kChan / 4; i += kThreads) {
      const int t = i / (kChan / 4), e = (i - t * (kChan / 4)) * 4;
      float vx[4], vd[4], st[4];
      widen4(raw(stage, 0) + t * kChan + e, vx);
      widen4(raw(stage, 1) + t * kChan + e, vd);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float v = vd[k] + (p.dt_bias != nullptr && e + k < there ? p.dt_bias[first + e + k] : 0.0f);
        // a step of no time leaves the states of a row that does not exist as they are
        st[k] = t < rows ? (p.softplus ? softplus_step(v) : v) : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) s_step[t * kChan + e + k] = make_float2(st[k], t < rows ? st[k] * vx[k] : 0.0f);
    }
    for (int i = tid; i < kTile * kPad / kVec; i += kThreads) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        s_b[i * kVec + k] = widen1(raw_n(stage, 0)[i * kVec + k]);
        s_c[i * kVec + k] = widen1(raw_n(stage, 1)[i * kVec + k]);
      }
    }
    __syncthreads();

#pragma unroll 1
    for (int t = 0; t < kTile; t += 4) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 step = s_step[(t + j) * kChan + ch];
        if ((starts >> (t + j)) & 1u) {
#pragma unroll
          for (int s = 0; s < S; ++s) h[s] = 0.0f;
        }
        y[j] = 0.0f;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const int n = state_of(s);
          h[s] = fmaf(exp2_fast(step.x * a2[s]), h[s], step.y * s_b[(t + j) * kPad + n]);
          y[j] = fmaf(h[s], s_c[(t + j) * kPad + n], y[j]);
        }
      }
      // sums over the channel's lanes: with every exchange a lane keeps half of its time steps
      int mine = 0;
      if constexpr (L >= 2) {
        const bool up = l & 1;
        const float g0 = __shfl_xor_sync(0xffffffffu, up ? y[0] : y[2], 1);
        const float g1 = __shfl_xor_sync(0xffffffffu, up ? y[1] : y[3], 1);
        y[0] = (up ? y[2] : y[0]) + g0;
        y[1] = (up ? y[3] : y[1]) + g1;
        mine = up ? 2 : 0;
      }
      if constexpr (L >= 4) {
        const bool up = l & 2;
        const float g0 = __shfl_xor_sync(0xffffffffu, up ? y[0] : y[1], 2);
        y[0] = (up ? y[1] : y[0]) + g0;
        mine += up ? 1 : 0;
      }
#pragma unroll
      for (int o = 4; o < L; o <<= 1) y[0] += __shfl_xor_sync(0xffffffffu, y[0], o);
      constexpr int kKept = L >= 4 ? 1 : L == 2 ? 2 : 4;
      if (l < 4) {
#pragma unroll
        for (int j = 0; j < kKept; ++j) s_y[(t + mine + j) * Sm::kPitchY + ch] = y[j];
      }
    }
    __syncthreads();

    for (int i = tid; i < kTile * kChan / 4; i += kThreads) {
      const int t = i / (kChan / 4), e = (i - t * (kChan / 4)) * 4;
      if (t >= rows || e >= there) continue;
      float vx[4], vz[4], out[4];
      widen4(raw(stage, 0) + t * kChan + e, vx);
      if (z != nullptr) widen4(raw(stage, 2) + t * kChan + e, vz);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        out[k] = s_y[t * Sm::kPitchY + e + k];
        if (p.d != nullptr && e + k < there) out[k] = fmaf(p.d[first + e + k], vx[k], out[k]);
        if (z != nullptr) out[k] *= silu_fast(vz[k]);
      }
      T* y = static_cast<T*>(p.y) + (b * p.T + t0 + t) * p.E + first + e;
      if (p.store4 && e + 4 <= there) {
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16x2(out[0], out[1]), pack_bf16x2(out[2], out[3]));
        else
          *reinterpret_cast<float4*>(y) = make_float4(out[0], out[1], out[2], out[3]);
      } else {
        for (int k = 0; k < 4 && e + k < there; ++k) y[k] = static_cast<T>(out[k]);
      }
    }
  }

  if (p.state_out != nullptr && ch < there) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int n = state_of(s);
      if (n < p.N) p.state_out[(b * p.E + first + ch) * p.N + n] = h[s];
    }
  }
}

template <typename T, int S, int L>
cudaError_t launch(SelectiveArgs p, cudaStream_t s) {
  using Sm = Smem<T, S, L>;
  static PerDeviceOnce once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(selective_scan_kernel<T, S, L>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sm::kBytes);
  });
  if (e != cudaSuccess) return e;
  p.copy_x = min(p.copy_x, Sm::kChan * (int)sizeof(T));
  const int blocks = (p.per_group + Sm::kChan - 1) / Sm::kChan;
  selective_scan_kernel<T, S, L><<<dim3((unsigned)(blocks * p.groups), (unsigned)p.B), kThreads, Sm::kBytes, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_states(const SelectiveArgs& p, cudaStream_t s) {
  if (p.N <= 4) return launch<T, 4, 1>(p, s);
  if (p.N <= 8) return launch<T, 4, 2>(p, s);
  if (p.N <= 16) return launch<T, 4, 4>(p, s);
  if (p.N <= 32) return launch<T, 4, 8>(p, s);
  if (p.N <= 64) return launch<T, 4, 16>(p, s);
  if (p.N <= 128) return launch<T, 4, 32>(p, s);
  return launch<T, 8, 32>(p, s);
}

// The largest copy (bytes) that every address base + i * batch + j * token + k * width (elements) allows.
int copy_bytes(const void* base, int64_t batch, int64_t token, int64_t width, int size) {
  const uint64_t all = (uint64_t)reinterpret_cast<uintptr_t>(base) | (uint64_t)(batch * size) | (uint64_t)(token * size) |
                       (uint64_t)(width * size);
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

}  // namespace

cudaError_t launch_selective_scan(SelectiveArgs p, int dtype, cudaStream_t s) {
  if (p.B == 0 || p.E == 0) return cudaSuccess;
  const int size = dtype == 1 ? 2 : 4;
  p.per_group = (int)(p.E / p.groups);
  p.copy_x = min(copy_bytes(p.x, p.x_batch, p.x_token, p.per_group, size),
                 copy_bytes(p.dt, p.dt_batch, p.dt_token, p.per_group, size));
  if (p.z != nullptr) p.copy_x = min(p.copy_x, copy_bytes(p.z, p.z_batch, p.z_token, p.per_group, size));
  p.copy_n = min(copy_bytes(p.b, p.b_batch, p.b_token, p.N, size), copy_bytes(p.c, p.c_batch, p.c_token, p.N, size));
  p.store4 = p.per_group % 4 == 0 && p.E % 4 == 0 && reinterpret_cast<uintptr_t>(p.y) % (4 * size) == 0;
  return dtype == 1 ? launch_states<__nv_bfloat16>(p, s) : launch_states<float>(p, s);
}

}  // namespace rgk
