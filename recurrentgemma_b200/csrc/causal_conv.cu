// The short causal convolution in front of a selective state space layer: depthwise, 2 to 4 taps, over rows
// that may continue a state, with an optional bias and silu:
//   X = state ++ x,   y_t = act(bias + sum_j w[j] X_{t - (W-1) + j}),
// a tap only where no document start lies behind it (a start at t' hides every row before t').  One rounding,
// at the end.  state_out = the last W-1 rows of X, zero where a start lies behind them.
//
// Bound: HBM, every element is read and written once.  A thread owns one pack of channels (16 bytes, or one
// channel where the rows are not 16-byte aligned) and kRows consecutive rows, whose loads are all asked for
// before the first is used; the W-1 rows in front of them come from L2, where the neighbour has just put them.
#include "rgk_common.cuh"
#include "rgk_internal.h"

namespace rgk {
namespace {

constexpr int kThreads = 128;

template <typename T, int kPer> struct Pack;                     // kPer channels as they lie in memory
template <> struct Pack<__nv_bfloat16, 8> { using Raw = uint4; };
template <> struct Pack<float, 4> { using Raw = uint4; };
template <> struct Pack<__nv_bfloat16, 1> { using Raw = uint16_t; };
template <> struct Pack<float, 1> { using Raw = uint32_t; };

template <typename T, int kPer>
__device__ __forceinline__ void widen(const typename Pack<T, kPer>::Raw& r, float* f) {
  if constexpr (kPer > 1) unpack<T>(r, f);
  else if constexpr (sizeof(T) == 2) f[0] = __uint_as_float((uint32_t)r << 16);
  else f[0] = __uint_as_float(r);
}
template <typename T, int kPer>
__device__ __forceinline__ typename Pack<T, kPer>::Raw narrow(const float* f) {
  if constexpr (kPer > 1) return pack<T>(f);
  else if constexpr (sizeof(T) == 2) return __bfloat16_as_ushort(__float2bfloat16_rn(f[0]));
  else return __float_as_uint(f[0]);
}
template <typename Raw> __device__ __forceinline__ Raw nothing() {
  if constexpr (sizeof(Raw) == 16) return make_uint4(0u, 0u, 0u, 0u);
  else return Raw(0);
}

template <bool kFast> __device__ __forceinline__ float silu(float v) {
  if constexpr (kFast) return v * sigmoid_<true>(v);
  return v / (1.0f + expf(-v));
}

template <typename T, int kPer, int kTaps, int kRows>
__global__ void __launch_bounds__(kThreads)
causal_conv_kernel(const ConvArgs p) {
  using Raw = typename Pack<T, kPer>::Raw;
  constexpr int kHalo = kTaps - 1;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int packs = (int)(p.E / kPer);
  const int64_t unit = at / packs;                               // (sequence, chunk of kRows rows)
  const int e = (int)(at - unit * packs) * kPer;
  const int64_t b = unit / p.chunks, t0 = (unit - b * p.chunks) * kRows;
  if (b >= p.B) return;

  const T* x = static_cast<const T*>(p.x) + b * p.x_batch + e;
  const T* state = p.state_in == nullptr ? nullptr : static_cast<const T*>(p.state_in) + b * kHalo * p.E + e;
  // row `t` of X: before the sequence the state, behind it nothing
  auto row = [&](int64_t t) -> Raw {
    if (t >= 0) return t < p.T ? *reinterpret_cast<const Raw*>(x + t * p.x_token) : nothing<Raw>();
    return state != nullptr && t >= -kHalo ? *reinterpret_cast<const Raw*>(state + (t + kHalo) * p.E) : nothing<Raw>();
  };
  auto starts = [&](int64_t t) { return p.pos != nullptr && t >= 0 && t < p.T && pos_is_zero(p.pos, p.pos64, b * p.T + t); };

  Raw raw[kRows + kHalo];
#pragma unroll
  for (int r = 0; r < kRows + kHalo; ++r) raw[r] = row(t0 - kHalo + r);
  uint32_t start = 0;                                            // bit r: row t0 - kHalo + r begins a document
  if (p.pos != nullptr) {
#pragma unroll
    for (int r = 0; r < kRows + kHalo; ++r) start |= (uint32_t)starts(t0 - kHalo + r) << r;
  }
  // the chunk that has read the state also writes the new one, which may lie over it
  Raw last[kHalo];
  if (t0 == 0 && p.state_out != nullptr) {
    bool hidden = false;
#pragma unroll
    for (int j = kHalo - 1; j >= 0; --j) {
      const int64_t t = p.T - kHalo + j;
      last[j] = hidden ? nothing<Raw>() : row(t);
      hidden = hidden || starts(t);
    }
    T* out = static_cast<T*>(p.state_out) + b * kHalo * p.E + e;
#pragma unroll
    for (int j = 0; j < kHalo; ++j) *reinterpret_cast<Raw*>(out + (int64_t)j * p.E) = last[j];
  }

  float w[kTaps][kPer], bias[kPer];
#pragma unroll
  for (int j = 0; j < kTaps; ++j)
    widen<T, kPer>(*reinterpret_cast<const Raw*>(static_cast<const T*>(p.w) + (int64_t)j * p.E + e), w[j]);
  if (p.bias != nullptr) {
    widen<T, kPer>(*reinterpret_cast<const Raw*>(static_cast<const T*>(p.bias) + e), bias);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) bias[i] = 0.0f;
  }

  T* y = static_cast<T*>(p.y) + (b * p.T + t0) * p.E + e;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (t0 + r >= p.T) break;
    float acc[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = bias[i];
    bool hidden = false;
#pragma unroll
    for (int j = kTaps - 1; j >= 0; --j) {
      float f[kPer];
      widen<T, kPer>(raw[r + j], f);
      if (!hidden) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] = fmaf(f[i], w[j][i], acc[i]);
      }
      hidden = hidden || ((start >> (r + j)) & 1u);
    }
    if (p.silu) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] = silu<sizeof(T) == 2>(acc[i]);
    }
    *reinterpret_cast<Raw*>(y + (int64_t)r * p.E) = narrow<T, kPer>(acc);
  }
}

template <typename T, int kPer, int kRows>
cudaError_t launch_rows(ConvArgs p, cudaStream_t s) {
  p.chunks = p.T > 0 ? (p.T + kRows - 1) / kRows : 1;            // (without a token the state still moves on)
  const int64_t blocks = (p.B * p.chunks * (p.E / kPer) + kThreads - 1) / kThreads;
  if (blocks >= ((int64_t)1 << 31)) return cudaErrorInvalidValue;
  const unsigned grid = (unsigned)blocks;
  if (p.taps == 4) causal_conv_kernel<T, kPer, 4, kRows><<<grid, kThreads, 0, s>>>(p);
  else if (p.taps == 3) causal_conv_kernel<T, kPer, 3, kRows><<<grid, kThreads, 0, s>>>(p);
  else causal_conv_kernel<T, kPer, 2, kRows><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int kPer>
cudaError_t launch_pack(const ConvArgs& p, cudaStream_t s) {
  // sixteen rows a thread where that still fills the device, four where it does not.  (From W-1 rows on a
  // sequence's first chunk is the only one that reads the state, so that it may be written in place.)
  if (p.T <= 1) return launch_rows<T, kPer, 1>(p, s);
  if (p.B * p.T * (p.E / kPer) >= 16 * (int64_t)148 * 512) return launch_rows<T, kPer, 16>(p, s);
  return launch_rows<T, kPer, 4>(p, s);
}

}  // namespace

cudaError_t launch_causal_conv(const ConvArgs& p, int dtype, cudaStream_t s) {
  if (p.B == 0 || p.E == 0) return cudaSuccess;
  const int per = dtype == 1 ? 8 : 4;
  auto fits = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
  const bool packs = p.E % per == 0 && p.x_token % per == 0 && p.x_batch % per == 0 && fits(p.x) && fits(p.w) &&
                     fits(p.bias) && fits(p.state_in) && fits(p.state_out) && fits(p.y);
  if (dtype == 1) return packs ? launch_pack<__nv_bfloat16, 8>(p, s) : launch_pack<__nv_bfloat16, 1>(p, s);
  return packs ? launch_pack<float, 4>(p, s) : launch_pack<float, 1>(p, s);
}

}  // namespace rgk
