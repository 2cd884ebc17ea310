// The short causal convolution in front of a selective state space layer: depthwise, 2 to 4 taps, over rows
// that may continue a state, with an optional bias and silu:
//   X = state ++ x,   y_t = act(bias + sum_j w[j] X_{t - (W-1) + j}),
// a tap only where no document start lies behind it (a start at t' hides every row before t').  One rounding,
// at the end.  state_out = the last W-1 rows of X, zero where a start lies behind them.
//
// Bound: HBM, every element is read and written once.  A thread owns one pack of channels (8 bytes, or one
// channel where the rows are not aligned to that) and kRows consecutive rows, whose loads are all asked for before
// the first is used; the W-1 rows in front of them come from L2, where the neighbour has just put them.  8 x 4096 x
// 5120 in bfloat16: 119 us, 86 % of the measured copy rate (with packs of 16 bytes, 160 registers a thread, 168).
#include "packed.cuh"
#include "rgk_common.cuh"
#include "rgk_internal.h"

namespace rgk {
namespace {

constexpr int kThreads = 128;

template <int kBytes> struct RawOf;                               // a pack as it lies in memory
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };

template <typename T, int kPer>
__device__ __forceinline__ void widen(const typename RawOf<kPer * sizeof(T)>::type& r, float* f) {
  if constexpr (kPer == 4) {
    f[0] = bf16_lo(r.x); f[1] = bf16_hi(r.x); f[2] = bf16_lo(r.y); f[3] = bf16_hi(r.y);
  } else if constexpr (kPer == 2) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y);
  } else if constexpr (sizeof(T) == 2) {
    f[0] = __uint_as_float((uint32_t)r << 16);
  } else {
    f[0] = __uint_as_float(r);
  }
}
template <typename T, int kPer>
__device__ __forceinline__ typename RawOf<kPer * sizeof(T)>::type narrow(const float* f) {
  if constexpr (kPer == 4) return make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
  else if constexpr (kPer == 2) return make_uint2(__float_as_uint(f[0]), __float_as_uint(f[1]));
  else if constexpr (sizeof(T) == 2) return __bfloat16_as_ushort(__float2bfloat16_rn(f[0]));
  else return __float_as_uint(f[0]);
}

// bfloat16 takes the hardware's exponential and reciprocal (2 units in the last place of float32, far below its own)
template <typename T, int kPer> __device__ __forceinline__ void silu(float (&v)[kPer]) {
  if constexpr (sizeof(T) == 2 && kPer > 1) {
#pragma unroll
    for (int i = 0; i < kPer; i += 2) {
      const float2 r = silu_fast(v[i], v[i + 1]);
      v[i] = r.x; v[i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = v[i] / (1.0f + expf(-v[i]));
  }
}

template <typename T, int kPer, int kTaps, int kRows, bool kDocs>
__global__ void __launch_bounds__(kThreads)
causal_conv_kernel(const ConvArgs p) {
  using Raw = typename RawOf<kPer * sizeof(T)>::type;
  constexpr int kHalo = kTaps - 1;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int packs = (int)(p.E / kPer);
  const int64_t unit = at / packs;                               // (sequence, chunk of kRows rows)
  const int e = (int)(at - unit * packs) * kPer;
  const int64_t b = unit / p.chunks, t0 = (unit - b * p.chunks) * kRows;

  const T* x = static_cast<const T*>(p.x) + b * p.x_batch + e;
  const T* state = p.state_in == nullptr ? nullptr : static_cast<const T*>(p.state_in) + b * kHalo * p.E + e;
  // row `t` of X: before the sequence the state, behind it nothing
  auto row = [&](int64_t t) -> Raw {
    if (t >= 0) return t < p.T ? *reinterpret_cast<const Raw*>(x + t * p.x_token) : Raw{};
    return state != nullptr && t >= -kHalo ? *reinterpret_cast<const Raw*>(state + (t + kHalo) * p.E) : Raw{};
  };
  auto starts = [&](int64_t t) { return kDocs && t >= 0 && t < p.T && pos_is_zero(p.pos, p.pos64, b * p.T + t); };

  uint32_t start = 0;                                            // bit r: row t0 - kHalo + r begins a document
  if constexpr (kDocs) {
    const int64_t here = b < p.B ? unit : -1;
    if (__all_sync(0xffffffffu, here == __shfl_sync(0xffffffffu, here, 0))) {        // a position a lane
      const int lane = threadIdx.x & 31;
      start = __ballot_sync(0xffffffffu, here >= 0 && lane < kRows + kHalo && starts(t0 - kHalo + lane));
    } else if (here >= 0) {
#pragma unroll 1
      for (int r = 0; r < kRows + kHalo; ++r) start |= (uint32_t)starts(t0 - kHalo + r) << r;
    }
  }
  if (b >= p.B) return;

  Raw raw[kRows + kHalo];
  if (t0 >= kHalo && t0 + kRows <= p.T) {                        // (a plain run of rows: most of them)
    const T* from = x + (t0 - kHalo) * p.x_token;
#pragma unroll
    for (int r = 0; r < kRows + kHalo; ++r) raw[r] = *reinterpret_cast<const Raw*>(from + r * p.x_token);
  } else {
#pragma unroll
    for (int r = 0; r < kRows + kHalo; ++r) raw[r] = row(t0 - kHalo + r);
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
  // the chunk that has read the state also writes the new one, which may lie over it
  if (t0 == 0 && p.state_out != nullptr) {
    Raw last[kHalo];
    bool hidden = false;
#pragma unroll
    for (int j = kHalo - 1; j >= 0; --j) {
      const int64_t t = p.T - kHalo + j;
      last[j] = hidden ? Raw{} : row(t);
      hidden = hidden || starts(t);
    }
    T* out = static_cast<T*>(p.state_out) + b * kHalo * p.E + e;
#pragma unroll
    for (int j = 0; j < kHalo; ++j) {
      if (RGK_IN_RANGE(out - static_cast<T*>(p.state_out) + j * p.E, p.B * kHalo * p.E - (kPer - 1), nullptr))
        *reinterpret_cast<Raw*>(out + (int64_t)j * p.E) = last[j];
    }
  }

  T* y = static_cast<T*>(p.y) + (b * p.T + t0) * p.E + e;
  float f[kTaps][kPer];                                          // the last kTaps rows, row r in f[r % kTaps]
#pragma unroll
  for (int r = 0; r < kHalo; ++r) widen<T, kPer>(raw[r], f[r]);
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (t0 + r >= p.T) break;
    widen<T, kPer>(raw[r + kHalo], f[(r + kHalo) % kTaps]);
    float acc[kPer];
    if constexpr (kPer > 1 && !kDocs) {
#pragma unroll
      for (int i = 0; i < kPer; i += 2) {
        Pair sum = pair(bias[i], bias[i + 1]);
#pragma unroll
        for (int j = kTaps - 1; j >= 0; --j) {
          const float* g = f[(r + j) % kTaps];
          sum = fma2(pair(g[i], g[i + 1]), pair(w[j][i], w[j][i + 1]), sum);
        }
        const float2 two = split(sum);
        acc[i] = two.x; acc[i + 1] = two.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] = bias[i];
      bool hidden = false;
#pragma unroll
      for (int j = kTaps - 1; j >= 0; --j) {
        if (!hidden) {
#pragma unroll
          for (int i = 0; i < kPer; ++i) acc[i] = fmaf(f[(r + j) % kTaps][i], w[j][i], acc[i]);
        }
        hidden = hidden || (kDocs && ((start >> (r + j)) & 1u));
      }
    }
    if (p.silu) silu<T, kPer>(acc);
    if (RGK_IN_RANGE(y - static_cast<T*>(p.y) + r * p.E, p.B * p.T * p.E - (kPer - 1), nullptr))
      *reinterpret_cast<Raw*>(y + (int64_t)r * p.E) = narrow<T, kPer>(acc);
  }
}

template <typename T, int kPer, int kRows, bool kDocs>
cudaError_t launch_taps(const ConvArgs& p, unsigned grid, cudaStream_t s) {
  if (p.taps == 4) causal_conv_kernel<T, kPer, 4, kRows, kDocs><<<grid, kThreads, 0, s>>>(p);
  else if (p.taps == 3) causal_conv_kernel<T, kPer, 3, kRows, kDocs><<<grid, kThreads, 0, s>>>(p);
  else causal_conv_kernel<T, kPer, 2, kRows, kDocs><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}
template <typename T, int kPer, int kRows>
cudaError_t launch_rows(ConvArgs p, cudaStream_t s) {
  p.chunks = p.T > 0 ? (p.T + kRows - 1) / kRows : 1;            // (without a token the state still moves on)
  const int64_t blocks = (p.B * p.chunks * (p.E / kPer) + kThreads - 1) / kThreads;
  if (blocks >= ((int64_t)1 << 31)) return cudaErrorInvalidValue;
  return p.pos != nullptr ? launch_taps<T, kPer, kRows, true>(p, (unsigned)blocks, s)
                          : launch_taps<T, kPer, kRows, false>(p, (unsigned)blocks, s);
}

template <typename T, int kPer>
cudaError_t launch_pack(const ConvArgs& p, int sms, cudaStream_t s) {
  // Many rows a thread where that still fills the device (8 x 4096 x 5120 in bfloat16 with 8 / 12 / 16 / 24 rows:
  // 139 / 130 / 124 / 127 us; 3 x 1237 x 2565 in float32, a channel a thread: 31 / 29 / 41 / 46), four where it
  // does not.  (From W-1 rows on a sequence's first chunk is the only one that reads the state, so that it may be
  // written in place.)
  constexpr int kMany = kPer > 1 ? 16 : 12;
  if (p.T <= 1) return launch_rows<T, kPer, 1>(p, s);
  if (p.B * p.T * (p.E / kPer) >= kMany * (int64_t)sms * 1024) return launch_rows<T, kPer, kMany>(p, s);
  return launch_rows<T, kPer, 4>(p, s);
}

}  // namespace

cudaError_t launch_causal_conv(const ConvArgs& p, int dtype, cudaStream_t s) {
  if (p.B == 0 || p.E == 0) return cudaSuccess;
  static PerDeviceOnce once;
  int sms = 0;
  const cudaError_t e = once.run([] { return cudaSuccess; }, &sms);
  if (e != cudaSuccess) return e;
  const int per = dtype == 1 ? 4 : 2;
  auto fits = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 7u) == 0; };
  const bool packs = p.E % per == 0 && p.x_token % per == 0 && p.x_batch % per == 0 && fits(p.x) && fits(p.w) &&
                     fits(p.bias) && fits(p.state_in) && fits(p.state_out) && fits(p.y);
  if (dtype == 1) return packs ? launch_pack<__nv_bfloat16, 4>(p, sms, s) : launch_pack<__nv_bfloat16, 1>(p, sms, s);
  return packs ? launch_pack<float, 2>(p, sms, s) : launch_pack<float, 1>(p, sms, s);
}

}  // namespace rgk
