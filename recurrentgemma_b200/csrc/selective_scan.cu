// The selective state space recurrence: N float32 states a channel, each with a decay of its own,
//   D_t = softplus(dt_t + dt_bias),  h_t[n] = exp(D_t a[n]) h_{t-1}[n] + D_t x_t b_t[n],
//   y_t = (sum_n h_t[n] c_t[n] + d x_t) silu(z_t),
// where a document start drops h_{t-1}.  b and c are shared by the channels of a group.
//
// Bound: the special functions.  An (element, state) takes one exponential and four multiply-adds' worth of
// float32 work, and an SM has 16 special-function results a clock but 128 multiply-adds: for 16 states (and
// three more for softplus and silu) 168 M elements take 0.71 ms where their bytes take 0.21.  8 x 4096 x 5120 in
// bfloat16: 995 us, 71 % of that rate.  (In float32 the decays take a polynomial as well: exact_decays.)
//
// The recurrence runs in time order in registers: L neighbouring lanes share a channel, each with S of its
// states, and time is not split - the lanes are, which leaves no work to do twice.  A CTA is two teams of 128 threads.
// The owners of the states do nothing but the recurrence, from float32 tiles in shared memory, and leave sums over
// their S states; the helpers turn the next tile (brought in by cp.async) into D, D x and widened b and c, and the sums of the tile
// before into outputs, so that one team's latencies lie under the other's work (one team for all three, tile
// after tile: 1023 us and, for one row of 2048 steps, 190 where the teams take 134).  A load from shared memory costs what
// arrives in registers, broadcast or not: a thread with two channels uses b and c twice (988 us; with one 1039, with 4
// states 1325).  Polynomials in place of a quarter of the exponentials made it slower (1104), and a shuffle's latency
// more than the parts of the sums in shared memory.
//
// Long calls of more channels than the CTAs hold are cut into chunks of time that are drawn by a ticket, so that no SM
// works on a fifth CTA while others have four (1090 -> 1023 us in the form with one team); a state goes from chunk to chunk through state_out.
#include <type_traits>

#include "packed.cuh"
#include "rgk_common.cuh"
#include "rgk_internal.h"

namespace rgk {
namespace {

constexpr int kTeam = 128;                                        // threads of each half of a CTA
constexpr int kMostBlocks = 1 << 16;                             // whose progress the workspace has room for
constexpr unsigned kWaitLimit = 1u << 23;                       // polls, 0.2 us and more each

// softplus(v) = max(v, 0) + log1p(e), e = exp(-|v|) in (0, 1]: log1p(e) / e by a polynomial fitted for the
// smallest largest relative error on [0, 1] (5e-9; 1.8e-7 in float32 arithmetic).  Steps of 1e-3 come out with their
// relative precision, which the hardware logarithm of 1 + e would lose.  (A NaN stays one: e is.)  kExact: e by exp_exact,
// for float32; the hardware's exponential of |v| log2(e) is 1.5e-7 off on average for steps of 1e-3 to 1.
constexpr float softplus_coefficient(int i) {
  constexpr float k[10] = {1.0f, -0.4999990165233612f, 0.3332996368408203f, -0.24954134225845337f,
                           0.1967593878507614f, -0.15305590629577637f, 0.10603651404380798f,
                           -0.056959498673677444f, 0.01985144428908825f, -0.0032440212089568377f};
  return k[i];
}
template <bool kExact>
__device__ __forceinline__ float2 softplus_steps(float v0, float v1) {
  Pair e;
  if constexpr (kExact) {
    e = exp_exact(-fabsf(v0), -fabsf(v1));
  } else {
    e = exp2_pair(mul2(pair(fabsf(v0), fabsf(v1)), pair(-kLog2e, -kLog2e)));
  }
  Pair p = pair(softplus_coefficient(9), softplus_coefficient(9));
#pragma unroll
  for (int i = 8; i >= 0; --i) p = fma2(p, e, pair(softplus_coefficient(i), softplus_coefficient(i)));
  return split(fma2(p, e, pair(fmaxf(v0, 0.0f), fmaxf(v1, 0.0f))));
}

// In float32, and up to 4 states (of a channel, rounded up), the decays are exp2_exact: slow states keep their terms for a
// thousand steps, and that the hardware's exponential is a little small shows in them.  2048 steps of 1 / 8 / 16 states in
// float32: 1.2e-6 / 7.8e-7 / 6.0e-7 off 64 bits with it, 2.1e-7 / 1.7e-7 / 1.5e-7 so, for 2 / 5 / 24 % more time (a step of
// 256 sequences 45 -> 48 us).  bfloat16 calls of more states keep the hardware's (30 % more time otherwise), of an argument
// that is 2e-8 larger, which costs nothing and takes most of the bias away: its mean error, in 1e-9, for |x| from 1e-5 / 1e-4 /
// 1e-3 / 1e-2 / 0.05 / 0.1 / 0.2 up to the next is -8 / -6 / -12 / -26 / -14 / -18 / -20, and +6 / +8 / +2 / -12 / +1 / -6 /
// -2 so (rms 30 to 47, and 30 to 35); a step of 0 still is a factor of 1.  One rule for sequences and single steps, so that they
// come to the same states.
constexpr float kDecayBias = 2.0e-8f;
template <typename T> constexpr bool exact_decays(int states) { return sizeof(T) == 4 || states <= 4; }
// 2^(step a) for two states
template <bool kExact> __device__ __forceinline__ Pair decays(Pair step, Pair a) {
  if constexpr (kExact) return exp2_exact(mul2(step, a));
  else return exp2_pair(fma2(step, a, pair(kDecayBias, kDecayBias)));
}
// (not packed without the polynomial: one register less for the constant)
template <bool kExact> __device__ __forceinline__ float2 decays(float step, float a0, float a1) {
  if constexpr (kExact) return split(decays<true>(pair(step, step), pair(a0, a1)));
  else return make_float2(exp2_fast(fmaf(step, a0, kDecayBias)), exp2_fast(fmaf(step, a1, kDecayBias)));
}

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

// kRows rows into rows of kPitch elements; rows from `rows` on and elements from `there` on become zero (elements
// from `width` on stay as they are).  kBytes: of one copy; 2: plain loads.
template <typename T, int kBytes, int kThreads, int kRows, int kPitch>
__device__ __forceinline__ void fetch(int tid, T* dst, const T* src, int64_t stride, int rows, int width, int there) {
  constexpr int kPer = kBytes / (int)sizeof(T), kCols = kPitch / kPer;
  static_assert(kPitch % kPer == 0, "whole copies");
#pragma unroll
  for (int k = 0; k < (kRows * kCols + kThreads - 1) / kThreads; ++k) {
    const int i = tid + k * kThreads;
    const int r = i / kCols, e = i % kCols * kPer;
    if ((kRows * kCols % kThreads != 0 && r >= kRows) || e >= width) continue;
    const bool in = r < rows && e < there;
    const T* s = in ? src + r * stride + e : src;
    if constexpr (kBytes >= 4) copy_async<kBytes>(dst + r * kPitch + e, s, in);
    else dst[r * kPitch + e] = in ? *s : T(0.0f);
  }
}
// `bytes`: the largest copy that all addresses allow; kAligned: it is 16, or a whole row
template <typename T, bool kAligned, int kThreads, int kRows, int kPitch>
__device__ __forceinline__ void fetch_rows(int tid, int bytes, T* dst, const T* src, int64_t stride, int rows, int width,
                                           int there) {
  constexpr int kMost = kPitch * (int)sizeof(T) < 16 ? kPitch * (int)sizeof(T) : 16;
  if (kAligned || bytes >= kMost) fetch<T, kMost, kThreads, kRows, kPitch>(tid, dst, src, stride, rows, width, there);
  else if (sizeof(T) == 4 || bytes >= 4) fetch<T, 4, kThreads, kRows, kPitch>(tid, dst, src, stride, rows, width, there);
  else fetch<T, (int)sizeof(T), kThreads, kRows, kPitch>(tid, dst, src, stride, rows, width, there);
}

// Named barriers of a CTA: `arrive` does not wait, `meet` does.
enum { kFull = 1, kDone = 3, kHelpersMeet = 5, kOwnersMeet = 6 };           // kFull, kDone: one for each of two buffers
template <int kCount> __device__ __forceinline__ void arrive(int id) {
  asm volatile("bar.arrive %0, %1;" :: "r"(id), "n"(kCount) : "memory");
}
template <int kCount> __device__ __forceinline__ void meet(int id) {
  asm volatile("bar.sync %0, %1;" :: "r"(id), "n"(kCount) : "memory");
}

// S states of each of C channels a thread, L lanes a channel, kTile time steps a tile.  128 threads run the recurrence
// (the owners of the states), 128 do what goes by element.  Shared memory: three stages of raw x, dt, z, b, c; two
// buffers each of D and D x, parts of sums, b and c in float32.  In what is by channel and float32, channel
// 4 q + k lies at k * kQuads + q: threads that work on four neighbouring channels store each of them next to what
// their neighbours store.
template <typename T, int S_, int C_, int L_, int kTile_> struct Shape {
  static constexpr int S = S_, C = C_, L = L_, kTile = kTile_;
  static constexpr int kOwners = kTeam / L;                      // (groups of lanes)
  static constexpr int kChan = kOwners * C, kQuads = kChan / 4;  // channels of a CTA
  static constexpr int kPad = S * L;                             // states, rounded up
  static constexpr int kRow = kTile * kChan * (int)sizeof(T);
  static constexpr int kRowN = kTile * kPad * (int)sizeof(T);
  static constexpr int kStage = 3 * kRow + 2 * kRowN;
  static constexpr int kStep = kTile * kChan * 8, kPart = kTile * kTeam * C * 4, kWide = kTile * kPad * 4;
  static constexpr int kOffStep = 3 * kStage;
  static constexpr int kOffPart = kOffStep + 2 * kStep;
  static constexpr int kOffB = kOffPart + 2 * kPart;
  static constexpr int kOffC = kOffB + 2 * kWide;
  static constexpr int kBytes = kOffC + 2 * kWide;
  static constexpr int kUnroll = 8;
  static_assert(kChan % 4 == 0 && kTile <= 32 && kTile % kUnroll == 0 && kBytes <= 227 * 1024, "a tile");
};

// Waits until chunk - 1 of a block of channels has left its states.  The CTA that has drawn it is running (all items are
// drawn in this order, the first one of a CTA too, by CTAs that have started), and none waits for a later one: however
// few of the CTAs find a place on the device, the item that was drawn first among the unfinished ones goes on.
__device__ __forceinline__ void wait_for(const int* done, int chunk, unsigned limit, int* status) {
  if (threadIdx.x == 0) {
    int seen = 0;
    for (unsigned n = 0; n < limit; ++n) {
      asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(seen) : "l"(done) : "memory");
      if (seen >= chunk) break;
      __nanosleep(200);
    }
    if (seen < chunk && status != nullptr) atomicExch(status, kStatusTimeout);
  }
  meet<kTeam>(kOwnersMeet);
}

template <typename T, typename Sh, bool kAligned>
__global__ void __launch_bounds__(2 * kTeam, 2)
selective_scan_kernel(const SelectiveArgs p) {
  constexpr int S = Sh::S, C = Sh::C, L = Sh::L, kTile = Sh::kTile;
  constexpr int kChan = Sh::kChan, kQuads = Sh::kQuads, kPad = Sh::kPad;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_item;
  __shared__ uint32_t s_starts[2];
  const bool helper = threadIdx.x >= kTeam;
  const int tid = threadIdx.x % kTeam, lane = tid & 31;          // in its team
  auto raw = [&](int stage, int which) { return reinterpret_cast<T*>(smem + stage * Sh::kStage + which * Sh::kRow); };
  auto raw_n = [&](int stage, int which) {
    return reinterpret_cast<T*>(smem + stage * Sh::kStage + 3 * Sh::kRow + which * Sh::kRowN);
  };
  auto steps = [&](int buf) { return reinterpret_cast<float2*>(smem + Sh::kOffStep + buf * Sh::kStep); };
  auto parts = [&](int buf) { return reinterpret_cast<float*>(smem + Sh::kOffPart + buf * Sh::kPart); };
  auto wide_b = [&](int buf) { return reinterpret_cast<float*>(smem + Sh::kOffB + buf * Sh::kWide); };
  auto wide_c = [&](int buf) { return reinterpret_cast<float*>(smem + Sh::kOffC + buf * Sh::kWide); };

  // the places of states that do not exist are never copied to: zero once
  if (p.N < kPad) {
    for (int stage = 0; stage < 3; ++stage) {
      for (int i = threadIdx.x; i < 2 * kTile * kPad; i += 2 * kTeam) raw_n(stage, 0)[i] = T(0.0f);
    }
    __syncthreads();
  }

  auto draw = [&]() -> int64_t {                                 // for all of the CTA; what it has done is published
    if (threadIdx.x == 0) s_item = (int)atomicAdd(p.ticket, 1u);
    __syncthreads();
    return s_item;
  };
  const int64_t items = p.chunks * p.blocks;
  for (int64_t item = p.chunks == 1 ? blockIdx.x : draw(); item < items;) {
    const int64_t chunk = item / p.blocks;
    const int block = (int)(item - chunk * p.blocks);
    const int per_row = p.groups * p.blocks_per_group;
    const int64_t b = block / per_row;
    const int in_row = block % per_row, g = in_row / p.blocks_per_group, e0 = (in_row - g * p.blocks_per_group) * kChan;
    const int there = min(kChan, p.per_group - e0);              // channels that exist
    const int64_t first = (int64_t)g * p.per_group + e0;         // the CTA's first channel
    const int64_t begin = chunk * p.chunk, end = min(p.T, begin + p.chunk);
    const int tiles = (int)((end - begin + kTile - 1) / kTile);

    if (helper) {
      constexpr int kRowsAtOnce = kTeam / kQuads;
      constexpr int kPasses = kTile > kRowsAtOnce ? kTile / kRowsAtOnce : 1;
      constexpr int kPassesN = (kTile * kPad + kTeam * 4 - 1) / (kTeam * 4);
      const T* x = static_cast<const T*>(p.x) + b * p.x_batch + first;
      const T* dt = static_cast<const T*>(p.dt) + b * p.dt_batch + first;
      const T* z = p.z == nullptr ? nullptr : static_cast<const T*>(p.z) + b * p.z_batch + first;
      const T* bb = static_cast<const T*>(p.b) + b * p.b_batch + (int64_t)g * p.N;
      const T* cc = static_cast<const T*>(p.c) + b * p.c_batch + (int64_t)g * p.N;
      T* y = static_cast<T*>(p.y) + b * p.T * p.E + first;
      // whole tiles of whole rows: a thread's copies start at fixed places, a tile further each time
      constexpr int kPer = 16 / (int)sizeof(T);
      constexpr int kCols = kChan >= kPer ? kChan / kPer : 1, kColsN = kPad >= kPer ? kPad / kPer : 1;  // copies of a row
      constexpr bool kQuick = kAligned && kChan >= kPer && kPad >= kPer && kTeam % kCols == 0 && kTeam % kColsN == 0;
      constexpr int kStepX = kTeam / kCols, kStepN = kTeam / kColsN;                                     // rows at once
      const int xr = tid / kCols, xc = tid % kCols * kPer, nr = tid / kColsN, nc = tid % kColsN * kPer;
      const T *qx = x + (begin + xr) * p.x_token + xc, *qd = dt + (begin + xr) * p.dt_token + xc;
      const T* qz = z == nullptr ? nullptr : z + (begin + xr) * p.z_token + xc;
      const T *qb = bb + (begin + nr) * p.b_token + nc, *qc = cc + (begin + nr) * p.c_token + nc;
      // b and c of two-byte elements whose rows begin anywhere: no copy takes them, so they come through registers, loaded
      // when the tile is asked for and stored when it is wanted
      constexpr bool kStaged = !kAligned && sizeof(T) == 2;
      constexpr int kHeld = kStaged ? (kTile * kPad + kTeam - 1) / kTeam : 1;
      T on_way[2][kHeld];
      auto load_rows = [&](const T* src, int64_t stride, int rows, T (&to)[kHeld]) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
          const int i = tid + k * kTeam, r = i / kPad, n = i % kPad;
          to[k] = r < rows && n < p.N ? src[r * stride + n] : T(0.0f);
        }
      };
      auto settle = [&](int tile) {
        if (kStaged && p.copy_n < 4) {
#pragma unroll
          for (int k = 0; k < kHeld; ++k) {
            const int i = tid + k * kTeam;
            if (kTile * kPad % kTeam == 0 || i < kTile * kPad) {
              raw_n(tile % 3, 0)[i] = on_way[0][k];
              raw_n(tile % 3, 1)[i] = on_way[1][k];
            }
          }
        }
      };
      auto ask = [&](int tile) {
        const int64_t t0 = begin + (int64_t)tile * kTile;
        const int stage = tile % 3, rows = (int)min((int64_t)kTile, end - t0);
        if (kQuick && rows == kTile && there == kChan) {
          auto copy = [&](T* dst, const T* src, int64_t stride, auto at_once, int r) {
            constexpr int kAtOnce = decltype(at_once)::value;
#pragma unroll
            for (int k = 0; k < (kTile + kAtOnce - 1) / kAtOnce; ++k) {
              if (kTile % kAtOnce == 0 || r + k * kAtOnce < kTile) copy_async<16>(dst + k * kTeam * kPer, src + k * kAtOnce * stride, true);
            }
          };
          std::integral_constant<int, kStepX> by_x;
          std::integral_constant<int, kStepN> by_n;
          copy(raw(stage, 0) + tid * kPer, qx, p.x_token, by_x, xr);
          copy(raw(stage, 1) + tid * kPer, qd, p.dt_token, by_x, xr);
          if (z != nullptr) copy(raw(stage, 2) + tid * kPer, qz, p.z_token, by_x, xr);
          if (nc < p.N) {
            copy(raw_n(stage, 0) + tid * kPer, qb, p.b_token, by_n, nr);
            copy(raw_n(stage, 1) + tid * kPer, qc, p.c_token, by_n, nr);
          }
          qx += kTile * p.x_token; qd += kTile * p.dt_token; qb += kTile * p.b_token; qc += kTile * p.c_token;
          if (z != nullptr) qz += kTile * p.z_token;
        } else {
          fetch_rows<T, kAligned, kTeam, kTile, kChan>(tid, p.copy_x, raw(stage, 0), x + t0 * p.x_token, p.x_token, rows, kChan, there);
          fetch_rows<T, kAligned, kTeam, kTile, kChan>(tid, p.copy_x, raw(stage, 1), dt + t0 * p.dt_token, p.dt_token, rows, kChan, there);
          if (z != nullptr)
            fetch_rows<T, kAligned, kTeam, kTile, kChan>(tid, p.copy_x, raw(stage, 2), z + t0 * p.z_token, p.z_token, rows, kChan, there);
          if (kStaged && p.copy_n < 4) {
            load_rows(bb + t0 * p.b_token, p.b_token, rows, on_way[0]);
            load_rows(cc + t0 * p.c_token, p.c_token, rows, on_way[1]);
          } else {
            fetch_rows<T, kAligned, kTeam, kTile, kPad>(tid, p.copy_n, raw_n(stage, 0), bb + t0 * p.b_token, p.b_token, rows, p.N, p.N);
            fetch_rows<T, kAligned, kTeam, kTile, kPad>(tid, p.copy_n, raw_n(stage, 1), cc + t0 * p.c_token, p.c_token, rows, p.N, p.N);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      auto starts_at = [&](int tile) {
        const int64_t t = begin + (int64_t)tile * kTile + lane;
        return p.pos != nullptr && lane < kTile && t < end && pos_is_zero(p.pos, p.pos64, b * p.T + t);
      };

      const int q = tid % kQuads, row0 = tid / kQuads;           // a thread's four channels, 4 q to 4 q + 3
      float bias[4], d[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = 4 * q + k < there;
        bias[k] = in && p.dt_bias != nullptr ? p.dt_bias[first + 4 * q + k] : 0.0f;
        d[k] = in && p.d != nullptr ? p.d[first + 4 * q + k] : 0.0f;
      }
      // what the recurrence reads of a tile
      auto prepare = [&](int tile, bool start) {
        const int stage = tile % 3, buf = tile & 1, rows = (int)min((int64_t)kTile, end - begin - (int64_t)tile * kTile);
        if (tid < 32) {
          const uint32_t all = __ballot_sync(0xffffffffu, start);
          if (lane == 0) s_starts[buf] = all;
        }
        // (all that is read before anything that is written: to the compiler they may overlap)
        float by_x[kPasses][4], by_step[kPasses][4], by_n[kPassesN][2][4];
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
          const int t = row0 + k * kRowsAtOnce;
          if (kRowsAtOnce > kTile && t >= kTile) break;
          widen4(raw(stage, 0) + t * kChan + 4 * q, by_x[k]);
          widen4(raw(stage, 1) + t * kChan + 4 * q, by_step[k]);
        }
#pragma unroll
        for (int k = 0; k < kPassesN; ++k) {
          const int i = (tid + k * kTeam) * 4;
          if (kTile * kPad % (kTeam * 4) != 0 && i >= kTile * kPad) break;
          widen4(raw_n(stage, 0) + i, by_n[k][0]);
          widen4(raw_n(stage, 1) + i, by_n[k][1]);
        }
#pragma unroll
        for (int k = 0; k < kPassesN; ++k) {
          const int i = (tid + k * kTeam) * 4;
          if (kTile * kPad % (kTeam * 4) != 0 && i >= kTile * kPad) break;
          *reinterpret_cast<float4*>(wide_b(buf) + i) = make_float4(by_n[k][0][0], by_n[k][0][1], by_n[k][0][2], by_n[k][0][3]);
          *reinterpret_cast<float4*>(wide_c(buf) + i) = make_float4(by_n[k][1][0], by_n[k][1][1], by_n[k][1][2], by_n[k][1][3]);
        }
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
          const int t = row0 + k * kRowsAtOnce;
          if (kRowsAtOnce > kTile && t >= kTile) break;
          float (&vx)[4] = by_x[k], (&step)[4] = by_step[k];
#pragma unroll
          for (int i = 0; i < 4; ++i) step[i] += bias[i];
          if (p.softplus) {
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float2 two = softplus_steps<sizeof(T) == 4>(step[i], step[i + 1]);
              step[i] = two.x; step[i + 1] = two.y;
            }
          }
          if (rows < kTile && t >= rows) {                       // a step of no time leaves the states as they are
#pragma unroll
            for (int i = 0; i < 4; ++i) step[i] = vx[i] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) steps(buf)[t * kChan + i * kQuads + q] = make_float2(step[i], step[i] * vx[i]);
        }
        if (tile == 0 && chunk == 0 && p.state_in == nullptr && row0 == 0) {     // as at a start, without a state
#pragma unroll
          for (int i = 0; i < 4; ++i) steps(buf)[i * kQuads + q].x = 0.0f;
        }
      };
      // its outputs
      auto finish = [&](int tile) {
        const int64_t t0 = begin + (int64_t)tile * kTile;
        const int stage = tile % 3, rows = (int)min((int64_t)kTile, end - t0);
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
          const int t = row0 + k * kRowsAtOnce;
          if (t >= rows || 4 * q >= there) continue;
          float vx[4], out[4];
          widen4(raw(stage, 0) + t * kChan + 4 * q, vx);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* part = parts(tile & 1) + (t * kChan + i * kQuads + q) * L;
            float sum;
            if constexpr (L == 1) {
              sum = part[0];
            } else if constexpr (L == 2) {
              const float2 v = *reinterpret_cast<const float2*>(part);
              sum = v.x + v.y;
            } else {
              sum = 0.0f;
#pragma unroll
              for (int j = 0; j < L; j += 4) {
                const float4 v = *reinterpret_cast<const float4*>(part + j);
                sum += (v.x + v.y) + (v.z + v.w);
              }
            }
            out[i] = fmaf(d[i], vx[i], sum);
          }
          if (z != nullptr) {
            float vz[4];
            widen4(raw(stage, 2) + t * kChan + 4 * q, vz);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float2 gate = silu_fast<sizeof(T) == 4>(vz[i], vz[i + 1]);
              out[i] *= gate.x; out[i + 1] *= gate.y;
            }
          }
          T* to = y + (t0 + t) * p.E + 4 * q;
          if (!RGK_IN_RANGE(to - static_cast<T*>(p.y), p.B * p.T * p.E - (min(there - 4 * q, 4) - 1), p.status)) continue;
          if (kAligned || (p.store4 && 4 * q + 4 <= there)) {
            if constexpr (sizeof(T) == 2)
              *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(out[0], out[1]), pack_bf16x2(out[2], out[3]));
            else
              *reinterpret_cast<float4*>(to) = make_float4(out[0], out[1], out[2], out[3]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (4 * q + i < there) to[i] = static_cast<T>(out[i]);
            }
          }
        }
      };

      // While the owners work on tile - 1: tile's inputs, then the outputs of tile - 1.  A buffer is written again two
      // tiles later, when the owners have long met for the tile in between.
      if (tiles > 0) ask(0);
      bool start = starts_at(0);
#pragma unroll 1
      for (int tile = 0; tile < tiles; ++tile) {
        settle(tile);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        meet<kTeam>(kHelpersMeet);                               // the tile is here, tile - 2 is done with
        if (tile + 1 < tiles) ask(tile + 1);
        prepare(tile, start);
        start = starts_at(tile + 1);
        arrive<2 * kTeam>(kFull + (tile & 1));
        if (tile > 0) {
          meet<2 * kTeam>(kDone + ((tile - 1) & 1));
          finish(tile - 1);
        }
      }
      if (tiles > 0) {
        meet<2 * kTeam>(kDone + ((tiles - 1) & 1));
        finish(tiles - 1);
      }
    } else {
      // A thread's channels, for each of its c the one at place owner + c * kOwners, and their states in runs of kRun
      // that lie next to its neighbours' (value kRun r + i is state kRun L r + kRun l + i).
      constexpr int kRun = S < 4 ? S : 4, kUnroll = Sh::kUnroll;
      constexpr bool kExact = exact_decays<T>(Sh::kPad);
      const int l = tid & (L - 1), owner = tid / L;
      auto channel_of = [&](int c) { const int at = owner + c * Sh::kOwners; return at % kQuads * 4 + at / kQuads; };
      auto state_of = [&](int s) { return s / kRun * kRun * L + l * kRun + s % kRun; };
      if (chunk > 0) wait_for(p.done + block, (int)chunk, p.wait_limit, p.status);
      const float* from = chunk > 0 ? p.state_out : p.state_in;
      Pair h[C][S / 2], a2[C][S / 2];
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int s = 0; s < S / 2; ++s) {
          float va[2], vh[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n = state_of(2 * s + i), ch = channel_of(c);
            const bool in = ch < there && n < p.N;
            va[i] = in ? p.a[(first + ch) * p.N + n] * kLog2e : 0.0f;
            vh[i] = in && from != nullptr && RGK_IN_RANGE((b * p.E + first + ch) * p.N + n, p.B * p.E * p.N, p.status)
                        ? __ldcg(from + (b * p.E + first + ch) * p.N + n) : 0.0f;
          }
          a2[c][s] = pair(va[0], va[1]);
          h[c][s] = pair(vh[0], vh[1]);
        }
      }
#pragma unroll 1
      for (int tile = 0; tile < tiles; ++tile) {
        const int buf = tile & 1;
        meet<2 * kTeam>(kFull + buf);
        const float2* s_step = steps(buf);
        const float *s_b = wide_b(buf), *s_c = wide_c(buf);
        float* s_part = parts(buf);
        const uint32_t starts = s_starts[buf];
        // (every lane leaves its part of a sum over states: the helpers join them, nothing here waits for another lane)
        auto recur = [&](auto with_starts) {
#pragma unroll 1
          for (int t0 = 0; t0 < kTile; t0 += kUnroll) {
            float sum[kUnroll][C];                               // (stored behind the loads of all of these steps)
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
              const int t = t0 + j, n = t * kPad + l * kRun;
              Pair vb[S / 2], vc[S / 2];
              if constexpr (S == 2) {
                vb[0] = *reinterpret_cast<const Pair*>(s_b + n);
                vc[0] = *reinterpret_cast<const Pair*>(s_c + n);
              } else {
#pragma unroll
                for (int r = 0; r < S / 4; ++r) {
                  const ulonglong2 b4 = *reinterpret_cast<const ulonglong2*>(s_b + n + r * 4 * L);
                  const ulonglong2 c4 = *reinterpret_cast<const ulonglong2*>(s_c + n + r * 4 * L);
                  vb[2 * r] = b4.x; vb[2 * r + 1] = b4.y;
                  vc[2 * r] = c4.x; vc[2 * r + 1] = c4.y;
                }
              }
#pragma unroll
              for (int c = 0; c < C; ++c) {
                const float2 step = s_step[t * kChan + owner + c * Sh::kOwners];
                // (at a start the factor is 1: one that has overflowed would not be dropped by what it multiplies)
                const float by = decltype(with_starts)::value && ((starts >> t) & 1u) ? 0.0f : step.x;
                const Pair step2 = pair(by, by), put2 = pair(step.y, step.y);
                Pair both = 0;
#pragma unroll
                for (int s = 0; s < S / 2; ++s) {
                  Pair before = h[c][s];
                  if (decltype(with_starts)::value && ((starts >> t) & 1u)) before = 0;
                  h[c][s] = fma2(decays<kExact>(step2, a2[c][s]), before, mul2(put2, vb[s]));
                  both = s == 0 ? mul2(h[c][s], vc[s]) : fma2(h[c][s], vc[s], both);
                }
                const float2 halves = split(both);
                sum[j][c] = halves.x + halves.y;
              }
            }
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
#pragma unroll
              for (int c = 0; c < C; ++c) s_part[((t0 + j) * C + c) * kTeam + tid] = sum[j][c];
            }
          }
        };
        if (starts != 0) recur(std::true_type{});
        else recur(std::false_type{});
        arrive<2 * kTeam>(kDone + buf);
      }
      if (p.state_out != nullptr) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int ch = channel_of(c);
          if (ch >= there) continue;
#pragma unroll
          for (int s = 0; s < S; ++s) {
            const int n = state_of(s);
            const float2 v = split(h[c][s / 2]);
            if (n < p.N && RGK_IN_RANGE((b * p.E + first + ch) * p.N + n, p.B * p.E * p.N, p.status))
              p.state_out[(b * p.E + first + ch) * p.N + n] = s % 2 == 0 ? v.x : v.y;
          }
        }
      }
    }
    if (p.chunks == 1) return;
    __syncthreads();
    if (threadIdx.x == 0) {
      if (chunk + 1 < p.chunks && RGK_IN_RANGE(block, kMostBlocks, p.status)) {
        __threadfence();
        asm volatile("st.release.gpu.global.s32 [%0], %1;" :: "l"(p.done + block), "r"((int)chunk + 1) : "memory");
      }
    }
    item = draw();
  }
}

template <typename T, typename Sh, bool kAligned>
cudaError_t launch_kernel(SelectiveArgs p, cudaStream_t s) {
  static PerDeviceOnce once;
  int sms = 0;
  cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(selective_scan_kernel<T, Sh, kAligned>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kBytes);
  }, &sms);
  if (e != cudaSuccess) return e;
  p.blocks_per_group = (p.per_group + Sh::kChan - 1) / Sh::kChan;
  p.blocks = (int64_t)p.blocks_per_group * p.groups * p.B;
  p.chunk = p.T;
  p.chunks = 1;
  if (p.blocks >= ((int64_t)1 << 31)) return cudaErrorInvalidValue;
  int64_t grid = p.blocks;
  if (p.wait_limit == 0) p.wait_limit = kWaitLimit;
  // Chunks of time drawn by a ticket.
  if (p.ticket != nullptr && p.state_out != nullptr && p.T >= kScanChunksFrom) {
    int per_sm = 0;
    if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, selective_scan_kernel<T, Sh, kAligned>, 2 * kTeam,
                                                           Sh::kBytes)) != cudaSuccess) return e;
    const int64_t most = min((int64_t)per_sm, p.blocks / sms);
    if ((p.skip_first || (most > 0 && most * sms < p.blocks)) && p.blocks <= kMostBlocks) {
      grid = p.skip_first ? p.blocks : most * sms;
      // (24 of them: the last round is short of 4 % at most; no longer than a wait for one is given)
      p.chunk = min((int64_t)4096, max((int64_t)128, (p.T / 24 + Sh::kTile - 1) / Sh::kTile * Sh::kTile));
      p.chunks = (p.T + p.chunk - 1) / p.chunk;
      p.done = reinterpret_cast<int*>(p.ticket) + 1;
      if ((e = cudaMemsetAsync(p.ticket, 0, (1 + p.blocks) * sizeof(int), s)) != cudaSuccess) return e;
      if (p.skip_first && (e = cudaMemsetAsync(p.ticket, (int)p.blocks, 1, s)) != cudaSuccess) return e;  // (below 256)
    }
  }
  selective_scan_kernel<T, Sh, kAligned><<<(unsigned)grid, 2 * kTeam, Sh::kBytes, s>>>(p);
  return cudaGetLastError();
}
template <typename T, int S, int C, int L, int kTile>
cudaError_t launch(const SelectiveArgs& p, cudaStream_t s) {
  using Sh = Shape<T, S, C, L, kTile>;
  // (with whole copies of x's rows there are whole quads of channels too)
  const bool aligned = p.copy_x >= min(16, Sh::kChan * (int)sizeof(T)) && p.copy_n >= min(16, Sh::kPad * (int)sizeof(T)) &&
                       p.store4;
  return aligned ? launch_kernel<T, Sh, true>(p, s) : launch_kernel<T, Sh, false>(p, s);
}

template <bool kExact>
__device__ __forceinline__ float softplus_step(float v) {        // softplus_steps for one
  const float e = kExact ? exp_exact(-fabsf(v)) : exp2_fast(-fabsf(v) * kLog2e);
  float q = softplus_coefficient(9);
#pragma unroll
  for (int i = 8; i >= 0; --i) q = fmaf(q, e, softplus_coefficient(i));
  return fmaf(q, e, fmaxf(v, 0.0f));
}

template <typename T> struct Four;                               // four elements as they lie in memory
template <> struct Four<float> { using type = float4; };
template <> struct Four<__nv_bfloat16> { using type = uint2; };
__device__ __forceinline__ void widen4(const float4& v, float* f) { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
__device__ __forceinline__ void widen4(const uint2& v, float* f) {
  f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x); f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
}

// One time step: the states are read and written once and bound it.  A lane holds four states (8 beyond 128) of each
// of kRows sequences, L lanes a channel, so that a, d and the bias are read once for kRows sequences and all that is
// read of kRows sequences is in flight at a time.  kVec: states, b and c are read and written four at a time.
template <typename T, int S, int L, int kRows, bool kVec>
__global__ void __launch_bounds__(256)
selective_step_kernel(const SelectiveArgs p) {
  using Raw = typename Four<T>::type;
  constexpr int Q = S / 4;
  constexpr bool kExact = exact_decays<T>(S * L);
  const int64_t at = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const int l = threadIdx.x % L;
  const bool in = at < p.E;
  const int64_t e = in ? at : p.E - 1;                           // (whole groups of lanes: they shuffle)
  const int64_t b0 = (int64_t)blockIdx.y * kRows;
  const int g = (int)(e / p.per_group);

  // a quad of the lane: states 4 L k + 4 l on; there: how many of them exist
  auto quad = [&](int k) { return k * 4 * L + l * 4; };
  float4 h[kRows][Q];
  Raw vb[kRows][Q], vc[kRows][Q];
  T x[kRows], dt[kRows], z[kRows];
  bool fresh[kRows];                                             // nothing of what was held counts
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t b = min(b0 + r, p.B - 1);
    fresh[r] = p.state_in == nullptr || (p.pos != nullptr && pos_is_zero(p.pos, p.pos64, b));
    const float* from = p.state_in + (b * p.E + e) * p.N;
    const T* rb = static_cast<const T*>(p.b) + b * p.b_batch + (int64_t)g * p.N;
    const T* rc = static_cast<const T*>(p.c) + b * p.c_batch + (int64_t)g * p.N;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      const int n = quad(k);
      h[r][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      vb[r][k] = vc[r][k] = Raw{};
      if (kVec) {
        if (n < p.N) {
          if (!fresh[r]) h[r][k] = *reinterpret_cast<const float4*>(from + n);
          vb[r][k] = *reinterpret_cast<const Raw*>(rb + n);
          vc[r][k] = *reinterpret_cast<const Raw*>(rc + n);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (n + i < p.N) {
            if (!fresh[r]) (&h[r][k].x)[i] = from[n + i];
            reinterpret_cast<T*>(&vb[r][k])[i] = rb[n + i];
            reinterpret_cast<T*>(&vc[r][k])[i] = rc[n + i];
          }
        }
      }
    }
    x[r] = static_cast<const T*>(p.x)[b * p.x_batch + e];
    dt[r] = static_cast<const T*>(p.dt)[b * p.dt_batch + e];
    z[r] = p.z != nullptr ? static_cast<const T*>(p.z)[b * p.z_batch + e] : T(0.0f);
  }
  float a2[S];
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    const int n = quad(k);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (kVec && p.N % 4 == 0 && reinterpret_cast<uintptr_t>(p.a) % 16 == 0) {
      if (n < p.N) v = *reinterpret_cast<const float4*>(p.a + e * p.N + n);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (n + i < p.N) (&v.x)[i] = p.a[e * p.N + n + i];
      }
    }
    a2[4 * k] = v.x * kLog2e; a2[4 * k + 1] = v.y * kLog2e; a2[4 * k + 2] = v.z * kLog2e; a2[4 * k + 3] = v.w * kLog2e;
  }
  const float bias = p.dt_bias != nullptr ? p.dt_bias[e] : 0.0f, d = p.d != nullptr ? p.d[e] : 0.0f;

#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t b = b0 + r;
    if (b >= p.B) break;
    const float xr = static_cast<float>(x[r]);
    float now = static_cast<float>(dt[r]) + bias;
    if (p.softplus) now = softplus_step<sizeof(T) == 4>(now);
    const float put = now * xr, by = fresh[r] ? 0.0f : now;       // (a factor that has overflowed multiplies nothing)
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      const int n = quad(k);
      float fb[4], fc[4], fh[4];
      widen4(vb[r][k], fb);
      widen4(vc[r][k], fc);
      widen4(h[r][k], fh);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float2 decay = decays<kExact>(by, a2[4 * k + i], a2[4 * k + i + 1]);
        fh[i] = fmaf(decay.x, fh[i], put * fb[i]);
        fh[i + 1] = fmaf(decay.y, fh[i + 1], put * fb[i + 1]);
        sum = fmaf(fh[i], fc[i], sum);
        sum = fmaf(fh[i + 1], fc[i + 1], sum);
      }
      if (p.state_out != nullptr && in) {
        float* to = p.state_out + (b * p.E + e) * p.N + n;
        if (kVec) {
          if (n < p.N) *reinterpret_cast<float4*>(to) = make_float4(fh[0], fh[1], fh[2], fh[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (n + i < p.N) to[i] = fh[i];
          }
        }
      }
    }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (l == 0 && in) {
      float out = fmaf(d, xr, sum);
      if (p.z != nullptr) out *= silu_fast<sizeof(T) == 4>(static_cast<float>(z[r]));
      static_cast<T*>(p.y)[b * p.E + e] = static_cast<T>(out);
    }
  }
}

// The same for many sequences: a thread goes through kDepth and more of them with the same four states of a channel, whose
// values come by copies that run kDepth sequences ahead into places of its own in shared memory (nobody else reads them:
// no barriers), the rest of a sequence a step ahead into registers.  256 x 5120 x 16 in bfloat16: 48 us with
// four sequences a thread, 44 so (63 % of the measured copy rate).
// (Addresses run along: products of 64 bits for every row were most of its 237 instructions, which bound it.)
template <typename T, int L>
__global__ void __launch_bounds__(256, 4)
selective_steps_kernel(const SelectiveArgs p, int per) {
  using Raw = typename Four<T>::type;
  constexpr int kDepth = 8;
  constexpr bool kExact = exact_decays<T>(4 * L);
  __shared__ float4 ring[kDepth][256];
  const int64_t at = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const int l = threadIdx.x % L;
  const bool in = at < p.E;
  const int64_t e = in ? at : p.E - 1;                           // (whole groups of lanes: they shuffle)
  const bool there = l * 4 < p.N, mine = in && there;
  const int n = there ? l * 4 : 0;                               // (a lane too many reads what the first one does)
  const int64_t b0 = (int64_t)blockIdx.y * per;
  const int rows = (int)min((int64_t)per, p.B - b0), g = (int)(e / p.per_group);

  const int64_t row = p.E * p.N, place = b0 * row + e * p.N + n; // of a state
  const bool held = p.state_in != nullptr, gated = p.z != nullptr;
  const float* from = held ? p.state_in + place : nullptr;
  float* to = mine && p.state_out != nullptr ? p.state_out + place : nullptr;
  const T *px = static_cast<const T*>(p.x) + b0 * p.x_batch + e, *pdt = static_cast<const T*>(p.dt) + b0 * p.dt_batch + e;
  const T* pz = gated ? static_cast<const T*>(p.z) + b0 * p.z_batch + e : px;
  const int64_t z_batch = gated ? p.z_batch : p.x_batch;
  const T* pb = static_cast<const T*>(p.b) + b0 * p.b_batch + (int64_t)g * p.N + n;
  const T* pc = static_cast<const T*>(p.c) + b0 * p.c_batch + (int64_t)g * p.N + n;
  T* y = static_cast<T*>(p.y) + b0 * p.E + e;

  int asked = 0;
  auto ask = [&]() {
    if (held && asked < rows) {
      copy_async<16>(&ring[asked % kDepth][threadIdx.x], from, true);
      from += row;
    }
    ++asked;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  struct Inputs { Raw b, c; T x, dt, z; };
  auto inputs = [&]() {
    Inputs v;
    v.b = *reinterpret_cast<const Raw*>(pb);
    v.c = *reinterpret_cast<const Raw*>(pc);
    v.x = *px; v.dt = *pdt; v.z = *pz;
    pb += p.b_batch; pc += p.c_batch; px += p.x_batch; pdt += p.dt_batch; pz += z_batch;
    return v;
  };
  for (int r = 0; r < kDepth - 1; ++r) ask();
  Inputs next = inputs();
  float a2[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) a2[i] = there ? p.a[e * p.N + n + i] * kLog2e : 0.0f;
  const float bias = p.dt_bias != nullptr ? p.dt_bias[e] : 0.0f, d = p.d != nullptr ? p.d[e] : 0.0f;

#pragma unroll 1
  for (int r = 0; r < rows; ++r) {
    ask();                                                       // (where the sequence before this one has been)
    const Inputs v = next;
    if (r + 1 < rows) next = inputs();
    asm volatile("cp.async.wait_group %0;" :: "n"(kDepth - 1) : "memory");
    float h[4] = {0.0f, 0.0f, 0.0f, 0.0f}, fb[4], fc[4];
    const bool fresh = !held || (p.pos != nullptr && pos_is_zero(p.pos, p.pos64, b0 + r));
    if (!fresh) {
      const float4 was = ring[r % kDepth][threadIdx.x];
      h[0] = was.x; h[1] = was.y; h[2] = was.z; h[3] = was.w;
    }
    widen4(v.b, fb);
    widen4(v.c, fc);
    const float x = static_cast<float>(v.x);
    float now = static_cast<float>(v.dt) + bias;
    if (p.softplus) now = softplus_step<sizeof(T) == 4>(now);
    const float put = now * x, by = fresh ? 0.0f : now;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float2 decay = decays<kExact>(by, a2[i], a2[i + 1]);
      h[i] = fmaf(decay.x, h[i], put * fb[i]);
      h[i + 1] = fmaf(decay.y, h[i + 1], put * fb[i + 1]);
      sum = fmaf(h[i], fc[i], sum);
      sum = fmaf(h[i + 1], fc[i + 1], sum);
    }
    if (to != nullptr) {
      *reinterpret_cast<float4*>(to) = make_float4(h[0], h[1], h[2], h[3]);
      to += row;
    }
    sum = there ? sum : 0.0f;
#pragma unroll
    for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (l == 0 && in) {
      float out = fmaf(d, x, sum);
      if (gated) out *= silu_fast<sizeof(T) == 4>(static_cast<float>(v.z));
      *y = static_cast<T>(out);
    }
    y += p.E;
  }
}

template <typename T, int S, int L>
cudaError_t launch_step(const SelectiveArgs& p, int sms, cudaStream_t s) {
  auto fits = [&](const void* q, int64_t batch, int size) {
    return (reinterpret_cast<uintptr_t>(q) | (uint64_t)(batch * size)) % (4 * size) == 0;
  };
  const bool vec = p.N % 4 == 0 && fits(p.state_in, 0, 4) && fits(p.state_out, 0, 4) && fits(p.b, p.b_batch, sizeof(T)) &&
                   fits(p.c, p.c_batch, sizeof(T));
  const unsigned across = (unsigned)((p.E + 256 / L - 1) / (256 / L));
  if constexpr (S == 4) {
    if (vec) {
      // eight sequences a thread and more where four CTAs an SM have that many
      const int64_t down = max((int64_t)1, (int64_t)4 * sms / across), per = (p.B + down - 1) / down;
      if (per >= 8)
        selective_steps_kernel<T, L><<<dim3(across, (unsigned)((p.B + per - 1) / per)), 256, 0, s>>>(p, (int)per);
      else
        selective_step_kernel<T, S, L, 1, true><<<dim3(across, (unsigned)p.B), 256, 0, s>>>(p);
      return cudaGetLastError();
    }
  }
  // four sequences a thread where they still give every SM its threads
  const bool many = across * p.B >= 4 * 8 * (int64_t)sms;
  const dim3 grid(across, (unsigned)(many ? (p.B + 3) / 4 : p.B));
  if constexpr (S != 4) {
    if (vec && many) selective_step_kernel<T, S, L, 4, true><<<grid, 256, 0, s>>>(p);
    else if (vec) selective_step_kernel<T, S, L, 1, true><<<grid, 256, 0, s>>>(p);
    if (vec) return cudaGetLastError();
  }
  if (many) selective_step_kernel<T, S, L, 4, false><<<grid, 256, 0, s>>>(p);
  else selective_step_kernel<T, S, L, 1, false><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch_step_states(const SelectiveArgs& p, int sms, cudaStream_t s) {
  if (p.N <= 4) return launch_step<T, 4, 1>(p, sms, s);
  if (p.N <= 8) return launch_step<T, 4, 2>(p, sms, s);
  if (p.N <= 16) return launch_step<T, 4, 4>(p, sms, s);
  if (p.N <= 32) return launch_step<T, 4, 8>(p, sms, s);
  if (p.N <= 64) return launch_step<T, 4, 16>(p, sms, s);
  if (p.N <= 128) return launch_step<T, 4, 32>(p, sms, s);
  return launch_step<T, 8, 32>(p, sms, s);
}

// There is a choice of shapes: few states a thread keep a step short where channels are few, many states and two channels
// share what is read from shared memory where they are many.  What a shape takes for 1024 steps, us: `alone` where every
// CTA has an SM, and for each round of SMs `some` up to two of them, `many` beyond (where time is cut into chunks).
struct Choice { double alone, some, many; int channels; };       // channels of a CTA
template <int kCount>
int quickest(const Choice (&of)[kCount], const SelectiveArgs& p, int sms) {
  int best = 0;
  double least = 0.0;
  for (int i = kCount - 1; i >= 0; --i) {
    const int64_t blocks = (p.per_group + of[i].channels - 1) / of[i].channels * p.groups * p.B;
    const double rounds = (double)blocks / sms;
    const double time = rounds <= 1.0 ? of[i].alone : rounds * (rounds < 2.0 ? of[i].some : of[i].many);
    // (more channels a CTA fetch b and c less often, which counts where those are not aligned: a tie goes to them)
    if (i == kCount - 1 || time < 0.96 * least) { best = i; least = time; }
  }
  return best;
}

// Measured on one B200 with 640 to 40960 channels, in the order of the shapes; a shape's three numbers come from 1024,
// 1280 to 4096, and 5120 and more.  For instance 2560 / 10240 / 40960 channels, 16 states in float32: 65 / 171 / 643, 54 /
// 123 / 436, 91 / 130 / 388, 165 / 167 / 439; in bfloat16: 58 / 148 / 553, 46 / 99 / 364, 69 / 103 / 282, 124 / 124 / 277.  64
// states in float32: 132 / 486 / 1900, 124 / 360 / 1382, 169 / 334 / 1240; in bfloat16: 122 / 450 / 1759, 103 / 283 / 1079,
// 114 / 237 / 873.
template <typename T>
cudaError_t launch_states(const SelectiveArgs& p, int sms, cudaStream_t s) {
  constexpr bool kF32 = sizeof(T) == 4;
  if (p.N <= 4) return launch<T, 4, 1, 1, 16>(p, s);
  if (p.N <= 8) {
    static constexpr Choice f32[] = {{67, 96, 63, 64}, {120, 153, 148, 128}};
    static constexpr Choice bf16[] = {{57, 79, 51, 64}, {96, 124, 87, 128}};
    return quickest(kF32 ? f32 : bf16, p, sms) == 0 ? launch<T, 4, 1, 2, 16>(p, s) : launch<T, 4, 2, 2, 16>(p, s);
  }
  if (p.N <= 16) {
    static constexpr Choice f32[] = {{42, 59, 40, 16}, {54, 77, 55, 32}, {91, 120, 95, 64}, {165, 210, 203, 128}};
    static constexpr Choice bf16[] = {{35, 53, 35, 16}, {45, 68, 45, 32}, {69, 95, 67, 64}, {124, 168, 128, 128}};
    switch (quickest(kF32 ? f32 : bf16, p, sms)) {
      case 0: return launch<T, 2, 1, 8, 32>(p, s);
      case 1: return launch<T, 4, 1, 4, 32>(p, s);
      case 2: return launch<T, 8, 1, 2, 16>(p, s);
      default: return launch<T, 8, 2, 2, 16>(p, s);
    }
  }
  if (p.N <= 32) {
    static constexpr Choice f32[] = {{56, 76, 54, 16}, {85, 111, 86, 32}, {171, 212, 155, 64}};
    static constexpr Choice bf16[] = {{47, 66, 45, 16}, {68, 92, 65, 32}, {118, 152, 108, 64}};
    switch (quickest(kF32 ? f32 : bf16, p, sms)) {
      case 0: return launch<T, 4, 1, 8, 32>(p, s);
      case 1: return launch<T, 8, 1, 4, 16>(p, s);
      default: return launch<T, 8, 2, 4, 16>(p, s);
    }
  }
  if (p.N <= 64) {
    static constexpr Choice f32[] = {{69, 88, 59, 8}, {89, 112, 87, 16}, {169, 203, 150, 32}};
    static constexpr Choice bf16[] = {{66, 84, 54, 8}, {71, 94, 67, 16}, {114, 143, 106, 32}};
    switch (quickest(kF32 ? f32 : bf16, p, sms)) {
      case 0: return launch<T, 4, 1, 16, 16>(p, s);
      case 1: return launch<T, 8, 1, 8, 16>(p, s);
      default: return launch<T, 8, 2, 8, 16>(p, s);
    }
  }
  if (p.N <= 128) {
    static constexpr Choice f32[] = {{105, 125, 95, 8}, {216, 243, 167, 16}};
    static constexpr Choice bf16[] = {{83, 104, 74, 8}, {148, 168, 117, 16}};
    return quickest(kF32 ? f32 : bf16, p, sms) == 0 ? launch<T, 8, 1, 16, 16>(p, s) : launch<T, 8, 2, 16, 8>(p, s);
  }
  return launch<T, 8, 1, 32, 8>(p, s);
}

// The largest copy (bytes) that every address base + i * batch + j * token + k * width (elements) allows.
int copy_bytes(const void* base, int64_t batch, int64_t token, int64_t width, int size) {
  const uint64_t all = (uint64_t)reinterpret_cast<uintptr_t>(base) | (uint64_t)(batch * size) | (uint64_t)(token * size) |
                       (uint64_t)(width * size);
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

}  // namespace

size_t selective_workspace_bytes() { return (1 + kMostBlocks) * sizeof(int); }

cudaError_t launch_selective_scan(SelectiveArgs p, int dtype, cudaStream_t s) {
  if (p.B == 0 || p.E == 0) return cudaSuccess;
  const int size = dtype == 1 ? 2 : 4;
  static PerDeviceOnce once;
  int sms = 0;
  const cudaError_t e = once.run([] { return cudaSuccess; }, &sms);
  if (e != cudaSuccess) return e;
  p.per_group = (int)(p.E / p.groups);
  if (p.T == 1) return dtype == 1 ? launch_step_states<__nv_bfloat16>(p, sms, s) : launch_step_states<float>(p, sms, s);
  p.copy_x = min(copy_bytes(p.x, p.x_batch, p.x_token, p.per_group, size),
                 copy_bytes(p.dt, p.dt_batch, p.dt_token, p.per_group, size));
  if (p.z != nullptr) p.copy_x = min(p.copy_x, copy_bytes(p.z, p.z_batch, p.z_token, p.per_group, size));
  p.copy_n = min(copy_bytes(p.b, p.b_batch, p.b_token, p.N, size), copy_bytes(p.c, p.c_batch, p.c_token, p.N, size));
  p.store4 = p.per_group % 4 == 0 && p.E % 4 == 0 && reinterpret_cast<uintptr_t>(p.y) % (4 * size) == 0;
  return dtype == 1 ? launch_states<__nv_bfloat16>(p, sms, s) : launch_states<float>(p, sms, s);
}

}  // namespace rgk
