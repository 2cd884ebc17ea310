// One token per row of logits: temperature, top-k, top-p and min-p, drawn by a given uniform number.
//
// Weights are integers: W(l) = 2^F exp((l - max) / T), rounded, with F = 44 or as many bits as keep the sum of a row
// below 2^62.  Sums of integers do not depend on their order, so that a row gives the same token whatever the launch,
// and 44 bits make the borders between tokens finer than a float32 sum over 256000 of them could (whose rounding would
// move a border by a few percent of such a token's width).  Order: logit descending, ties by lowest index.
//   top-k   the cut is the largest key (the logit's bits, made monotonic) above which fewer than k logits lie
//   top-p   the same with weights instead of counts, and p of the kept weight instead of k
//   min-p   W(l) >= min_p 2^F
//   draw    the first index at which the kept weights sum to more than u times all of them
// A cut is found by histograms over a narrowing range of keys; ties at the cut are kept up to an index.
#include "rgk_common.cuh"
#include "rgk_internal.h"

namespace rgk {
namespace {

using u64 = unsigned long long;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kSlice = 256;                                       // tokens whose weights are summed before the last walk

// The order of the floats as an order of integers (-0 counts as 0, NaN below everything).
__device__ __forceinline__ uint32_t key_of(float l) {
  if (l != l) return 0u;
  const uint32_t b = __float_as_uint(l + 0.0f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}
constexpr uint32_t kKeyNothing = 0x007fffffu;                     // key of -inf

struct Weights {
  double scale;                                                   // log2(e) / T
  double max;
  float fmax;
  double unit;                                                    // 2^F
  // exp2 on [-1/2, 1/2] by its Taylor polynomial of degree 11 (6e-15)
  __device__ u64 operator()(float l) const {
    if (l == fmax) return (u64)unit;
    const double t = ((double)l - max) * scale;
    if (!(t > -50.0)) return 0;                                   // (NaN too)
    const double n = rint(t), f = (t - n) * 0.6931471805599453;
    double p = 1.0 / 39916800.0;
    p = fma(p, f, 1.0 / 3628800.0);
    p = fma(p, f, 1.0 / 362880.0);
    p = fma(p, f, 1.0 / 40320.0);
    p = fma(p, f, 1.0 / 5040.0);
    p = fma(p, f, 1.0 / 720.0);
    p = fma(p, f, 1.0 / 120.0);
    p = fma(p, f, 1.0 / 24.0);
    p = fma(p, f, 1.0 / 6.0);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    return (u64)__double2ll_rn(p * unit * __hiloint2double((1023 + (int)n) << 20, 0));
  }
};

// What is kept: keys above `key`, and those equal to it up to index `last`.
struct Cut {
  uint32_t key;
  u64 ties;                                                       // how many of those equal to it
  int last;
};

struct Shared {
  u64 hist[kBins];
  u64 part[kWarps];
  float part_f[kWarps];
  int part_i[kWarps];
  u64 total;
  int found;
  u64 above;
  u64 at;
};

__device__ u64 block_sum(u64 v, Shared& sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 s = 0;
  for (int w = 0; w < kWarps; ++w) s += sh.part[w];
  return s;
}

// The entry of `n` values v[0..n) at which their running sum first exceeds `target`: into sh.found, and the sum in
// front of it into sh.above (found stays -1 where the whole sum does not exceed it).  n <= 4 * kThreads.
__device__ void find_first(const u64* v, int n, bool backwards, u64 target, Shared& sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  u64 mine[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = tid * 4 + i;
    mine[i] = at < n ? v[backwards ? n - 1 - at : at] : 0;
    sum += mine[i];
  }
  u64 upto = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 q = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += q;
  }
  __syncthreads();
  if (tid == 0) sh.found = -1;
  if (lane == 31) sh.part[warp] = upto;
  __syncthreads();
  u64 before = upto - sum;
  for (int w = 0; w < warp; ++w) before += sh.part[w];
  if (before <= target) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before <= target && before + mine[i] > target) {
        sh.found = backwards ? n - 1 - (tid * 4 + i) : tid * 4 + i;
        sh.above = before;
      }
      before += mine[i];
    }
  }
  __syncthreads();
}

// The cut that keeps the shortest prefix whose measure (weights, or counts) reaches `target` among what `was` keeps.
template <bool kCount, typename T>
__device__ Cut select(const T* row, int V, uint32_t lo, uint32_t hi, u64 target, const Cut& was, const Weights& weight,
                      Shared& sh) {
  u64 above = 0;
  if (lo <= was.key) lo = was.key;
  while (true) {
    int shift = 0;
    while (((hi - lo) >> shift) >= (uint32_t)kBins) ++shift;
    const int bins = (int)((hi - lo) >> shift) + 1;
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += kThreads) sh.hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float l = static_cast<float>(row[i]);
      const uint32_t k = key_of(l);
      if (k < lo || k > hi || (k == was.key && i > was.last)) continue;
      atomicAdd(&sh.hist[(k - lo) >> shift], kCount ? 1ull : weight(l));
    }
    __syncthreads();
    find_first(sh.hist, bins, true, target - 1 - above, sh);      // (the sum has to reach target - above)
    const int bin = sh.found;
    if (bin < 0) return was;                                      // all of it does not reach the target
    above += sh.above;
    lo += (uint32_t)bin << shift;
    hi = min(hi, lo + (uint32_t)((1ull << shift) - 1));
    if (shift == 0) break;
  }
  const u64 there = sh.hist[sh.found];
  const float l = __uint_as_float((lo >> 31) ? lo & 0x7fffffffu : ~lo);
  const u64 each = kCount ? 1ull : weight(l);
  const u64 ties = (target - above + each - 1) / each;
  Cut cut{lo, ties, V};
  if (ties * each < there) {                                      // not all of them: up to which index
    u64* count = sh.hist;
    const int slices = (V + kSlice - 1) / kSlice;
    __syncthreads();
    // (per slice, at most 4096 of them: two counts to a word of the histogram)
    uint32_t* counts = reinterpret_cast<uint32_t*>(count);
    for (int s = threadIdx.x >> 5; s < slices; s += kWarps) {
      int n = 0;
      for (int i = s * kSlice + (threadIdx.x & 31); i < min(V, (s + 1) * kSlice); i += 32)
        n += key_of(static_cast<float>(row[i])) == lo;
      n = __reduce_add_sync(0xffffffffu, n);
      if ((threadIdx.x & 31) == 0) counts[s] = (uint32_t)n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 left = ties;
      int s = 0;
      while (left > counts[s]) left -= counts[s++];
      int i = s * kSlice;
      for (;; ++i) {
        if (key_of(static_cast<float>(row[i])) == lo && --left == 0) break;
      }
      sh.found = i;
    }
    __syncthreads();
    cut.last = sh.found;
  }
  return cut;
}

template <typename V> __device__ __forceinline__ V setting(const V* p, V value, int64_t m) { return p != nullptr ? p[m] : value; }

template <typename T>
__global__ void __launch_bounds__(kThreads)
sample_kernel(const SampleArgs p) {
  __shared__ Shared sh;
  extern __shared__ u64 slices[];
  const int64_t m = blockIdx.x;
  const int V = (int)p.V, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* row = static_cast<const T*>(p.logits) + m * p.row_stride;

  // the first maximum
  float best = -INFINITY;
  int at = V;
  for (int i = tid; i < V; i += kThreads) {
    const float l = static_cast<float>(row[i]);
    if (l > best) { best = l; at = i; }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ob = __shfl_xor_sync(0xffffffffu, best, o);
    const int oa = __shfl_xor_sync(0xffffffffu, at, o);
    if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
  }
  if (lane == 0) { sh.part_f[warp] = best; sh.part_i[warp] = at; }
  __syncthreads();
  best = sh.part_f[0]; at = sh.part_i[0];
  for (int w = 1; w < kWarps; ++w) {
    if (sh.part_f[w] > best || (sh.part_f[w] == best && sh.part_i[w] < at)) { best = sh.part_f[w]; at = sh.part_i[w]; }
  }
  const float temperature = setting(p.temperature, p.temperature_value, m);
  if (best == -INFINITY || !(temperature > 0.0f)) {
    if (tid == 0) p.out[m] = best == -INFINITY ? 0 : at;
    return;
  }
  best += 0.0f;
  const Weights weight{1.4426950408889634 / (double)temperature, (double)best, best, (double)(1ull << p.bits)};

  // what weighs nothing needs no place in the ranges: W = 0 from (bits + 1) ln 2 temperatures below the maximum
  const uint32_t hi = key_of(best);
  const uint32_t lo = min(hi, key_of(__fsub_rd(best, __fmul_ru(32.0f, temperature))));
  Cut cut{max(lo, kKeyNothing + 1) - 1, 0, -1};
  const int top_k = setting(p.top_k, p.top_k_value, m);
  if (top_k > 0 && top_k < V) cut = select<true>(row, V, cut.key + 1, hi, (u64)top_k, cut, weight, sh);
  const float top_p = setting(p.top_p, p.top_p_value, m);
  if (top_p < 1.0f) {
    u64 sum = 0;
    for (int i = tid; i < V; i += kThreads) {
      const float l = static_cast<float>(row[i]);
      const uint32_t k = key_of(l);
      if (k > cut.key || (k == cut.key && i <= cut.last)) sum += weight(l);
    }
    const double want = ceil((double)top_p * (double)block_sum(sum, sh));
    cut = select<false>(row, V, cut.key, hi, want > 1.0 ? (u64)want : 1ull, cut, weight, sh);
  }
  const double min_p = (double)setting(p.min_p, p.min_p_value, m);
  const u64 least = min_p > 0.0 ? (u64)ceil(fmin(min_p, 1.0) * weight.unit) : 0ull;
  auto kept = [&](float l, int i) -> u64 {
    const uint32_t k = key_of(l);
    if (!(k > cut.key || (k == cut.key && i <= cut.last))) return 0;
    const u64 w = weight(l);
    return w >= least ? w : 0;
  };

  const int n = (V + kSlice - 1) / kSlice;
  u64 total = 0;
  for (int s = warp; s < n; s += kWarps) {
    u64 sum = 0;
    for (int i = s * kSlice + lane; i < min(V, (s + 1) * kSlice); i += 32) sum += kept(static_cast<float>(row[i]), i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) { slices[s] = sum; total += sum; }
  }
  total = block_sum(total, sh);
  const float u = p.uniforms[m];
  u64 target = u > 0.0f ? (u64)((double)fminf(u, 1.0f) * (double)total) : 0ull;
  if (target >= total) target = total - 1;
  find_first(slices, n, false, target, sh);
  if (warp == 0) {
    const int s = sh.found;
    u64 before = sh.above;
    for (int i0 = s * kSlice; i0 < V; i0 += 32) {
      const int i = i0 + lane;
      u64 upto = i < V ? kept(static_cast<float>(row[i]), i) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 q = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += q;
      }
      const unsigned over = __ballot_sync(0xffffffffu, before + upto > target);
      if (over != 0) {
        if (lane == 0) p.out[m] = i0 + __ffs(over) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& p, int dtype, cudaStream_t s) {
  if (p.M == 0) return cudaSuccess;
  const size_t smem = (size_t)((p.V + kSlice - 1) / kSlice) * sizeof(u64);
  static PerDeviceOnce once;
  const cudaError_t e = once.run([] {
    const cudaError_t a = cudaFuncSetAttribute(sample_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
    if (a != cudaSuccess) return a;
    return cudaFuncSetAttribute(sample_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
  });
  if (e != cudaSuccess) return e;
  if (dtype == 1) sample_kernel<__nv_bfloat16><<<(unsigned)p.M, kThreads, smem, s>>>(p);
  else sample_kernel<float><<<(unsigned)p.M, kThreads, smem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace rgk
