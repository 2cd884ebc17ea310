// One token per row of logits: temperature, top-k, top-p and min-p, drawn by a given uniform number.
//
// Weights are integers: W(l) = 2^F exp((l - max) / T), rounded, with F = 44 or as many bits as keep the sum of a row
// below 2^62.  Sums of integers do not depend on their order, so that a row gives the same token whatever the launch,
// and 44 bits make the borders between tokens finer than a float32 sum over 256000 of them could (whose rounding would
// move a border by a few percent of such a token's width).  Order: logit descending, ties by lowest index.
//   top-k   the longest prefix of k tokens
//   top-p   the shortest prefix with p of the weight of those
//   min-p   W(l) >= min_p 2^F
//   draw    the first index at which the kept weights sum to more than u times all of them
//
// Nothing is sorted but short lists.  A cluster of CTAs shares a row, every warp a run of it that it reads again for
// each pass (HBM the first time, L2 or L1 after that).  A prefix is found by a histogram of counts and weights over the
// distance from the maximum: 2048 bins of 1/64 temperature, added up over the cluster.  Where the bins up to the one
// that it ends in hold at most 2048 tokens, those are brought together in index order, and one CTA sorts them and does
// the rest; otherwise the bin's own tokens are, which gives the last token kept, and the draw runs over the row.  A bin
// with more tokens than that (ties, huge temperatures) is cut into 2048 ranges of keys, and again if need be; a single
// key is cut by counting.
//
// Bound: 2 or 4 bytes a token from HBM, and for whole rows and top-p without top-k the 64-bit exponential of every token
// within 31 temperatures of the maximum (11 double-precision operations, 2 cycles of a scheduler each).
#include "rgk_common.cuh"
#include "rgk_internal.h"
#include "tc_common.cuh"

namespace rgk {
namespace {

using u64 = unsigned long long;
#ifndef MINB
#define MINB 1
#endif
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;                                       // four to a thread
constexpr int kList = 2048;                                       // longest list that is sorted, four to a thread
constexpr int kMostParts = 8;
constexpr float kRange = 32.0f;                                   // temperatures below the maximum: W = 0 from 31.2 on
constexpr int kTable = 64;

// The order of the floats as an order of integers (-0 counts as 0, NaN below everything).
__device__ __forceinline__ uint32_t key_of(float l) {
  if (l != l) return 0u;
  const uint32_t b = __float_as_uint(l + 0.0f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key >> 31) ? key & 0x7fffffffu : ~key);
}
constexpr uint32_t kKeyNothing = 0x007fffffu;                     // key of -inf

// 2^F exp((l - max) / T): 2^t with t = n + j / 64 + f, |f| <= 1/128, as 2^n, a table of 2^(j / 64) and the Taylor
// polynomial of 2^f to degree 4 (4e-14 of the value).
struct Weights {
  double scale;                                                   // log2(e) / T
  double max;
  float fmax;
  int bits;                                                       // F
  const double* table;
  __device__ __forceinline__ u64 unit() const { return 1ull << bits; }
  __device__ __forceinline__ u64 operator()(float l) const {
    if (l == fmax) return unit();
    const double t = ((double)l - max) * scale;
    if (!(t > -50.0)) return 0;                                   // (NaN too)
    constexpr double kMagic = 105553116266496.0;                  // 1.5 2^46: sums with it are multiples of 1/64
    const double rounded = t + kMagic;
    const int j = __double2loint(rounded);
    const double f = t - (rounded - kMagic);
    double q = fma(f, 0.009618129107628477, 0.05550410866482158);
    q = fma(q, f, 0.2402265069591007);
    q = fma(q, f, 0.6931471805599453);
    q = fma(q, f, 1.0);
    q *= table[j & (kTable - 1)];
    q = __hiloint2double(__double2hiint(q) + (((j >> 6) + bits) << 20), __double2loint(q));
    q += 4503599627370496.0;                                      // 2^52: the integer in the low bits
    return (u64)__double_as_longlong(q) & ((1ull << 52) - 1);
  }
};

// What is kept: keys above `key`, and those equal to it up to index `last`.
struct Cut {
  uint32_t key;
  int last;
  __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};

// How a pass sorts tokens into bins: by distance from the maximum (linear, monotonic in the logit), or by key.
struct Binning {
  bool by_key;
  float max4, scale4, fmax;                                       // (max - l) / 4, which does not overflow, times 4 bins
  uint32_t lo, hi;                                                // keys
  int shift;
  __device__ __forceinline__ int operator()(float l, uint32_t k) const {
    if (by_key) return k >= lo && k <= hi ? (int)((hi - k) >> shift) : kBins;
    if (l == fmax) return 0;
    const float at = fmaf(l, -0.25f, max4) * scale4;
    return at < (float)kBins ? (int)at : kBins;                   // (NaN is in none)
  }
};

struct Found {                                                    // by a histogram, or for all of a cluster otherwise
  int bin;                                                        // -1: all of it does not reach the target
  unsigned in_bin, upto;                                          // tokens
  u64 above, target;                                              // in front of the bin
};

struct Shared {
  union {
    struct {
      unsigned count[kBins], lo[kBins], hi[kBins];                // of this CTA; weights as two words
      unsigned all_count[kBins];                                  // of the cluster, in its first CTA
      u64 all_weight[kBins];
    };
    struct {
      u64 order[kList];                                           // list: in the first CTA
      u64 kept[kList];
      float value[kList];
      int index[kList];
    };
  };
  double table[kTable];
  u64 part[kWarps + 1];
  u64 total[kMostParts];                                          // one from each CTA of the cluster
  float best[kMostParts];
  int best_at[kMostParts];
  unsigned key_lo[kMostParts], key_hi[kMostParts];
  Found found;
  int walked;                                                     // an index that a warp of the cluster has found
};

template <typename P> __device__ __forceinline__ P* peer(P* p, int rank) {
  P* r;
  asm("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(p), "r"(rank));
  return r;
}

// A row's CTAs, and the calling warp's run of it in 16-byte packs.
template <typename T> struct Row {
  static constexpr int kPer = 16 / (int)sizeof(T);
  const T* row;                                                   // its first token
  int V, head;                                                    // tokens in front of it in its first pack
  int parts, rank;
  int begin, end;                                                 // packs
  __device__ __forceinline__ void sync() const {
    if (parts > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads();
  }
  // fn(values, first index, ...) of every pack, all lanes together; what does not exist is NaN
  template <typename F> __device__ __forceinline__ void each(F&& fn) const {
    const int lane = threadIdx.x & 31;
    for (int g0 = begin; g0 < end; g0 += 128) {
      uint4 raw[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = (g0 + 32 * u + lane) * kPer - head;
        if (i >= 0 && i + kPer <= V && g0 + 32 * u + lane < end) raw[u] = *reinterpret_cast<const uint4*>(row + i);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (g0 + 32 * u >= end) break;
        const bool mine = g0 + 32 * u + lane < end;
        const int i = (g0 + 32 * u + lane) * kPer - head;
        float v[kPer];
        if (mine && i >= 0 && i + kPer <= V) {
          unpack<T>(raw[u], v);
        } else {
#pragma unroll
          for (int j = 0; j < kPer; ++j) v[j] = mine && i + j >= 0 && i + j < V ? static_cast<float>(row[i + j]) : NAN;
        }
        if (fn(v, i)) return;
      }
    }
  }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_upto(u64 v) {                 // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 q = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += q;
  }
  return v;
}

// Sums over the CTA of one value a thread: what lies in front of the thread, and all of it.
__device__ __forceinline__ u64 block_before(u64 v, Shared& sh, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64 upto = warp_upto(v);
  __syncthreads();
  if (lane == 31) sh.part[warp] = upto;
  __syncthreads();
  u64 before = upto - v, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sh.part[w];
    all += sh.part[w];
  }
  *total = all;
  return before;
}
// Sums over the cluster of one value a warp (the same in all its lanes).
template <typename T>
__device__ __forceinline__ u64 cluster_before(u64 v, const Row<T>& row, Shared& sh, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) sh.part[warp] = v;
  __syncthreads();
  u64 before = 0, mine = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sh.part[w];
    mine += sh.part[w];
  }
  if ((int)threadIdx.x < row.parts) peer(&sh, threadIdx.x)->total[row.rank] = mine;
  row.sync();
  u64 all = 0;
  for (int r = 0; r < row.parts; ++r) {
    if (r < row.rank) before += sh.total[r];
    all += sh.total[r];
  }
  row.sync();                                                     // (before anyone's next total arrives)
  *total = all;
  return before;
}

// The first index at which the running sum of weight(l, i) exceeds `target(total)`, for all of the cluster.
template <typename T, typename F, typename G>
__device__ int walk(const Row<T>& row, Shared& sh, F&& weight, G&& target) {
  const int lane = threadIdx.x & 31;
  u64 mine = 0;
  row.each([&](const float (&v)[Row<T>::kPer], int i) {
#pragma unroll
    for (int j = 0; j < Row<T>::kPer; ++j) mine += weight(v[j], i + j);
    return false;
  });
  mine = warp_sum(mine);
  u64 total;
  u64 before = cluster_before(mine, row, sh, &total);
  const u64 limit = target(total);
  if (before <= limit && before + mine > limit) {                 // one warp of the cluster
    row.each([&](const float (&v)[Row<T>::kPer], int i) {
      u64 w[Row<T>::kPer], sum = 0;
#pragma unroll
      for (int j = 0; j < Row<T>::kPer; ++j) sum += w[j] = weight(v[j], i + j);
      const u64 upto = before + warp_upto(sum);
      const unsigned over = __ballot_sync(0xffffffffu, upto > limit);
      if (over == 0) {
        before = __shfl_sync(0xffffffffu, upto, 31);
        return false;
      }
      if (lane == __ffs(over) - 1) {
        u64 at = upto - sum;
        int found = i;
#pragma unroll
        for (int j = 0; j < Row<T>::kPer; ++j) {
          if (at <= limit) found = i + j;
          at += w[j];
        }
        for (int r = 0; r < row.parts; ++r) peer(&sh, r)->walked = found;
      }
      return true;
    });
  }
  row.sync();
  return sh.walked;
}

// The bin in which the prefix with `target` of the tokens (kCount) or of their weight ends.  Without kCount the target is
// a share of all that `eligible` keeps (share >= 0), or what is left of it.
template <bool kCount, typename T, typename E>
__device__ Found histogram(const Row<T>& row, Shared& sh, const Binning& bins, const Weights& weight, E&& eligible,
                           double share, u64 target) {
  const int tid = threadIdx.x;
  __syncthreads();
  for (int i = tid; i < kBins; i += kThreads) sh.count[i] = sh.lo[i] = sh.hi[i] = 0;
  __syncthreads();
  row.each([&](const float (&v)[Row<T>::kPer], int i) {
#pragma unroll
    for (int j = 0; j < Row<T>::kPer; ++j) {
      const uint32_t k = key_of(v[j]);
      const int bin = bins(v[j], k);
      if (bin >= kBins || !eligible(k, i + j)) continue;
      atomicAdd(&sh.count[bin], 1u);
      if (!kCount) {
        const u64 w = weight(v[j]);
        const unsigned lo = (unsigned)w;
        const unsigned carry = atomicAdd(&sh.lo[bin], lo) + lo < lo;
        const unsigned hi = (unsigned)(w >> 32) + carry;
        if (hi != 0) atomicAdd(&sh.hi[bin], hi);
      }
    }
    return false;
  });
  row.sync();
  {                                                               // every CTA adds up its share of the bins
    const int each = kBins / row.parts;
    for (int i = row.rank * each + tid; i < (row.rank + 1) * each; i += kThreads) {
      unsigned count = 0;
      u64 w = 0;
      for (int r = 0; r < row.parts; ++r) {
        const Shared* s = row.parts > 1 ? peer(&sh, r) : &sh;
        count += s->count[i];
        if (!kCount) w += ((u64)s->hi[i] << 32) + s->lo[i];
      }
      Shared* first = row.parts > 1 ? peer(&sh, 0) : &sh;
      first->all_count[i] = count;
      first->all_weight[i] = kCount ? count : w;
    }
  }
  row.sync();
  if (row.rank == 0) {
    u64 mine[4], sum = 0, counts = 0, total, all;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum += mine[j] = sh.all_weight[tid * 4 + j];
      counts += sh.all_count[tid * 4 + j];
    }
    u64 before = block_before(sum, sh, &total), upto = block_before(counts, sh, &all);
    if (share >= 0.0) target = max(1ull, (u64)ceil(share * (double)total));
    Found f{-1, 0, 0, 0, target};
    if (tid == 0 && total < target) {
      for (int r = 0; r < row.parts; ++r) peer(&sh, r)->found = f;
    }
    if (before < target && before + sum >= target) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned n = sh.all_count[tid * 4 + j];
        upto += n;
        if (before < target && before + mine[j] >= target) {
          f.bin = tid * 4 + j;
          f.in_bin = n;
          f.upto = (unsigned)upto;
          f.above = before;
          for (int r = 0; r < row.parts; ++r) peer(&sh, r)->found = f;
        }
        before += mine[j];
      }
    }
  }
  row.sync();
  const Found f = sh.found;
  row.sync();
  return f;
}

// Brings the tokens that `wanted` picks, 2048 at most, together in the first CTA, in the order of their indices.
template <typename T, typename F>
__device__ int gather(const Row<T>& row, Shared& sh, F&& wanted) {
  u64 mine = 0;
  row.each([&](const float (&v)[Row<T>::kPer], int i) {
#pragma unroll
    for (int j = 0; j < Row<T>::kPer; ++j) mine += wanted(v[j], i + j);
    return false;
  });
  mine = warp_sum(mine);
  u64 total;
  unsigned at = (unsigned)cluster_before(mine, row, sh, &total);
  Shared* first = row.parts > 1 ? peer(&sh, 0) : &sh;
  if (mine != 0) {
    row.each([&](const float (&v)[Row<T>::kPer], int i) {
      unsigned picked = 0;
#pragma unroll
      for (int j = 0; j < Row<T>::kPer; ++j) picked |= (unsigned)wanted(v[j], i + j) << j;
      if (__any_sync(0xffffffffu, picked != 0)) {
        const unsigned n = __popc(picked), upto = (unsigned)warp_upto(n);
        unsigned to = at + upto - n;
#pragma unroll
        for (int j = 0; j < Row<T>::kPer; ++j) {
          if (((picked >> j) & 1u) && to < kList) {
            first->value[to] = v[j];
            first->index[to] = i + j;
            ++to;
          }
        }
        at += __shfl_sync(0xffffffffu, upto, 31);
      }
      return false;
    });
  }
  row.sync();
  return (int)min(total, (u64)kList);
}

// order[] = places in the list by key descending, then by place; padded to a power of two, which it returns.
__device__ int sort_list(Shared& sh, int n) {
  int size = 32;
  while (size < n) size <<= 1;
  for (int i = threadIdx.x; i < size; i += kThreads)
    sh.order[i] = i < n ? (u64)~key_of(sh.value[i]) << 32 | (unsigned)i : ~0ull;
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < size / 2; i += kThreads) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const u64 x = sh.order[a], y = sh.order[b];
        if ((x > y) == ((a & k) == 0)) { sh.order[a] = y; sh.order[b] = x; }
      }
    }
  }
  __syncthreads();
  return size;
}

// The first place at which the running sum of four values a thread reaches `target` (sum >= target), for the whole CTA.
__device__ __forceinline__ int first_reaching(const u64 (&v)[4], u64 before, u64 target, Shared& sh) {
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (before < target && before + v[j] >= target) sh.walked = threadIdx.x * 4 + j;
    before += v[j];
  }
  __syncthreads();
  return sh.walked;
}

struct Settings {
  int top_k;                                                      // 0: all
  float top_p;
  u64 least;
  float uniform;
  // the sum that the running one has to exceed
  __device__ __forceinline__ u64 limit(u64 total) const {
    const u64 t = uniform > 0.0f ? (u64)((double)fminf(uniform, 1.0f) * (double)total) : 0ull;
    return min(t, total - 1);
  }
};

// The token, from a list that holds every token that can be kept.  wanted: what top-p has to reach, where top-k does not
// come before it.
__device__ int finish_list(Shared& sh, int n, const Weights& weight, const Settings& set, u64 wanted) {
  const int tid = threadIdx.x;
  sort_list(sh, n);
  u64 w[4], sum = 0, total, before;
  const int first = tid * 4, longest = set.top_k > 0 ? min(n, set.top_k) : n;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w[j] = first + j < longest ? weight(sh.value[(unsigned)sh.order[first + j]]) : 0ull;
    sum += w[j];
  }
  before = block_before(sum, sh, &total);
  int length = longest;
  if (set.top_p < 1.0f) {
    if (set.top_k > 0) wanted = max(1ull, (u64)ceil((double)set.top_p * (double)total));
    if (wanted <= total) length = min(length, first_reaching(w, before, wanted, sh) + 1);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (first + j < n) sh.kept[(unsigned)sh.order[first + j]] = first + j < length && w[j] >= set.least ? w[j] : 0ull;
  }
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) sum += w[j] = first + j < n ? sh.kept[first + j] : 0ull;
  before = block_before(sum, sh, &total);
  return sh.index[first_reaching(w, before, set.limit(total) + 1, sh)];
}

// The shortest prefix of what `was` keeps with `target` tokens, or with `share` of the weight.  True: it, and everything
// in front of it, is in a list of `*n` tokens, where `*wanted` is to be reached; else *cut is its end.
template <bool kCount, typename T>
__device__ bool prefix(const Row<T>& row, Shared& sh, const Weights& weight, Binning bins, const Cut& was, double share,
                       u64 target, Cut* cut, int* n, u64* wanted) {
  *cut = was;
  auto eligible = [&](uint32_t k, int i) { return was.keeps(k, i); };
  Found f = histogram<kCount>(row, sh, bins, weight, eligible, share, target);
  if (f.bin < 0) return false;                                    // all of it
  *wanted = f.target;
  auto upto = [&](float l, int i) {
    const uint32_t k = key_of(l);
    return bins(l, k) <= f.bin && f.bin < kBins && eligible(k, i);
  };
  auto within = [&](float l, int i) {
    const uint32_t k = key_of(l);
    return bins(l, k) == f.bin && eligible(k, i);
  };
  if (f.upto <= kList) {
    *n = gather(row, sh, upto);
    return true;
  }
  u64 left = f.target - f.above;                                  // to be reached within the bin
  while (f.in_bin > kList) {
    uint32_t lo = ~0u, hi = 0;
    row.each([&](const float (&v)[Row<T>::kPer], int i) {
#pragma unroll
      for (int j = 0; j < Row<T>::kPer; ++j) {
        if (within(v[j], i + j)) {
          const uint32_t k = key_of(v[j]);
          lo = min(lo, k);
          hi = max(hi, k);
        }
      }
      return false;
    });
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (threadIdx.x == 0) { sh.count[0] = ~0u; sh.count[1] = 0; }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) { atomicMin(&sh.count[0], lo); atomicMax(&sh.count[1], hi); }
    __syncthreads();
    if ((int)threadIdx.x < row.parts) {
      peer(&sh, threadIdx.x)->key_lo[row.rank] = sh.count[0];
      peer(&sh, threadIdx.x)->key_hi[row.rank] = sh.count[1];
    }
    row.sync();
    for (int r = 0; r < row.parts; ++r) { lo = min(lo, sh.key_lo[r]); hi = max(hi, sh.key_hi[r]); }
    row.sync();
    if (lo == hi) {                                               // ties: the first of them, by counting
      const u64 w = kCount ? 1ull : weight(value_of(lo));
      const u64 ties = (left + w - 1) / w;
      cut->key = lo;
      cut->last = ties >= f.in_bin ? row.V : walk(row, sh, [&](float l, int i) -> u64 {
        return key_of(l) == lo && eligible(lo, i);
      }, [&](u64) { return ties - 1; });
      return false;
    }
    bins.by_key = true;
    bins.lo = lo;
    bins.hi = hi;
    bins.shift = max(0, 32 - __clz(hi - lo) - 11);
    f = histogram<kCount>(row, sh, bins, weight, eligible, -1.0, left);
    left -= f.above;
  }
  *n = gather(row, sh, within);
  if (row.rank == 0) {
    sort_list(sh, *n);
    u64 w[4], sum = 0, total;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = threadIdx.x * 4 + j;
      sum += w[j] = at >= *n ? 0ull : kCount ? 1ull : weight(sh.value[(unsigned)sh.order[at]]);
    }
    const u64 before = block_before(sum, sh, &total);
    const int at = (unsigned)sh.order[first_reaching(w, before, left, sh)];
    const Found end{sh.index[at], key_of(sh.value[at]), 0, 0, 0};
    if ((int)threadIdx.x < row.parts) peer(&sh, threadIdx.x)->found = end;
  }
  row.sync();
  cut->key = sh.found.in_bin;
  cut->last = sh.found.bin;
  row.sync();
  return false;
}

template <typename V> __device__ __forceinline__ V setting(const V* p, V value, int64_t m) { return p != nullptr ? p[m] : value; }

template <typename T>
__global__ void __launch_bounds__(kThreads, MINB)
sample_kernel(const SampleArgs p, int parts) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t m = blockIdx.x / parts;
  Row<T> row;
  row.row = static_cast<const T*>(p.logits) + m * p.row_stride;
  row.V = (int)p.V;
  row.head = (int)((reinterpret_cast<uintptr_t>(row.row) & 15u) / sizeof(T));
  row.parts = parts;
  row.rank = (int)(blockIdx.x - m * parts);
  const int packs = (row.head + row.V + Row<T>::kPer - 1) / Row<T>::kPer;
  const int run = ((packs + parts * kWarps - 1) / (parts * kWarps) + 31) & ~31;
  row.begin = min(packs, (row.rank * kWarps + warp) * run);
  row.end = min(packs, row.begin + run);
  if (parts > 1) cluster_arrive();                                // "this CTA runs"
  if (tid < kTable) sh.table[tid] = exp2((double)tid / kTable);

  // the first maximum
  float best = -INFINITY;
  int at = row.V;
  row.each([&](const float (&v)[Row<T>::kPer], int i) {
#pragma unroll
    for (int j = 0; j < Row<T>::kPer; ++j) {
      if (v[j] > best) { best = v[j]; at = i + j; }
    }
    return false;
  });
  auto better = [&](float ob, int oa) {
    if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, at, o));
  if (lane == 0) {
    sh.kept[warp] = (u64)__float_as_uint(best) << 32 | (unsigned)at;
  }
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) better(__uint_as_float((unsigned)(sh.kept[w] >> 32)), (int)(unsigned)sh.kept[w]);
  if (parts > 1) cluster_wait();
  if (tid < parts) {
    peer(&sh, tid)->best[row.rank] = best;
    peer(&sh, tid)->best_at[row.rank] = at;
  }
  row.sync();
  for (int r = 0; r < parts; ++r) better(sh.best[r], sh.best_at[r]);

  const float temperature = setting(p.temperature, p.temperature_value, m);
  if (best == -INFINITY || !(temperature > 0.0f)) {
    if (row.rank == 0 && tid == 0) p.out[m] = best == -INFINITY ? 0 : at;
    return;                                                       // (nothing remote is under way)
  }
  best += 0.0f;
  const Weights weight{1.4426950408889634 / (double)temperature, (double)best, best, p.bits, sh.table};
  Settings set;
  set.top_k = setting(p.top_k, p.top_k_value, m);
  if (set.top_k < 0 || set.top_k >= row.V) set.top_k = 0;
  set.top_p = setting(p.top_p, p.top_p_value, m);
  const double min_p = (double)setting(p.min_p, p.min_p_value, m);
  set.least = min_p > 0.0 ? (u64)ceil(fmin(min_p, 1.0) * (double)weight.unit()) : 0ull;
  set.uniform = p.uniforms[m];
  const Binning bins{false, 0.25f * best, 4.0f * kBins / kRange / temperature, best, 0, 0, 0};

  Cut cut{kKeyNothing, row.V};                                    // all but -inf and NaN
  int n = 0;
  u64 wanted = 0;
  bool listed = false;
  if (set.top_k > 0) listed = prefix<true>(row, sh, weight, bins, cut, -1.0, (u64)set.top_k, &cut, &n, &wanted);
  if (!listed && set.top_p < 1.0f) {
    set.top_k = 0;                                                // (in the cut by now)
    listed = prefix<false>(row, sh, weight, bins, cut, fmax((double)set.top_p, 0.0), 0, &cut, &n, &wanted);
  }
  int token = 0;
  if (!listed) {
    token = walk(row, sh, [&](float l, int i) -> u64 {
      if (!cut.keeps(key_of(l), i)) return 0;
      const u64 w = weight(l);
      return w >= set.least ? w : 0;
    }, [&](u64 total) { return set.limit(total); });
  } else if (row.rank == 0) {
    token = finish_list(sh, n, weight, set, wanted);
  }
  if (row.rank == 0 && tid == 0) p.out[m] = token;
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& p, int dtype, cudaStream_t s) {
  if (p.M == 0) return cudaSuccess;
  static PerDeviceOnce once;
  int sms = 0;
  cudaError_t e = once.run([] {
    const cudaError_t a = cudaFuncSetAttribute(sample_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
    if (a != cudaSuccess) return a;
    return cudaFuncSetAttribute(sample_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
  }, &sms);
  if (e != cudaSuccess) return e;
  // CTAs of a row: as long as each has 4096 tokens and they do not fill the device twice
  int parts = kMostParts;
  while (parts > 1 && (p.V < parts * 4096 || p.M * parts > 4 * sms)) parts /= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.M * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = dtype == 1 ? cudaLaunchKernelEx(&cfg, sample_kernel<__nv_bfloat16>, p, parts)
                 : cudaLaunchKernelEx(&cfg, sample_kernel<float>, p, parts);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace rgk
