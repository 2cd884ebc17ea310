// One token per row of logits: temperature, top-k, top-p and min-p, drawn by a given uniform number.
//
// Weights are integers: W(l) = 2^F exp((l - max) / T), to within one, with F = 44 or as many bits as keep the sum of a row
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
// key is cut by counting.  For top-k up to 128 there is mostly no histogram: the k-th largest of the maxima of 128 parts of
// the row, or more, bounds what can be among the first k (unless more than 2048 tokens are as large as that).
//
// Bound: 2 or 4 bytes a token from HBM, and for whole rows and top-p without top-k the 64-bit exponential of every token
// within 31 temperatures of the maximum (11 double-precision operations, 2 cycles of a scheduler each).
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "rgk_common.cuh"
#include "rgk_internal.h"
#include "tc_common.cuh"

namespace rgk {
namespace {

using u64 = unsigned long long;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 2048;                                       // longest list that is sorted
constexpr int kEach = kBins / kThreads;                           // bins, or tokens of a list, to a thread
static_assert(kList == kBins, "one number a thread for both");
constexpr int kMostParts = 8;
constexpr float kRange = 32.0f;                                   // temperatures below the maximum: W = 0 from 31.2 on
constexpr int kTable = 64;
constexpr int kStretches = 16;
constexpr int kMostK = 128, kMostGroups = 320;                    // of top-k by groups of a row's lanes

// The order of the floats as an order of integers (-0 counts as 0, NaN below everything).
__device__ __forceinline__ uint32_t key_of(float l) {
  if (l != l) return 0u;
  const uint32_t b = __float_as_uint(l + 0.0f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key >> 31) ? key & 0x7fffffffu : ~key);
}

// 2^F exp((l - max) / T): 2^t with t = n + j / 64 + f, |f| <= 1/128, as 2^n, a table of 2^(j / 64) and the Taylor
// polynomial of 2^f to degree 4 (4e-14 of the value, 0.7 of the last bit of the largest weight).  Of tokens within 44 temperatures of the maximum: the callers
// drop what it says of others.  No branches: the tokens of a pack are evaluated side by side.
struct Weights {
  double scale;                                                   // log2(e) / T
  double max;
  int bits;                                                       // F
  const double* table;
  __device__ __forceinline__ u64 unit() const { return 1ull << bits; }
  __device__ __forceinline__ u64 operator()(float l) const {
    const double t = ((double)l - max) * scale;
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

// What is kept: logits above `end`, and those equal to it up to index `last`.  (NaN is not.)
struct Cut {
  float end;
  int last;
  __device__ __forceinline__ bool keeps(float l, int i) const { return l > end || (l == end && i <= last); }
};
// The same as a test for the passes over a row: without ties at the end it is one comparison.
template <bool kTies> struct Test {
  Cut cut;
  __device__ __forceinline__ bool operator()(float l, int i) const { return kTies ? cut.keeps(l, i) : l > cut.end; }
};

// How a pass sorts tokens into bins: by distance from the maximum (linear, monotonic in the logit; of tokens within
// kRange temperatures of it), or by key.
struct Binning {
  bool by_key;
  float max4, scale4;                                             // (max - l) / 4, which does not overflow, times 4 bins
  uint32_t lo, hi;                                                // keys
  int shift;
  __device__ __forceinline__ int operator()(float l) const {
    if (by_key) {
      const uint32_t k = key_of(l);
      return k >= lo && k <= hi ? (int)((hi - k) >> shift) : kBins;
    }
    // (rounded down by the sum with 2^23)
    return min((int)(__float_as_uint(__fadd_rd(fmaf(l, -0.25f, max4) * scale4, 8388608.0f)) & 0xffffu), kBins - 1);
  }
  // The smallest logit that `was` may keep whose bin is at most `bin`, by halving the keys below the maximum.
  __device__ float smallest(int bin, const Cut& was, float largest) const {
    uint32_t out = key_of(was.end) - (was.last >= 0), in = key_of(largest);  // (the maximum is in bin 0)
    while (in - out > 1) {
      const uint32_t mid = out + (in - out) / 2;
      if ((*this)(value_of(mid)) <= bin) in = mid; else out = mid;
    }
    return value_of(in);
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
      u64 order[kList], kept[kList];                              // the list: in the first CTA
    };
  };
  double table[kTable];
  u64 part[kWarps];
  u64 stretch[kWarps][kStretches];                                // sums of the pieces of a warp's run
  u64 total[kMostParts];                                          // one from each CTA of the cluster
  float best[kMostParts];
  int best_at[kMostParts];
  unsigned key_lo[kMostParts], key_hi[kMostParts];
  alignas(16) float groups[kMostGroups + 4];                      // maxima of parts of the row
  float least;                                                    // one of them
  Found found;
  unsigned length;                                                // of the list
  unsigned mine, place;                                           // of it in this CTA: how many, and from where on
  int walked;                                                     // an index that a warp of the cluster has found
};

template <typename P> __device__ __forceinline__ P* peer(P* p, int rank) {
  P* r;
  asm("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(p), "r"(rank));
  return r;
}

// A row's CTAs, and the calling warp's run of it in packs of four tokens.
constexpr int kPer = 4, kAhead = 4;                               // packs that a lane asks for at a time
template <typename T> struct Row {
  const T* row;                                                   // its first token
  int V, head;                                                    // tokens in front of it in its first pack
  int parts, rank;
  int begin, end;                                                 // packs
  __device__ __forceinline__ void sync() const {
    if (parts > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads();
  }
  using Raw = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
  __device__ __forceinline__ bool whole(int g) const { return g < end && g * kPer >= head && (g + 1) * kPer - head <= V; }
  static __device__ __forceinline__ void unpack4(const Raw& raw, float (&v)[kPer]) {
    if constexpr (sizeof(T) == 4) {
      unpack<T>(raw, v);
    } else {
      v[0] = bf16_lo(raw.x); v[1] = bf16_hi(raw.x); v[2] = bf16_lo(raw.y); v[3] = bf16_hi(raw.y);
    }
  }
  __device__ __forceinline__ void widen(const Raw& raw, int g, float (&v)[kPer]) const {
    if (whole(g)) {
      unpack4(raw, v);
    } else {
      const int i = g * kPer - head;
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] = g < end && i + j >= 0 && i + j < V ? static_cast<float>(row[i + j]) : NAN;
    }
  }
  // fn(values, first index) of every pack, all lanes together; what does not exist is NaN.  Packs are taken 32 kAhead
  // at a time, after which done(the first of them) is called.
  template <typename F, typename G> __device__ __forceinline__ void each(F&& fn, G&& done) const {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int g0 = begin; g0 < end; g0 += 32 * kAhead) {
      const int g = g0 + lane;
      const T* at = row + ((int64_t)g * kPer - head);
      Raw raw[kAhead];
      if (g0 * kPer >= head && g0 + 32 * kAhead <= end && (g0 + 32 * kAhead) * kPer - head <= V) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) raw[u] = *reinterpret_cast<const Raw*>(at + 32 * u * kPer);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          float v[kPer];
          unpack4(raw[u], v);
          fn(v, (g + 32 * u) * kPer - head);
        }
      } else {
#pragma unroll 1
        for (int u = 0; u < kAhead; ++u) {
          raw[0] = {};
          if (whole(g + 32 * u)) raw[0] = *reinterpret_cast<const Raw*>(at + 32 * u * kPer);
          float v[kPer];
          widen(raw[0], g + 32 * u, v);
          fn(v, (g + 32 * u) * kPer - head);
        }
      }
      done(g0);
    }
  }
  template <typename F> __device__ __forceinline__ void each(F&& fn) const { each(fn, [](int) {}); }
};

// How many packs a warp takes of a row.
__host__ __device__ __forceinline__ int run_of(int packs, int parts) {
  const int run = (packs + parts * kWarps - 1) / (parts * kWarps);
  return run > 64 ? (run + 32 * kAhead - 1) / (32 * kAhead) * (32 * kAhead) : run;       // (whole rounds of `each`)
}

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
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // every lane's sums, stretch after stretch of the run, so that the last stage reads one stretch again and no more
  u64 mine = 0, stretch = 0;
  const int per = (row.end - row.begin + 32 * kAhead * kStretches - 1) / (32 * kAhead * kStretches) * 32 * kAhead;
  row.each([&](const float (&v)[kPer], int i) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) stretch += weight(v[j], i + j);
  }, [&](int g0) {
    const int behind = g0 + 32 * kAhead - row.begin;
    if (behind % per == 0 || g0 + 32 * kAhead >= row.end) {
      stretch = warp_sum(stretch);
      if (lane == 0) sh.stretch[warp][(behind - 1) / per] = stretch;
      mine += stretch;
      stretch = 0;
    }
  });
  u64 total;
  u64 before = cluster_before(mine, row, sh, &total);
  const u64 limit = target(total);
  if (before <= limit && before + mine > limit) {                 // one warp of the cluster
    int at = 0;
    while (at + 1 < kStretches && before + sh.stretch[warp][at] <= limit) before += sh.stretch[warp][at++];
    for (int g0 = row.begin + at * per; g0 < row.end; g0 += 32) {
      const int g = g0 + lane, i = g * kPer - row.head;
      typename Row<T>::Raw raw = {};
      if (row.whole(g)) raw = *reinterpret_cast<const typename Row<T>::Raw*>(row.row + i);
      float v[kPer];
      row.widen(raw, g, v);
      u64 w[kPer], sum = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) sum += w[j] = weight(v[j], i + j);
      const u64 upto = before + warp_upto(sum);
      const unsigned over = __ballot_sync(0xffffffffu, upto > limit);
      if (over == 0) {
        before = __shfl_sync(0xffffffffu, upto, 31);
        continue;
      }
      if (lane == __ffs(over) - 1) {
        u64 sofar = upto - sum;
        int found = i;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (sofar <= limit) found = i + j;
          sofar += w[j];
        }
        for (int r = 0; r < row.parts; ++r) peer(&sh, r)->walked = found;
      }
      break;
    }
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
  row.each([&](const float (&v)[kPer], int i) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int bin = bins(v[j]);
      const u64 w = kCount ? 0ull : weight(v[j]);
      if (bin >= kBins || !eligible(v[j], i + j)) continue;
      atomicAdd(&sh.count[bin], 1u);
      if (!kCount) {
        const unsigned lo = (unsigned)w;
        const unsigned carry = atomicAdd(&sh.lo[bin], lo) + lo < lo;
        const unsigned hi = (unsigned)(w >> 32) + carry;
        if (hi != 0) atomicAdd(&sh.hi[bin], hi);
      }
    }
  });
  row.sync();
  {                                                               // every CTA adds up its share of the bins
    const int each = kBins / row.parts;
    for (int i = row.rank * each + tid; i < (row.rank + 1) * each; i += kThreads) {
      unsigned counts[kMostParts], los[kMostParts], his[kMostParts], count = 0;
      u64 w = 0;
#pragma unroll
      for (int r = 0; r < kMostParts; ++r) {                      // (asked for all at once)
        counts[r] = los[r] = his[r] = 0;
        if (r < row.parts) {
          const Shared* s = peer(&sh, r);
          counts[r] = s->count[i];
          if (!kCount) { los[r] = s->lo[i]; his[r] = s->hi[i]; }
        }
      }
#pragma unroll
      for (int r = 0; r < kMostParts; ++r) {
        count += counts[r];
        w += ((u64)his[r] << 32) + los[r];
      }
      Shared* first = row.parts > 1 ? peer(&sh, 0) : &sh;
      first->all_count[i] = count;
      first->all_weight[i] = kCount ? count : w;
    }
  }
  row.sync();
  if (row.rank == 0) {
    u64 mine[kEach], sum = 0, counts = 0, total, all;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      sum += mine[j] = sh.all_weight[tid * kEach + j];
      counts += sh.all_count[tid * kEach + j];
    }
    u64 before = block_before(sum, sh, &total), upto = block_before(counts, sh, &all);
    if (share >= 0.0) target = max(1ull, (u64)ceil(share * (double)total));
    Found f{-1, 0, 0, 0, target};
    if (tid == 0 && total < target) {
      for (int r = 0; r < row.parts; ++r) peer(&sh, r)->found = f;
    }
    if (before < target && before + sum >= target) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const unsigned n = sh.all_count[tid * kEach + j];
        upto += n;
        if (before < target && before + mine[j] >= target) {
          f.bin = tid * kEach + j;
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

// Brings the tokens that `wanted` picks, 2048 at most, together in the first CTA, in any order, as sort_list's words:
// in each CTA first (in `kept`), then with one place for all of a CTA's in the first one's `order`.  How many there are,
// which may be more than the list holds: then it is of no use.
template <typename T, typename F>
__device__ int gather(const Row<T>& row, Shared& sh, F&& wanted) {
  if (threadIdx.x == 0) sh.mine = sh.length = 0;
  row.sync();
  row.each([&](const float (&v)[kPer], int i) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < kPer; ++j) any |= wanted(v[j], i + j);
    if (any) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (!wanted(v[j], i + j)) continue;
        const unsigned to = atomicAdd(&sh.mine, 1u);
        if (to < kList) sh.kept[to] = (u64)~key_of(v[j]) << 32 | (unsigned)(i + j);
      }
    }
  });
  __syncthreads();
  const unsigned n = min(sh.mine, (unsigned)kList);
  Shared* first = row.parts > 1 ? peer(&sh, 0) : &sh;
  if (threadIdx.x == 0) sh.place = atomicAdd(&first->length, sh.mine);
  __syncthreads();
  for (unsigned i = threadIdx.x; i < n; i += kThreads) {
    if (sh.place + i < kList) first->order[sh.place + i] = sh.kept[i];
  }
  row.sync();
  const int all = (int)first->length;
  row.sync();
  return all;
}

// Sorts the first n words of `words`, which are all different, ascending: short lists by counting what is smaller, long
// ones by exchanges, those over less than 64 places within a warp's own.
__device__ void sort_list(u64* words, int n) {
  if (n <= 256) {
    const u64 mine = threadIdx.x < n ? words[threadIdx.x] : ~0ull;
    int place = 0;
    if (threadIdx.x < n) {
#pragma unroll 8
      for (int i = 0; i < n; ++i) place += words[i] < mine;
    }
    __syncthreads();
    if (threadIdx.x < n) words[place] = mine;
    __syncthreads();
    return;
  }
  int size = 512;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kThreads) words[i] = ~0ull;
  __syncthreads();
  bool wide = false;
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j >= 64 || wide) __syncthreads(); else __syncwarp();
      wide = j >= 64;
#pragma unroll 2
      for (int i = threadIdx.x; i < size / 2; i += kThreads) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const u64 x = words[a], y = words[b];
        if ((x > y) == ((a & k) == 0)) { words[a] = y; words[b] = x; }
      }
    }
  }
  __syncthreads();
}
// Of a list's word: the logit, descending in the order of the words, and the index.
__device__ __forceinline__ float logit_of(u64 word) { return value_of(~(uint32_t)(word >> 32)); }

// The first place at which the running sum of kEach values a thread reaches `target` (sum >= target), for the whole CTA.
__device__ __forceinline__ int first_reaching(const u64 (&v)[kEach], u64 before, u64 target, Shared& sh) {
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (before < target && before + v[j] >= target) sh.walked = threadIdx.x * kEach + j;
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
  const int tid = threadIdx.x, first = tid * kEach, longest = set.top_k > 0 ? min(n, set.top_k) : n;
  sort_list(sh.order, n);
  u64 w[kEach], sum = 0, total, before;
#pragma unroll
  for (int j = 0; j < kEach; ++j) sum += w[j] = first + j < longest ? weight(logit_of(sh.order[first + j])) : 0ull;
  before = block_before(sum, sh, &total);
  int length = longest;
  if (set.top_p < 1.0f) {
    if (set.top_k > 0) wanted = max(1ull, (u64)ceil((double)set.top_p * (double)total));
    if (wanted <= total) length = min(length, first_reaching(w, before, wanted, sh) + 1);
  }
  // those that are kept by index, each with its place in the list
  for (int i = tid; i < length; i += kThreads) sh.kept[i] = sh.order[i] << 32 | (unsigned)i;
  __syncthreads();
  sort_list(sh.kept, length);
  sum = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    w[j] = first + j < length ? weight(logit_of(sh.order[(unsigned)sh.kept[first + j]])) : 0ull;
    sum += w[j] = w[j] >= set.least ? w[j] : 0ull;
  }
  before = block_before(sum, sh, &total);
  return (int)(sh.kept[first_reaching(w, before, set.limit(total) + 1, sh)] >> 32);
}

// The shortest prefix of what `was` keeps with `target` tokens, or with `share` of the weight.  True: it, and everything
// in front of it, is in a list of `*n` tokens, where `*wanted` is to be reached; else *cut is its end.
template <bool kCount, bool kTies, typename T>
__device__ bool prefix(const Row<T>& row, Shared& sh, const Weights& weight, Binning bins, float largest, const Cut was,
                       double share, u64 target, Cut* cut, int* n, u64* wanted) {
  *cut = was;
  const Test<kTies> eligible{was};
  Found f = histogram<kCount>(row, sh, bins, weight, eligible, share, target);
  if (f.bin < 0) return false;                                    // all of it
  *wanted = f.target;
  // the bin as a range of logits: from `least` to below `above`
  float least = bins.smallest(f.bin, was, largest);
  if (f.upto <= kList) {
    *n = gather(row, sh, [&](float l, int i) { return l >= least && eligible(l, i); });
    return true;
  }
  float above = f.bin > 0 ? bins.smallest(f.bin - 1, was, largest) : INFINITY;
  auto within = [&](float l, int i) { return l >= least && l < above && eligible(l, i); };
  u64 left = f.target - f.above;                                  // to be reached within the bin
  while (f.in_bin > kList) {
    uint32_t lo = ~0u, hi = 0;
    row.each([&](const float (&v)[kPer], int i) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (within(v[j], i + j)) {
          const uint32_t k = key_of(v[j]);
          lo = min(lo, k);
          hi = max(hi, k);
        }
      }
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
      cut->end = value_of(lo);
      cut->last = ties >= f.in_bin ? row.V : walk(row, sh, [&](float l, int i) -> u64 {
        return l == cut->end && eligible(l, i);
      }, [&](u64) { return ties - 1; });
      return false;
    }
    bins.by_key = true;
    bins.lo = lo;
    bins.hi = hi;
    bins.shift = max(0, 32 - __clz(hi - lo) - 11);
    f = histogram<kCount>(row, sh, bins, weight, eligible, -1.0, left);
    left -= f.above;
    const uint32_t from = hi - ((uint32_t)f.bin << bins.shift);   // the bin's largest key
    least = value_of(max(lo, from - ((1u << bins.shift) - 1)));
    above = value_of(from + 1);
  }
  *n = gather(row, sh, within);
  if (row.rank == 0) {
    sort_list(sh.order, *n);
    u64 w[kEach], sum = 0, total;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int at = threadIdx.x * kEach + j;
      sum += w[j] = at >= *n ? 0ull : kCount ? 1ull : weight(logit_of(sh.order[at]));
    }
    const u64 before = block_before(sum, sh, &total);
    const u64 last = sh.order[first_reaching(w, before, left, sh)];
    const Found end{(int)(unsigned)last, ~(uint32_t)(last >> 32), 0, 0, 0};
    if ((int)threadIdx.x < row.parts) peer(&sh, threadIdx.x)->found = end;
  }
  row.sync();
  cut->end = value_of(sh.found.in_bin);
  cut->last = sh.found.bin;
  row.sync();
  return false;
}

template <typename V> __device__ __forceinline__ V setting(const V* p, V value, int64_t m) { return p != nullptr ? p[m] : value; }
__device__ __forceinline__ int top_k_of(const SampleArgs& p, int64_t m) { return setting(p.top_k, p.top_k_value, m); }

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
sample_kernel(const SampleArgs p, int parts) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t m = blockIdx.x / parts;
  Row<T> row;
  row.row = static_cast<const T*>(p.logits) + m * p.row_stride;
  row.V = (int)p.V;
  row.head = (int)(reinterpret_cast<uintptr_t>(row.row) / sizeof(T) % kPer);
  row.parts = parts;
  row.rank = (int)(blockIdx.x - m * parts);
  const int packs = (row.head + row.V + kPer - 1) / kPer;
  const int run = run_of(packs, parts);
  row.begin = min(packs, (row.rank * kWarps + warp) * run);
  row.end = min(packs, row.begin + run);
  if (parts > 1) cluster_arrive();                                // "this CTA runs"
  if (tid < kTable) sh.table[tid] = exp2((double)tid / kTable);

  // the first maximum
  float best = -INFINITY;
  int at = row.V;
  row.each([&](const float (&v)[kPer], int i) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (v[j] > best) { best = v[j]; at = i + j; }
    }
  });
  auto better = [&](float ob, int oa) {
    if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
  };
  // (In a row that begins inside of a pack a group may be without a token, or not be asked: a bound it is all the same.)
  const int k = top_k_of(p, m);
  const bool fine = k > p.coarse.most_k && k <= kMostK;
  const int group = fine ? p.fine.lanes : p.coarse.lanes;
  float of_group = best;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, at, o));
    if (2 * o == group) of_group = best;
  }
  if (lane == 0) {
    sh.part[warp] = (u64)__float_as_uint(best) << 32 | (unsigned)at;
  }
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) better(__uint_as_float((unsigned)(sh.part[w] >> 32)), (int)(unsigned)sh.part[w]);
  if (parts > 1) cluster_wait();
  if (tid < parts) {
    peer(&sh, tid)->best[row.rank] = best;
    peer(&sh, tid)->best_at[row.rank] = at;
  }
  {
    const int per_warp = fine ? p.fine.per_warp : p.coarse.per_warp, groups = fine ? p.fine.groups : p.coarse.groups;
    const int at_group = (row.rank * kWarps + warp) * per_warp + lane / group;
    if (lane % group == 0 && lane / group < per_warp && at_group < groups) {
      for (int r = 0; r < parts; ++r) peer(&sh, r)->groups[at_group] = of_group;
    }
    if (tid < 4) sh.groups[groups + tid] = -INFINITY;             // (read in fours)
  }
  row.sync();
  for (int r = 0; r < parts; ++r) better(sh.best[r], sh.best_at[r]);

  const float temperature = setting(p.temperature, p.temperature_value, m);
  if (best == -INFINITY || !(temperature > 0.0f)) {
    if (row.rank == 0 && tid == 0) p.out[m] = best == -INFINITY ? 0 : at;
    return;                                                       // (nothing remote is under way)
  }
  best += 0.0f;
  const Weights weight{1.4426950408889634 / (double)temperature, (double)best, p.bits, sh.table};
  Settings set;
  set.top_k = top_k_of(p, m);
  if (set.top_k < 0 || set.top_k >= row.V) set.top_k = 0;
  set.top_p = setting(p.top_p, p.top_p_value, m);
  if (set.top_p < 0.0f) set.top_p = 0.0f;
  const double min_p = (double)setting(p.min_p, p.min_p_value, m);
  set.least = min_p > 0.0 ? (u64)ceil(fmin(min_p, 1.0) * (double)weight.unit()) : 0ull;
  set.uniform = p.uniforms[m];
  const Binning bins{false, 0.25f * best, fminf(4.0f * kBins / kRange / temperature, FLT_MAX), 0, 0, 0};

  if (best == INFINITY) {                                         // they share evenly, nothing else weighs anything
    const int token = walk(row, sh, [&](float l, int) -> u64 { return l == INFINITY; }, [&](u64 total) {
      u64 kept = set.top_k > 0 ? min(total, (u64)set.top_k) : total;
      if (set.top_p < 1.0f) kept = min(kept, max(1ull, (u64)ceil((double)set.top_p * (double)kept)));
      return set.limit(kept);
    });
    if (row.rank == 0 && tid == 0) p.out[m] = token;
    return;
  }

  // all but NaN, -inf and what weighs nothing
  Cut cut{__fmaf_rd(-kRange, temperature, best), -1};
  int n = 0;
  u64 wanted = 0;
  bool listed = false;
  if (set.top_k > 0 && set.top_k <= kMostK) {
    // The k-th largest of the groups' maxima: k tokens are at least that, so the first k of all are among those that
    // are.  Mostly they are few (some 60 for k = 50, 200 for k = 100 or 128).  Fewer than k groups are there only in rows of
    // fewer than 512 tokens: all of those.
    const int groups = fine ? p.fine.groups : p.coarse.groups;
    if (tid < groups) {
      const float mine = sh.groups[tid];
      int place = 0;
#pragma unroll 4
      for (int i = 0; i < groups; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(sh.groups + i);
        place += (v.x > mine || (v.x == mine && i < tid)) + (v.y > mine || (v.y == mine && i + 1 < tid)) +
                 (v.z > mine || (v.z == mine && i + 2 < tid)) + (v.w > mine || (v.w == mine && i + 3 < tid));
      }
      if (place == min(set.top_k, groups) - 1) sh.least = set.top_k <= groups ? mine : -INFINITY;
    }
    __syncthreads();
    const float least = sh.least;
    n = gather(row, sh, [&](float l, int) { return l >= least && l > cut.end; });
    listed = n <= kList;
  }
  if (!listed && set.top_k > 0)
    listed = prefix<true, false>(row, sh, weight, bins, best, cut, -1.0, (u64)set.top_k, &cut, &n, &wanted);
  if (!listed && set.top_p < 1.0f) {
    set.top_k = 0;                                                // (in the cut by now)
    const double share = (double)set.top_p;
    listed = cut.last < 0 ? prefix<false, false>(row, sh, weight, bins, best, cut, share, 0, &cut, &n, &wanted)
                          : prefix<false, true>(row, sh, weight, bins, best, cut, share, 0, &cut, &n, &wanted);
  }
  int token = 0;
  if (!listed) {
    auto draw = [&](auto keeps) {
      return walk(row, sh, [&](float l, int i) -> u64 {
        const u64 w = weight(l);
        return keeps(l, i) && w >= set.least ? w : 0ull;
      }, [&](u64 total) { return set.limit(total); });
    };
    token = cut.last < 0 ? draw(Test<false>{cut}) : draw(Test<true>{cut});
  } else if (row.rank == 0) {
    token = finish_list(sh, n, weight, set, wanted);
  }
  if (row.rank == 0 && tid == 0) p.out[m] = token;
}

}  // namespace

// Groups of neighbouring lanes of a row, for top-k: a quarter more than k of them that have tokens, if there are as many
// such lanes.  A warp's run is rounded up, so that the last warps may be without: counted are the whole runs and what
// is left of a row, one run at most (of 128 groups by threads alone 65 have tokens of 33000, 99 of 151936).  One row of 151936
// tokens takes 14 us for k = 50 with coarse groups, and for k = 100 16 us with fine ones; where there are fewer groups than k, a
// histogram has to find the k-th: 31 us.
static void group_lanes(SampleArgs* p, int parts) {
  const int packs = (int)((p->V + kPer - 1) / kPer), run = run_of(packs, parts);
  auto groups_by = [&](int lanes) {
    const int per_warp = (std::min(run, 32) + lanes - 1) / lanes;
    const int groups = packs / run * per_warp + (std::min(packs % run, 32) + lanes - 1) / lanes;
    return SampleArgs::Groups{lanes, per_warp, groups, groups * 4 / 5};
  };
  int lanes = kThreads * parts / kMostK;                          // 4, 8, 16 or 32: 128 groups, where all have tokens
  p->coarse = groups_by(lanes);
  // (never more than kMostGroups: with twice the lanes there are fewer than 5/4 of kMostK)
  while (lanes > 1 && groups_by(lanes).most_k < kMostK) lanes /= 2;
  p->fine = groups_by(lanes);
}

cudaError_t launch_sample(SampleArgs p, int dtype, cudaStream_t s) {
  if (p.M == 0) return cudaSuccess;
  static PerDeviceOnce once;
  int sms = 0;
  cudaError_t e = once.run([] {
    const cudaError_t a = cudaFuncSetAttribute(sample_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
    if (a != cudaSuccess) return a;
    return cudaFuncSetAttribute(sample_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
  }, &sms);
  if (e != cudaSuccess) return e;
  // CTAs of a row: as many as are on the device at a time, each with 4096 tokens at least.  A CTA more costs a row its
  // barriers and its share of the merging; 256000 tokens with 1, 2, 4 and 8 of them: top-p on 256 rows 359 / 387 / 426 /
  // 567 us, on 64 rows 209 / 125 / 110 / 149, on 16 rows 208 / 125 / 79 / 74, on one row 199 / 117 / 72 / 52.
  int parts = kMostParts;
  while (parts > 1 && (p.V < parts * 4096 || p.M * parts > 2 * sms)) parts /= 2;
  group_lanes(&p, parts);
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
