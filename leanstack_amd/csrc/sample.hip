// A token from each row of logits, for gfx950: temperature, top-k, min-p, top-p, and
// the draw by a random number that the caller gives.
//
//   w_v = 2^-44 round(2^44 e^((x_v - max x) / T)),  order: larger x, then lower index;
//   kept: the first top_k; of those w_v >= min_p; of those the shortest prefix whose sum
//   reaches top_p times their sum (at least one);
//   the token is the first, by index, at which the kept weights' running sum exceeds u
//   times their sum.
// Weights are whole numbers of 2^-44 and every sum is one of 64-bit integers: no order
// of additions, no atomics' timing and no split moves a border between two tokens.
//
// Every filter keeps a prefix of the order, so the kept set is a smallest (x, index),
// as one 64-bit number ("place").  It is found without sorting: weights and counts
// by 2048 bins, even in x, down from the maximum to where weights vanish; then the
// places of the one bin in which the cut lies, ranked against each other, or, where
// they are many (ties, narrow logits), binned again by their bits first.
//
// One workgroup per row.  With top-k or min-p few tokens can be kept, and two sweeps over the
// row do: the first takes the maximum of each of 4096 groups of values, of which the k-th
// largest is a bound below which none of the first k lies; the second lists what is above
// it.  All else works on the list, in LDS.  Without either (top-p or the temperature alone)
// every weight counts, and a workgroup is bound by the arithmetic of the weights.  Few rows
// are cut into slices, a workgroup each, which leave lists or sums for the row's own.
//
// 128 rows of 151936 fp32 values with all filters: 24 + 9 us, 6.4 TB/s in the first launch, which
// reads them twice (kept in registers between the sweeps, 40 of them, they are read once by one
// workgroup to a CU instead of two: 20 us here and 23 for 21 with 37 rows); 1 row 6 + 8 us, the chain
// of sweep, groups, list, gathering, ranks and draw.  Without top-k and min-p 64 rows 32 us, with
// top-p 60..70: the arithmetic of two or three passes of weights (some 30 instructions for a
// value, half of them in 64 bits).

#include <hip/hip_runtime.h>

#include "lsk_internal.h"

namespace lsk {
namespace {

typedef unsigned long long u64;
typedef u64 u64x2_t __attribute__((ext_vector_type(2)));

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = kSampleBins;
static_assert(kBins == 2 * kThreads, "two to a thread");
constexpr int kRanked = 1024;               // places ranked against each other
constexpr int kRankedListed = 64;           // .. of a list, which is quickly binned again
constexpr int kListed = 4096;               // tokens that may be kept
constexpr int kFew = 256;                   // of them, compared each with each
constexpr int kGroups = 4;                  // of values per thread, whose maxima bound the k-th
constexpr int kMostK = kGroups * kThreads / 2;
constexpr int kAhead = 8;                   // 16-byte loads of a thread in flight
constexpr int kAheadDense = 2;              // ... where much is done with each value
constexpr int kParts = kSampleMaxVocab / 256 + 2;
constexpr double kUnit = 17592186044416.0;  // 2^44
constexpr float kOctaves = 46.f;            // below the maximum, in the bins
constexpr int kLastBin = kBins * 45 / 46 + 1;  // from 45 on weights round to zero
static_assert(kLastBin < kBins - 1, "what lies below all bins is in the last");

// Larger order: larger value; -0 equals +0.  (NaN is seen to apart.)
__device__ __forceinline__ unsigned value_order(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.f);
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float ordered_value(unsigned o) {
  return __builtin_bit_cast(float, o ^ ((unsigned)((int)~o >> 31) | 0x80000000u));
}

__device__ __forceinline__ u64 place_of(float x, int v) { return (u64)value_order(x) << 32 | (0xffffffffu - (unsigned)v); }
__device__ __forceinline__ int index_of(u64 place) { return (int)(0xffffffffu - (unsigned)place); }
__device__ __forceinline__ float value_of(u64 place) { return ordered_value((unsigned)(place >> 32)); }

// 2^(j / 64), j = 0..63, and then 2^t by the nearest of them below it, 2^n, and the series of
// e^(f ln(2) / 64), |f| <= 1/2: to 2^-50 of it.
constexpr int kPowers = 64;
__device__ __forceinline__ double root_power(int j) {
  // ln(2)^i / i!, for 2^(j / 64 - 1 / 2)
  constexpr double c[] = {1.0, 0.69314718055994531, 0.24022650695910072, 0.055504108664821580, 0.0096181291076284772,
                          0.0013333558146428443, 0.00015403530393381610, 1.5252733804059840e-05, 1.3215486790144309e-06,
                          1.0178086009239699e-07, 7.0549116208011233e-09, 4.4455382718708115e-10, 2.5678435993488206e-11};
  const double f = (double)j / kPowers - 0.5;
  double p = c[12];
#pragma unroll
  for (int i = 11; i >= 0; --i) p = __builtin_fma(p, f, c[i]);
  return p * 1.4142135623730951;
}
// Units of 2^(t64 / 64), t64 in -46 * 64..0, as a whole number: the sum with 2^52 rounds it.
__device__ __forceinline__ u64 units_of(double t64, const double* powers) {
  const double n = __builtin_rint(t64), f = t64 - n;
  const int i = (int)n;
  // (ln(2) / 64)^i / i!
  constexpr double l = 0.69314718055994531 / kPowers;
  constexpr double c[] = {1.0, l, l * l / 2, l * l * l / 6, l * l * l * l / 24, l * l * l * l * l / 120};
  double p = c[5];
#pragma unroll
  for (int e = 4; e >= 0; --e) p = __builtin_fma(p, f, c[e]);
  const double w = __builtin_ldexp(p * powers[i & (kPowers - 1)], 44 + (i >> 6));
  return __builtin_bit_cast(u64, w + 0x1p52) & ((1ull << 52) - 1);
}

// Inclusive sums over a wave's lanes: within rows of 16 (row_shr 1, 2, 4, 8), then rows 1 and 3
// the row in front of them (row_bcast 15), then the upper half the lower (row_bcast 31).
template <int kCtrl, int kRows>
__device__ __forceinline__ unsigned moved(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xf, false);
}
template <int kCtrl, int kRows>
__device__ __forceinline__ u64 moved(u64 v) {
  return (u64)moved<kCtrl, kRows>((unsigned)(v >> 32)) << 32 | moved<kCtrl, kRows>((unsigned)v);
}
template <typename V>
__device__ __forceinline__ V wave_inclusive(V v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}

struct Counts {
  unsigned count[kBins], wave_count[kWaves];
  int found;
};
struct Shared : Counts {
  double powers[kPowers];
  u64 weight[kBins], before[kBins];  // of the bins; and of those in front
  unsigned counted[kBins];
  union {
    struct {
      u64 weight[kBins];
      unsigned count[kBins];
    } sub;
    u64 parts[kParts];
  };
  u64 ranked[kRanked], ranked_weight[kRanked];
  u64 listed[kListed];
  u64 wave_weight[kWaves];
  float wave_max[kWaves];
  u64 lo, hi, kept, total, total_listed;
  unsigned n, listed_n;
};

// Accesses [first, end) of a row, and the values in front of the first and behind the last.
struct Range {
  int first, end;
  bool head, tail;
};

// A row in accesses of 16 bytes from its first aligned value on: access q holds the kVec
// values from head + q kVec on; those around them are taken one by one.
template <typename T>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(kVec)));
  const T* at;
  int V, head, vecs;
  __device__ __forceinline__ Row(const T* p, int n) : at(p), V(n) {
    head = min((int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T), n);
    vecs = (n - head) / kVec;
  }
  __device__ __forceinline__ float value(int v) const { return static_cast<float>(at[v]); }
  // access(v0, x): kVec values from index v0 on; one(v, x): a value apart.  All threads.
  template <int kAhead, typename Access, typename One>
  __device__ __forceinline__ void sweep(Access access, One one) const {
    sweep<kAhead>(Range{0, vecs, true, true}, access, one);
  }
  template <int kAhead, typename Access, typename One>
  __device__ __forceinline__ void sweep(const Range& r, Access access, One one) const {
    const int tid = threadIdx.x, first = r.first, end = r.end;
    if (r.head && tid < head) one(tid, value(tid));
    const vec_t* body = reinterpret_cast<const vec_t*>(at + head);
    for (int q0 = first + tid; q0 < end; q0 += kAhead * kThreads) {
      vec_t x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) x[k] = body[min(q0 + k * kThreads, end - 1)];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (q0 + k * kThreads >= end) break;
        float f[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) f[e] = static_cast<float>(x[k][e]);
        access(head + (q0 + k * kThreads) * kVec, f);
      }
    }
    const int tail = head + vecs * kVec + tid;
    if (r.tail && tail < V) one(tail, value(tail));
  }
  template <typename Each>
  __device__ __forceinline__ void each(const Range& r, Each f) const {
    sweep<kAheadDense>(r, [&](int v0, const float (&x)[kVec]) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) f(v0 + e, x[e]);
    }, f);
  }
  template <typename Each>
  __device__ __forceinline__ void each(Each f) const { each(Range{0, vecs, true, true}, f); }
  // Parts of the row in index order: the values in front of the first access, the accesses by
  // 64 (a wave's), the values behind the last.
  __device__ __forceinline__ int parts() const { return (vecs + 63) / 64 + 2; }
  __device__ __forceinline__ int part_of(int v) const {
    return v < head ? 0 : v >= head + vecs * kVec ? parts() - 1 : (v - head) / (64 * kVec) + 1;
  }
};

// The maxima of the thread's groups of values (NaN if one is), and the wave's.
template <typename T>
__device__ __forceinline__ float group_maxima(const Row<T>& row, const Range& r, float (&maxima)[kGroups]) {
  constexpr int kVec = Row<T>::kVec;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) maxima[g] = -__builtin_huge_valf();
  row.template sweep<kAhead>(r, [&](int, const float (&x)[kVec]) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) maxima[e % kGroups] = __builtin_elementwise_maximum(maxima[e % kGroups], x[e]);
  }, [&](int, float x) { maxima[0] = __builtin_elementwise_maximum(maxima[0], x); });
  float top = maxima[0];
#pragma unroll
  for (int g = 1; g < kGroups; ++g) top = __builtin_elementwise_maximum(top, maxima[g]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, d));
  return top;
}

// How a row's values weigh, and the bins that they fall into.
struct Rule {
  float top, per_bin;
  float part, part_top;  // distances from the maximum are taken of half the values where they could overflow
  double to_base2;  // and to 64ths
  double least;
  const double* powers;
  // Weight in units; 0 also for what min_p drops (a token without weight counts for nothing).
  __device__ __forceinline__ u64 weight(float x) const {
    if (x == top) return 1ull << 44;
    const double t = ((double)x - (double)top) * to_base2;
    if (!(t > -(double)kOctaves * kPowers)) return 0;
    const u64 w = units_of(t, powers);
    return (double)w >= least ? w : 0;
  }
  // Bins down from the maximum, monotone in x.
  __device__ __forceinline__ float in_bins(float x) const { return __builtin_fmaf(x, -part, part_top) * per_bin; }
  __device__ __forceinline__ int bin(float x) const {
    const float f = in_bins(x);
    return x == top ? 0 : f < (float)(kBins - 1) ? (int)f : kBins - 1;
  }
};

__device__ __forceinline__ Rule rule_of(float top, float temperature, float min_p, const double* powers) {
  const float part = top > 0x1p100f ? 0.5f : 1.f;
  return {top, (float)kBins * 1.44269504f / (kOctaves * part) / temperature, part, top * part,
          kPowers * 1.4426950408889634 / (double)temperature, min_p > 0.f ? (double)fminf(min_p, 1.f) * kUnit : 0.0, powers};
}

// Exclusive sums of count and weight over the bins; found: the first bin at which `reached`
// (count and weight up to and with it), kBins if there is none.
template <typename Reached>
__device__ void scan_bins(Shared& s, const unsigned* count, const u64* weight, unsigned* counted, u64* before,
                          Reached reached) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const unsigned c0 = count[2 * tid], c1 = count[2 * tid + 1];
  const u64 w0 = weight[2 * tid], w1 = weight[2 * tid + 1];
  const unsigned c = wave_inclusive(c0 + c1);
  const u64 w = wave_inclusive(w0 + w1);
  if (tid == 0) s.found = kBins;
  if (lane == 63) s.wave_count[wave] = c, s.wave_weight[wave] = w;
  __syncthreads();
  unsigned cb = c - c0 - c1;
  u64 wb = w - w0 - w1;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    cb += i < wave ? s.wave_count[i] : 0;
    wb += i < wave ? s.wave_weight[i] : 0;
  }
  if (counted) {
    counted[2 * tid] = cb, counted[2 * tid + 1] = cb + c0;
    before[2 * tid] = wb, before[2 * tid + 1] = wb + w0;
  }
  if (c0 && reached(cb + c0, wb + w0))
    atomicMin(&s.found, 2 * tid);
  else if (c1 && reached(cb + c0 + c1, wb + w0 + w1))
    atomicMin(&s.found, 2 * tid + 1);
  __syncthreads();
}

// The first bin at which the count reaches k (kBins: none).
__device__ __forceinline__ int bin_of_kth(Counts& s, unsigned k) {
  const int tid = threadIdx.x, wave = tid >> 6;
  const unsigned c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
  const unsigned up_to = wave_inclusive(c0 + c1);
  if ((tid & 63) == 63) s.wave_count[wave] = up_to;
  if (tid == 0) s.found = kBins;
  __syncthreads();
  unsigned c = up_to - c0 - c1;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) c += i < wave ? s.wave_count[i] : 0;
  if (c < k && c + c0 >= k)
    s.found = 2 * tid;
  else if (c + c0 < k && c + c0 + c1 >= k)
    s.found = 2 * tid + 1;
  __syncthreads();
  return s.found;
}

// The lowest kept place of the bin in which a cut lies: the first `want` by count, or those with
// less than `target` in front of them.  each(f): f(v, x) for all tokens, the bins filled and
// scanned.  More than `most` places are binned again.  Returns the place; s.kept: the weight up to it.
template <typename Each>
__device__ u64 cut_in_bin(Shared& s, const Rule& rule, Each each, int bin, bool by_count, unsigned want, double target, unsigned most) {
  const int tid = threadIdx.x;
  unsigned n = s.count[bin], base_c = s.counted[bin];
  u64 lo = 0, hi = ~0ull, base_w = s.before[bin];
  if (n > most) {
    if (tid == 0) s.lo = ~0ull, s.hi = 0;
    __syncthreads();
    u64 least = ~0ull, top = 0;
    each([&](int v, float x) {
      if (rule.bin(x) == bin && rule.weight(x)) {
        const u64 p = place_of(x, v);
        least = p < least ? p : least, top = p > top ? p : top;
      }
    });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const u64 l = __shfl_xor(least, d), h = __shfl_xor(top, d);
      least = l < least ? l : least, top = h > top ? h : top;
    }
    if ((tid & 63) == 0 && top) atomicMin(&s.lo, least), atomicMax(&s.hi, top);
    __syncthreads();
    lo = s.lo, hi = s.hi;
  }
  __syncthreads();
  while (n > most) {
    const int bits = 64 - __clzll((long long)(hi - lo));
    const int shift = bits > 11 ? bits - 11 : 0;
    for (int i = tid; i < kBins; i += kThreads) s.sub.count[i] = 0, s.sub.weight[i] = 0;
    __syncthreads();
    each([&](int v, float x) {
      if (rule.bin(x) != bin) return;
      const u64 p = place_of(x, v);
      if (p < lo || p > hi) return;
      const u64 w = rule.weight(x);
      if (!w) return;
      const int at = (int)((hi - p) >> shift);
      atomicAdd(&s.sub.count[at], 1u);
      atomicAdd(&s.sub.weight[at], w);
    });
    __syncthreads();
    scan_bins(s, s.sub.count, s.sub.weight, nullptr, nullptr, [&](unsigned c, u64 w) {
      return by_count ? base_c + c >= want : (double)(base_w + w) >= target;
    });
    // (rounding can leave the target out of reach: then the last)
    int at = s.found;
    if (at == kBins) at = (int)((hi - lo) >> shift);
    if (tid == 0) s.lo = 0, s.hi = 0;
    __syncthreads();
    u64 c = 0, w = 0;
    for (int i = tid; i < at; i += kThreads) c += s.sub.count[i], w += s.sub.weight[i];
    c = wave_inclusive(c), w = wave_inclusive(w);
    if ((tid & 63) == 63 && c) atomicAdd(&s.lo, c), atomicAdd(&s.hi, w);
    __syncthreads();
    base_c += (unsigned)s.lo, base_w += s.hi;
    n = s.sub.count[at];
    const u64 width = (1ull << shift) - 1;
    hi -= (u64)at << shift;
    lo = hi >= width && hi - width > lo ? hi - width : lo;
    __syncthreads();
  }
  if (tid == 0) s.n = 0, s.lo = ~0ull, s.kept = base_w;
  __syncthreads();
  each([&](int v, float x) {
    if (rule.bin(x) != bin) return;
    const u64 p = place_of(x, v);
    if (p < lo || p > hi) return;
    const u64 w = rule.weight(x);
    if (!w) return;
    const unsigned at = atomicAdd(&s.n, 1u);
    if (at < kRanked) s.ranked[at] = p, s.ranked_weight[at] = w;
  });
  __syncthreads();
  n = min(s.n, (unsigned)kRanked);
  if (tid < (int)n) {
    const u64 mine = s.ranked[tid];
    unsigned c = base_c;
    u64 w = base_w;
    for (unsigned i = 0; i < n; ++i)
      if (s.ranked[i] > mine) ++c, w += s.ranked_weight[i];
    if (by_count ? c < want : c == 0 || (double)w < target) {
      atomicMin(&s.lo, mine);
      atomicAdd(&s.kept, s.ranked_weight[tid]);
    }
  }
  __syncthreads();
  return s.lo;
}

// The lowest kept place under top-k (k below the number of tokens) and top-p (below 1).
// total: of all tokens' weights, where each() leaves some out (else 0).
template <typename Each>
__device__ u64 lowest_kept(Shared& s, const Rule& rule, Each each, bool by_k, unsigned k, bool by_p, float top_p, u64 total,
                           unsigned most) {
  const int tid = threadIdx.x;
  __syncthreads();
  for (int i = tid; i < kBins; i += kThreads) s.count[i] = 0, s.weight[i] = 0;
  __syncthreads();
  each([&](int, float x) {
    const u64 w = rule.weight(x);
    if (!w) return;
    const int at = rule.bin(x);
    atomicAdd(&s.count[at], 1u);
    atomicAdd(&s.weight[at], w);
  });
  __syncthreads();
  scan_bins(s, s.count, s.weight, s.counted, s.before, [&](unsigned c, u64) { return by_k && c >= k; });
  u64 sum = total ? total : s.before[kBins - 1] + s.weight[kBins - 1], lowest = 0;
  const int bin = s.found;
  if (by_k && bin < kBins) {  // (fewer than k have weight: no cut)
    lowest = cut_in_bin(s, rule, each, bin, true, k, 0.0, most);
    sum = s.kept;
  }
  if (by_p) {
    const double target = top_p > 0.f ? (double)top_p * (double)sum : 0.0;
    __syncthreads();
    scan_bins(s, s.count, s.weight, s.counted, s.before, [&](unsigned, u64 w) { return (double)w >= target; });
    const int at = s.found;
    if (at < kBins) {
      const u64 p = cut_in_bin(s, rule, each, at, false, 0, target, most);
      lowest = p > lowest ? p : lowest;
    }
  }
  __syncthreads();
  return lowest;
}

// Where in a sum of kept weights the random number falls.
__device__ __forceinline__ u64 drawn(float u, u64 total) {
  const u64 at = u > 0.f ? (u64)((double)fminf(u, 1.f) * (double)total) : 0;
  return at < total ? at : total - 1;
}

// Which of `count` (up to kParts) sums in s.parts the drawn token lies in, what is in front
// of it and all of them: the first at which the running sum exceeds u times the total.
struct Drawn {
  int part;
  u64 before, total, target;
};
__device__ Drawn draw_part(Shared& s, int count, float u) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int each = (count + kThreads - 1) / kThreads;
  const int i0 = min(tid * each, count), i1 = min(i0 + each, count);
  u64 mine = 0;
  for (int i = i0; i < i1; ++i) mine += s.parts[i];
  const u64 up_to = wave_inclusive(mine);
  if (lane == 63) s.wave_weight[wave] = up_to;
  __syncthreads();
  u64 before = up_to - mine, total = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    before += i < wave ? s.wave_weight[i] : 0;
    total += s.wave_weight[i];
  }
  const u64 target = drawn(u, total);
  if (before <= target && target < before + mine) {
    int i = i0;
    for (; i < i1 - 1; ++i) {
      if (target < before + s.parts[i]) break;
      before += s.parts[i];
    }
    s.found = i;
    s.lo = before;
  }
  __syncthreads();
  return {s.found, s.lo, total, target};
}

// Sums over four neighbouring lanes (quad_perm).
template <typename V>
__device__ __forceinline__ V quad_sum(V v) {
  v += moved<0xb1, 0xf>(v);
  v += moved<0x4e, 0xf>(v);
  return v;
}

// Up to kFew listed tokens, each compared with each by four lanes: its rank and what is in
// front of it, then what is kept in front of its index.
template <typename Write>
__device__ __forceinline__ void few_tokens(Shared& s, const Rule& rule, int n, unsigned k, bool by_p, float top_p, u64 all,
                                           float u, Write write) {
  static_assert(4 * kFew == kThreads, "four lanes to a token");
  constexpr int kStep = 8;  // tokens of a lane at a time
  const int tid = threadIdx.x, me = tid >> 2, q = tid & 3;
  const bool here = me < n;
  const u64 mine = here ? s.listed[me] : 0, w = here ? rule.weight(value_of(mine)) : 0;
  const int rounded = (n + 4 * kStep - 1) / (4 * kStep) * (4 * kStep);
  __syncthreads();
  if (me < rounded && q == 0) {  // (places of zero are behind all others)
    s.listed[me] = mine;
    s.ranked_weight[me] = w;
  }
  __syncthreads();
  unsigned rank = 0;
  u64 before = 0;
  if (here) {
    for (int i0 = q; i0 < n; i0 += 4 * kStep) {
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        const bool larger = s.listed[i0 + 4 * i] > mine;
        rank += larger ? 1u : 0u;
        before += larger ? s.ranked_weight[i0 + 4 * i] : 0;
      }
    }
  }
  rank = quad_sum(rank);
  before = quad_sum(before);
  if (here && rank == min(k, (unsigned)n) - 1) s.kept = before + w;  // the sum of the first k
  __syncthreads();
  const double target = top_p > 0.f ? (double)top_p * (double)(all ? all : s.kept) : 0.0;
  const bool kept = here && rank < k && (!by_p || rank == 0 || (double)before < target);
  if (me < rounded && q == 0) s.ranked[me] = kept ? w : 0;
  __syncthreads();
  u64 in_front = 0, total = 0;
  if (here) {
    for (int i0 = q; i0 < n; i0 += 4 * kStep) {
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        const u64 other = s.ranked[i0 + 4 * i];
        total += other;
        in_front += (unsigned)s.listed[i0 + 4 * i] > (unsigned)mine ? other : 0;  // (a lower index)
      }
    }
  }
  total = quad_sum(total);
  in_front = quad_sum(in_front);
  if (!kept || q != 0) return;
  const u64 at = drawn(u, total);
  if (in_front <= at && at < in_front + w) write(index_of(mine), w, total);
}

// Tokens that top-k and min-p may keep are in the first `last` bins or none: where the lowest lies whose
// weight rounds up to min-p's least whole units (half a unit less; two bins for what the logarithm is
// off), and where weights vanish.
__device__ __forceinline__ int last_bin(float min_p) {
  if (!(min_p > 0.f)) return kLastBin;
  const float least = fmaxf(__builtin_ceilf(fminf(min_p, 1.f) * (float)kUnit), 1.f);
  return (int)fminf((float)kLastBin, 2.f + (44.f - __log2f(least - 0.5f)) * ((float)kBins / kOctaves));
}

// The bin of the k-th largest of the threads' maxima: at least k values are in it or above.
__device__ __forceinline__ int bin_of_maxima(Counts& s, const Rule& rule, const float (&maxima)[kGroups], unsigned k) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = 0;
  __syncthreads();
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int at = rule.bin(maxima[g]);
    if (at <= kLastBin) atomicAdd(&s.count[at], 1u);
  }
  __syncthreads();
  return bin_of_kth(s, k);
}

// ------------------------------------------------------------------ few rows, in slices

// What a row's slices leave for each other and for the row's own workgroup: their maxima; the bin
// in which top-p cuts (kBins: no cut) and the weight in front of it; and of each slice the first index of
// the maximum (for rows without a temperature) and how many tokens it has listed (more than
// the list holds: too many).
struct RowSums {
  u64 before, total;
  int bin;
  float max[kSampleMaxSlices];
  int first[kSampleMaxSlices];
  unsigned n[kSampleMaxSlices];
};
static_assert(sizeof(RowSums) <= kSampleRowBytes, "as the host counts it");
struct Space {
  RowSums* row;
  u64* listed;  // [slices][kSampleRankListed] places that top-k or min-p may keep; or
  u64* parts;   // [parts] weights in front of top-p's cut, by the row's parts,
  u64* cut;     // [slices][kSampleSliceListed] places of the bin of the cut
  u64* bins;    // [slices][kBins] weights
};
__device__ __forceinline__ Space space_of(const SampleArgs& a, int m) {
  unsigned char* at = a.workspace + (size_t)m * a.row_bytes;
  Space s;
  s.row = reinterpret_cast<RowSums*>(at);
  s.listed = s.parts = reinterpret_cast<u64*>(at + kSampleRowBytes);
  s.cut = s.parts + a.max_parts;
  s.bins = s.cut + (size_t)a.slices * kSampleSliceListed;
  return s;
}
// Slice i of a row: whole parts.
template <typename T>
__device__ __forceinline__ Range slice_of(const SampleArgs& a, const Row<T>& row, int i) {
  const int each = ((row.vecs + 63) / 64 + a.slices - 1) / a.slices * 64;
  const int first = min(i * each, row.vecs);
  return {first, min(first + each, row.vecs), i == 0, i == a.slices - 1};
}
// The row's maximum (NaN if there is one), in all threads.
__device__ __forceinline__ float row_top(const SampleArgs& a, const RowSums& r) {
  float top = r.max[min((int)(threadIdx.x & (kSampleMaxSlices - 1)), a.slices - 1)];
#pragma unroll
  for (int d = 1; d < kSampleMaxSlices; d <<= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, d));
  return top;
}

// Grid of these: slice (fastest), row.

// Of rows with top-k or min-p: a slice's tokens that they may keep, by the slice's own maxima.
template <typename T>
__global__ __launch_bounds__(kThreads) void slice_list_kernel(SampleArgs a) {
  constexpr int kVec = Row<T>::kVec;
  __shared__ Counts s;
  __shared__ float wave_max[kWaves];
  __shared__ unsigned listed;
  __shared__ int found;
  const int m = blockIdx.x / a.slices, i = blockIdx.x % a.slices, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Space at = space_of(a, m);
  const Row<T> row(static_cast<const T*>(a.logits) + (size_t)m * a.logits_ld, a.V);
  const Range sl = slice_of(a, row, i);
  float maxima[kGroups];
  float top = group_maxima(row, sl, maxima);
  if (lane == 0) wave_max[wave] = top;
  if (tid == 0) listed = 0, found = a.V;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = __builtin_elementwise_maximum(top, wave_max[w]);
  if (tid == 0) at.row->max[i] = top;
  const float temperature = a.temperature ? a.temperature[m] : 1.f;
  if (!(temperature > 0.f)) {
    int first = a.V;
    row.each(sl, [&](int v, float x) { first = x == top ? min(first, v) : first; });
    if (first < a.V) atomicMin(&found, first);
    __syncthreads();
    if (tid == 0) at.row->first[i] = found;
    return;
  }
  const int k = a.top_k && a.top_k[m] > 0 ? a.top_k[m] : a.V;
  const float min_p = a.min_p ? a.min_p[m] : 0.f;
  const bool by_k = k < a.V && k <= kMostK;
  if ((by_k || min_p > 0.f) && top > -__builtin_huge_valf()) {
    const Rule rule = rule_of(top, temperature, min_p, nullptr);
    int last = last_bin(min_p);
    if (by_k) last = min(bin_of_maxima(s, rule, maxima, (unsigned)k), last);
    const float end = (float)(last + 1);
    auto list = [&](int v, float x) {
      if (!(rule.in_bins(x) < end || x == top)) return;
      const unsigned to = atomicAdd(&listed, 1u);
      if (to < kSampleRankListed) at.listed[(size_t)i * kSampleRankListed + to] = place_of(x, v);
    };
    row.template sweep<kAheadDense>(sl, [&](int v0, const float (&x)[kVec]) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) list(v0 + e, x[e]);
    }, list);
  }
  __syncthreads();
  if (tid == 0) at.row->n[i] = listed;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void slice_top_kernel(SampleArgs a) {
  __shared__ float wave_max[kWaves];
  const int m = blockIdx.x / a.slices, i = blockIdx.x % a.slices;
  const Row<T> row(static_cast<const T*>(a.logits) + (size_t)m * a.logits_ld, a.V);
  const Range sl = slice_of(a, row, i);
  float top = -__builtin_huge_valf();
  row.template sweep<kAheadDense>(sl, [&](int, const float (&x)[Row<T>::kVec]) {
#pragma unroll
    for (int e = 0; e < Row<T>::kVec; ++e) top = __builtin_elementwise_maximum(top, x[e]);
  }, [&](int, float x) { top = __builtin_elementwise_maximum(top, x); });
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) top = __builtin_elementwise_maximum(top, wave_max[w]);
    space_of(a, m).row->max[i] = top;
  }
}

// Weights by bins, of rows that top-p cuts.
template <typename T>
__global__ __launch_bounds__(kThreads) void slice_bins_kernel(SampleArgs a) {
  __shared__ u64 weight[kBins];
  __shared__ double powers[kPowers];
  const int m = blockIdx.x / a.slices, i = blockIdx.x % a.slices, tid = threadIdx.x;
  const Space at = space_of(a, m);
  const float temperature = a.temperature ? a.temperature[m] : 1.f, top = row_top(a, *at.row);
  if (!(top > -__builtin_huge_valf()) || !(temperature > 0.f) || !(a.top_p[m] < 1.f)) return;
  if (tid < kPowers) powers[tid] = root_power(tid);
  weight[2 * tid] = weight[2 * tid + 1] = 0;
  __syncthreads();
  const Rule rule = rule_of(top, temperature, 0.f, powers);
  const Row<T> row(static_cast<const T*>(a.logits) + (size_t)m * a.logits_ld, a.V);
  const Range sl = slice_of(a, row, i);
  row.each(sl, [&](int, float x) {
    const u64 w = rule.weight(x);
    if (w) atomicAdd(&weight[rule.bin(x)], w);
  });
  __syncthreads();
  u64* out = at.bins + (size_t)i * kBins;
  out[2 * tid] = weight[2 * tid], out[2 * tid + 1] = weight[2 * tid + 1];
}

// Weights by parts: all, or those in front of the bin in which top-p cuts, whose tokens are listed.
template <typename T>
__global__ __launch_bounds__(kThreads) void slice_parts_kernel(SampleArgs a) {
  constexpr int kVec = Row<T>::kVec;
  __shared__ double powers[kPowers];
  __shared__ u64 wave_weight[kWaves], before_bin;
  __shared__ int found;
  __shared__ unsigned listed;
  const int m = blockIdx.x / a.slices, i = blockIdx.x % a.slices, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Space at = space_of(a, m);
  const float temperature = a.temperature ? a.temperature[m] : 1.f, top = row_top(a, *at.row);
  if (!(top > -__builtin_huge_valf())) return;
  const Row<T> row(static_cast<const T*>(a.logits) + (size_t)m * a.logits_ld, a.V);
  const Range sl = slice_of(a, row, i);
  if (tid < kPowers) powers[tid] = root_power(tid);
  if (tid == 0) found = a.V > kBins ? a.V : kBins, listed = 0;
  __syncthreads();
  if (!(temperature > 0.f)) {
    int first = a.V;
    row.each(sl, [&](int v, float x) { first = x == top ? min(first, v) : first; });
    if (first < a.V) atomicMin(&found, first);
    __syncthreads();
    if (tid == 0) at.row->first[i] = found;
    return;
  }
  const Rule rule = rule_of(top, temperature, 0.f, powers);
  const float top_p = a.top_p ? a.top_p[m] : 1.f;
  int bin = kBins;
  if (top_p < 1.f) {
    u64 w0 = 0, w1 = 0;
    const auto* bins = reinterpret_cast<const u64x2_t*>(at.bins) + tid;
    constexpr int kHeld = 8;  // (16 of them cost the second workgroup of a CU)
    for (int s0 = 0; s0 < a.slices; s0 += kHeld) {
      u64x2_t held[kHeld];
#pragma unroll
      for (int s = 0; s < kHeld; ++s) held[s] = bins[min(s0 + s, a.slices - 1) * (kBins / 2)];
#pragma unroll
      for (int s = 0; s < kHeld; ++s)
        if (s0 + s < a.slices) w0 += held[s][0], w1 += held[s][1];
    }
    const u64 up_to = wave_inclusive(w0 + w1);
    if (lane == 63) wave_weight[wave] = up_to;
    __syncthreads();
    u64 before = up_to - w0 - w1, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      before += w < wave ? wave_weight[w] : 0;
      total += wave_weight[w];
    }
    const double target = top_p > 0.f ? (double)top_p * (double)total : 0.0;
    const bool first = w0 && (double)(before + w0) >= target, second = w1 && (double)(before + w0 + w1) >= target;
    if (first || second) atomicMin(&found, first ? 2 * tid : 2 * tid + 1);
    __syncthreads();
    bin = found;  // (the sum of all is no less than the target)
    if (bin >> 1 == tid) before_bin = before + (bin & 1 ? w0 : 0);
    __syncthreads();
    if (i == 0 && tid == 0) at.row->before = before_bin, at.row->total = total;
  }
  if (i == 0 && tid == 0) at.row->bin = bin;
  auto kept = [&](int v, float x) -> u64 {
    const u64 w = rule.weight(x);
    if (bin == kBins || !w) return w;
    const int here = rule.bin(x);
    if (here == bin) {
      const unsigned to = atomicAdd(&listed, 1u);
      if (to < kSampleSliceListed) at.cut[(size_t)i * kSampleSliceListed + to] = place_of(x, v);
    }
    return here < bin ? w : 0;
  };
  const auto* body = reinterpret_cast<const typename Row<T>::vec_t*>(row.at + row.head);
  const int tail = row.head + row.vecs * kVec;
  if (i == 0 && wave == 0) {
    const u64 w = wave_inclusive(lane < row.head ? kept(lane, row.value(lane)) : 0);
    if (lane == 63) at.parts[0] = w;
  }
  if (i == a.slices - 1 && wave == 0) {
    const u64 w = wave_inclusive(tail + lane < a.V ? kept(tail + lane, row.value(tail + lane)) : 0);
    if (lane == 63) at.parts[row.parts() - 1] = w;
  }
  for (int q0 = sl.first + 64 * wave; q0 < sl.end; q0 += kThreads) {
    u64 w = 0;
    if (q0 + lane < sl.end) {
      const auto x = body[q0 + lane];
#pragma unroll
      for (int e = 0; e < kVec; ++e) w += kept(row.head + (q0 + lane) * kVec + e, static_cast<float>(x[e]));
    }
    w = wave_inclusive(w);
    if (lane == 63) at.parts[q0 / 64 + 1] = w;
  }
  __syncthreads();
  if (tid == 0) at.row->n[i] = listed;
}

// The drawn token of a row whose kept weights are in s.parts.
template <typename T, typename Write>
__device__ __forceinline__ void draw_of_parts(Shared& s, const Rule& rule, const Row<T>& row, u64 lowest, float u, Write write) {
  constexpr int kVec = Row<T>::kVec;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int parts = row.parts(), tail = row.head + row.vecs * kVec;
  const Drawn d = draw_part(s, parts, u);
  if (wave != 0) return;
  const int begin = d.part == 0 ? 0 : d.part == parts - 1 ? tail : row.head + (d.part - 1) * 64 * kVec;
  const int end = d.part == 0 ? row.head : d.part == parts - 1 ? row.V : min(begin + 64 * kVec, tail);
  u64 sum = d.before;
  for (int v0 = begin; v0 < end; v0 += 64) {
    const int v = v0 + lane;
    const float x = row.value(min(v, end - 1));
    const u64 w = v < end && place_of(x, v) >= lowest ? rule.weight(x) : 0;
    const u64 c = sum + wave_inclusive(w);
    const u64 there = __ballot(c > d.target);
    if (there) {
      if (lane == __builtin_ctzll(there)) write(v, w, d.total);
      return;
    }
    sum = __shfl(c, 63);
  }
}

// The end of a row whose slices have been summed; false: too many tokens in the bin of the cut.
template <typename T, typename Write>
__device__ bool draw_of_slices(Shared& s, const SampleArgs& a, const Rule& rule, const Row<T>& row, const Space& at, float top_p,
                               float u, Write write) {
  const int tid = threadIdx.x, bin = at.row->bin;
  u64 lowest = 0;
  unsigned n = 0;
  if (bin < kBins) {
    // A wave per slice: the lists one behind the other.
    static_assert(kWaves == kSampleMaxSlices, "a wave per slice");
    const int lane = tid & 63, slice = tid >> 6;
    const unsigned here = lane < a.slices ? at.row->n[lane] : 0, up_to = wave_inclusive(here);
    n = (unsigned)__builtin_amdgcn_readlane((int)up_to, 63);
    if (__ballot(here > kSampleSliceListed) || n > kListed) return false;
    const unsigned mine = (unsigned)__builtin_amdgcn_readlane((int)here, slice);
    const unsigned from = (unsigned)__builtin_amdgcn_readlane((int)up_to, slice) - mine;
    for (unsigned i = lane; i < mine; i += 64) s.listed[from + i] = at.cut[(size_t)slice * kSampleSliceListed + i];
    if (tid == 0) s.count[bin] = n, s.counted[bin] = 0, s.before[bin] = at.row->before;
    __syncthreads();
    const double target = top_p > 0.f ? (double)top_p * (double)at.row->total : 0.0;
    lowest = cut_in_bin(s, rule, [&](auto f) {
      for (int i = tid; i < (int)n; i += kThreads) f(index_of(s.listed[i]), value_of(s.listed[i]));
    }, bin, false, 0, target, kRankedListed);
    __syncthreads();
  }
  for (int i = tid; i < row.parts(); i += kThreads) s.parts[i] = at.parts[i];
  __syncthreads();
  for (int i = tid; i < (int)n; i += kThreads)
    if (s.listed[i] >= lowest) atomicAdd(&s.parts[row.part_of(index_of(s.listed[i]))], rule.weight(value_of(s.listed[i])));
  __syncthreads();
  draw_of_parts(s, rule, row, lowest, u, write);
  return true;
}

// The first index of the row's maximum, from its slices'.
__device__ __forceinline__ int first_of_slices(const SampleArgs& a, const RowSums& r, float top) {
  const int i = min((int)(threadIdx.x & (kSampleMaxSlices - 1)), a.slices - 1);
  int first = r.max[i] == top ? r.first[i] : a.V;
#pragma unroll
  for (int d = 1; d < kSampleMaxSlices; d <<= 1) first = min(first, __shfl_xor(first, d));
  return first;
}

// The slices' lists brought together in s.listed, without what cannot be kept by the whole row's
// counts; false: too many tokens.
__device__ __forceinline__ bool gather_lists(Shared& s, const SampleArgs& a, const Rule& rule, const Space& at, bool by_k,
                                             unsigned k, float min_p) {
  const int tid = threadIdx.x, lane = tid & 63, slice = tid >> 6;
  const unsigned here = lane < a.slices ? at.row->n[lane] : 0;
  if (__ballot(here > kSampleRankListed)) return false;
  const unsigned n = slice < a.slices ? (unsigned)__shfl((int)here, slice) : 0;
  const u64* from = at.listed + (size_t)slice * kSampleRankListed;
  int last = last_bin(min_p);
  if (by_k) {
    for (int i = tid; i < kBins; i += kThreads) s.count[i] = 0;
    __syncthreads();
    for (unsigned i = lane; i < n; i += 64) {
      const int bin = rule.bin(value_of(from[i]));
      if (bin <= kLastBin) atomicAdd(&s.count[bin], 1u);
    }
    __syncthreads();
    last = min(bin_of_kth(s, k), last);
  }
  const float end = (float)(last + 1);
  for (unsigned i = lane; i < n; i += 64) {
    const u64 place = from[i];
    const float x = value_of(place);
    if (!(rule.in_bins(x) < end || x == rule.top)) continue;
    const unsigned to = atomicAdd(&s.listed_n, 1u);
    if (to < kListed) s.listed[to] = place;
  }
  __syncthreads();
  return s.listed_n <= kListed;
}

// Whole rows by themselves, or with what their slices' kernels have left.
enum Sliced { kWhole, kSummed, kRankedLists };
template <typename T, Sliced SLICED>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  Shared& s = *reinterpret_cast<Shared*>(shared_bytes);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m = blockIdx.x, V = a.V;
  const Row<T> row(static_cast<const T*>(a.logits) + (size_t)m * a.logits_ld, V);
  constexpr int kVec = Row<T>::kVec;
  auto write = [&](int v, u64 w, u64 total) {
    a.tokens[m] = v;
    a.logprobs[m] = (float)log((double)w / (double)total);
  };
  if constexpr (SLICED == kSummed) {
    const Space at = space_of(a, m);
    const float top = row_top(a, *at.row), temperature = a.temperature ? a.temperature[m] : 1.f;
    if (!(top > -__builtin_huge_valf())) {
      if (tid == 0) a.tokens[m] = -1, a.logprobs[m] = __builtin_nanf("");
      return;
    }
    if (!(temperature > 0.f)) {
      const int first = first_of_slices(a, *at.row, top);
      if (tid == 0) a.tokens[m] = first, a.logprobs[m] = 0.f;
      return;
    }
    if (tid < kPowers) s.powers[tid] = root_power(tid);
    __syncthreads();
    const Rule rule = rule_of(top, temperature, 0.f, s.powers);
    if (draw_of_slices(s, a, rule, row, at, a.top_p ? a.top_p[m] : 1.f, a.uniforms[m], write)) return;
    __syncthreads();
  }

  float maxima[kGroups], top;
  if constexpr (SLICED == kRankedLists)
    top = row_top(a, *space_of(a, m).row);
  else
    top = group_maxima(row, Range{0, row.vecs, true, true}, maxima);
  if (lane == 0) s.wave_max[wave] = top;
  if (tid == 0) s.found = V, s.listed_n = 0, s.total = s.total_listed = 0;
  if (tid < kPowers) s.powers[tid] = root_power(tid);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) top = __builtin_elementwise_maximum(top, s.wave_max[i]);
  if (__builtin_expect(!(top > -__builtin_huge_valf()), 0)) {  // NaN, or -inf alone: no distribution
    if (tid == 0) a.tokens[m] = -1, a.logprobs[m] = __builtin_nanf("");
    return;
  }
  const float temperature = a.temperature ? a.temperature[m] : 1.f;
  if (__builtin_expect(!(temperature > 0.f), 0)) {  // greedy
    int first = V;
    if constexpr (SLICED == kRankedLists)
      first = first_of_slices(a, *space_of(a, m).row, top);
    else
      row.each([&](int v, float x) { first = x == top ? min(first, v) : first; });
    if (first < V) atomicMin(&s.found, first);
    __syncthreads();
    if (tid == 0) a.tokens[m] = s.found, a.logprobs[m] = 0.f;
    return;
  }
  const int k = a.top_k && a.top_k[m] > 0 ? a.top_k[m] : V;
  const float min_p = a.min_p ? a.min_p[m] : 0.f;
  const float top_p = a.top_p ? a.top_p[m] : 1.f;
  const bool by_k = k < V, by_p = top_p < 1.f;  // (NaN: off)
  const Rule rule = rule_of(top, temperature, min_p, s.powers);
  const float u = a.uniforms[m];

  // Top-p alone: the sum is one of all weights, and the cut mostly among the first few thousand.
  const bool sums = by_p && !by_k && !(min_p > 0.f);
  u64 all = 0;
  const bool few_k = by_k && k <= kMostK;
  bool listed = few_k || min_p > 0.f || V <= kListed || sums;
  if (SLICED == kRankedLists && (few_k || min_p > 0.f)) {
    listed = gather_lists(s, a, rule, space_of(a, m), few_k, (unsigned)k, min_p);
  } else if (listed) {
    int last = last_bin(min_p);
    if constexpr (SLICED == kRankedLists) group_maxima(row, Range{0, row.vecs, true, true}, maxima);
    if (few_k || sums) last = min(bin_of_maxima(s, rule, maxima, (unsigned)(sums ? kMostK : k)), last);
    // (some may weigh nothing: they change nothing)
    const float end = (float)(last + 1);
    auto in_reach = [&](float x) { return rule.in_bins(x) < end || x == top; };
    auto list = [&](int v, float x) {
      if (in_reach(x)) {
        const unsigned at = atomicAdd(&s.listed_n, 1u);
        if (at < kListed) s.listed[at] = place_of(x, v);
      }
    };
    if (sums) {
      u64 total = 0, reached = 0;
      row.each([&](int v, float x) {
        const u64 w = rule.weight(x);
        total += w;
        if (in_reach(x)) reached += w;
        list(v, x);
      });
      total = wave_inclusive(total), reached = wave_inclusive(reached);
      if (lane == 63) atomicAdd(&s.total, total), atomicAdd(&s.total_listed, reached);
    } else row.template sweep<kAhead>([&](int v0, const float (&x)[kVec]) {
      float most = x[0];
#pragma unroll
      for (int e = 1; e < kVec; ++e) most = fmaxf(most, x[e]);
      if (!in_reach(most)) return;
#pragma unroll
      for (int e = 0; e < kVec; ++e) list(v0 + e, x[e]);
    }, list);
    __syncthreads();
    all = s.total;
    listed = s.listed_n <= kListed &&  // (else ties, or logits too flat)
             (!sums || s.total_listed == all || (double)s.total_listed >= (double)top_p * (double)all);
  }
  const int n = (int)s.listed_n;
  if (__builtin_expect(listed && n <= kFew, 1)) {
    few_tokens(s, rule, n, (unsigned)k, by_p, top_p, all, u, write);
    return;
  }
  auto each_listed = [&](auto f) {
    for (int i = tid; i < n; i += kThreads) f(index_of(s.listed[i]), value_of(s.listed[i]));
  };
  auto each_of_row = [&](auto f) { row.each(f); };
  u64 lowest = 0;
  if (by_k || by_p)
    lowest = listed ? lowest_kept(s, rule, each_listed, by_k, (unsigned)k, by_p, top_p, all, kRankedListed)
                    : lowest_kept(s, rule, each_of_row, by_k, (unsigned)k, by_p, top_p, 0, kRanked);

  __syncthreads();
  if (listed) {
    // Kept weights by ranges of the vocabulary, then token by token in the drawn range.
    const int width = (V + kRanked - 1) / kRanked;  // (at most 512)
    for (int i = tid; i < kRanked; i += kThreads) s.parts[i] = 0;
    if (tid == 0) s.n = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads)
      if (s.listed[i] >= lowest) atomicAdd(&s.parts[index_of(s.listed[i]) / width], rule.weight(value_of(s.listed[i])));
    __syncthreads();
    const Drawn d = draw_part(s, kRanked, u);
    for (int i = tid; i < n; i += kThreads)
      if (s.listed[i] >= lowest && index_of(s.listed[i]) / width == d.part) {
        const unsigned at = atomicAdd(&s.n, 1u);
        s.ranked[at] = s.listed[i];
        s.ranked_weight[at] = rule.weight(value_of(s.listed[i]));
      }
    __syncthreads();
    if (tid < (int)s.n) {
      const int mine = index_of(s.ranked[tid]);
      u64 before = d.before;
      for (unsigned i = 0; i < s.n; ++i)
        if (index_of(s.ranked[i]) < mine) before += s.ranked_weight[i];
      const u64 w = s.ranked_weight[tid];
      if (before <= d.target && d.target < before + w) write(mine, w, d.total);
    }
    return;
  }
  // Kept weights by the row's parts.
  auto kept = [&](int v, float x) -> u64 { return place_of(x, v) >= lowest ? rule.weight(x) : 0; };
  const int parts = row.parts(), tail = row.head + row.vecs * kVec;
  if (tid == 0) s.parts[0] = 0, s.parts[parts - 1] = 0;
  __syncthreads();
  if (tid < row.head) atomicAdd(&s.parts[0], kept(tid, row.value(tid)));
  if (tail + tid < V) atomicAdd(&s.parts[parts - 1], kept(tail + tid, row.value(tail + tid)));
  for (int p = wave; p < parts - 2; p += kWaves) {
    const int q = p * 64 + lane;
    u64 w = 0;
    if (q < row.vecs) {
      const auto x = reinterpret_cast<const typename Row<T>::vec_t*>(row.at + row.head)[q];
#pragma unroll
      for (int e = 0; e < kVec; ++e) w += kept(row.head + q * kVec + e, static_cast<float>(x[e]));
    }
    w = wave_inclusive(w);
    if (lane == 63) s.parts[p + 1] = w;
  }
  __syncthreads();
  draw_of_parts(s, rule, row, lowest, u, write);
}

template <typename T>
hipError_t launch(const SampleArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.M * (unsigned)a.slices), threads(kThreads);
  if (a.slices > 1 && (a.top_k || a.min_p)) {
    launch_kernel(slice_list_kernel<T>, grid, threads, 0, stream, a);
    launch_kernel(sample_kernel<T, kRankedLists>, dim3((unsigned)a.M), threads, sizeof(Shared), stream, a);
  } else if (a.slices > 1) {
    launch_kernel(slice_top_kernel<T>, grid, threads, 0, stream, a);
    if (a.top_p) launch_kernel(slice_bins_kernel<T>, grid, threads, 0, stream, a);
    launch_kernel(slice_parts_kernel<T>, grid, threads, 0, stream, a);
    launch_kernel(sample_kernel<T, kSummed>, dim3((unsigned)a.M), threads, sizeof(Shared), stream, a);
  } else {
    launch_kernel(sample_kernel<T, kWhole>, dim3((unsigned)a.M), threads, sizeof(Shared), stream, a);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, bool bf16, hipStream_t stream) {
  static_assert(sizeof(Shared) <= 160 * 1024, "LDS of a CU");
  return bf16 ? launch<__bf16>(a, stream) : launch<float>(a, stream);
}

}  // namespace lsk
