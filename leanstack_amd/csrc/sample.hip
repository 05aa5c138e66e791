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

#include <hip/hip_runtime.h>

#include "lsk_internal.h"

namespace lsk {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kList = 1024;
constexpr int kParts = 16;      // of a wave's share of the row, for the draw
constexpr double kUnit = 17592186044416.0;  // 2^44
constexpr float kOctaves = 46.f;            // below the maximum: weights round to zero

// Larger order: larger value; -0 equals +0.  (NaN is seen to apart.)
__device__ __forceinline__ unsigned value_order(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.f);
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ u64 place_of(float x, int v) { return (u64)value_order(x) << 32 | (0xffffffffu - (unsigned)v); }

template <typename V>
__device__ __forceinline__ V wave_inclusive(V v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const V o = __shfl_up(v, s);
    if (lane >= s) v += o;
  }
  return v;
}

struct Shared {
  u64 weight[kBins], before[kBins];      // of the bins; and of those in front
  unsigned count[kBins], counted[kBins];
  u64 sub_weight[kBins];
  unsigned sub_count[kBins];
  u64 list[kList], list_weight[kList];
  u64 wave_weight[kWaves];
  unsigned wave_count[kWaves];
  u64 parts[kWaves * kParts];
  u64 lo, hi, kept;
  unsigned n;
  int found, nan;
};

// Exclusive sums of count and weight over the bins; found: the first bin at which `reached`
// (count and weight up to and with it), kBins if there is none.  Returns whether there is.
template <typename Reached>
__device__ void scan_bins(Shared& s, const unsigned* count, const u64* weight, unsigned* counted, u64* before,
                          Reached reached) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const unsigned c0 = count[2 * tid], c1 = count[2 * tid + 1];
  const u64 w0 = weight[2 * tid], w1 = weight[2 * tid + 1];
  const unsigned c = wave_inclusive(c0 + c1);
  const u64 w = wave_inclusive(w0 + w1);
  if (tid == 0) s.found = kBins;
  __syncthreads();
  if (lane == 63) s.wave_count[wave] = c, s.wave_weight[wave] = w;
  __syncthreads();
  unsigned cb = c - c0 - c1;
  u64 wb = w - w0 - w1;
  for (int i = 0; i < wave; ++i) cb += s.wave_count[i], wb += s.wave_weight[i];
  if (counted) {
    counted[2 * tid] = cb, counted[2 * tid + 1] = cb + c0;
    before[2 * tid] = wb, before[2 * tid + 1] = wb + w0;
  }
  if (c0 && reached(cb + c0, wb + w0)) atomicMin(&s.found, 2 * tid);
  if (c1 && reached(cb + c0 + c1, wb + w0 + w1)) atomicMin(&s.found, 2 * tid + 1);
  __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  Shared& s = *reinterpret_cast<Shared*>(shared_bytes);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x;
  const T* logits = static_cast<const T*>(a.logits) + (size_t)row * a.logits_ld;
  const int V = a.V;

  // The largest place.
  if (tid == 0) s.nan = 0, s.hi = 0;
  __syncthreads();
  u64 best = 0;
  bool nan = false;
  for (int v = tid; v < V; v += kThreads) {
    const float x = static_cast<float>(logits[v]);
    nan |= x != x;
    const u64 p = place_of(x, v);
    best = p > best ? p : best;
  }
  atomicMax(&s.hi, best);
  if (nan) s.nan = 1;
  __syncthreads();
  best = s.hi;
  const int best_at = (int)(0xffffffffu - (unsigned)best);
  const float top = static_cast<float>(logits[best_at]);
  if (s.nan || top == -__builtin_huge_valf()) {  // no distribution
    if (tid == 0) a.tokens[row] = -1, a.logprobs[row] = __builtin_nanf("");
    return;
  }
  const float temperature = a.temperature ? a.temperature[row] : 1.f;
  if (!(temperature > 0.f)) {  // greedy
    if (tid == 0) a.tokens[row] = best_at, a.logprobs[row] = 0.f;
    return;
  }
  const int k = a.top_k && a.top_k[row] > 0 ? a.top_k[row] : V;
  const float min_p = a.min_p ? a.min_p[row] : 0.f;
  const float top_p = a.top_p ? a.top_p[row] : 1.f;
  const double least = min_p > 0.f ? (double)fminf(min_p, 1.f) * kUnit : 0.0;  // (NaN: off)
  const bool by_k = k < V, by_p = top_p < 1.f;                                // (NaN: off)

  const double to_base2 = 1.4426950408889634 / (double)temperature;
  // Weight in units; 0 also for what min_p drops (a token without weight counts for nothing).
  auto weight_of = [&](float x) -> u64 {
    if (x == top) return 1ull << 44;
    const double t = ((double)x - (double)top) * to_base2;
    if (!(t > -kOctaves)) return 0;
    const double w = __builtin_rint(exp2(t) * kUnit);
    return w >= least ? (u64)w : 0;
  };
  // Bins down from the maximum, monotone in x.
  const float per_bin = (float)kBins * 1.44269504f / (kOctaves * temperature);
  auto bin_of = [&](float x) {
    const float f = (top - x) * per_bin;
    return x == top ? 0 : f < (float)(kBins - 1) ? (int)f : kBins - 1;
  };
  auto each = [&](auto f) {
    for (int v = tid; v < V; v += kThreads) f(v, static_cast<float>(logits[v]));
  };

  // The lowest kept place of the bin in which a cut lies: the first k by count, or those with
  // less than `target` in front of them.  base_c, base_w: what lies in front of the bin.
  // Returns the place; s.kept: the weight up to it.
  auto cut_in_bin = [&](int bin, unsigned base_c, u64 base_w, bool count, unsigned want, double target) -> u64 {
    if (tid == 0) s.lo = ~0ull, s.hi = 0, s.n = 0;
    __syncthreads();
    {
      u64 lo = ~0ull, hi = 0;
      unsigned n = 0;
      each([&](int v, float x) {
        if (bin_of(x) == bin && weight_of(x)) {
          const u64 p = place_of(x, v);
          lo = p < lo ? p : lo, hi = p > hi ? p : hi, ++n;
        }
      });
      if (n) atomicMin(&s.lo, lo), atomicMax(&s.hi, hi), atomicAdd(&s.n, n);
    }
    __syncthreads();
    u64 lo = s.lo, hi = s.hi;
    unsigned n = s.n;
    while (n > kList) {
      const int bits = 64 - __clzll((long long)(hi - lo));
      const int shift = bits > 11 ? bits - 11 : 0;
      for (int i = tid; i < kBins; i += kThreads) s.sub_count[i] = 0, s.sub_weight[i] = 0;
      __syncthreads();
      each([&](int v, float x) {
        if (bin_of(x) != bin) return;
        const u64 p = place_of(x, v);
        if (p < lo || p > hi) return;
        const u64 w = weight_of(x);
        if (!w) return;
        const int at = (int)((hi - p) >> shift);
        atomicAdd(&s.sub_count[at], 1u);
        atomicAdd(&s.sub_weight[at], w);
      });
      __syncthreads();
      scan_bins(s, s.sub_count, s.sub_weight, nullptr, nullptr, [&](unsigned c, u64 w) {
        return count ? base_c + c >= want : (double)(base_w + w) >= target;
      });
      // (rounding can leave the target out of reach: then the last)
      int at = s.found;
      if (at == kBins) at = (int)((hi - lo) >> shift);
      __syncthreads();
      if (tid == 0) s.lo = 0, s.hi = 0;
      __syncthreads();
      u64 c = 0, w = 0;
      for (int i = tid; i < at; i += kThreads) c += s.sub_count[i], w += s.sub_weight[i];
      if (c) atomicAdd(&s.lo, c), atomicAdd(&s.hi, w);
      __syncthreads();
      base_c += (unsigned)s.lo, base_w += s.hi;
      n = s.sub_count[at];
      hi -= (u64)at << shift;
      const u64 low = hi - ((1ull << shift) - 1);
      lo = hi >= ((1ull << shift) - 1) && low > lo ? low : lo;
      __syncthreads();
    }
    if (tid == 0) s.n = 0, s.lo = ~0ull, s.kept = base_w;
    __syncthreads();
    each([&](int v, float x) {
      if (bin_of(x) != bin) return;
      const u64 p = place_of(x, v);
      if (p < lo || p > hi) return;
      const u64 w = weight_of(x);
      if (!w) return;
      const unsigned at = atomicAdd(&s.n, 1u);
      if (at < kList) s.list[at] = p, s.list_weight[at] = w;
    });
    __syncthreads();
    n = min(s.n, (unsigned)kList);
    if (tid < (int)n) {
      const u64 mine = s.list[tid];
      unsigned c = base_c;
      u64 w = base_w;
      for (unsigned i = 0; i < n; ++i)
        if (s.list[i] > mine) ++c, w += s.list_weight[i];
      if (count ? c < want : c == 0 || (double)w < target) {
        atomicMin(&s.lo, mine);
        atomicAdd(&s.kept, s.list_weight[tid]);
      }
    }
    __syncthreads();
    return s.lo;
  };

  u64 lowest = 0;  // kept place
  if (by_k || by_p) {
    for (int i = tid; i < kBins; i += kThreads) s.count[i] = 0, s.weight[i] = 0;
    __syncthreads();
    each([&](int, float x) {
      const u64 w = weight_of(x);
      if (!w) return;
      const int at = bin_of(x);
      atomicAdd(&s.count[at], 1u);
      atomicAdd(&s.weight[at], w);
    });
    __syncthreads();
    scan_bins(s, s.count, s.weight, s.counted, s.before,
              [&](unsigned c, u64) { return c > (unsigned)k; });  // more than k: a cut
    u64 sum = s.before[kBins - 1] + s.weight[kBins - 1];
    // The bin of the k-th: the first at which the count reaches k.
    if (by_k && s.found < kBins) {
      __syncthreads();
      scan_bins(s, s.count, s.weight, s.counted, s.before, [&](unsigned c, u64) { return c >= (unsigned)k; });
      const int bin = s.found;
      __syncthreads();
      lowest = cut_in_bin(bin, s.counted[bin], s.before[bin], true, (unsigned)k, 0.0);
      sum = s.kept;
    }
    if (by_p) {
      const double target = top_p > 0.f ? (double)top_p * (double)sum : 0.0;
      __syncthreads();
      scan_bins(s, s.count, s.weight, s.counted, s.before, [&](unsigned, u64 w) { return (double)w >= target; });
      const int bin = s.found;
      __syncthreads();
      if (bin < kBins) {
        const u64 p = cut_in_bin(bin, s.counted[bin], s.before[bin], false, 0, target);
        lowest = p > lowest ? p : lowest;
      }
    }
    __syncthreads();
  }

  // The draw: sums of kParts parts of each wave's share of the row, in index order.
  const int share = (V + kWaves * kParts - 1) / (kWaves * kParts);
  auto kept = [&](int v) -> u64 {
    const float x = static_cast<float>(logits[v]);
    return place_of(x, v) >= lowest ? weight_of(x) : 0;
  };
  for (int i = 0; i < kParts; ++i) {
    const int begin = min((wave * kParts + i) * share, V), end = min(begin + share, V);
    u64 w = 0;
    for (int v = begin + lane; v < end; v += 64) w += kept(v);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) w += __shfl_xor(w, d);
    if (lane == 0) s.parts[wave * kParts + i] = w;
  }
  __syncthreads();
  if (wave != 0) return;
  constexpr int kMine = kWaves * kParts / 64;
  u64 mine = 0;
#pragma unroll
  for (int i = 0; i < kMine; ++i) mine += s.parts[lane * kMine + i];
  const u64 up_to = wave_inclusive(mine);
  const u64 total = __shfl(up_to, 63);
  const float u = a.uniforms[row];
  u64 target = u > 0.f ? (u64)((double)fminf(u, 1.f) * (double)total) : 0;
  if (target >= total) target = total - 1;
  const u64 here = __ballot(up_to > target);
  const int from = __builtin_ctzll(here);
  u64 sum = __shfl(up_to - mine, from);
  int part = from * kMine;
  for (int i = 0; i < kMine - 1; ++i) {
    const u64 w = s.parts[part];
    if (sum + w > target) break;
    sum += w, ++part;
  }
  const int begin = part * share, end = min(begin + share, V);
  for (int v0 = begin; v0 < end; v0 += 64) {
    const int v = v0 + lane;
    const u64 w = v < end ? kept(v) : 0;
    const u64 c = sum + wave_inclusive(w);
    const u64 there = __ballot(c > target);
    if (there) {
      if (lane == __builtin_ctzll(there)) {
        a.tokens[row] = v;
        a.logprobs[row] = (float)log((double)w / (double)total);
      }
      return;
    }
    sum = __shfl(c, 63);
  }
}

template <typename T>
hipError_t launch(const SampleArgs& a, hipStream_t stream) {
  launch_kernel(sample_kernel<T>, dim3((unsigned)a.M), dim3(kThreads), sizeof(Shared), stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, bool bf16, hipStream_t stream) {
  return bf16 ? launch<__bf16>(a, stream) : launch<float>(a, stream);
}

}  // namespace lsk
