// Per-request constraints on the logits in front of the greedy choice, and the
// choice, for gfx950: penalties for repeated tokens, biases and grammar masks.
//
// Per value, in this order (fp32, one rounding per step):
//   z = l;  token seen: z = z > 0 ? z / rho : z * rho;
//   c > 0 in the answer: z = (z - alpha_f c) - alpha_p;  z += bias;
//   not allowed: z = -inf;  rounded once to the logits' type.
// The token is the lowest index of the largest rounded value.
//
// One workgroup per (row, slice of the vocabulary).  What a request has said is
// a list of tokens; a slice's workgroup reads the whole list and counts those in
// its slice in LDS, one word per vocabulary entry:
//   bit 31: in the prompt;  bits 21..30: bias entry + 1;  bits 0..20: c
// by integer atomics, whose order does not matter (a table of counts per row in
// memory would be read beside the logits, twice their bytes in bf16, and kept up
// to date by the caller).  The logits are then read and written once, 16 bytes a
// lane, with the values' words and mask bits beside them.  A workgroup's best
// (value, index) is one 64-bit key, the largest of a row's keys its token: the
// workgroup that counts itself the row's last reads them all.  Nothing waits.
//
// Bound by the logits' bytes for many rows: 128 rows of 151936 fp32 logits with 8000
// tokens, 300 biases and masks 42.2 us, 3.8 TB/s (a copy reaches 4.8).  For few rows
// by its chain of latencies (list, counts, logits, the last workgroup): 5.8 us for
// one row with 600 tokens, 5.0 for five with masks alone.  37 rows of 50257 in bf16 with
// 2000 tokens take 10.5 us for 8 MB: each of a row's 25 slices reads its whole list.
// Rows whose logits and results lie differently against 16 bytes (a view of a padded
// vocabulary) go value by value, in about the same time: 128 rows of 50257 with 8000
// tokens 20.2 us (fp32) and 20.3 (bf16) of a view 50272 wide, 21.4 and 19.9 dense.

#include <hip/hip_runtime.h>

#include "lsk_internal.h"

namespace lsk {
namespace {

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kThreads = kConstrainThreads;
constexpr int kWaves = kThreads / 64;
constexpr int kAhead = 4;  // history accesses of a thread in flight
constexpr unsigned kSeen = 0x80000000u;
constexpr int kBiasShift = 21;
constexpr unsigned kCountMask = (1u << kBiasShift) - 1;
static_assert(kConstrainMaxBias < (1 << (31 - kBiasShift)), "a bias entry's number fits its bits");
static_assert(kConstrainMaxHistory <= kCountMask, "a count fits its bits");

// Larger order: larger value.  NaN is the largest (as torch.argmax takes it), -0
// equals +0.
__device__ __forceinline__ unsigned value_order(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.f);
  return v != v ? 0xffffffffu : b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
constexpr unsigned kOrderNegInf = ~0xff800000u;  // value_order(-inf): no value is smaller

// Of two keys (value_order, then ~index) the larger is the larger value, or the lower index.
__device__ __forceinline__ unsigned long long max_key(unsigned long long a, unsigned long long b) {
  return a > b ? a : b;
}

__device__ __forceinline__ unsigned long long wave_max_key(unsigned long long k) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) k = max_key(k, __shfl_xor(k, s));
  return k;
}

struct RowRule {
  float rho, alpha_f, alpha_p;
};

// One value under its slice word `w` (0 without a history or biases).
template <bool HIST>
__device__ __forceinline__ float constrain_value(float z, unsigned w, const RowRule& r, const float* bias_values,
                                                 bool allowed) {
#pragma clang fp contract(off)
  if constexpr (HIST) {
    if (w != 0) {
      const unsigned count = w & kCountMask;
      if ((w & kSeen) || count) z = z > 0.f ? z / r.rho : z * r.rho;
      if (count) z = (z - r.alpha_f * static_cast<float>(count)) - r.alpha_p;
      const unsigned entry = (w & ~kSeen) >> kBiasShift;
      if (entry) z = z + bias_values[entry - 1];
    }
  }
  return allowed ? z : -__builtin_huge_valf();
}

template <typename T, bool HIST>
__global__ __launch_bounds__(kThreads) void constrain_kernel(ConstrainArgs a) {
#pragma clang fp contract(off)
  constexpr int kHold = HIST ? 5 : 1;  // logits accesses of a thread in flight
  constexpr int kVec = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(kVec)));
  extern __shared__ __align__(16) unsigned words[];  // HIST: one per vocabulary entry of the slice, from `shift` on
  __shared__ unsigned long long best[kWaves];

  const int row = blockIdx.x / a.slices;
  const int slice = blockIdx.x - row * a.slices;
  const int v0 = slice * a.slice;
  const int n = min(a.slice, a.V - v0);
  const int tid = threadIdx.x;
  const T* src = static_cast<const T*>(a.logits) + (size_t)row * a.logits_ld + v0;
  T* dst = static_cast<T*>(a.out) + (size_t)row * a.V + v0;
  // 16-byte accesses from the first aligned value of the slice to the last; the
  // values around them one by one.  Rows of an odd vocabulary start anywhere.
  const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / (int)sizeof(T);
  const int head = ((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & 15) ? n : min(lead, n);
  const int vecs = (n - head) / kVec;
  const int shift = (kVec - head % kVec) % kVec;  // the words of an access are aligned too

  // The first logits are on their way while the history is counted (a slice of
  // kConstrainMaxSlice fp32 values is five accesses per thread: 106 -> 84 us at 300
  // rows of 151936 with 2000 tokens); without one a single access is as fast.
  vec_t held[kHold];
  auto load_round = [&](int q0) {
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (q0 + k * kThreads < vecs) held[k] = *reinterpret_cast<const vec_t*>(src + head + (q0 + k * kThreads) * kVec);
  };
  load_round(tid);

  RowRule rule = {1.f, 0.f, 0.f};
  const float* bias_values = nullptr;
  if constexpr (HIST) {
    for (int i = 4 * tid; i < n + kVec; i += 4 * kThreads) *reinterpret_cast<u32x4_t*>(words + i) = u32x4_t{0u, 0u, 0u, 0u};
    __syncthreads();
    unsigned* mine = words + shift;
    if (a.bias_count > 0) {
      const int* ids = a.bias_ids + (size_t)row * a.bias_ld;
      bias_values = a.bias_values + (size_t)row * a.bias_ld;
      for (int i = tid; i < a.bias_count; i += kThreads) {
        const unsigned at = (unsigned)(ids[i] - v0);
        // Of several entries for one token the last counts.
        if (at < (unsigned)n) atomicMax(&mine[at], (unsigned)(i + 1) << kBiasShift);
      }
      __syncthreads();
    }
    if (a.history != nullptr) {
      if (a.repetition) rule.rho = a.repetition[row];
      if (a.frequency) rule.alpha_f = a.frequency[row];
      if (a.presence) rule.alpha_p = a.presence[row];
      const int* history = a.history + (size_t)row * a.history_ld;
      const int length = a.history_lens ? min(max(a.history_lens[row], 0), a.history_len) : a.history_len;
      const int prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
      auto count = [&](int token, int i) {
        const unsigned at = (unsigned)(token - v0);
        if (at < (unsigned)n) {
          if (i < prompt)
            atomicOr(&mine[at], kSeen);
          else
            atomicAdd(&mine[at], 1u);
        }
      };
      // 16 bytes a load from the first aligned token on, four loads in flight.
      const int first = min((int)((16 - (reinterpret_cast<uintptr_t>(history) & 15)) & 15) / 4, length);
      const int fours = (length - first) / 4;
      const u32x4_t* list = reinterpret_cast<const u32x4_t*>(history + first);
      if (tid < first) count(history[tid], tid);
      for (int q = tid; q < fours; q += kAhead * kThreads) {
        u32x4_t token[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) token[k] = list[min(q + k * kThreads, fours - 1)];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          if (q + k * kThreads >= fours) break;
#pragma unroll
          for (int e = 0; e < 4; ++e) count((int)token[k][e], first + 4 * (q + k * kThreads) + e);
        }
      }
      for (int i = first + 4 * fours + tid; i < length; i += kThreads) count(history[i], i);
    }
    __syncthreads();
  }

  const unsigned* allowed = a.allowed ? a.allowed + (size_t)row * a.allowed_ld : nullptr;
  unsigned top = 0;  // value_order of the thread's largest value: at its lowest index, as indices rise
  int top_at = 0;
  auto one = [&](float l, int i, unsigned w, bool ok) {
    const T o = static_cast<T>(constrain_value<HIST>(l, w, rule, bias_values, ok));
    const unsigned order = value_order(static_cast<float>(o));
    if (order > top) top = order, top_at = v0 + i;
    return o;
  };
  auto single = [&](int i) {
    const int v = v0 + i;
    unsigned w = 0;
    if constexpr (HIST) w = words[i + shift];
    dst[i] = one(static_cast<float>(src[i]), i, w, allowed == nullptr || (allowed[v >> 5] >> (v & 31) & 1u));
  };
  for (int i = tid; i < head; i += kThreads) single(i);
  auto access = [&](int q, vec_t l) {
    const int i0 = head + q * kVec;
    unsigned bits = 0xffffffffu;
    if (allowed != nullptr) {
      const int v = v0 + i0;
      const int last = v + kVec - 1;  // in the next word where the access straddles two
      bits = (unsigned)(((unsigned long long)allowed[last >> 5] << 32 | allowed[v >> 5]) >> (v & 31));
    }
    unsigned w[kVec] = {};
    if constexpr (HIST) {
#pragma unroll
      for (int e = 0; e < kVec; e += 4) {
        const u32x4_t four = *reinterpret_cast<const u32x4_t*>(words + shift + i0 + e);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[e + k] = four[k];
      }
    }
    vec_t o;
#pragma unroll
    for (int e = 0; e < kVec; ++e) o[e] = one(static_cast<float>(l[e]), i0 + e, w[e], bits >> e & 1u);
    *reinterpret_cast<vec_t*>(dst + i0) = o;
  };
  for (int q0 = tid; q0 < vecs; q0 += kHold * kThreads) {
    if (q0 != tid) load_round(q0);
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (q0 + k * kThreads < vecs) access(q0 + k * kThreads, held[k]);
  }
  for (int i = head + vecs * kVec + tid; i < n; i += kThreads) single(i);

  unsigned long long key = (unsigned long long)top << 32 | (0xffffffffu - (unsigned)top_at);
  key = wave_max_key(key);
  if ((tid & 63) == 0) best[tid >> 6] = key;
  __syncthreads();
  if (tid >= 64) return;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) key = max_key(key, best[w]);
  if (a.slices > 1) {
    // The key is where every workgroup sees it before this one counts itself.
    unsigned long long* keys = a.keys + (size_t)row * a.slices;
    unsigned arrived = 0;
    if (tid == 0) {
      __hip_atomic_store(keys + slice, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      arrived = __hip_atomic_fetch_add(a.arrived + (size_t)row * kConstrainCounterWords, 1u, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
    }
    if (__builtin_amdgcn_readfirstlane(arrived) != (unsigned)a.slices - 1) return;
    for (int i = tid; i < a.slices; i += 64) {
      key = max_key(key, __hip_atomic_load(keys + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      __hip_atomic_store(keys + i, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    key = wave_max_key(key);
    if (tid == 0)
      __hip_atomic_store(a.arrived + (size_t)row * kConstrainCounterWords, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (tid == 0) a.tokens[row] = (unsigned)(key >> 32) == kOrderNegInf ? -1LL : (long long)(0xffffffffu - (unsigned)key);
}

template <typename T, bool HIST>
hipError_t launch(const ConstrainArgs& a, hipStream_t stream) {
  // four workgroups per CU
  constexpr int kMostLds = (kConstrainMaxSlice + 16) * 4;
  static_assert(4 * (kMostLds + kWaves * 8) <= 160 * 1024 && kConstrainMaxSlice % 64 == 0, "their LDS");
  const size_t lds = HIST ? (size_t)(a.slice + 2 * (16 / sizeof(T))) * 4 : 0;
  launch_kernel(constrain_kernel<T, HIST>, dim3((unsigned)a.M * a.slices), dim3(kThreads), lds, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_constrain(const ConstrainArgs& a, bool bf16, hipStream_t stream) {
  const bool hist = a.history != nullptr || a.bias_count > 0;
  if (bf16) return hist ? launch<__bf16, true>(a, stream) : launch<__bf16, false>(a, stream);
  return hist ? launch<float, true>(a, stream) : launch<float, false>(a, stream);
}

}  // namespace lsk
