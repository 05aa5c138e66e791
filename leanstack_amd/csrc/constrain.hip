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
// to date by the caller).  The logits are then read and written once; each
// workgroup leaves its best (value, index) as one 64-bit key, and a wave per row
// takes the largest.
// Bound by the logits' bytes.

#include <hip/hip_runtime.h>

#include "lsk_internal.h"

namespace lsk {
namespace {

constexpr int kThreads = kConstrainThreads;
constexpr int kWaves = kThreads / 64;
constexpr unsigned kSeen = 0x80000000u;
constexpr int kBiasShift = 21;
constexpr unsigned kCountMask = (1u << kBiasShift) - 1;
static_assert(kConstrainMaxBias < (1 << (31 - kBiasShift)), "a bias entry's number fits its bits");
static_assert(kConstrainMaxHistory <= kCountMask, "a count fits its bits");

// Larger key: larger value, then lower index.  NaN is the largest value (as
// torch.argmax takes it), -0 equals +0.
__device__ __forceinline__ unsigned long long choice_key(float v, int index) {
  unsigned b = __builtin_bit_cast(unsigned, v == 0.f ? 0.f : v);
  b = v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (unsigned long long)b << 32 | (0xffffffffu - (unsigned)index);
}
// choice_key's upper word of -inf: no value is smaller.
constexpr unsigned kKeyNegInf = ~0xff800000u;

__device__ __forceinline__ unsigned long long max_key(unsigned long long a, unsigned long long b) {
  return a > b ? a : b;
}

__device__ __forceinline__ unsigned long long wave_max_key(unsigned long long k) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) k = max_key(k, __shfl_xor(k, s));
  return k;
}

__device__ __forceinline__ float load_value(const float* p) { return *p; }
__device__ __forceinline__ float load_value(const __bf16* p) { return static_cast<float>(*p); }

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
  constexpr int kVec = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(kVec)));
  extern __shared__ unsigned words[];  // HIST: one per vocabulary entry of the slice
  __shared__ unsigned long long best[kWaves];

  const int row = blockIdx.x / a.slices;
  const int slice = blockIdx.x - row * a.slices;
  const int v0 = slice * a.slice;
  const int n = min(a.slice, a.V - v0);
  const int tid = threadIdx.x;

  RowRule rule = {1.f, 0.f, 0.f};
  const float* bias_values = nullptr;
  if constexpr (HIST) {
    for (int i = tid; i < n; i += kThreads) words[i] = 0;
    __syncthreads();
    if (a.bias_count > 0) {
      const int* ids = a.bias_ids + (size_t)row * a.bias_ld;
      bias_values = a.bias_values + (size_t)row * a.bias_ld;
      for (int i = tid; i < a.bias_count; i += kThreads) {
        const unsigned at = (unsigned)(ids[i] - v0);
        // Of several entries for one token the last counts.
        if (at < (unsigned)n) atomicMax(&words[at], (unsigned)(i + 1) << kBiasShift);
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
      for (int i = tid; i < length; i += kThreads) {
        const unsigned at = (unsigned)(history[i] - v0);
        if (at < (unsigned)n) {
          if (i < prompt)
            atomicOr(&words[at], kSeen);
          else
            atomicAdd(&words[at], 1u);
        }
      }
    }
    __syncthreads();
  }

  const T* src = static_cast<const T*>(a.logits) + (size_t)row * a.logits_ld + v0;
  T* dst = static_cast<T*>(a.out) + (size_t)row * a.V + v0;
  const unsigned* allowed = a.allowed ? a.allowed + (size_t)row * a.allowed_ld : nullptr;
  unsigned long long key = 0;

  auto one = [&](float l, int i) {
    const int v = v0 + i;
    const bool ok = allowed == nullptr || (allowed[v >> 5] >> (v & 31) & 1u);
    unsigned w = 0;
    if constexpr (HIST) w = words[i];
    const T o = static_cast<T>(constrain_value<HIST>(l, w, rule, bias_values, ok));
    key = max_key(key, choice_key(static_cast<float>(o), v));
    return o;
  };
  // 16-byte accesses from the first aligned value of the slice to the last; the
  // values around them one by one.  Rows of an odd vocabulary start anywhere.
  const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / (int)sizeof(T);
  const int head = ((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & 15) ? n : min(lead, n);
  for (int i = tid; i < head; i += kThreads) dst[i] = one(load_value(src + i), i);
  const int vecs = (n - head) / kVec;
  for (int q = tid; q < vecs; q += kThreads) {
    const int i0 = head + q * kVec;
    const vec_t l = *reinterpret_cast<const vec_t*>(src + i0);
    vec_t o;
#pragma unroll
    for (int e = 0; e < kVec; ++e) o[e] = one(static_cast<float>(l[e]), i0 + e);
    *reinterpret_cast<vec_t*>(dst + i0) = o;
  }
  for (int i = head + vecs * kVec + tid; i < n; i += kThreads) dst[i] = one(load_value(src + i), i);

  key = wave_max_key(key);
  if ((tid & 63) == 0) best[tid >> 6] = key;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) key = max_key(key, best[w]);
    a.keys[blockIdx.x] = key;
  }
}

// A wave per row: the largest key of its slices.
__global__ __launch_bounds__(64) void choose_kernel(const unsigned long long* keys, int slices, long long* tokens) {
  const unsigned long long* row = keys + (size_t)blockIdx.x * slices;
  unsigned long long key = 0;
  for (int i = threadIdx.x; i < slices; i += 64) key = max_key(key, row[i]);
  key = wave_max_key(key);
  if (threadIdx.x == 0)
    tokens[blockIdx.x] = (unsigned)(key >> 32) == kKeyNegInf ? -1LL : (long long)(0xffffffffu - (unsigned)key);
}

template <typename T, bool HIST>
hipError_t launch(const ConstrainArgs& a, hipStream_t stream) {
  const size_t lds = HIST ? (size_t)a.slice * 4 : 0;  // at most 64 KB: two workgroups per CU
  launch_kernel(constrain_kernel<T, HIST>, dim3((unsigned)a.M * a.slices), dim3(kThreads), lds, stream, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  launch_kernel(choose_kernel, dim3(a.M), dim3(64), 0, stream, a.keys, a.slices, a.tokens);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_constrain(const ConstrainArgs& a, bool bf16, hipStream_t stream) {
  const bool hist = a.history != nullptr || a.bias_count > 0;
  if (bf16) return hist ? launch<__bf16, true>(a, stream) : launch<__bf16, false>(a, stream);
  return hist ? launch<float, true>(a, stream) : launch<float, false>(a, stream);
}

}  // namespace lsk
