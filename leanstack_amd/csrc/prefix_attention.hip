// Attention of a batch of requests that share a prefix, for gfx950: T query
// tokens of each request over P prefix rows, held once, and over the rows that
// the request has cached since (causal within them).
//
//   out = sum_i e^(s_i - m) v_i / sum_i e^(s_i - m),  s = scale q . k,
// over the prefix rows and the request's own visible rows.  The prefix is read
// once for many requests' heads instead of once per request, which is what
// makes a long one cheap.
//
// Work is cut into items: 32 (or 4 x 32) query rows of one kv head over a
// range of key rows.  Query rows of a prefix item are those of any requests (row
// (b T + t) G + g of the kv head); an own item's are one request's.  A wave
// holds 32 query rows and takes 32 key rows a step:
//   S^T = K Q^T on v_mfma_f32_32x32x16_bf16, so that a lane holds 16 scores of
//     one query row, and the other 16 are in the other half-wave;
//   the running maximum m and sum l of the softmax, in base 2, in fp32.  m is
//     raised only where a step exceeds it by 2^8 (weights up to 2^8 are as exact
//     as weights up to 1, and the sums, rescaled on a raise, stay in range of
//     values up to some 2^110);
//   O^T += V^T P^T on the same MFMA.  The scores' lanes are those of the B operand
//     if the 16 key rows of a product are taken in the order that the lanes hold
//     them in, so P needs no transposition; V^T comes from LDS by
//     ds_read_b64_tr_b16.
// P is rounded to bf16, at most 2^-8 of each weight, and l sums the rounded
// weights: the result is exactly that of slightly other weights, whose errors
// average out over the rows (the output's own rounding is as large: 0.0018 to 0.0022
// from 64 bits in all, relative 2-norm, 0.0017 with weights in fp32, which P V
// on matrix instructions would take twice the products for).
//
// K and V rows go to LDS by DMA, their 16-byte chunks permuted by row so that
// neither 16 lanes' reads of K (one row per lane) nor of V (four rows) meet in a
// bank.  Rows past the last visible one are out of the buffers' range and come as
// zeros: what lies behind the written rows is never read.
//
// Items whose waves share query rows (own rows; a prefix with few query rows) split
// the key rows, each wave with a slot of its own and no barrier: the next step's K
// is on its way while P V is multiplied, the next V during the next scores.  Items
// of 128 query rows share each step's rows among the waves through a ring of slots.
//
// An item leaves (m, l, O) in fp32 in the workspace and a second launch adds a
// row's items up; a short context runs in one launch, each request's items
// reading the prefix and its own rows.
//
// What it measured (32 q, 8 kv heads; B requests of T tokens, P + S rows; medians of
// the launches by themselves):
//   1x5 300+64       8.8 us, one launch: latency (the bytes are 0.3 us)
//   12x1 1024+512    7.0 + 4.0 us
//   64x1 8191+1088  41.4 + 5.0 us: 166 MB, 4.0 TB/s in the first launch (a copy reaches 4.8)
//   48x4 16000+320  65.4 + 8.5 us: 51 GFLOP, 777 TFLOP/s in the first launch (a large matrix
//     product reaches 1214).  A step of a wave is 512 cycles of MFMA; by the counters
//     products are under way in 42 % of the cycles of a busy CU, vector instructions
//     (most of them the softmax's) in 52 %, its LDS pipe in 34 % (105 cycles a step, 33
//     of them bank conflicts): the first two take turns more than they overlap.
//     Tried and no faster: 8 waves with 256 query rows (74 us for 67), pairs of steps,
//     half the waves a barrier behind the others (79), 64 query rows per wave (70).
//   prompts: 1x256 1024+256  21.0 + 7.7 us; 1x512 4096+512  57.2 + 14.6 us, 640 TFLOP/s;
//     4x256 2048+256  59.5 + 23.2 us

#include <hip/hip_runtime.h>

#include <type_traits>

#include "lsk_internal.h"

namespace lsk {
namespace {

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

constexpr int D = kAttnHeadDim;
constexpr int kStep = 32;                  // key rows, and query rows of a wave
constexpr int kHalfSlot = kStep * D * 2;   // bytes of a step's K, or V
constexpr int kSlot = 2 * kHalfSlot;
constexpr float kRaise = 8.f;
constexpr float kFar = 0x1p30f;
constexpr int kJointWaves = 8;             // of an item of a short context
constexpr int kWaves = 4;                  // of another item
static_assert(kPrefixSharedRows == 32 * kWaves, "query rows of an item whose waves have some of their own");

__device__ __forceinline__ float neg_inf() { return -__builtin_huge_valf(); }

// Both halves' values of a lane pair 32 apart, in both lanes.  (The compiler takes
// a swap of a value with itself for two equal results: it is given a copy that it
// does not know to be one.)
struct Halves {
  float low, high;
};
__device__ __forceinline__ Halves both_halves(float v) {
  const unsigned a = __builtin_bit_cast(unsigned, v);
  unsigned b = a;
  asm("" : "+v"(b));
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  return {__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1])};
}
__device__ __forceinline__ float other_half_max(float v) {
  const Halves h = both_halves(v);
  return fmaxf(h.low, h.high);
}
__device__ __forceinline__ float other_half_sum(float v) {
  const Halves h = both_halves(v);
  return h.low + h.high;
}

// Rows that request b has cached, and those of them that its query t sees.
__device__ __forceinline__ int own_written(const PrefixArgs& a, int b) { return min(max(a.lens[b], 0), a.S); }
__device__ __forceinline__ int own_visible(const PrefixArgs& a, int b, int t) {
  return max(own_written(a, b) - (a.T - 1 - t), 0);
}

// Key rows [begin, end) of one kv head.
struct Rows {
  const __bf16 *k, *v;
  int stride;  // elements from a row to the next
  int begin, end;
};

// A wave's softmax state for its 32 query rows: lane (h, c) holds row c, of O the
// dims 32 db + 8 (i / 4) + 4 h + i % 4, of l the share of the lane's scores, and
// of m the factor c2 that takes its scores to base 2.
struct State {
  float m, l, c2;
  f32x16_t o[4];
};

// Addresses of a lane in a step's rows, the same for every step.
struct Lane {
  unsigned k_at[4], v_at[2];  // DMA: byte offsets from the step's first row, K loads 0..3 and V loads 0..1
  unsigned k_read;            // LDS: row c, chunk h
  unsigned v_read;            // LDS: transposing read of 4 rows x 16 dims per 16 lanes
};

// Chunk (16 bytes) `ch` of row r is at position ch ^ (r % 16) for K and
// ch ^ 2 (r % 8) for V.
__device__ __forceinline__ Lane lane_addresses(int stride) {
  const int lane = threadIdx.x & 63;
  Lane a;
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // load i: rows 4 i + lane / 16
    const int r = 4 * i + (lane >> 4);
    a.k_at[i] = (unsigned)(r * stride * 2 + (((lane & 15) ^ r) << 4));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 4 * i + (lane >> 4);
    a.v_at[i] = (unsigned)(r * stride * 2 + (((lane & 15) ^ (2 * r)) << 4));
  }
  const int c = lane & 31, h = lane >> 5;
  a.k_read = (unsigned)(c * 256 + ((h ^ (c & 15)) << 4));
  const int i = lane & 15, q = lane >> 4;
  const int r = 4 * (q >> 1) + (i >> 2);
  a.v_read = (unsigned)(r * 256 + (((2 * (q & 1) + ((i & 3) >> 1)) ^ (2 * r)) << 4) + ((i & 1) << 3));
  return a;
}

// K and V rows up to `end` from 16 (K) or 8 (V) row boundaries of a step on: each load
// of a step is then the lane's offset, the step's and a buffer.  Rows from `end` on
// are out of range: zeros to LDS, and no memory access.
struct Buffers {
  lds_load_words_t k[2], v[4];
};
__device__ __forceinline__ lds_load_words_t rows_from(const __bf16* p, int stride, int end, int first) {
  const long long bytes = ((long long)(end - 1 - first) * stride + D) * 2;
  lds_load_words_t w = buffer_words(p + (size_t)first * stride, end > first ? (size_t)bytes : 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_readfirstlane(w[i]);  // wave-uniform; says so to the compiler
  return w;
}
__device__ __forceinline__ Buffers row_buffers(const Rows& src) {
  Buffers b;
#pragma unroll
  for (int i = 0; i < 2; ++i) b.k[i] = rows_from(src.k, src.stride, src.end, 16 * i);
#pragma unroll
  for (int i = 0; i < 4; ++i) b.v[i] = rows_from(src.v, src.stride, src.end, 8 * i);
  return b;
}

// A step's K, V to LDS (8 loads of 1 KB, 4 rows each); `off`: byte offset of its first row.
__device__ __forceinline__ void load_k(const Buffers& b, const Lane& a, unsigned off, unsigned lds) {
#pragma unroll
  for (int u = 0; u < 8; ++u) dma_1k<false>(b.k[u >> 2], a.k_at[u & 3] + off, 0, lds + u * 1024);
}
__device__ __forceinline__ void load_v(const Buffers& b, const Lane& a, unsigned off, unsigned lds) {
#pragma unroll
  for (int u = 0; u < 8; ++u) dma_1k<false>(b.v[u >> 1], a.v_at[u & 1] + off, 0, lds + u * 1024);
}

typedef __attribute__((address_space(3))) const unsigned char lds_byte_t;

__device__ __forceinline__ bf16x8_t k_operand(lds_byte_t* k, const Lane& a, int ks) {
  return *reinterpret_cast<__attribute__((address_space(3))) const bf16x8_t*>(k + (a.k_read ^ (unsigned)(ks << 5)));
}

// S^T = K Q^T of a step's key rows.  A product waits twice its time for the one that it
// adds to: two half sums by turns.
__device__ __forceinline__ f32x16_t step_scores(lds_byte_t* k, const Lane& a, const bf16x8_t (&qf)[8]) {
  f32x16_t c[2] = {};
#pragma unroll
  for (int ks = 0; ks < 8; ++ks)
    c[ks & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_operand(k, a, ks), qf[ks], c[ks & 1], 0, 0, 0);
  return c[0] + c[1];
}

// V^T of rows 16 s .. + 15 (in the lanes' order: slot e of half h is row
// 16 s + 8 (e / 4) + 4 h + e % 4), dims 32 db .. + 31.
__device__ __forceinline__ bf16x8_t v_operand(lds_byte_t* v, const Lane& a, int s, int db) {
  typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4_t;
  auto* at = (lds_bf16x4_t*)(v + (a.v_read ^ (unsigned)(db << 6)) + s * 16 * 256);
  const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(at);
  const bf16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(at + 8 * 256 / 8);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The weights P of a step (bf16, the B operands of two products), and m, l, O
// brought to the new maximum.  limit: key rows of the step that the lane's query row
// sees.
//
// Exponents are s c2 - m with one rounding, m being the rounded top c2: far from zero
// (kFar) its rounding error would be more than 2^x holds.  There scores that are not
// equal are 2^6 and more apart in base 2, so any factor gives the same weights, if m's
// order stays: the next power of two above c2, whose products are exact.
template <bool MASK>
__device__ __forceinline__ void step_weights(f32x16_t s, float c2, int limit, State& st, bf16x8_t (&p)[2]) {
  const int h = (threadIdx.x & 63) >> 5;
  auto seen = [&](int i) { return 8 * (i / 4) + 4 * h + i % 4 < limit; };
  if constexpr (MASK) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!seen(i)) s[i] = neg_inf();
  }
  float top = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
  top = other_half_max(top);
  float mx = top * st.c2;
  if (MASK && limit <= 0) mx = neg_inf();  // (-inf times a scale of zero)
  const bool raise = mx > st.m + kRaise;
  if (__ballot(raise)) {  // (a query row's maximum goes by its own scores alone)
    const float above = __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, c2) + 0x007fffffu) & 0x7f800000u);
    st.c2 = !raise ? st.c2 : fabsf(top * c2) < kFar ? c2 : above;
    mx = top * st.c2;
    const float f = raise ? __builtin_amdgcn_exp2f(st.m - mx) : 1.f;
    st.m = raise ? mx : st.m;
    st.l *= f;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[db][i] *= f;
  }
  const float m = st.m == neg_inf() ? 0.f : st.m;
  const bf16x2_t ones = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], st.c2, -m));
    if (MASK && !seen(i)) e = 0.f;
    p[i / 8][i % 8] = static_cast<__bf16>(e);
  }
#pragma unroll
  for (int i = 0; i < 16; i += 2)
    st.l = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{p[i / 8][i % 8], p[i / 8][i % 8 + 1]}, ones, st.l, false);
}

__device__ __forceinline__ void step_accumulate(lds_byte_t* v, const Lane& a, const bf16x8_t (&p)[2], State& st) {
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int db = 0; db < 4; ++db)
      st.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v_operand(v, a, s, db), p[s], st.o[db], 0, 0, 0);
}

// V of a step's rows that only some query rows see (from `all` to `end`): a weight
// of zero does not take an infinity or a NaN out of a product, so those become
// zero, and write_item adds them to the query rows that see them.  Returns whether there
// were any.
__device__ __forceinline__ bool mask_values(unsigned char* v, int all, int end) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63;
  bool found = false;
#pragma unroll
  for (int i = 0; i < kHalfSlot / 1024; ++i) {
    const int r = 4 * i + (lane >> 4);
    u32x4* at = reinterpret_cast<u32x4*>(v + i * 1024 + lane * 16);
    if (r >= all && r < end) {
      u32x4 w = *at;
      bool here = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool low = (w[e] & 0x00007f80u) == 0x00007f80u, high = (w[e] & 0x7f800000u) == 0x7f800000u;
        w[e] &= (low ? 0xffff0000u : 0xffffffffu) & (high ? 0x0000ffffu : 0xffffffffu);
        here |= low | high;
      }
      if (here) *at = w;
      found |= here;
    }
  }
  wave_lds_order();
  return __ballot(found) != 0;
}

// vmcnt(8): all but the 8 loads last issued have landed; and what the wave read
// from LDS before is in registers, so its slot may be written.
__device__ __forceinline__ void wait_half() { asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void wait_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

// Rows of `src`, the steps w, w + NW, .. for wave w of NW, counted from the `first`-th
// wave on, in the wave's own slot.  limit: key rows that the lane's query row sees;
// `least`, the least of them (CAUSAL).  Returns whether mask_values took values out.
template <int NW, bool CAUSAL>
__device__ __forceinline__ bool attend_split(const Rows& src, const bf16x8_t (&qf)[8], float c2, int limit,
                                             int least, int first, unsigned char* slots, State& st) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (uniform: so are the branches on it)
  int row0 = src.begin + ((wave - first) & (NW - 1)) * kStep;
  if (row0 >= src.end) return false;
  bool special = false;
  const Lane a = lane_addresses(src.stride);
  const Buffers buf = row_buffers(src);
  auto* slot = (lds_byte_t*)(slots + wave * kSlot);
  const unsigned at = (unsigned)(size_t)slot;
  unsigned off = (unsigned)row0 * (unsigned)(src.stride * 2);
  wait_all();  // (loads counted by the compiler are not among those counted here)
  load_k(buf, a, off, at);
  load_v(buf, a, off, at + kHalfSlot);
  auto step = [&](auto masked) __attribute__((always_inline)) {
    constexpr bool kMask = decltype(masked)::value;
    wait_half();  // K is here
    const f32x16_t s = step_scores(slot, a, qf);
    wait_reads();
    off += (unsigned)(NW * kStep) * (unsigned)(src.stride * 2);
    load_k(buf, a, off, at);
    bf16x8_t p[2];
    step_weights<kMask>(s, c2, min(limit, src.end) - row0, st, p);
    wait_half();  // V is here
    if constexpr (kMask && CAUSAL)
      special |= mask_values(slots + wave * kSlot + kHalfSlot, least - row0, src.end - row0);
    step_accumulate(slot + kHalfSlot, a, p, st);
    wait_reads();
    load_v(buf, a, off, at + kHalfSlot);
    row0 += NW * kStep;
  };
  const int full = CAUSAL ? min(least, src.end) : src.end;
  while (row0 + kStep <= full) step(std::false_type{});
  while (row0 < src.end) step(std::true_type{});
  wait_all();
  return special;
}

// Rows of `src` for four waves with query rows of their own: steps through a ring of
// four slots, two K and two V loads of each step by each wave.
__device__ __forceinline__ void attend_shared(const Rows& src, const bf16x8_t (&qf)[8], float c2, unsigned char* slots,
                                              State& st) {
  constexpr int kRing = kWaves * kSlot;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Lane a = lane_addresses(src.stride);
  // rows 8 wave .. + 7 of a step
  const lds_load_words_t kb = rows_from(src.k, src.stride, src.end, 16 * (wave >> 1));
  const lds_load_words_t vb = rows_from(src.v, src.stride, src.end, 8 * wave);
  const unsigned k0 = wave & 1 ? a.k_at[2] : a.k_at[0], k1 = wave & 1 ? a.k_at[3] : a.k_at[1];
  auto* ring = (lds_byte_t*)slots;
  const unsigned at = (unsigned)(size_t)ring + 2048u * wave;
  unsigned off = (unsigned)src.begin * (unsigned)(src.stride * 2);
  unsigned to = 0;  // slot of the next load
  auto load = [&]() __attribute__((always_inline)) {
    // (past the last row: zeros, so that the count of loads in flight stays the same)
    dma_1k<false>(kb, k0 + off, 0, at + to);
    dma_1k<false>(kb, k1 + off, 0, at + to + 1024);
    dma_1k<false>(vb, a.v_at[0] + off, 0, at + to + kHalfSlot);
    dma_1k<false>(vb, a.v_at[1] + off, 0, at + to + kHalfSlot + 1024);
    off += (unsigned)kStep * (unsigned)(src.stride * 2);
    to = (to + kSlot) & (kRing - 1);
  };
  wait_all();
#pragma unroll
  for (int i = 0; i < kWaves - 1; ++i) load();
  unsigned from = 0;
  int row0 = src.begin;
  auto step = [&](auto masked) __attribute__((always_inline)) {
    // Steps up to this one have landed here (two of 4 loads each are behind it), and
    // with the barrier everywhere; every wave is done with the step before it, whose
    // slot the next load takes.
    asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    load();
    const f32x16_t s = step_scores(ring + from, a, qf);
    bf16x8_t p[2];
    step_weights<decltype(masked)::value>(s, c2, src.end - row0, st, p);
    step_accumulate(ring + from + kHalfSlot, a, p, st);
    from = (from + kSlot) & (kRing - 1);
    row0 += kStep;
  };
  while (row0 + kStep <= src.end) step(std::false_type{});
  if (row0 < src.end) step(std::true_type{});
  wait_all();
}

// Query row r of kv head j: request, token and q head.
struct Query {
  int b, t, h;
};

// What the NW waves leave, to rows of the output or of the workspace.
//   SPLIT: the waves hold the same 32 query rows over different key rows, added
//   here; else 32 rows each.
// find(i): query row i of the item, or b = -1 behind the last one.  add(q, d, l, o): what
// mask_values took out of dims d .. d + 3 for query row q, whose weights sum to l.
template <int NW, bool SPLIT, bool DIRECT, typename Find, typename Add>
__device__ __forceinline__ void write_item(const PrefixArgs& a, const State& st, unsigned char* slots, float (*ms)[32],
                                           float (*ls)[32], int part, Find find, Add add) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = lane & 31, h = lane >> 5;
  const float l = other_half_sum(st.l);
  __syncthreads();  // the slots' last reads and loads are done in every wave
  // O to LDS as rows of 512 bytes, chunk ch of row c at ch ^ c.
  unsigned char* mine = slots + wave * kSlot + c * 512;
  if (find(SPLIT ? c : wave * 32 + c).b >= 0) {
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int ch = 8 * db + 2 * q + h;
        *reinterpret_cast<f32x4_t*>(mine + ((ch ^ c) << 4)) =
            f32x4_t{st.o[db][4 * q], st.o[db][4 * q + 1], st.o[db][4 * q + 2], st.o[db][4 * q + 3]};
      }
    if (h == 0) {
      ms[wave][c] = st.m;
      ls[wave][c] = l;
    }
  }
  __syncthreads();
  constexpr int kLanes = SPLIT ? 2 * NW : 8;  // to a query row
  constexpr int kPasses = SPLIT ? 1 : 4;
  constexpr int kFrom = SPLIT ? NW : 1;
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    const int r = SPLIT ? tid / kLanes : pass * 8 + (lane >> 3);  // of the wave's 32
    const Query q = find(SPLIT ? r : wave * 32 + r);
    if (q.b < 0) continue;
    float w[kFrom], m = neg_inf(), sum = 0.f;
#pragma unroll
    for (int i = 0; i < kFrom; ++i) m = fmaxf(m, ms[SPLIT ? i : wave][r]);
#pragma unroll
    for (int i = 0; i < kFrom; ++i) {
      const float mi = ms[SPLIT ? i : wave][r];
      w[i] = mi == m ? 1.f : __builtin_amdgcn_exp2f(mi - m);
      sum += w[i] * ls[SPLIT ? i : wave][r];
    }
    const size_t row = ((size_t)q.b * a.T + q.t) * a.n_q + q.h;
    const size_t slot_row = (size_t)part * a.rows + row;
    // (no row at all: zero; rows that all score -inf: 0 / 0)
    const bool none = a.P == 0 && own_visible(a, q.b, q.t) == 0;
#pragma unroll
    for (int k = 0; k < 32 / kLanes; ++k) {
      const int ch = (lane & (kLanes - 1)) + kLanes * k;
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kFrom; ++i)
        o += w[i] * *reinterpret_cast<const f32x4_t*>(slots + (SPLIT ? i : wave) * kSlot + r * 512 + ((ch ^ r) << 4));
      add(q, 4 * ch, sum, o);
      if constexpr (DIRECT) {
        bf16x4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = static_cast<__bf16>(none ? 0.f : o[e] / sum);
        *reinterpret_cast<bf16x4_t*>(a.out + row * D + 4 * ch) = v;
      } else {
        *reinterpret_cast<f32x4_t*>(a.part_o + slot_row * D + 4 * ch) = o;
      }
    }
    if (!DIRECT && (lane & (kLanes - 1)) == 0) *reinterpret_cast<f32x2_t*>(a.part_ml + slot_row * 2) = f32x2_t{m, sum};
  }
}

// B operands of a wave's 32 query rows, the sign of the scale in them.
__device__ __forceinline__ void load_q(const PrefixArgs& a, const Query& q, bf16x8_t (&qf)[8]) {
  const int h = (threadIdx.x & 63) >> 5;
  const __bf16* at = a.q + (size_t)q.b * a.q_b + (size_t)q.h * a.q_h + (size_t)q.t * a.q_t + 8 * h;
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const unsigned flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    u32x4 w = *reinterpret_cast<const u32x4*>(at + 16 * ks);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] ^= flip;
    qf[ks] = __builtin_bit_cast(bf16x8_t, w);
  }
}

__device__ __forceinline__ State empty_state(float c2) {
  State st;
  st.m = neg_inf();
  st.l = 0.f;
  st.c2 = c2;
#pragma unroll
  for (int db = 0; db < 4; ++db) st.o[db] = f32x16_t{};
  return st;
}

// One request's query rows r0 .. r0 + 31 of kv head j over its own rows [begin, end),
// with JOINT over the prefix in front of them.
template <int NW, bool CAUSAL, bool JOINT>
__device__ __forceinline__ void own_item(const PrefixArgs& a, int j, int b, int r0, int begin, int end, int part,
                                         unsigned char* slots, float (*ms)[32], float (*ls)[32]) {
  const int c = threadIdx.x & 31;
  const int rows = a.T * a.G;
  auto find = [&](int i) __attribute__((always_inline)) {
    const int r = r0 + i;
    return r < rows ? Query{b, r / a.G, j * a.G + r % a.G} : Query{-1, 0, 0};
  };
  const Query mine = find(min(c, rows - 1 - r0));
  bf16x8_t qf[8];
  load_q(a, mine, qf);
  const int written = __builtin_amdgcn_readfirstlane(own_written(a, b));
  if (!JOINT && begin >= written) return;  // (the second launch knows this, too)
  const float c2 = fabsf(a.scale) * 1.44269504088896341f;
  State st = empty_state(c2);
  if (JOINT && a.P > 0) {
    const Rows src = {a.pk + (size_t)j * a.p_h, a.pv + (size_t)j * a.p_h, a.p_row, 0, a.P};
    attend_split<NW, false>(src, qf, c2, a.P, a.P, 0, slots, st);
  }
  // The rows that the item's first query row sees all of them see, and none is read
  // that its last one does not.
  const int least = max(written - (a.T - 1 - r0 / a.G), 0);
  const int stop = min(end, max(written - (a.T - 1 - min(r0 + 31, rows - 1) / a.G), 0));
  const size_t base = (size_t)b * a.k_b + (size_t)j * a.k_h;
  bool special = false;
  if (begin < stop) {
    const Rows src = {a.k + base, a.v + base, a.k_row, begin, stop};
    // (the waves that had one step less of the prefix come first)
    special = attend_split<NW, CAUSAL>(src, qf, c2, max(written - (a.T - 1 - mine.t), 0), least,
                                       JOINT ? (a.P + kStep - 1) / kStep : 0, slots, st);
  }
  if constexpr (CAUSAL) {
    // Infinite and NaN values of rows that only some query rows see: to those.
    const bool any = __syncthreads_or(special);
    int first = max(begin, least);
    asm("" : "+v"(first));  // (a vector register: scalar ones are short in the loops before)
    write_item<NW, true, JOINT>(a, st, slots, ms, ls, part, find,
                                [&](const Query& q, int d, float sum, f32x4_t& o) __attribute__((always_inline)) {
      if (!any) return;
      for (int i = first; i < min(stop, written - (a.T - 1 - q.t)); ++i) {
        const unsigned row = (unsigned)i * (unsigned)a.k_row;  // (a head's rows span less than 2^30 values)
        const bf16x4_t v = *reinterpret_cast<const bf16x4_t*>(a.v + base + (row + (unsigned)d));
        // 0, or NaN for what is not finite.  A row whose key is not finite scores -inf, and 0
        // times the value is NaN, too, or makes all of the query's output NaN.
        float key = 0.f;
#pragma unroll 1
        for (int e = 0; e < D; e += 4) {
          const bf16x4_t k = *reinterpret_cast<const bf16x4_t*>(a.k + base + (row + (unsigned)e));
#pragma unroll
          for (int u = 0; u < 4; ++u) key += static_cast<float>(k[u]) * 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = static_cast<float>(v[e]);
          if (!(fabsf(f) < __builtin_huge_valf())) o[e] += sum != 0.f ? f + key : f * 0.f;  // (of no weight: NaN)
        }
      }
    });
  } else {
    write_item<NW, true, JOINT>(a, st, slots, ms, ls, part, find, [](const Query&, int, float, f32x4_t&) {});
  }
}

// Query rows r0 .. r0 + (SHARED ? 127 : 31) of kv head j over prefix rows [begin, end).
template <bool SHARED>
__device__ __forceinline__ void prefix_item(const PrefixArgs& a, int j, int r0, int begin, int end, int part,
                                            unsigned char* slots, float (*ms)[32], float (*ls)[32]) {
  const int rows = a.B * a.T * a.G;
  auto find = [&](int i) __attribute__((always_inline)) {
    const int r = r0 + i;
    if (r >= rows) return Query{-1, 0, 0};
    const int bt = r / a.G;
    return Query{bt / a.T, bt % a.T, j * a.G + r % a.G};
  };
  const int i = (SHARED ? (threadIdx.x >> 6) * 32 : 0) + (threadIdx.x & 31);
  bf16x8_t qf[8];
  load_q(a, find(min(i, rows - 1 - r0)), qf);
  const float c2 = fabsf(a.scale) * 1.44269504088896341f;
  State st = empty_state(c2);
  const Rows src = {a.pk + (size_t)j * a.p_h, a.pv + (size_t)j * a.p_h, a.p_row, begin, end};
  if constexpr (SHARED)
    attend_shared(src, qf, c2, slots, st);
  else
    attend_split<kWaves, false>(src, qf, c2, end, end, 0, slots, st);
  write_item<kWaves, !SHARED, false>(a, st, slots, ms, ls, part, find, [](const Query&, int, float, f32x4_t&) {});
}

// Grid: prefix items (kv head fastest: with 8 of them each XCD's L2 holds one
// head's rows; then key ranges, then query rows), then own items (kv head,
// request, query rows, key ranges).
template <bool SHARED, bool CAUSAL>
__global__ __launch_bounds__(64 * kWaves, 2) void prefix_attention_kernel(PrefixArgs a) {
  __shared__ __align__(1024) unsigned char slots[kWaves * kSlot];
  __shared__ float ms[kWaves][32], ls[kWaves][32];
  int id = blockIdx.x;
  if (id < a.prefix_items) {
    const int j = id % a.n_kv;
    id /= a.n_kv;
    const int part = id % a.prefix_parts;
    const int tile = id / a.prefix_parts;
    const int begin = part * a.prefix_chunk;
    prefix_item<SHARED>(a, j, tile * (SHARED ? kPrefixSharedRows : 32), begin, min(begin + a.prefix_chunk, a.P), part,
                            slots, ms, ls);
    return;
  }
  id -= a.prefix_items;
  const int j = id % a.n_kv;
  id /= a.n_kv;
  const int b = id % a.B;
  id /= a.B;
  const int tile = id % a.own_tiles;
  const int part = id / a.own_tiles;
  const int begin = part * a.own_chunk;
  own_item<kWaves, CAUSAL, false>(a, j, b, tile * 32, begin, begin + a.own_chunk, a.prefix_parts + part, slots, ms, ls);
}

// Short contexts, one launch.  Grid: (kv head, request, query rows), the head fastest.
template <bool CAUSAL>
__global__ __launch_bounds__(64 * kJointWaves, 2) void joint_attention_kernel(PrefixArgs a) {
  __shared__ __align__(1024) unsigned char slots[kJointWaves * kSlot];
  __shared__ float ms[kJointWaves][32], ls[kJointWaves][32];
  int id = blockIdx.x;
  const int j = id % a.n_kv;
  id /= a.n_kv;
  const int b = id % a.B;
  own_item<kJointWaves, CAUSAL, true>(a, j, b, id / a.B * 32, 0, a.S, 0, slots, ms, ls);
}

// Adds a row's items up: kGroups times 32 lanes per row, 4 dims each, group g the items
// g, g + kGroups, .., kPartsAhead of them on their way at a time (past the last the last
// again, unused); then the groups, in their order.
constexpr int kCombineThreads = 256;
constexpr int kGroups = 4;
constexpr int kCombineRows = kCombineThreads / (32 * kGroups);
constexpr int kPartsAhead = 4;
__global__ __launch_bounds__(kCombineThreads) void combine_kernel(PrefixArgs a) {
  __shared__ float gm[kCombineRows][kGroups], gl[kCombineRows][kGroups];
  __shared__ f32x4_t go[kCombineRows][kGroups][32];
  const int g = (threadIdx.x >> 5) % kGroups, mine = threadIdx.x / (32 * kGroups), lane = threadIdx.x & 31;
  const size_t want = (size_t)blockIdx.x * kCombineRows + mine;
  const size_t row = want < (size_t)a.rows ? want : a.rows - 1;
  const int d = 4 * lane;
  const int bt = (int)(row / a.n_q);
  const int b = bt / a.T;
  const int parts = a.prefix_parts + (own_written(a, b) + a.own_chunk - 1) / a.own_chunk;
  float m = neg_inf(), l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  auto join = [&](float pm, float pl, f32x4_t po) __attribute__((always_inline)) {
    const float top = fmaxf(m, pm);
    const float was = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
    const float now = pm == top ? 1.f : __builtin_amdgcn_exp2f(pm - top);
    l = l * was + pl * now;
    o = o * was + po * now;
    m = top;
  };
  for (int first = g; first < parts; first += kGroups * kPartsAhead) {
    f32x2_t ml[kPartsAhead];
    f32x4_t v[kPartsAhead];
#pragma unroll
    for (int i = 0; i < kPartsAhead; ++i) {
      const size_t at = (size_t)min(first + i * kGroups, parts - 1) * a.rows + row;
      ml[i] = *reinterpret_cast<const f32x2_t*>(a.part_ml + at * 2);
      v[i] = *reinterpret_cast<const f32x4_t*>(a.part_o + at * D + d);
    }
#pragma unroll
    for (int i = 0; i < kPartsAhead; ++i)
      if (first + i * kGroups < parts) join(ml[i][0], ml[i][1], v[i]);
  }
  if (lane == 0) {
    gm[mine][g] = m;
    gl[mine][g] = l;
  }
  go[mine][g][lane] = o;
  __syncthreads();
  if (g != 0 || want >= (size_t)a.rows) return;
#pragma unroll
  for (int i = 1; i < kGroups; ++i) join(gm[mine][i], gl[mine][i], go[mine][i][lane]);
  const bool none = a.P == 0 && own_visible(a, b, bt % a.T) == 0;
  bf16x4_t v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = static_cast<__bf16>(none ? 0.f : o[e] / l);
  *reinterpret_cast<bf16x4_t*>(a.out + row * D + d) = v;
}

template <bool CAUSAL>
hipError_t launch(const PrefixArgs& a, const PrefixPlan& plan, hipStream_t stream) {
  const unsigned own = (unsigned)a.n_kv * a.B * a.own_tiles;
  if (plan.joint) {
    launch_kernel(joint_attention_kernel<CAUSAL>, dim3(own), dim3(64 * kJointWaves), 0, stream, a);
    return hipGetLastError();
  }
  const dim3 items((unsigned)a.prefix_items + own * plan.own_parts);
  if (plan.shared)
    launch_kernel(prefix_attention_kernel<true, CAUSAL>, items, dim3(64 * kWaves), 0, stream, a);
  else
    launch_kernel(prefix_attention_kernel<false, CAUSAL>, items, dim3(64 * kWaves), 0, stream, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  launch_kernel(combine_kernel, dim3((unsigned)((a.rows + kCombineRows - 1) / kCombineRows)), dim3(kCombineThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_prefix_attention(const PrefixArgs& a, const PrefixPlan& plan, hipStream_t stream) {
  return a.T > 1 ? launch<true>(a, plan, stream) : launch<false>(a, plan, stream);
}

}  // namespace lsk
