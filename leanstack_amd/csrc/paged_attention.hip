// Attention over the pages of an 8-bit cache for gfx950: T query tokens of each of B
// requests over the rows that the request has cached, its new ones the last of them
// (causal within them).
//
//   out = sum_i e^(s_i - m) v_i / sum_i e^(s_i - m),  s = scale q . k,
// k and v being e4m3 bytes times a power of two per 16 rows and head (paged_cache.hip
// has the format).
//
// An item is 16 or 32 query rows (T n_q / n_kv are few; up to 64 in one launch) or 128 of one
// request and kv head, over the rows that its last one sees.  How many those are only the device
// knows; every wave counts the items' units of key rows (lens is read once more by each).
// Few query rows: an item is cut into chunks of equal length, as many as let all the
// chunks run at once, one wave each.  Many: a kv head's items are laid end to end and
// its workgroups take equal shares of the line (the end of one item, whole items, the start
// of another), because an item more or less per CU would cost a whole round.  Whole items
// are written to the output, parts as (m, l, O) in fp32 to the workspace, and a second
// launch adds an item's parts up in their order.  A context that is short for certain runs
// in one launch, an item per workgroup.  (paged_plan in lsk_host.h has the rules.)
//
// Bound by: single tokens and a few, the cache's bytes (64 requests over 17..8001 rows, 527 MB: 88 us,
// 6.0 TB/s, and 4 for the second launch), where there is little to read the chain of lens,
// table, rows, sums and the second launch (1 request over 32768 rows 17 + 6 us); prompts, the
// chain of products, exponentials and conversions of two waves that share a SIMD (2 x 1500
// tokens, the last of 4000 and 7001 rows: 261 us, 897 TFLOP/s, and 13 for the parts' 110 MB).
//
// Few query rows (decode, verify).  A wave takes two blocks, 32 key rows, a step, for up to
// 4 x 16 query rows:
//   bytes to bf16 with their scale, two values an instruction, exact;
//   S = K Q^T on v_mfma_f32_16x16x32_bf16: a lane holds 2 x 4 scores of one query row;
//   the running maximum m and sum l of the softmax in base 2, in fp32, m raised only
//     where a step exceeds it by 2^8;
//   O^T += V^T P^T on the same instruction: the scores' lanes are those of its operand
//     if the 32 key rows are taken in the order in which the lanes hold them, and the
//     blocks of V lie in memory as the other operand's lanes take them.
// Nothing goes through LDS but the waves' sums at the end.
//
// Many query rows (prompts).  Four waves of 32 query rows share the key rows of a step (64)
// through a ring in LDS, filled by DMA.  K and V are converted on their way out of LDS, each wave for
// itself, for v_mfma_f32_32x32x16_bf16.  (K as it is stored, against q as the sum of two e4m3 numbers on
// v_mfma_scale_f32_32x32x64_f8f6f4, takes as long on the matrix units and saves the conversion: 239 us for the 264 of
// 2 x 1500 tokens over 4000 and 7001 rows.  But that instruction drops of eight products what is below 2^-13 of the largest, where
// the bf16 one keeps 24 bits: scores were off by hundredths beside a few large dims.)
//
// P: up to 16 query rows (single tokens) two bf16 numbers a weight, the second what the first leaves,
// 2^-16 of it at most; with more of them one, 2^-8 at most: a second product would be as long as the
// first.  l sums what is multiplied, so the result is exactly that of slightly other weights.

#include <hip/hip_runtime.h>

#include <type_traits>

#include "lsk_internal.h"

namespace lsk {
namespace {

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

constexpr int D = kAttnHeadDim;
constexpr int kFewWaves = 4, kShortWaves = 8;  // of a workgroup for few query rows
constexpr float kRaise = 8.f, kMostWeight = 256.f;  // in base 2
constexpr float kFar = 0x1p30f;
constexpr int kJoinThreads = 256, kJoinWide = 1024;
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ float neg_inf() { return -__builtin_huge_valf(); }

__device__ __forceinline__ float power_of_two(int n) {
  return n < -126 ? 0.f : __builtin_bit_cast(float, (unsigned)(n + 127) << 23);
}

// Four bytes times a power of two.
__device__ __forceinline__ bf16x4_t four(unsigned w, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
  return bf16x4_t{a[0], a[1], b[0], b[1]};
}
__device__ __forceinline__ bf16x8_t eight(unsigned w0, unsigned w1, float scale0, float scale1) {
  return __builtin_shufflevector(four(w0, scale0), four(w1, scale1), 0, 1, 2, 3, 4, 5, 6, 7);
}

// Bytes of a word that are NaN, as 0xff each.
__device__ __forceinline__ unsigned nan_bytes(unsigned w) {
  const unsigned t = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  return (t >> 7) * 0xffu;
}
// ... as ones (e4m3 0x38).
__device__ __forceinline__ unsigned nan_ones(unsigned w) { return nan_bytes(w) & 0x38383838u; }

// What a request has, and what its query token t sees (those behind the last real one: as
// many rows as that).
struct Request {
  int len, count, most;
  __device__ __forceinline__ int visible(int t) const { return min(max(len - max(count - 1 - t, 0), 0), most); }
};
__device__ __forceinline__ Request request_of(const PagedAttentionArgs& a, int b) {
  return {max(a.lens[b], 0), a.counts ? min(max(a.counts[b], 0), a.T) : a.T, 16 * a.pool.blocks};
}

// An item's request.  Up to 64 query rows are one item (paged_plan).
template <bool MANY>
__device__ __forceinline__ int request_at(const PagedAttentionArgs& a, int item) {
  return !MANY || a.tiles == 1 ? item : item / a.tiles;
}
// The rows that the last query row of a tile of a request sees.
template <bool MANY>
__device__ __forceinline__ int item_rows(const PagedAttentionArgs& a, const Request& q, int tile) {
  if (!MANY || a.tiles == 1) return q.count > 0 ? q.visible(a.T - 1) : 0;
  const int r0 = tile * kPagedManyRows;
  if (q.count <= r0 / a.G) return 0;
  return q.visible((min(r0 + kPagedManyRows, a.T * a.G) - 1) / a.G);
}
template <bool MANY>
__device__ __forceinline__ int item_units(const PagedAttentionArgs& a, int item) {
  constexpr int kUnit = MANY ? kPagedManyUnit : kPagedFewUnit;
  const int b = request_at<MANY>(a, item);
  return max((item_rows<MANY>(a, request_of(a, b), MANY ? item - b * a.tiles : 0) + kUnit - 1) / kUnit, 1);
}

// Inclusive sums over a wave's lanes.
__device__ __forceinline__ int wave_sums(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int o = __shfl_up(v, s);
    if (lane >= s) v += o;
  }
  return v;
}

// The items in 64 runs, one per lane: each(i) adds up over a lane's.
template <typename Each>
__device__ __forceinline__ int lane_items(const PagedAttentionArgs& a, Each each) {
  const int lane = threadIdx.x & 63, n = (a.items + 63) / 64;
  const int i0 = min(lane * n, a.items), i1 = min(i0 + n, a.items);
  int sum = 0;
  for (int i = i0; i < i1; ++i) sum += each(i);
  return sum;
}

// The item at `place` of a line on which each(i) places are item i's, and the place where
// that one begins; mine, before: the lane's items' places, and those in front of them.
struct Found {
  int item, begin;
};
template <typename Each>
__device__ __forceinline__ Found item_at(const PagedAttentionArgs& a, int place, int mine, int before, Each each) {
  const int lane = threadIdx.x & 63, n = (a.items + 63) / 64;
  const int i1 = min((lane + 1) * n, a.items);
  // the last lane whose items do not begin behind it
  const int from = 63 - __builtin_clzll(__ballot(mine > 0 && before <= place));
  int i = min(lane * n, a.items), at = before;
  for (; i < i1 - 1; ++i) {
    const int here = each(i);
    if (place < at + here) break;
    at += here;
  }
  return {__builtin_amdgcn_readlane(i, from), __builtin_amdgcn_readlane(at, from)};
}

// Where the items begin, for the second launch.
template <typename Each>
__device__ __forceinline__ void write_begins(const PagedAttentionArgs& a, int before, int total, Each each) {
  const int lane = threadIdx.x & 63, n = (a.items + 63) / 64;
  const int i1 = min((lane + 1) * n, a.items);
  for (int i = min(lane * n, a.items), at = before; i < i1; ++i) {
    a.begins[i] = at;
    at += each(i);
  }
  if (lane == 0) a.begins[a.items] = total;
}

// Worker w's chunk: units [first, last) of an item (none: first = last).
struct Chunk {
  int item, first, last;
  bool whole;
};
__device__ __forceinline__ Chunk chunk_of(const PagedAttentionArgs& a, int w, bool write) {
  auto units_of = [&](int i) { return item_units<false>(a, i); };
  const int total = __builtin_amdgcn_readlane(wave_sums(lane_items(a, units_of)), 63);
  const int most = max((total + a.places - 1) / a.places, a.least_units);  // units of a chunk
  auto chunks_of = [&](int i) { return (item_units<false>(a, i) + most - 1) / most; };
  const int mine = lane_items(a, chunks_of), up_to = wave_sums(mine);
  const int chunks = __builtin_amdgcn_readlane(up_to, 63);
  if (write) write_begins(a, up_to - mine, chunks, chunks_of);
  if (w >= chunks) return {0, 0, 0, false};
  const Found f = item_at(a, w, mine, up_to - mine, chunks_of);
  const int units = item_units<false>(a, f.item), n = (units + most - 1) / most;
  const int each = (units + n - 1) / n;  // (at most `most`: none of the n is empty)
  const int first = (w - f.begin) * each;
  return {f.item, first, min(first + each, units), n == 1};
}

// Where worker w's share of the line begins.
__device__ __forceinline__ int share_begin(long long units, int w, int workers) { return (int)(units * w / workers); }

// The item in which worker w's share begins, the places of it in front of the share, and the
// share's length.  An item's places: kPagedManyStart for its beginning and its end, then its units.
// cuts: whether it is the first share to begin behind the item's first unit.
struct Share {
  int item, skip, places;
  bool cuts;
};
__device__ __forceinline__ Share share_of(const PagedAttentionArgs& a, int w, bool write) {
  auto places_of = [&](int i) { return item_units<true>(a, i) + kPagedManyStart; };
  const int mine = lane_items(a, places_of), up_to = wave_sums(mine);
  const int total = __builtin_amdgcn_readlane(up_to, 63);
  if (write) write_begins(a, up_to - mine, total, places_of);
  const int begin = share_begin(total, w, a.workers);
  const Found f = item_at(a, begin, mine, up_to - mine, places_of);
  const int unit0 = f.begin + kPagedManyStart;
  return {f.item, begin - f.begin, share_begin(total, w + 1, a.workers) - begin,
          begin > unit0 && share_begin(total, w - 1, a.workers) <= unit0};
}

struct Part {
  float* o;   // [rows][D]
  float* ml;  // [rows][2]
};
__device__ __forceinline__ Part part_of(const PagedAttentionArgs& a, size_t slot) {
  return {a.part_o + slot * a.slot_rows * D, a.part_ml + slot * a.slot_rows * 2};
}

// The weights of V and the running sums.
//
// Exponents are s c2 - m with one rounding, m being the rounded top c2: far from zero
// (kFar) its rounding error would be more than 2^x holds.  There scores that are not
// equal are 2^6 and more apart in base 2, so any factor gives the same weights, if m's
// order stays: the next power of two above c2, whose products are exact.
// m starts at the lowest finite number, so that scores of -inf have no weight; whether any row
// was seen is known apart.
struct Sums {
  float m, l, c2;
};
__device__ __forceinline__ Sums no_sums(float c2) { return {kLowest, 0.f, c2}; }

// Raises m to the row's maximum `top` and returns what the sums so far are multiplied by.
__device__ __forceinline__ float raised(Sums& st, float top, float c2) {
  const bool raise = top * st.c2 > st.m + kRaise;
  const float above = __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, c2) + 0x007fffffu) & 0x7f800000u);
  st.c2 = !raise ? st.c2 : fabsf(top * c2) < kFar ? c2 : above;
  const float mx = top * st.c2;
  const float f = raise ? __builtin_amdgcn_exp2f(st.m - mx) : 1.f;
  st.m = raise ? mx : st.m;
  st.l *= f;
  return f;
}

// What brings scores to base 2, and what is done to q's bits: a negative scale's sign goes
// into q, and a scale of zero leaves zeros (an unseen row's score of -inf has to
// meet a factor above zero), infinities and NaN of q aside.
struct Scale {
  float c2;
  unsigned flip;
  bool zero;
};
__device__ __forceinline__ Scale scale_of(float scale) {
  const bool zero = scale == 0.f;
  return {zero ? 1.f : fabsf(scale) * 1.44269504088896341f, scale < 0.f ? 0x80008000u : 0u, zero};
}
__device__ __forceinline__ unsigned scaled_bits(unsigned w, const Scale& sc) {
  w ^= sc.flip;
  if (sc.zero) {
    const bool low = (w & 0x7f80u) == 0x7f80u, high = (w & 0x7f800000u) == 0x7f800000u;
    w &= (low ? 0xffffu : 0u) | (high ? 0xffff0000u : 0u);
  }
  return w;
}

// ------------------------------------------------------------------ few query rows

// The four lanes that hold a query row's scores: c, c + 16, c + 32, c + 48.
__device__ __forceinline__ float rows_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float rows_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// A wave's state for 16 query rows: lane (c, g) holds row c, of O the dims 16 i + 4 g .. + 3,
// of l the share of the lane's scores.
struct State {
  Sums sums;
  f32x4_t o[8];
};

// 1 KB of a block, 16 bytes a lane; zeros and no access where there is none.  Past the caches
// (nt): a block is read once, by the four waves of a workgroup by turns (64 requests over 17..8001 rows:
// 105 us for 116).
constexpr int kStream = 2;
__device__ __forceinline__ u32x4_t load_1k(const unsigned char* blocks, int at, int half) {
  const __amdgpu_buffer_rsrc_t block = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(blocks) + (size_t)(at < 0 ? 0 : at) * kPagedBlockBytes, (short)0,
      at < 0 ? 0 : kPagedBlockBytes, 0x00020000);
  return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(block, (threadIdx.x & 63) * 16, half * 1024, kStream));
}

// The weights P of a step as operands of the second product, and m, l, O brought to
// the new maximum.  s[m][i]: row 16 m + 4 g + i of the step, -inf where it is not seen.
struct Weights {
  bf16x8_t high, low;  // low: what high leaves of them
};
template <bool FINE>
__device__ __forceinline__ Weights step_weights(const f32x4_t (&s)[2], float c2, State& st) {
  float top = fmaxf(s[0][0], s[0][1]);
#pragma unroll
  for (int i = 2; i < 8; ++i) top = fmaxf(top, s[i / 4][i % 4]);
  if (__ballot(top * st.sums.c2 > st.sums.m + kRaise)) {
    const float f = raised(st.sums, rows_max(top), c2);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[i][e] *= f;
  }
  Weights p;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4], st.sums.c2, -st.sums.m));
    p.high[i] = static_cast<__bf16>(w);
    if constexpr (FINE) p.low[i] = static_cast<__bf16>(w - static_cast<float>(p.high[i]));
  }
  const bf16x2_t ones = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    st.sums.l = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{p.high[i], p.high[i + 1]}, ones, st.sums.l, false);
    if constexpr (FINE) st.sums.l = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{p.low[i], p.low[i + 1]}, ones, st.sums.l, false);
  }
  return p;
}

// What the wave's lane l knows of block 2 (first + NW (l / 2)) + l % 2: its place in the pool
// (-1: no row of it is read) and its scales.
struct Blocks {
  int at;
  float ks, vs;
};
template <int NW>
__device__ __forceinline__ Blocks blocks_from(const PagedPool& p, int b, int j, int first, int end) {
  const int lane = threadIdx.x & 63;
  const int block = 2 * (first + NW * (lane >> 1)) + (lane & 1);
  Blocks r = {-1, 1.f, 1.f};
  if (block < end) {
    const int page = p.table[(size_t)b * p.table_ld + (block >> p.page_shift)];
    if ((unsigned)page < (unsigned)p.pages) {
      r.at = ((page * p.n_kv + j) << p.page_shift) | (block & ((1 << p.page_shift) - 1));  // (a pool has fewer than 2^31)
      r.ks = power_of_two((int)p.k_exp[r.at] - 127);
      r.vs = power_of_two((int)p.v_exp[r.at] - 127);
    }
  }
  return r;
}

// threadIdx.x, anew: what is made of it is not kept in registers from one item to the next.
__device__ __forceinline__ int own_thread() {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid;
}

// The weights as two bf16 numbers, not one.  The second product of 16 query rows runs while the next rows are on their
// way: 1 request over 900 rows 10.0 us for 9.5, 64 over 17..8001 95 for 94; of 32 rows it would not (24 x 5 tokens over
// 5..3001 rows 29.5 us for 27.3, 8 x 8 over 8192 38.8 for 36.3).
template <int NT>
constexpr bool kFine = NT == 1;

// Query rows of more than one tile are kept in LDS (16 registers each).
template <int NT>
constexpr bool kQueriesInLds = NT > 1;
template <int NT>
struct Queries {
  u32x4_t q[kQueriesInLds<NT> ? NT : 1][4][64];
};

// A wave's steps first_step + i NW (up to stop_step), i = 0, 1, .., for the query rows of
// kv head j of request b.  any[n]: whether the lane has met a row that its query row sees.
template <int NT, int NW>
__device__ __forceinline__ void few_steps(const PagedAttentionArgs& a, Queries<NT>& lds, int j, int b, int first_step, int stop_step,
                                          const Request& rq, State (&st)[NT], bool (&any)[NT]) {
  constexpr bool kInLds = kQueriesInLds<NT>;
  constexpr int kAhead = NT > 2 ? 1 : 2;  // steps on their way
  const PagedPool& p = a.pool;
  const int lane = own_thread() & 63, c = lane & 15, g = lane >> 4;
  const int rows = a.T * a.G;
  const int least = rq.count > 0 ? rq.visible(0) : 0;
  const int end_block = (item_rows<false>(a, rq, 0) + 15) / 16, stop = min(stop_step, (end_block + 1) / 2);
  // 32 steps' blocks in the lanes at a time; the first steps' rows are on their way before anything else.
  Blocks blocks;
  int here = 0;
  struct Held {
    u32x4_t k[2][2], v[2][2];
  } held[kAhead];
  auto load_k = [&](int i, u32x4_t (&kq)[2][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int at = i < here ? __builtin_amdgcn_readlane(blocks.at, 2 * i + m) : -1;
#pragma unroll
      for (int h = 0; h < 2; ++h) kq[m][h] = load_1k(p.k, at, h);
    }
  };
  auto load_v = [&](int i, u32x4_t (&vq)[2][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int at = i < here ? __builtin_amdgcn_readlane(blocks.at, 2 * i + m) : -1;
#pragma unroll
      for (int h = 0; h < 2; ++h) vq[m][h] = load_1k(p.v, at, h);
    }
  };
  auto begin_group = [&](int first) __attribute__((always_inline)) {
    blocks = blocks_from<NW>(p, b, j, first, end_block);
    here = min(32, (stop - first + NW - 1) / NW);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      load_k(i, held[i].k);
      load_v(i, held[i].v);
    }
  };
  begin_group(first_step);

  const Scale sc = scale_of(a.scale);
  bf16x8_t q[kInLds ? 1 : NT][4];
  int limit[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    any[n] = false;
    const int r = min(16 * n + c, rows - 1);
    const int t = r / a.G, h = j * a.G + r % a.G;
    limit[n] = rq.visible(t);
    st[n].sums = no_sums(sc.c2);
#pragma unroll
    for (int i = 0; i < 8; ++i) st[n].o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const __bf16* from = a.q + (size_t)b * a.q_b + (size_t)h * a.q_h + (size_t)t * a.q_t + 16 * g;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u32x4_t w = *reinterpret_cast<const u32x4_t*>(from + 64 * (k >> 1) + 8 * (k & 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = scaled_bits(w[e], sc);
      if constexpr (kInLds)
        lds.q[n][k][lane] = w;  // (a wave's own)
      else
        q[n][k] = __builtin_bit_cast(bf16x8_t, w);
    }
  }
  if constexpr (kInLds) wave_lds_order();

  for (int first = first_step; first < stop; first += 32 * NW) {
    if (first != first_step) begin_group(first);
    auto step = [&](int i, Held& hold) __attribute__((always_inline)) {
      u32x4_t (&kq)[2][2] = hold.k;
      u32x4_t (&vq)[2][2] = hold.v;
      const int row0 = 32 * (first + NW * i);
      int at[2];
      float ks[2], vs[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        at[m] = __builtin_amdgcn_readlane(blocks.at, 2 * i + m);
        ks[m] = row_lane(blocks.ks, 2 * i + m);
        vs[m] = row_lane(blocks.vs, 2 * i + m);
      }
      f32x4_t s[NT][2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        bf16x8_t key[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) key[m] = eight(kq[m][k >> 1][2 * (k & 1)], kq[m][k >> 1][2 * (k & 1) + 1], ks[m], ks[m]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          bf16x8_t query;
          if constexpr (kInLds)
            query = __builtin_bit_cast(bf16x8_t, lds.q[n][k][lane]);
          else
            query = q[n][k];
#pragma unroll
          for (int m = 0; m < 2; ++m)
            s[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key[m], query, k ? s[n][m] : f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
        }
      }
      load_k(i + kAhead, kq);  // on its way while this step's weights and second product run
      const bool masked = row0 + 32 > least || at[0] < 0 || at[1] < 0;
      auto seen = [&](int n, int i) { return row0 + 16 * (i / 4) + 4 * g + i % 4 < limit[n] && at[i / 4] >= 0; };
      if (masked) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool ok = seen(n, i);
            any[n] |= ok;
            s[n][i / 4][i % 4] = ok ? s[n][i / 4][i % 4] : neg_inf();
          }
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n) any[n] = true;
      }
      Weights w[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) w[n] = step_weights<kFine<NT>>(s[n], sc.c2, st[n]);
      if (masked) {
        // A weight of zero does not take a NaN out of a product: those become zero here and
        // come back for the query rows that see them.
        unsigned found = 0;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) found |= nan_bytes(vq[m][h][e]);
        if (__ballot(found != 0)) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            bf16x8_t sees;
#pragma unroll
            for (int e = 0; e < 8; ++e) sees[e] = static_cast<__bf16>(seen(n, e) ? 1.f : 0.f);
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              const bf16x8_t nans = eight(nan_ones(vq[0][d & 1][d >> 1]), nan_ones(vq[1][d & 1][d >> 1]), 1.f, 1.f);
              const f32x4_t met =
                  __builtin_amdgcn_mfma_f32_16x16x32_bf16(nans, sees, f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (met[e] > 0.f) st[n].o[d][e] = __builtin_nanf("");
              __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers)
            }
          }
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 4; ++e) vq[m][h][e] &= ~nan_bytes(vq[m][h][e]);
        }
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const bf16x8_t value = eight(vq[0][d & 1][d >> 1], vq[1][d & 1][d >> 1], vs[0], vs[1]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (kFine<NT>) st[n].o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value, w[n].low, st[n].o[d], 0, 0, 0);
          st[n].o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value, w[n].high, st[n].o[d], 0, 0, 0);
        }
      }
      load_v(i + kAhead, vq);
    };
    for (int i = 0; i < here; i += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (u == 0 || i + u < here) step(i + u, held[u]);
    }
  }

}

// Whether one of the row's four lanes has met a row; all lanes of the wave ask.
__device__ __forceinline__ bool met_any(bool any, int c) { return (__ballot(any) >> c & 0x0001000100010001ull) != 0; }

// Grid: kv head (fastest), four of its workers: a wave each.
template <int NT>
__global__ __launch_bounds__(64 * kFewWaves, 2) void few_attention_kernel(PagedAttentionArgs a) {
  __shared__ Queries<NT> queries[kFewWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = blockIdx.x % a.pool.n_kv, w = (blockIdx.x / a.pool.n_kv) * kFewWaves + wave;
  if (w >= a.workers) return;
  const Chunk ch = chunk_of(a, w, j == 0 && w == 0);
  if (ch.first == ch.last) return;
  const int b = ch.item;
  State st[NT];
  bool any[NT];
  const Request rq = request_of(a, b);
  few_steps<NT, 1>(a, queries[wave], j, b, ch.first, ch.last, rq, st, any);
  const int lane = own_thread() & 63, c = lane & 15, g = lane >> 4;
  const Part part = part_of(a, (size_t)j * a.workers + w);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = 16 * n + c;
    const float l = rows_sum(st[n].sums.l);
    const bool met = met_any(any[n], c);
    if (row >= a.T * a.G) continue;
    if (ch.whole) {
      const int t = row / a.G, h = j * a.G + row % a.G;
      const bool none = t >= rq.count || !met;
      const float share = none ? 0.f : 1.f / l;  // (of a sum of 0: infinite, and 0 times that NaN)
      __bf16* out = a.out + (((size_t)b * a.T + t) * a.n_q + h) * D + 4 * g;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        bf16x4_t o;
#pragma unroll
        for (int u = 0; u < 4; ++u) o[u] = static_cast<__bf16>(none ? 0.f : st[n].o[d][u] * share);
        *reinterpret_cast<bf16x4_t*>(out + 16 * d) = o;
      }
    } else {
      float* out = part.o + (size_t)row * D + 4 * g;
#pragma unroll
      for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4_t*>(out + 16 * d) = st[n].o[d];
      if (g == 0) *reinterpret_cast<f32x2_t*>(part.ml + row * 2) = f32x2_t{met ? st[n].sums.m : neg_inf(), l};
    }
  }
}

// One launch, an item per workgroup whose waves take its steps by turns.  Grid: kv head (fastest), request.
template <int NT>
__global__ __launch_bounds__(64 * kShortWaves, 2) void short_attention_kernel(PagedAttentionArgs a) {
  constexpr int NW = kShortWaves;
  __shared__ union {
    Queries<NT> queries[NW];
    float os[NW][16][D + 4];
  } sh;
  __shared__ float ms[NW][16], ls[NW][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = blockIdx.x % a.pool.n_kv, b = blockIdx.x / a.pool.n_kv;
  State st[NT];
  bool any[NT];
  const Request rq = request_of(a, b);
  few_steps<NT, NW>(a, sh.queries[wave], j, b, wave, 1 << 26, rq, st, any);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    __syncthreads();  // the queries, or the last tile's sums, have been read
    const int tid = own_thread();
    const float l = rows_sum(st[n].sums.l);
    {
      const int c = tid & 15, g = tid >> 4 & 3;
#pragma unroll
      for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4_t*>(&sh.os[wave][c][16 * d + 4 * g]) = st[n].o[d];
      const bool met = met_any(any[n], c);
      if (g == 0) {
        ms[wave][c] = met ? st[n].sums.m : neg_inf();
        ls[wave][c] = l;
      }
    }
    __syncthreads();
    // 32 lanes to a query row, 4 dims each
    static_assert(NW * 64 == 16 * 32, "lanes to a query row");
    const int r = tid >> 5, d0 = (tid & 31) * 4;
    const int row = n * 16 + r;
    if (row < a.T * a.G) {
      const int t = row / a.G, h = j * a.G + row % a.G;
      float m = neg_inf(), sum = 0.f, w[NW];
#pragma unroll
      for (int i = 0; i < NW; ++i) m = fmaxf(m, ms[i][r]);
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        w[i] = ms[i][r] == m ? 1.f : __builtin_amdgcn_exp2f(ms[i][r] - m);
        sum += w[i] * ls[i][r];
      }
      const bool none = t >= rq.count || m == neg_inf();
      const float share = none ? 0.f : 1.f / sum;
      f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NW; ++i) x += w[i] * *reinterpret_cast<const f32x4_t*>(&sh.os[i][r][d0]);
      bf16x4_t o;
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = static_cast<__bf16>(none ? 0.f : x[u] * share);
      *reinterpret_cast<bf16x4_t*>(a.out + (((size_t)b * a.T + t) * a.n_q + h) * D + d0) = o;
    }
  }
}

// Adds up the parts of items that were cut.  Grid: kv head (fastest), item (MANY and more items than
// workers: worker, whose share may be the first to begin inside one), `1 << a.join_shift` query rows of it; 16 threads take 8 dims each of a part's row, and the rest of the workgroup other rows
// or, with few rows, further parts: stream s the parts s, s + streams, ..
template <bool MANY, int THREADS, int PASSES>
__global__ __launch_bounds__(THREADS) void join_kernel(PagedAttentionArgs a, int rows) {
  constexpr int kSlots = THREADS / 16;
  __shared__ __align__(16) float os[kSlots][D];
  __shared__ float ms[kSlots], ls[kSlots];
  int id = blockIdx.x;
  const int j = id % a.pool.n_kv;
  id /= a.pool.n_kv;
  const int own = 1 << a.join_shift, streams = kSlots >> a.join_shift;  // rows at a time; and of each
  const int groups = (min(rows, a.T * a.G) + own * PASSES - 1) / (own * PASSES);
  const int nth = id / groups, group = id - nth * groups, item = MANY && a.items > a.workers ? a.cuts[nth] : nth;
  if (item < 0) return;
  const int begin = a.begins[item], end = a.begins[item + 1];
  // parts `from` .. `last`: a slot per chunk, or the second slot of the worker that has the first unit
  // and the first slots of those up to the last unit's
  int from = begin, last = end - 1;
  const int places = MANY ? a.begins[a.items] : 0;
  if constexpr (MANY) {
    auto worker_of = [&](int place) {
      int w = (int)((long long)place * a.workers / places);
      while (share_begin(places, w + 1, a.workers) <= place) ++w;
      while (share_begin(places, w, a.workers) > place) --w;
      return w;
    };
    from = worker_of(begin + kPagedManyStart), last = worker_of(end - 1);
  }
  if (from == last) return;
  const int b = request_at<MANY>(a, item), tile = MANY ? item - b * a.tiles : 0;
  const int slot = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * 8;
  const int stream = slot >> a.join_shift;
  const int r0 = group * own * PASSES + (slot & (own - 1)), end_row = min(rows, a.T * a.G - tile * rows);
  float m[PASSES], l[PASSES];
  f32x4_t o[PASSES][2];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) m[p] = neg_inf(), l[p] = 0.f, o[p][0] = o[p][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // kJoinAhead parts of each row on their way at a time (past the last the last again, unused)
  constexpr int kJoinAhead = PASSES > 1 ? 2 : 4;
  for (int w0 = from + stream; w0 <= last; w0 += kJoinAhead * streams) {
    f32x2_t ml[kJoinAhead][PASSES];
    f32x4_t x[kJoinAhead][PASSES][2];
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i) {
      const int w = min(w0 + i * streams, last);
      const size_t at = (size_t)j * a.workers + w;
      const Part part = part_of(a, MANY ? at * 2 + (w == from ? 1 : 0) : at);
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int r = min(r0 + p * own, end_row - 1);
        ml[i][p] = *reinterpret_cast<const f32x2_t*>(part.ml + r * 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) x[i][p][e] = *reinterpret_cast<const f32x4_t*>(part.o + (size_t)r * D + d0 + 4 * e);
      }
    }
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i) {
      const int w = w0 + i * streams;
      if (w > last) break;
      if (MANY && share_begin(places, w, a.workers) == share_begin(places, w + 1, a.workers))
        continue;  // (fewer places than workers: one without a share)
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const float top = fmaxf(m[p], ml[i][p][0]);
        const float was = m[p] == top ? 1.f : __builtin_amdgcn_exp2f(m[p] - top);
        const float now = ml[i][p][0] == top ? 1.f : __builtin_amdgcn_exp2f(ml[i][p][0] - top);
        l[p] = l[p] * was + ml[i][p][1] * now;
#pragma unroll
        for (int e = 0; e < 2; ++e) o[p][e] = o[p][e] * was + x[i][p][e] * now;
        m[p] = top;
      }
    }
  }
  auto place = [&](int of) {
    const int t = of / a.G, h = j * a.G + of % a.G;
    return a.out + (((size_t)b * a.T + t) * a.n_q + h) * D;
  };
  const int count = request_of(a, b).count;
  if (PASSES > 1 || streams == 1) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int r = r0 + p * own, row = tile * rows + r;
      if (r >= end_row) break;
      const bool none = row / a.G >= count || m[p] == neg_inf();
      const float share = none ? 0.f : 1.f / l[p];
      bf16x8_t x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = static_cast<__bf16>(none ? 0.f : o[p][e / 4][e % 4] * share);
      *reinterpret_cast<bf16x8_t*>(place(row) + d0) = x;
    }
    return;
  }
  // The streams' sums in their order: a thread per row and dim.
#pragma unroll
  for (int e = 0; e < 2; ++e) *reinterpret_cast<f32x4_t*>(&os[slot][d0 + 4 * e]) = o[0][e];
  if (d0 == 0) ms[slot] = m[0], ls[slot] = l[0];
  __syncthreads();
  for (int i = threadIdx.x; i < own * D; i += THREADS) {
    const int mine = i / D, d = i % D, to = tile * rows + group * own + mine;
    if (group * own + mine >= end_row) continue;
    float most = ms[mine];
    for (int s = 1; s < streams; ++s) most = fmaxf(most, ms[s * own + mine]);
    float sum = 0.f, x = 0.f;
    for (int s = 0; s < streams; ++s) {
      const float part = ms[s * own + mine];
      const float weight = part == most ? 1.f : __builtin_amdgcn_exp2f(part - most);
      sum += ls[s * own + mine] * weight;
      x += os[s * own + mine][d] * weight;
    }
    const bool none = to / a.G >= count || most == neg_inf();
    place(to)[d] = static_cast<__bf16>(none ? 0.f : x * (1.f / sum));
  }
}

// ------------------------------------------------------------------ many query rows

constexpr int kManyWaves = 4;
constexpr int kManyRows = 32 * kManyWaves;
constexpr int kStep = 64;                           // key rows, one block per wave
constexpr int kRing = 4;
constexpr int kSlot = 2 * 4 * kPagedBlockBytes;     // K, then V, of a step
static_assert(kManyRows == kPagedManyRows && kStep == kPagedManyUnit, "as the host counts them");

// Both halves' values of a lane pair 32 apart, in both lanes.  (The compiler takes
// a swap of a value with itself for two equal results: it is given a copy that it
// does not know to be one.)
__device__ __forceinline__ f32x2_t both_halves(float v) {
  const unsigned a = __builtin_bit_cast(unsigned, v);
  unsigned b = a;
  asm("" : "+v"(b));
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  return f32x2_t{__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1])};
}

struct ManyShared {
  unsigned char ring[kRing * kSlot];
};

typedef __attribute__((address_space(3))) const unsigned char lds_byte_t;
__device__ __forceinline__ u32x4_t lds_16(lds_byte_t* at) {
  return *reinterpret_cast<__attribute__((address_space(3))) const u32x4_t*>(at);
}

// A lane's half of a query row: values 64 k + 32 h + 8 i .. + 7.
struct Query {
  bf16x8_t q[2][4];
};

// 32 key rows of K, blocks 2 m and 2 m + 1 of a slot, as the lanes multiply them.
struct Keys {
  unsigned k[2][8];  // dims 64 k + 32 h + 4 i .. + 3
};
__device__ __forceinline__ Keys many_keys(lds_byte_t* slot, int m) {
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  lds_byte_t* at = slot + (2 * m + (c >> 4)) * kPagedBlockBytes + (32 * h + (c & 15)) * 16;
  Keys keys;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const u32x4_t lo = lds_16(at + k * 1024), hi = lds_16(at + k * 1024 + 256);
#pragma unroll
    for (int i = 0; i < 4; ++i) keys.k[k][i] = lo[i], keys.k[k][4 + i] = hi[i];
  }
  return keys;
}

// S^T of 32 key rows: lane (h, c) holds query row c, key rows 8 (i / 4) + 4 h + i % 4.  scale:
// exponent byte of the block that key row c is in.
__device__ __forceinline__ f32x16_t many_scores(const Keys& keys, const Query& query, int scale) {
  const float ks = power_of_two(scale - 127);
  f32x16_t s = {};
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(eight(keys.k[k][2 * i], keys.k[k][2 * i + 1], ks, ks), query.q[k][i], s, 0, 0, 0);
  return s;
}

struct ManyState {
  Sums sums;
  f32x16_t o[4];  // dims 32 d + 8 (i / 4) + 4 h + i % 4 of query row c
};

// The weights of 32 key rows, p[u] those of the u-th block, and their sum.
__device__ __forceinline__ float many_weights(const f32x16_t& s, const Sums& sums, bf16x8_t (&p)[2]) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    p[i / 8][i % 8] = static_cast<__bf16>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sums.c2, -sums.m)));
  const bf16x2_t ones = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2)
    sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{p[i / 8][i % 8], p[i / 8][i % 8 + 1]}, ones, sum, false);
  return sum;
}

// V of block `block` of a slot: dims 32 d .. of lane c, rows 4 h .. + 3 and 8 + 4 h .. + 3.
struct Values {
  u32x4_t lo, hi;
};
__device__ __forceinline__ Values many_values(lds_byte_t* slot, int block) {
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  lds_byte_t* at = slot + (4 + block) * kPagedBlockBytes + (c >> 4) * 1024 + (16 * h + (c & 15)) * 16;
  return {lds_16(at), lds_16(at + 512)};
}

// NaN of rows that some query row does not see: to those that do (as for few query rows).
// sees(e): whether the lane's query row sees the e-th of its eight.
template <typename Sees>
__device__ __forceinline__ void many_nans(Values& v, Sees sees, ManyState& st) {
  unsigned found = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) found |= nan_bytes(v.lo[e]) | nan_bytes(v.hi[e]);
  if (__ballot(found != 0) == 0) return;
  bf16x8_t one;
#pragma unroll
  for (int e = 0; e < 8; ++e) one[e] = static_cast<__bf16>(sees(e) ? 1.f : 0.f);
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const f32x16_t met =
        __builtin_amdgcn_mfma_f32_32x32x16_bf16(eight(nan_ones(v.lo[d]), nan_ones(v.hi[d]), 1.f, 1.f), one, f32x16_t{}, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (met[i] > 0.f) st.o[d][i] = __builtin_nanf("");
    v.lo[d] &= ~nan_bytes(v.lo[d]);
    v.hi[d] &= ~nan_bytes(v.hi[d]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Lane l: block `first` + l of the item (-1: none of its rows is read) and its exponent bytes.
struct ManyBlocks {
  int at, ke, ve;
};
__device__ __forceinline__ ManyBlocks many_blocks(const PagedPool& p, int b, int j, int first, int end) {
  const int block = first + (threadIdx.x & 63);
  ManyBlocks r = {-1, 127, 127};
  if (block < end) {
    const int page = p.table[(size_t)b * p.table_ld + (block >> p.page_shift)];
    if ((unsigned)page < (unsigned)p.pages) {
      r.at = ((page * p.n_kv + j) << p.page_shift) | (block & ((1 << p.page_shift) - 1));
      r.ke = p.k_exp[r.at];
      r.ve = p.v_exp[r.at];
    }
  }
  return r;
}

// Query rows of a tile over steps [first_step, stop_step) of 64 key rows.
__device__ __forceinline__ void many_rows(const PagedAttentionArgs& a, ManyShared& sh, int j, int b, int tile, int first_step,
                                          int stop_step, bool whole, size_t slot_index) {
  const PagedPool& p = a.pool;
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = a.T * a.G, row = tile * kManyRows + 32 * wave + c;
  const Request rq = request_of(a, b);
  const int most = item_rows<true>(a, rq, tile);
  const int end_block = (most + 15) / 16;
  const int stop = min(stop_step, (end_block + 3) / 4);
  const int t = min(row, rows - 1) / a.G, head = j * a.G + min(row, rows - 1) % a.G;
  const int limit = rq.visible(t);
  // (the wave's first row sees the fewest)
  const int least = rq.visible(min(tile * kManyRows + 32 * wave, rows - 1) / a.G);
  const Scale sc = scale_of(a.scale);
  Query q;
  const __bf16* from = a.q + (size_t)b * a.q_b + (size_t)head * a.q_h + (size_t)t * a.q_t + 32 * h;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4_t w = *reinterpret_cast<const u32x4_t*>(from + 64 * k + 8 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = scaled_bits(w[e], sc);
      q.q[k][i] = __builtin_bit_cast(bf16x8_t, w);
    }
  bool any = false;
  ManyState st;
  st.sums = no_sums(sc.c2);
#pragma unroll
  for (int d = 0; d < 4; ++d) st.o[d] = f32x16_t{};

  auto* ring = (lds_byte_t*)sh.ring;
  const unsigned ring_at = (unsigned)(size_t)ring;
  // 16 steps' blocks in the lanes, this group's and the next one's
  ManyBlocks now = many_blocks(p, b, j, 4 * first_step, end_block), next = now;
  int group = first_step;  // the step of lane 0
  auto load = [&](int step, unsigned slot) __attribute__((always_inline)) {
    const int i = 4 * (step - group) + wave;  // (0..127)
    const int at = step < stop ? __builtin_amdgcn_readlane(i < 64 ? now.at : next.at, i & 63) : -1;
    const size_t from = (size_t)(at < 0 ? 0 : at) * kPagedBlockBytes;
    lds_load_words_t k = buffer_words(p.k + from, at < 0 ? 0 : kPagedBlockBytes);
    lds_load_words_t v = buffer_words(p.v + from, at < 0 ? 0 : kPagedBlockBytes);
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = __builtin_amdgcn_readfirstlane(k[e]), v[e] = __builtin_amdgcn_readfirstlane(v[e]);
    const unsigned to = ring_at + slot * kSlot + wave * kPagedBlockBytes;
    dma_1k<false>(k, lane * 16, 0, to);
    dma_1k<false>(k, lane * 16 + 1024, 0, to + 1024);
    dma_1k<false>(v, lane * 16, 0, to + 4 * kPagedBlockBytes);
    dma_1k<false>(v, lane * 16 + 1024, 0, to + 4 * kPagedBlockBytes + 1024);
  };
  __syncthreads();  // (the ring of the item before has been read)
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // (loads counted by the compiler are not among those counted here)
  // Half steps of 32 key rows.  A wave issues in order, so the products of the next half's
  // scores stand between the exponentials of this one's weights.
  auto key_scale = [&](int step, int m) __attribute__((always_inline)) {
    const int i = 4 * (step - group) + 2 * m;
    const int lo = __builtin_amdgcn_readlane(now.ke, i), hi = __builtin_amdgcn_readlane(now.ke, i + 1);
    return c < 16 ? lo : hi;
  };
  // The step's loads have landed (the next ones' are behind them), and with the barrier
  // every wave's; every wave is done with the step two before it, whose slot the load takes.
  auto begin_step = [&](int step) __attribute__((always_inline)) {
    if (step - group == 12) next = many_blocks(p, b, j, 4 * (group + 16), end_block);
    asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    load(step + 2, (step - first_step + 2) & (kRing - 1));
  };
  if (first_step < stop) {
    load(first_step, 0);
    load(first_step + 1, 1);
    begin_step(first_step);
    Keys keys = many_keys(ring, 0);
    f32x16_t s = many_scores(keys, q, key_scale(first_step, 0));
    keys = many_keys(ring, 1);
    for (int step = first_step; step < stop; ++step) {
      lds_byte_t* slot = ring + ((step - first_step) & (kRing - 1)) * kSlot;
      lds_byte_t* after = ring + ((step + 1 - first_step) & (kRing - 1)) * kSlot;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int i = 4 * (step - group) + 2 * m, row0 = kStep * step + 32 * m;
        int at[2], ve[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          at[u] = __builtin_amdgcn_readlane(now.at, i + u);
          ve[u] = __builtin_amdgcn_readlane(now.ve, i + u);
        }
        Values v[2] = {many_values(slot, 2 * m), many_values(slot, 2 * m + 1)};
        if (m == 1 && step + 1 - group == 16) {  // (this step's have been taken out)
          now = next;
          group = step + 1;
        }
        const int scale = key_scale(m == 0 ? step : step + 1, 1 - m);
        const bool masked = row0 + 32 > least || (at[0] | at[1]) < 0;
        auto seen = [&](int e) { return row0 + 8 * (e / 4) + 4 * h + e % 4 < limit && at[e / 8] >= 0; };
        if (masked) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool ok = seen(e);
            any |= ok;
            s[e] = ok ? s[e] : neg_inf();
          }
        } else {
          any = true;
        }
        bf16x8_t w[2];
        const f32x16_t then = many_scores(keys, q, scale);
        float sum = many_weights(s, st.sums, w);
        asm volatile("" : "+v"(sum) : "v"(then[0]));  // (the products stay in front of the branch)
        // A weight above 2^8 shows in their sum: then m is raised, and they are computed again.
        if (__ballot(sum > 16.f * kMostWeight)) {
          float top = s[0];
#pragma unroll
          for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
          const f32x2_t tops = both_halves(top);
          const float f = raised(st.sums, fmaxf(tops[0], tops[1]), sc.c2);
#pragma unroll
          for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) st.o[d][e] *= f;
          sum = many_weights(s, st.sums, w);
        }
        st.sums.l += sum;
        // The half after the next: of this step, or of the one that begins here.
        if (m == 0) {
          begin_step(step + 1);
          keys = many_keys(after, 0);
        } else {
          keys = many_keys(after, 1);
        }
        if (masked) {
#pragma unroll
          for (int u = 0; u < 2; ++u) many_nans(v[u], [&](int e) { return seen(8 * u + e); }, st);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float vs = power_of_two(ve[u] - 127);
          if (u == 0) __builtin_amdgcn_s_setprio(1);  // products before the other wave's exponentials
#pragma unroll
          for (int d = 0; d < 4; ++d)
            st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(eight(v[u].lo[d], v[u].hi[d], vs, vs), w[u], st.o[d], 0, 0, 0);
        }
        __builtin_amdgcn_s_setprio(0);
        s = then;
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");

  const f32x2_t ls = both_halves(st.sums.l);
  const float l = ls[0] + ls[1];
  const bool met = (__ballot(any) >> c & 0x0000000100000001ull) != 0;  // one of the row's two lanes has
  const float m = met ? st.sums.m : neg_inf();
  if (row >= rows) return;
  const bool none = t >= rq.count || m == neg_inf();
  const float share = none ? 0.f : 1.f / l;
  const Part part = part_of(a, slot_index);
  const int r = 32 * wave + c;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int dim = 32 * d + 8 * i + 4 * h;
      if (whole) {
        bf16x4_t o;
#pragma unroll
        for (int u = 0; u < 4; ++u) o[u] = static_cast<__bf16>(none ? 0.f : st.o[d][4 * i + u] * share);
        *reinterpret_cast<bf16x4_t*>(a.out + (((size_t)b * a.T + t) * a.n_q + head) * D + dim) = o;
      } else {
        *reinterpret_cast<f32x4_t*>(part.o + (size_t)r * D + dim) =
            f32x4_t{st.o[d][4 * i], st.o[d][4 * i + 1], st.o[d][4 * i + 2], st.o[d][4 * i + 3]};
      }
    }
  if (!whole && h == 0) *reinterpret_cast<f32x2_t*>(part.ml + r * 2) = f32x2_t{m, l};
}

// Grid: kv head (fastest: with 8 of them each XCD's L2 holds one head's rows), worker.
// A share that does not reach an item's start leaves its part in the worker's slot 0, one
// that starts the item and does not end it in slot 1.
__global__ __launch_bounds__(64 * kManyWaves, 2) void many_attention_kernel(PagedAttentionArgs a) {
  __shared__ __align__(1024) ManyShared sh;
  const int j = blockIdx.x % a.pool.n_kv, w = blockIdx.x / a.pool.n_kv;
  const Share s = share_of(a, w, blockIdx.x == 0 && threadIdx.x < 64);
  if (j == 0 && threadIdx.x == 0) a.cuts[w] = s.cuts ? s.item : -1;
  int item = s.item, skip = s.skip, left = s.places;
  while (left > 0) {
    const int b = request_at<true>(a, item);
    const int units = item_units<true>(a, item);
    const int stop = min(skip + left, units + kPagedManyStart);
    const int first = max(skip - kPagedManyStart, 0), last = stop - kPagedManyStart;
    if (first < last)
      many_rows(a, sh, j, b, item - b * a.tiles, first, last, first == 0 && last == units,
                ((size_t)j * a.workers + w) * 2 + (first == 0 ? 1 : 0));
    left -= stop - skip;
    skip = 0;
    ++item;
  }
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttentionArgs& a, const PagedPlan& plan, hipStream_t stream) {
  const unsigned n_kv = (unsigned)a.pool.n_kv;
  if (plan.one_launch) {
    const dim3 grid(n_kv * a.items);
    if (plan.rows == 16) launch_kernel(short_attention_kernel<1>, grid, dim3(64 * kShortWaves), 0, stream, a);
    if (plan.rows == 32) launch_kernel(short_attention_kernel<2>, grid, dim3(64 * kShortWaves), 0, stream, a);
    if (plan.rows == 64) launch_kernel(short_attention_kernel<4>, grid, dim3(64 * kShortWaves), 0, stream, a);
    return hipGetLastError();
  }
  const dim3 grid(n_kv * (plan.rows == kManyRows ? a.workers : ceil_div(a.workers, kFewWaves)));
  if (plan.rows == 16) launch_kernel(few_attention_kernel<1>, grid, dim3(64 * kFewWaves), 0, stream, a);
  if (plan.rows == 32) launch_kernel(few_attention_kernel<2>, grid, dim3(64 * kFewWaves), 0, stream, a);
  if (plan.rows == kManyRows) launch_kernel(many_attention_kernel, grid, dim3(64 * kManyWaves), 0, stream, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const dim3 joins((unsigned)plan.joins * n_kv * (unsigned)ceil_div(plan.slot_rows, plan.join_passes << plan.join_shift));
  auto join = [&](auto kernel, int threads) { launch_kernel(kernel, joins, dim3(threads), 0, stream, a, plan.rows); };
  if (plan.rows != kManyRows)
    plan.join_wide ? join(join_kernel<false, kJoinWide, 1>, kJoinWide) : join(join_kernel<false, kJoinThreads, 1>, kJoinThreads);
  else if (plan.join_passes > 1)
    join(join_kernel<true, kJoinThreads, kPagedJoinPasses>, kJoinThreads);
  else
    plan.join_wide ? join(join_kernel<true, kJoinWide, 1>, kJoinWide) : join(join_kernel<true, kJoinThreads, 1>, kJoinThreads);
  return hipGetLastError();
}

}  // namespace lsk
