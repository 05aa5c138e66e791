// Low-rank adapters of many requests beside a shared projection, for gfx950:
//   z[m] = y[m] + s_a (x[m] . A_a^T) . B_a^T,  a = index[m],
// out = z, or SiLU(z_gate) * z_up for gate_up rows in their packed column order.
//
// A group of work is (16 or 64 rows, one of the adapters that they name).  Its
// workgroup's 8 waves split K for h^T = A_a x^T on v_mfma_f32_16x16x32_bf16 (the
// adapter's rank rows are the A operand, 16 rows of x the B operand; rows that name
// another adapter are neither read nor kept) and add their partial tiles through
// LDS in wave order.  h^T leaves those products in exactly the lanes where
// v_mfma_f32_16x16x16_bf16 takes its B operand from, so z^T = y^T + B_a h^T
// follows without a transposition: the waves split the output columns, and each
// lane ends with 8 neighbouring columns of its row (for gate_up with 8 gate and
// their 8 up columns).
//
// h is held in fp32 and multiplied as the sum of two bf16 parts, h = hi + lo
// (lo the rounding error of hi, itself rounded): 2^-17 of h is lost instead of
// 2^-8, for one more MFMA per tile, which the bytes hide.  z is rounded once.
// A row's result depends on its own x, y and adapter alone: products of other
// rows or adapters are dropped by selection, never multiplied by zero.
//
// Two forms.  One launch: every workgroup of a group computes h anew from x and
// A (which come from L2) for its range of output columns.  Two launches: the
// first splits K over workgroups too and leaves h, one partial per K range, in
// the workspace; the second adds the partials in order.  adapter_plan chooses,
// and the rows of a group: 64 share an adapter's tiles among four times the
// rows, 16 keep a small batch's groups small.
//
// Bound by bytes for many rows or adapters, by the chain x, A, h, B, z for few (medians
// of the launches by themselves):
//   1 row, o (2560 x 4096), rank 8                     5.2 us
//   16 rows, QKV (6144 x 2560), 24 of rank 16          6.4 us (4.1 MB)
//   64 rows, down (2560 x 9728), 32 of rank 64         9.9 + 4.9 us (52 MB, most of them
//     A: 41 MB fetched by the first launch, each adapter's once)
//   2000 rows, gate_up (19456 x 2560), 8 of rank 32    7.6 + 35.1 us (135 MB: the second
//     launch 117 MB, 3.3 TB/s; a copy reaches 4.8)
// 17 to 128 rows that name few adapters of a store of many leave workgroups idle, and
// above 128 rows the time grows with the adapters that 64 neighbouring rows name:
// adapter_plan has the figures.

#include <hip/hip_runtime.h>

#include "lsk_internal.h"

namespace lsk {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * 64;
constexpr int kXcds = 8;
constexpr unsigned kRawBufferDword3 = 0x00020000u;
// A buffer offset past every row: the load returns zero without a memory access.
constexpr unsigned kOutOfRange = 0x80000000u;

__device__ __forceinline__ f32x4_t mfma_k16(bf16x4_t a, bf16x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, a), __builtin_bit_cast(s16x4_t, b), c,
                                                   0, 0, 0);
}

// Rows m0 .. m0 + 16 CB - 1: the slot-th adapter that they name, in the order of the
// first row that names it, with a bit for every row that does; `plain`, a bit for
// every row without an adapter.  adapter = -1: there are not so many.
struct Group {
  int adapter;
  unsigned long long rows, plain;
};
template <int CB>
__device__ __forceinline__ Group find_group(const AdapterArgs& a, int m0, int slot) {
  const int lane = threadIdx.x & 63;
  const bool row = lane < 16 * CB && m0 + lane < a.M;
  int v = row ? a.index[m0 + lane] : -1;
  if ((unsigned)v >= (unsigned)a.count) v = -1;
  unsigned long long left = __ballot(v >= 0);
  Group g = {-1, 0ull, __ballot(row && v < 0)};
  for (int n = 0; left != 0; ++n) {
    const int candidate = __builtin_amdgcn_readlane(v, __builtin_ctzll(left));
    const unsigned long long same = __ballot(v == candidate);
    if (n == slot) {
      g.adapter = candidate;
      g.rows = same;
      break;
    }
    left &= ~same;
  }
  return g;
}

// Whether any of the 16 rows of block cb is in `rows`; whether the lane's row of it is.
__device__ __forceinline__ bool block_any(unsigned long long rows, int cb) { return (rows >> (16 * cb) & 0xffffu) != 0; }
__device__ __forceinline__ bool lane_in(unsigned long long rows, int cb) {
  return rows >> (16 * cb + (threadIdx.x & 15)) & 1u;
}

// h^T over k-tiles [kt0, kt1): tile (rt, cb) of the rank and the rows, number
// rt CB + cb, in the wave `number % 8`'s lanes, for done(number, h).
template <int RT, int CB, typename Done>
__device__ __forceinline__ void shrink(const AdapterArgs& a, const Group& grp, int m0, int kt0, int kt1,
                                       f32x4_t (*part)[RT * CB < kWaves ? RT * CB : kWaves][64], Done done) {
  constexpr int kTiles = RT * CB;
  constexpr int kRound = kTiles < kWaves ? kTiles : kWaves;
  // k-tiles whose loads are issued together: some 16 KB per wave
  constexpr int U = RT + CB <= 2 ? 8 : RT + CB <= 4 ? 4 : RT + CB <= 8 ? 2 : 1;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int rows = min(16 * CB, a.M - m0);
  const __amdgpu_buffer_rsrc_t xbuf =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(a.x) + (size_t)m0 * a.ldx, (short)0,
                                        (int)(((rows - 1) * a.ldx + a.K) * 2), (int)kRawBufferDword3);
  unsigned xoff[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb)
    xoff[cb] = lane_in(grp.rows, cb) ? (unsigned)((16 * cb + (lane & 15)) * a.ldx + 8 * (lane >> 4)) * 2u : kOutOfRange;
  const bf16x8_t* at = reinterpret_cast<const bf16x8_t*>(a.a_tiles + (size_t)grp.adapter * a.a_stride) + lane;
  const int KT = a.K / kTileK;
  f32x4_t acc[RT][CB];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) acc[rt][cb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int kt = kt0 + wave; kt < kt1; kt += U * kWaves) {
    bf16x8_t xf[U][CB], af[U][RT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(kt + u * kWaves, kt1 - 1);  // past the end: the last tile again, not multiplied
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
        xf[u][cb] = __builtin_bit_cast(
            bf16x8_t, __builtin_amdgcn_raw_buffer_load_b128(xbuf, xoff[cb] + (unsigned)k * (kTileK * 2), 0, 0));
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) af[u][rt] = at[((size_t)rt * KT + k) * 64];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kt + u * kWaves >= kt1) break;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        if (CB > 1 && !block_any(grp.rows, cb)) continue;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          acc[rt][cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[u][rt], xf[u][cb], acc[rt][cb], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int first = 0; first < kTiles; first += kRound) {
    if (first > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < kRound; ++i)
      if (first + i < kTiles) part[wave][i][lane] = acc[(first + i) / CB][(first + i) % CB];
    __syncthreads();
    if (wave < kRound && first + wave < kTiles) {
      f32x4_t h = part[0][wave][lane];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) h += part[w][wave][lane];
      done(first + wave, h);
    }
  }
}

// Tile `number` of s_a h^T, split into two bf16 parts, to LDS for every wave.  Ranks
// past the adapter's own are zero whatever x holds.
template <int CB>
__device__ __forceinline__ void split_h(int number, f32x4_t h, float scale, int rank, bf16x8_t (*hs)[64]) {
  const int lane = threadIdx.x & 63;
  bf16x8_t o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v = 16 * (number / CB) + 4 * (lane >> 4) + i < rank ? h[i] * scale : 0.f;
    const float hi = bf16_round(v);
    o[i] = static_cast<__bf16>(hi);
    // (of an infinity nothing is left over)
    o[4 + i] = static_cast<__bf16>(fabsf(hi) < __builtin_huge_valf() ? v - hi : 0.f);
  }
  hs[number][lane] = o;
}

__device__ __forceinline__ bf16x4_t low_half(bf16x8_t v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3); }
__device__ __forceinline__ bf16x4_t high_half(bf16x8_t v) { return __builtin_shufflevector(v, v, 4, 5, 6, 7); }

// SiLU(g) * u, rounded once (sigmoid as in silu_mul_bf16).
__device__ __forceinline__ __bf16 silu_mul_once(float g, float u) {
  const float d = 1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896341f);
  const float sc = d > 0x1p96f ? 0x1p-32f : 1.0f;
  return static_cast<__bf16>(sc * (g * __builtin_amdgcn_rcpf(d * sc)) * u);
}

// The output columns a wave takes at a time: 32, or 64 of a gate_up projection (two
// blocks of 16 gate and 16 up columns), so that a lane's accesses are 16 bytes.
template <bool SILU>
struct Columns {
  static constexpr int kWidth = SILU ? 64 : 32;
  static constexpr int kPieces = SILU ? 2 : 1;  // of 8 columns: gate, up
};

// The output side of the rows `live` of a tile.
template <int RT, int CB, bool SILU>
struct Output {
  static constexpr int P = Columns<SILU>::kPieces;
  struct Y {
    bf16x8_t v[CB][P];
  };
  const AdapterArgs& a;
  __amdgpu_buffer_rsrc_t ybuf;
  unsigned yoff[CB];
  unsigned long long live;
  int at;  // the lane's first column of a block (gate_up: in y)
  __bf16* out;

  __device__ __forceinline__ Output(const AdapterArgs& args, unsigned long long rows_live, int m0) : a(args) {
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int rows = min(16 * CB, a.M - m0);
    live = rows_live;
    ybuf = __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(a.y) + (size_t)m0 * a.ldy, (short)0,
                                             (int)(((rows - 1) * a.ldy + a.N) * 2), (int)kRawBufferDword3);
    at = SILU ? 32 * (g >> 1) + 8 * (g & 1) : 8 * g;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
      yoff[cb] = lane_in(live, cb) ? (unsigned)((16 * cb + c) * a.ldy + at) * 2u : kOutOfRange;
    out = a.out + (size_t)(m0 + c) * (SILU ? a.N / 2 : a.N) + (SILU ? 8 * g : at);
  }

  // The last block may be half a block.
  __device__ __forceinline__ bool inside(int nb) const { return nb * Columns<SILU>::kWidth + at < a.N; }

  // (No load under a condition: behind one the compiler cannot count the loads in
  // flight and would wait for all of them.  Rows without work are out of range.)
  __device__ __forceinline__ void load(int nb, Y& y) const {
    const unsigned past = inside(nb) ? 0u : kOutOfRange;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int p = 0; p < P; ++p)
        y.v[cb][p] = __builtin_bit_cast(
            bf16x8_t, __builtin_amdgcn_raw_buffer_load_b128(
                          ybuf, (yoff[cb] | past) + (unsigned)nb * (Columns<SILU>::kWidth * 2) + 32u * p, 0, 0));
  }

  __device__ __forceinline__ void load_b(int adapter, int nb, bf16x8_t (&b)[RT][P]) const {
    const bf16x8_t* bt =
        reinterpret_cast<const bf16x8_t*>(a.b_tiles + (size_t)adapter * a.b_stride) + (threadIdx.x & 63);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int p = 0; p < P; ++p) b[rt][p] = bt[(((size_t)nb * RT + rt) * P + p) * 64];
  }

  // z of rows 16 cb ..: halves 0 and 1 of piece p are z[2 p] and z[2 p + 1].
  __device__ __forceinline__ void multiply(const bf16x8_t (&b)[RT][P], const bf16x8_t (*hs)[64], int cb,
                                           f32x4_t (&z)[2 * P]) const {
#pragma unroll
    for (int i = 0; i < 2 * P; ++i) z[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const bf16x8_t h = hs[rt * CB + cb][threadIdx.x & 63];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        z[2 * p] = mfma_k16(low_half(b[rt][p]), low_half(h), z[2 * p]);
        z[2 * p + 1] = mfma_k16(high_half(b[rt][p]), low_half(h), z[2 * p + 1]);
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        z[2 * p] = mfma_k16(low_half(b[rt][p]), high_half(h), z[2 * p]);
        z[2 * p + 1] = mfma_k16(high_half(b[rt][p]), high_half(h), z[2 * p + 1]);
      }
    }
  }

  __device__ __forceinline__ void store(int nb, int cb, const f32x4_t (&z)[2 * P]) const {
    if (!lane_in(live, cb) || !inside(nb)) return;
    bf16x8_t o;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      o[i] = SILU ? silu_mul_once(z[i / 4][i % 4], z[(2 * P - 2) + i / 4][i % 4]) : static_cast<__bf16>(z[i / 4][i % 4]);
    *reinterpret_cast<bf16x8_t*>(out + (size_t)(16 * cb) * (SILU ? a.N / 2 : a.N) + nb * 32) = o;
  }
};

__device__ __forceinline__ float half_of(const bf16x8_t& y, int half, int i) { return static_cast<float>(y[4 * half + i]); }

// Blocks [first, last) of share i of n.
__device__ __forceinline__ int share_begin(int total, int i, int n) { return (int)((long long)total * i / n); }

// Whether the column ranges of a group, which all read its A, go to one XCD's L2 (workgroups
// go to the XCDs by turns): of up to 16 rows in one launch, with a slot or more for each
// XCD.  16 rows with 16 adapters, o, rank 16: 9.0 -> 6.3 us, rank 32 12.3 -> 7.7,
// gate_up, rank 16 9.3 -> 7.9.  Several tiles leave XCDs idle where rows name few
// adapters (100 rows, gate_up: 17.5 -> 21.2).
__host__ __device__ inline bool by_xcd(const AdapterArgs& a, bool two) {
  return !two && a.tiles == 1 && a.slots >= kXcds;
}

// A decode batch: 16 rows and one of the adapters that they name.  Grid: (tile,
// slot, column range), the range fastest, or with by_xcd the slot's last three bits.
template <int RT, bool SILU, bool TWO>
__global__ __launch_bounds__(kThreads) void adapter_group_kernel(AdapterArgs a) {
  constexpr int CB = 1;
  __shared__ f32x4_t part[TWO ? 1 : kWaves][RT][64];
  __shared__ bf16x8_t hs[RT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int id = blockIdx.x, range;
  if (by_xcd(a, TWO)) {
    range = id / kXcds % a.ranges;
    id = id / kXcds / a.ranges * kXcds + id % kXcds;
    if (id >= a.slots) return;
  } else {
    range = id % a.ranges;
    id /= a.ranges;
  }
  const int tile = id / a.slots, slot = id % a.slots;
  const int m0 = tile * 16;
  const Group grp = find_group<CB>(a, m0, slot);
  if (grp.adapter < 0 && !(slot == 0 && grp.plain != 0)) return;
  const int blocks = (a.N + Columns<SILU>::kWidth - 1) / Columns<SILU>::kWidth;
  const int nb0 = share_begin(blocks, range, a.ranges) + wave, nb1 = share_begin(blocks, range + 1, a.ranges);
  using Out = Output<RT, CB, SILU>;
  const Out output(a, grp.rows | (slot == 0 ? grp.plain : 0ull), m0);
  const int adapter = max(grp.adapter, 0);  // (its B is loaded in any case)
  typename Out::Y even, odd;
  bf16x8_t bv[RT][Out::P];
  output.load(min(nb0, blocks - 1), even);
  output.load_b(adapter, min(nb0, blocks - 1), bv);
  if (grp.adapter >= 0) {
    const float scale = a.scale[grp.adapter];
    const int rank = a.ranks[grp.adapter];
    if constexpr (TWO) {
      if (wave < RT) {
        const f32x4_t* src = reinterpret_cast<const f32x4_t*>(a.h) + ((size_t)tile * RT + wave) * 64 + lane;
        const size_t step = (size_t)a.tiles * RT * 64;
        f32x4_t v[kAdapterMaxSplits];  // all on their way together; past the last the last again
#pragma unroll
        for (int s = 0; s < kAdapterMaxSplits; ++s) v[s] = src[(size_t)min(s, a.splits - 1) * step];
        f32x4_t h = v[0];
#pragma unroll
        for (int s = 1; s < kAdapterMaxSplits; ++s)
          if (s < a.splits) h += v[s];
        split_h<CB>(wave, h, scale, rank, hs);
      }
    } else {
      shrink<RT, CB>(a, grp, m0, 0, a.K / kTileK, part, [&](int n, f32x4_t h) { split_h<CB>(n, h, scale, rank, hs); });
    }
    __syncthreads();
  }
  auto finish = [&](int nb, const typename Out::Y& y) {
    f32x4_t z[2 * Out::P] = {};
    if (grp.adapter >= 0) output.multiply(bv, hs, 0, z);
    output.load_b(adapter, min(nb + kWaves, nb1 - 1), bv);
    const bool adapted = lane_in(grp.rows, 0);
#pragma unroll
    for (int j = 0; j < 2 * Out::P; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = half_of(y.v[0][j / 2], j % 2, i);
        z[j][i] = adapted ? v + z[j][i] : v;
      }
    output.store(nb, 0, z);
  };
  // y of two blocks by turns: one handed on in registers would be waited for at once.
  for (int nb = nb0; nb < nb1; nb += 2 * kWaves) {
    output.load(min(nb + kWaves, nb1 - 1), odd);
    finish(nb, even);
    output.load(min(nb + 2 * kWaves, nb1 - 1), even);
    if (nb + kWaves < nb1) finish(nb + kWaves, odd);
  }
}

// Prompt rows: 64 rows a workgroup with all the adapters that they name (mostly one
// or two), so that y is read and written once, in full columns, whoever's rows they
// are.  Grid: (tile, column range), the range fastest.
template <int RT, bool SILU>
__global__ __launch_bounds__(kThreads) void adapter_rows_kernel(AdapterArgs a) {
  constexpr int CB = 4;
  __shared__ bf16x8_t hs[RT * CB][64];
  __shared__ int named[16 * CB];
  __shared__ unsigned long long named_rows[16 * CB];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int range = blockIdx.x % a.ranges, tile = blockIdx.x / a.ranges;
  const int m0 = tile * 16 * CB;
  const bool row = m0 + lane < a.M;
  int mine = row ? a.index[m0 + lane] : -1;
  if ((unsigned)mine >= (unsigned)a.count) mine = -1;
  int count = 0;
  for (unsigned long long left = __ballot(mine >= 0); left != 0; ++count) {
    const int adapter = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const unsigned long long same = __ballot(mine == adapter);
    if (threadIdx.x == 0) named[count] = adapter, named_rows[count] = same;
    left &= ~same;
  }
  for (int n = wave; n < RT * CB; n += kWaves) {
    const int adapter = __shfl(mine, 16 * (n % CB) + c);
    const f32x4_t* src = reinterpret_cast<const f32x4_t*>(a.h) + ((size_t)tile * RT * CB + n) * 64 + lane;
    const size_t step = (size_t)a.tiles * RT * CB * 64;
    f32x4_t v[kAdapterMaxSplits];  // all on their way together; past the last the last again
#pragma unroll
    for (int s = 0; s < kAdapterMaxSplits; ++s) v[s] = src[(size_t)min(s, a.splits - 1) * step];
    f32x4_t h = v[0];
#pragma unroll
    for (int s = 1; s < kAdapterMaxSplits; ++s)
      if (s < a.splits) h += v[s];
    // (rows without an adapter were not written: their rank is zero)
    split_h<CB>(n, h, a.scale[max(adapter, 0)], adapter >= 0 ? a.ranks[adapter] : 0, hs);
  }
  __syncthreads();

  const int blocks = (a.N + Columns<SILU>::kWidth - 1) / Columns<SILU>::kWidth;
  const int nb0 = share_begin(blocks, range, a.ranges) + wave, nb1 = share_begin(blocks, range + 1, a.ranges);
  if (nb0 >= nb1) return;
  using Out = Output<RT, CB, SILU>;
  const Out output(a, __ballot(row), m0);
  const int first = count > 0 ? __builtin_amdgcn_readfirstlane(named[0]) : 0;  // (its B is loaded in any case)
  // Where a tile's rows name several adapters, B of two by turns (300 rows that name 16 per
  // tile, QKV, rank 16: 13.1 -> 11.5 us); gate_up is bound by its vector work and
  // gains nothing.
  constexpr bool kTwoB = !SILU;
  typename Out::Y even, odd;
  bf16x8_t bv[RT][Out::P], bw[RT][Out::P];
  output.load(nb0, even);
  output.load_b(first, nb0, bv);
  auto finish = [&](int nb, const typename Out::Y& y) {
    f32x4_t z[CB][2 * Out::P];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int j = 0; j < 2 * Out::P; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) z[cb][j][i] = half_of(y.v[cb][j / 2], j % 2, i);
    auto add = [&](int n, const bf16x8_t (&b)[RT][Out::P]) {
      const unsigned long long rows = named_rows[n];
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        if (!block_any(rows, cb)) continue;
        f32x4_t d[2 * Out::P];
        output.multiply(b, hs, cb, d);
        const bool adapted = lane_in(rows, cb);
#pragma unroll
        for (int j = 0; j < 2 * Out::P; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) z[cb][j][i] = adapted ? z[cb][j][i] + d[j][i] : z[cb][j][i];
      }
    };
    auto name = [&](int n) { return __builtin_amdgcn_readfirstlane(named[n]); };
    const int next = min(nb + kWaves, nb1 - 1);
    if (!(kTwoB && count > 1)) {
      for (int n = 0; n < count; ++n) {
        if (n > 0) output.load_b(name(n), nb, bv);
        add(n, bv);
      }
      output.load_b(first, next, bv);
    } else {
      for (int n = 0; n < count; n += 2) {
        output.load_b(name(min(n + 1, count - 1)), nb, bw);
        add(n, bv);
        const bool more = n + 2 < count;
        output.load_b(more ? name(n + 2) : first, more ? nb : next, bv);
        if (n + 1 < count) add(n + 1, bw);
      }
    }
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) output.store(nb, cb, z[cb]);
  };
  // y of two blocks by turns: one handed on in registers would be waited for at once.
  for (int nb = nb0; nb < nb1; nb += 2 * kWaves) {
    output.load(min(nb + kWaves, nb1 - 1), odd);
    finish(nb, even);
    output.load(min(nb + 2 * kWaves, nb1 - 1), even);
    if (nb + kWaves < nb1) finish(nb + kWaves, odd);
  }
}

// The first of two launches.  Grid: (tile, slot, K range), the range fastest.
template <int RT, int CB>
__global__ __launch_bounds__(kThreads) void adapter_shrink_kernel(AdapterArgs a) {
  constexpr int kRound = RT * CB < kWaves ? RT * CB : kWaves;
  __shared__ f32x4_t part[kWaves][kRound][64];
  const int lane = threadIdx.x & 63;
  int id = blockIdx.x;
  const int split = id % a.splits;
  id /= a.splits;
  const int tile = id / a.slots;
  const int KT = a.K / kTileK;
  for (int slot = id % a.slots;; slot += a.slots) {
    const Group grp = find_group<CB>(a, tile * 16 * CB, slot);
    if (grp.adapter < 0) return;
    shrink<RT, CB>(a, grp, tile * 16 * CB, share_begin(KT, split, a.splits), share_begin(KT, split + 1, a.splits), part,
                   [&](int n, f32x4_t h) {
                     if (lane_in(grp.rows, n % CB))
                       reinterpret_cast<f32x4_t*>(a.h)[(((size_t)split * a.tiles + tile) * RT * CB + n) * 64 + lane] = h;
                   });
    __syncthreads();  // the partial tiles are read before the next adapter's
  }
}

template <int RT, bool SILU>
hipError_t launch_silu(const AdapterArgs& a, int rows, hipStream_t stream) {
  const unsigned tiles = (unsigned)a.tiles, groups = tiles * a.slots;
  const dim3 block(kThreads);
  if (rows == 16 && a.splits == 0) {
    const unsigned whole = by_xcd(a, false) ? (groups + kXcds - 1) / kXcds * kXcds : groups;
    launch_kernel(adapter_group_kernel<RT, SILU, false>, dim3(whole * a.ranges), block, 0, stream, a);
    return hipGetLastError();
  }
  if (rows == 16)
    launch_kernel(adapter_shrink_kernel<RT, 1>, dim3(groups * a.splits), block, 0, stream, a);
  else
    launch_kernel(adapter_shrink_kernel<RT, 4>, dim3(groups * a.splits), block, 0, stream, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  if (rows == 16)
    launch_kernel(adapter_group_kernel<RT, SILU, true>, dim3(groups * a.ranges), block, 0, stream, a);
  else
    launch_kernel(adapter_rows_kernel<RT, SILU>, dim3(tiles * a.ranges), block, 0, stream, a);
  return hipGetLastError();
}

template <int RT>
hipError_t launch_rank(const AdapterArgs& a, int rows, bool silu, hipStream_t stream) {
  return silu ? launch_silu<RT, true>(a, rows, stream) : launch_silu<RT, false>(a, rows, stream);
}

}  // namespace

hipError_t launch_adapters(const AdapterArgs& a, int rank_tiles, int rows, bool silu, hipStream_t stream) {
  switch (rank_tiles) {
    case 1: return launch_rank<1>(a, rows, silu, stream);
    case 2: return launch_rank<2>(a, rows, silu, stream);
    case 3: return launch_rank<3>(a, rows, silu, stream);
    case 4: return launch_rank<4>(a, rows, silu, stream);
    case 6: return launch_rank<6>(a, rows, silu, stream);
    case 8: return launch_rank<8>(a, rows, silu, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace lsk
