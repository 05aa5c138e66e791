// Low-rank adapters of many requests beside a shared projection, for gfx950:
//   z[m] = y[m] + s_a (x[m] . A_a^T) . B_a^T,  a = index[m],
// out = z, or SiLU(z_gate) * z_up for gate_up rows in their packed column order.
//
// A group of work is (16 rows, one of the adapters that they name).  Its
// workgroup's 8 waves split K for h^T = A_a x^T on v_mfma_f32_16x16x32_bf16 (the
// adapter's rank rows are the A operand, the 16 rows of x the B operand; rows
// that name another adapter are neither read nor kept) and add their partial
// tiles through LDS in wave order.  h^T leaves those products in exactly the
// lanes where v_mfma_f32_16x16x16_bf16 takes its B operand from, so
// z^T = y^T + B_a h^T follows without a transposition: the waves split the
// output columns, 32 at a time, and each lane ends with 8 neighbouring columns
// of its row (for gate_up with 4 gate and their 4 up columns).
//
// h is held in fp32 and multiplied as the sum of two bf16 parts, h = hi + lo
// (lo the rounding error of hi, itself rounded): 2^-17 of h is lost instead of
// 2^-9, for one more MFMA per tile, which the bytes hide.  z is rounded once.
// A row's result depends on its own x, y and adapter alone: products of other
// rows or adapters are dropped by selection, never multiplied by zero.
//
// Two forms.  One launch: every workgroup of a group computes h anew from x and
// A (which come from L2) for its range of output columns.  Two launches: the
// first splits K over workgroups too and leaves h, one partial per K range, in
// the workspace; the second adds the partials in order.  The plan
// (adapter_plan) takes the second form when reading A anew would cost more than
// a launch.

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
constexpr unsigned kRawBufferDword3 = 0x00020000u;
// A buffer offset past every row: the load returns zero without a memory access.
constexpr unsigned kOutOfRange = 0x80000000u;

__device__ __forceinline__ f32x4_t mfma_k16(bf16x4_t a, bf16x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, a), __builtin_bit_cast(s16x4_t, b), c,
                                                   0, 0, 0);
}

// Rows 16 * tile .. + 15: the slot-th adapter that they name, in the order of
// the first row that names it, with a bit for every row that does; `plain`, a bit
// for every row without an adapter.  adapter = -1: there are not so many.
struct Group {
  int adapter;
  unsigned rows, plain;
};
__device__ __forceinline__ Group find_group(const AdapterArgs& a, int m0, int slot) {
  const int lane = threadIdx.x & 63;
  const bool row = lane < 16 && m0 + lane < a.M;
  int v = row ? a.index[m0 + lane] : -1;
  if ((unsigned)v >= (unsigned)a.count) v = -1;
  unsigned left = (unsigned)__ballot(v >= 0);
  Group g = {-1, 0u, (unsigned)__ballot(row && v < 0)};
  for (int n = 0; left != 0; ++n) {
    const int candidate = __builtin_amdgcn_readlane(v, __builtin_ctz(left));
    const unsigned same = (unsigned)__ballot(v == candidate);
    if (n == slot) {
      g.adapter = candidate;
      g.rows = same;
      break;
    }
    left &= ~same;
  }
  return g;
}

// Each wave's share of h^T over k-tiles [kt0, kt1), to LDS: [wave][rt][lane].
template <int RT>
__device__ __forceinline__ void shrink(const AdapterArgs& a, const Group& grp, int m0, int kt0, int kt1,
                                       f32x4_t (*part)[RT][64]) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int g = lane >> 4, c = lane & 15;
  constexpr int U = RT <= 2 ? 4 : 2;  // k-tiles whose loads are issued together
  const int rows = min(16, a.M - m0);
  const __amdgpu_buffer_rsrc_t xbuf =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(a.x) + (size_t)m0 * a.ldx, (short)0,
                                        (int)(((rows - 1) * a.ldx + a.K) * 2), (int)kRawBufferDword3);
  const unsigned xoff = (grp.rows >> c & 1u) ? (unsigned)(c * a.ldx + 8 * g) * 2u : kOutOfRange;
  const bf16x8_t* at = reinterpret_cast<const bf16x8_t*>(a.a_tiles + (size_t)grp.adapter * a.a_stride) + lane;
  const int KT = a.K / kTileK;
  f32x4_t acc[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) acc[rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int kt = kt0 + wave; kt < kt1; kt += U * kWaves) {
    bf16x8_t xf[U], af[U][RT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(kt + u * kWaves, kt1 - 1);  // past the end: the last tile again, its x zero
      const unsigned off = kt + u * kWaves < kt1 ? xoff + (unsigned)k * (kTileK * 2) : kOutOfRange;
      xf[u] = __builtin_bit_cast(bf16x8_t, __builtin_amdgcn_raw_buffer_load_b128(xbuf, off, 0, 0));
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) af[u][rt] = at[((size_t)rt * KT + k) * 64];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kt + u * kWaves >= kt1) break;  // (an infinite A value times the zero x would be NaN)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[u][rt], xf[u], acc[rt], 0, 0, 0);
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) part[wave][rt][lane] = acc[rt];
  __syncthreads();
}

// The waves' shares added in wave order: thread t < 64 RT holds lane t % 64 of rank tile t / 64.
template <int RT>
__device__ __forceinline__ f32x4_t sum_waves(f32x4_t (*part)[RT][64]) {
  const int rt = threadIdx.x >> 6, lane = threadIdx.x & 63;
  f32x4_t h = {0.f, 0.f, 0.f, 0.f};
  if (rt < RT) {
    h = part[0][rt][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) h += part[w][rt][lane];
  }
  return h;
}

// s_a h, split into two bf16 parts, to every wave through LDS.  Ranks past the
// adapter's own are zero whatever x holds.
template <int RT>
__device__ __forceinline__ void share_h(const AdapterArgs& a, const Group& grp, f32x4_t h, bf16x8_t (*hs)[64]) {
  const int rt = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (rt < RT) {
    const float s = a.scale[grp.adapter];
    const int rank = a.ranks[grp.adapter];
    bf16x8_t o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = 16 * rt + 4 * (lane >> 4) + i < rank ? h[i] * s : 0.f;
      const float hi = bf16_round(v);
      o[i] = static_cast<__bf16>(hi);
      // (of an infinity nothing is left over)
      o[4 + i] = static_cast<__bf16>(fabsf(hi) < __builtin_huge_valf() ? v - hi : 0.f);
    }
    hs[rt][lane] = o;
  }
  __syncthreads();
}

__device__ __forceinline__ bf16x4_t low_half(bf16x8_t v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3); }
__device__ __forceinline__ bf16x4_t high_half(bf16x8_t v) { return __builtin_shufflevector(v, v, 4, 5, 6, 7); }

// SiLU(g) * u, rounded once (sigmoid as in silu_mul_bf16).
__device__ __forceinline__ __bf16 silu_mul_once(float g, float u) {
  const float d = 1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896341f);
  const float sc = d > 0x1p96f ? 0x1p-32f : 1.0f;
  return static_cast<__bf16>(sc * (g * __builtin_amdgcn_rcpf(d * sc)) * u);
}

// Column blocks [nb0, nb1) of 32 columns of the group's rows; with kPlain set,
// of the rows without an adapter too, which keep y.
template <int RT, bool SILU>
__device__ __forceinline__ void expand(const AdapterArgs& a, const Group& grp, bool plain, int m0, int nb0, int nb1,
                                       bf16x8_t (*hs)[64]) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int g = lane >> 4, c = lane & 15;
  const bool adapted = grp.rows >> c & 1u;
  const bool live = adapted || (plain && (grp.plain >> c & 1u));
  const int rows = min(16, a.M - m0);
  const __amdgpu_buffer_rsrc_t ybuf =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(a.y) + (size_t)m0 * a.ldy, (short)0,
                                        (int)(((rows - 1) * a.ldy + a.N) * 2), (int)kRawBufferDword3);
  const unsigned yoff = live ? (unsigned)(c * a.ldy + (SILU ? 4 : 8) * g) * 2u : kOutOfRange;
  const int n_out = SILU ? a.N / 2 : a.N;
  __bf16* out = a.out + (size_t)(m0 + c) * n_out + (SILU ? 4 : 8) * g;
  bf16x8_t h[RT];
  if (grp.adapter >= 0) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) h[rt] = hs[rt][lane];
  }
  const bf16x8_t* bt = reinterpret_cast<const bf16x8_t*>(a.b_tiles + (size_t)max(grp.adapter, 0) * a.b_stride) + lane;
  for (int nb = nb0 + wave; nb < nb1; nb += kWaves) {
    f32x4_t z0 = {0.f, 0.f, 0.f, 0.f}, z1 = z0;
    f32x4_t y0, y1;
    if constexpr (SILU) {
      const bf16x4_t lo = __builtin_bit_cast(bf16x4_t, __builtin_amdgcn_raw_buffer_load_b64(ybuf, yoff + (unsigned)nb * 64u, 0, 0));
      const bf16x4_t hi = __builtin_bit_cast(bf16x4_t, __builtin_amdgcn_raw_buffer_load_b64(ybuf, yoff + (unsigned)nb * 64u + 32u, 0, 0));
#pragma unroll
      for (int i = 0; i < 4; ++i) y0[i] = static_cast<float>(lo[i]), y1[i] = static_cast<float>(hi[i]);
    } else {
      // (the last block of an odd number of 16-column blocks has 16 columns)
      const unsigned off = nb * 32 + 8 * g < a.N ? yoff + (unsigned)nb * 64u : kOutOfRange;
      const bf16x8_t y = __builtin_bit_cast(bf16x8_t, __builtin_amdgcn_raw_buffer_load_b128(ybuf, off, 0, 0));
#pragma unroll
      for (int i = 0; i < 4; ++i) y0[i] = static_cast<float>(y[i]), y1[i] = static_cast<float>(y[4 + i]);
    }
    if (grp.adapter >= 0) {
      bf16x8_t b[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) b[rt] = bt[((size_t)nb * RT + rt) * 64];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        z0 = mfma_k16(low_half(b[rt]), low_half(h[rt]), z0);
        z1 = mfma_k16(high_half(b[rt]), low_half(h[rt]), z1);
        z0 = mfma_k16(low_half(b[rt]), high_half(h[rt]), z0);
        z1 = mfma_k16(high_half(b[rt]), high_half(h[rt]), z1);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      z0[i] = adapted ? y0[i] + z0[i] : y0[i];
      z1[i] = adapted ? y1[i] + z1[i] : y1[i];
    }
    if constexpr (SILU) {
      bf16x4_t o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = silu_mul_once(z0[i], z1[i]);
      if (live) *reinterpret_cast<bf16x4_t*>(out + nb * 16) = o;
    } else {
      bf16x8_t o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = static_cast<__bf16>(z0[i]), o[4 + i] = static_cast<__bf16>(z1[i]);
      if (live && nb * 32 + 8 * g < a.N) *reinterpret_cast<bf16x8_t*>(out + nb * 32) = o;
    }
  }
}

// Blocks [first, last) of share i of n.
__device__ __forceinline__ int share_begin(int total, int i, int n) { return (int)((long long)total * i / n); }

// Grid: (16-row tile, slot, column range), the range fastest.
template <int RT, bool SILU, bool TWO>
__global__ __launch_bounds__(kThreads) void adapter_kernel(AdapterArgs a) {
  __shared__ f32x4_t part[TWO ? 1 : kWaves][RT][64];
  __shared__ bf16x8_t hs[RT][64];
  int id = blockIdx.x;
  const int range = id % a.ranges;
  id /= a.ranges;
  const int slot = id % a.slots;
  const int tile = id / a.slots;
  const int m0 = tile * 16;
  const Group grp = find_group(a, m0, slot);
  const bool plain = slot == 0;
  if (grp.adapter < 0 && !(plain && grp.plain != 0)) return;
  if (grp.adapter >= 0) {
    f32x4_t h = {0.f, 0.f, 0.f, 0.f};
    if constexpr (TWO) {
      const int rt = threadIdx.x >> 6, lane = threadIdx.x & 63;
      if (rt < RT && (grp.rows >> (lane & 15) & 1u)) {
        const f32x4_t* src = reinterpret_cast<const f32x4_t*>(a.h) + ((size_t)tile * RT + rt) * 64 + lane;
        const size_t step = (size_t)a.tiles * RT * 64;
        h = src[0];
        for (int s = 1; s < a.splits; ++s) h += src[(size_t)s * step];
      }
    } else {
      shrink<RT>(a, grp, m0, 0, a.K / kTileK, part);
      h = sum_waves<RT>(part);
    }
    share_h<RT>(a, grp, h, hs);
  }
  const int blocks = (a.N + 31) / 32;
  expand<RT, SILU>(a, grp, plain, m0, share_begin(blocks, range, a.ranges), share_begin(blocks, range + 1, a.ranges), hs);
}

// The first of two launches.  Grid: (16-row tile, slot, K range), the range fastest.
template <int RT>
__global__ __launch_bounds__(kThreads) void adapter_shrink_kernel(AdapterArgs a) {
  __shared__ f32x4_t part[kWaves][RT][64];
  int id = blockIdx.x;
  const int split = id % a.splits;
  id /= a.splits;
  const int slot = id % a.slots;
  const int tile = id / a.slots;
  const Group grp = find_group(a, tile * 16, slot);
  if (grp.adapter < 0) return;
  const int KT = a.K / kTileK;
  shrink<RT>(a, grp, tile * 16, share_begin(KT, split, a.splits), share_begin(KT, split + 1, a.splits), part);
  const f32x4_t h = sum_waves<RT>(part);
  const int rt = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (rt < RT && (grp.rows >> (lane & 15) & 1u))
    reinterpret_cast<f32x4_t*>(a.h)[((size_t)split * a.tiles + tile) * RT * 64 + rt * 64 + lane] = h;
}

template <int RT, bool SILU>
hipError_t launch_silu(const AdapterArgs& a, hipStream_t stream) {
  const unsigned groups = (unsigned)a.tiles * a.slots;
  if (a.splits == 0) {
    launch_kernel(adapter_kernel<RT, SILU, false>, dim3(groups * a.ranges), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  }
  launch_kernel(adapter_shrink_kernel<RT>, dim3(groups * a.splits), dim3(kThreads), 0, stream, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  launch_kernel(adapter_kernel<RT, SILU, true>, dim3(groups * a.ranges), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

template <int RT>
hipError_t launch_rank(const AdapterArgs& a, bool silu, hipStream_t stream) {
  return silu ? launch_silu<RT, true>(a, stream) : launch_silu<RT, false>(a, stream);
}

}  // namespace

hipError_t launch_adapters(const AdapterArgs& a, int rank_tiles, bool silu, hipStream_t stream) {
  switch (rank_tiles) {
    case 1: return launch_rank<1>(a, silu, stream);
    case 2: return launch_rank<2>(a, silu, stream);
    case 3: return launch_rank<3>(a, silu, stream);
    case 4: return launch_rank<4>(a, silu, stream);
    case 6: return launch_rank<6>(a, silu, stream);
    case 8: return launch_rank<8>(a, silu, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace lsk
