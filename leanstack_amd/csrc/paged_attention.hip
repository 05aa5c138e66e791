// Attention over the pages of an 8-bit cache for gfx950: T query tokens of each of B
// requests over the rows that the request has cached, its new ones the last of them
// (causal within them).
//
//   out = sum_i e^(s_i - m) v_i / sum_i e^(s_i - m),  s = scale q . k,
// k and v being e4m3 bytes times a power of two per 16 rows and head (paged_cache.hip
// has the format).  A wave takes two blocks, 32 key rows, a step, for up to 4 x 16 query
// rows of one kv head:
//   bytes to bf16 with their scale, two values an instruction, exact;
//   S = K Q^T on v_mfma_f32_16x16x32_bf16: a lane holds 2 x 4 scores of one query row;
//   the running maximum m and sum l of the softmax in base 2, in fp32, m raised only
//     where a step exceeds it by 2^8;
//   O^T += V^T P^T on the same instruction: the scores' lanes are those of its operand
//     if the 32 key rows are taken in the order in which the lanes hold them, and the
//     blocks of V lie in memory as the other operand's lanes take them.
// Nothing goes through LDS but the waves' sums at the end.
//
// P is rounded to bf16, at most 2^-9 of each weight, and l sums the rounded weights: the
// result is exactly that of slightly other weights.

#include <hip/hip_runtime.h>

#include "lsk_internal.h"

namespace lsk {
namespace {

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

constexpr int D = kAttnHeadDim;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr float kRaise = 8.f;
constexpr float kFar = 0x1p30f;
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ float neg_inf() { return -__builtin_huge_valf(); }

__device__ __forceinline__ float power_of_two(int n) {
  return n < -126 ? 0.f : __builtin_bit_cast(float, (unsigned)(n + 127) << 23);
}

// The four lanes that hold a query row's scores: c, c + 16, c + 32, c + 48.
__device__ __forceinline__ float rows_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float rows_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Eight bytes times a power of two.
__device__ __forceinline__ bf16x8_t eight(unsigned w0, unsigned w1, float scale0, float scale1) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale0, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale0, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale1, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale1, true);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Bytes of a word that are NaN, as 0xff each.
__device__ __forceinline__ unsigned nan_bytes(unsigned w) {
  const unsigned t = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  return (t >> 7) * 0xffu;
}

// A wave's softmax state for 16 query rows: lane (c, g) holds row c, of O the dims
// 16 i + 4 g .. + 3, of l the share of the lane's scores, and of m the factor c2 that
// takes its scores to base 2.  m = -inf: no row seen.
struct State {
  float m, l, c2;
  f32x4_t o[8];
};

__device__ __forceinline__ State empty_state(float c2) {
  State st;
  st.m = neg_inf();
  st.l = 0.f;
  st.c2 = c2;
#pragma unroll
  for (int i = 0; i < 8; ++i) st.o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  return st;
}

// 1 KB of a block, 16 bytes a lane; zeros and no access where there is none.
__device__ __forceinline__ u32x4_t load_1k(const unsigned char* blocks, int at, int half) {
  const __amdgpu_buffer_rsrc_t block = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(blocks) + (size_t)(at < 0 ? 0 : at) * kPagedBlockBytes, (short)0,
      at < 0 ? 0 : kPagedBlockBytes, 0x00020000);
  return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(block, (threadIdx.x & 63) * 16, half * 1024, 0));
}

// The weights P of a step as the operand of the second product, and m, l, O brought to
// the new maximum.  s[m][i]: row 16 m + 4 g + i of the step.  seen(m, i): whether the lane's
// query row sees it (MASK).
//
// Exponents are s c2 - m with one rounding, m being the rounded top c2: far from zero
// (kFar) its rounding error would be more than 2^x holds.  There scores that are not
// equal are 2^6 and more apart in base 2, so any factor gives the same weights, if m's
// order stays: the next power of two above c2, whose products are exact.
template <bool MASK, typename Seen>
__device__ __forceinline__ bf16x8_t step_weights(f32x4_t (&s)[2], float c2, State& st, Seen seen) {
  bool any = !MASK;
  if constexpr (MASK) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool ok = seen(i / 4, i % 4);
      any |= ok;
      if (!ok) s[i / 4][i % 4] = neg_inf();
    }
  }
  float top = fmaxf(s[0][0], s[0][1]);
#pragma unroll
  for (int i = 2; i < 8; ++i) top = fmaxf(top, s[i / 4][i % 4]);
  // (a row that is seen raises m from -inf whatever its score: sums of 0 are then NaN)
  const float mine = any ? fmaxf(top * st.c2, kLowest) : neg_inf();
  if (__ballot(mine > st.m + kRaise)) {
    top = rows_max(top);
    const bool raise = rows_max(mine) > st.m + kRaise;
    const float above = __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, c2) + 0x007fffffu) & 0x7f800000u);
    st.c2 = !raise ? st.c2 : fabsf(top * c2) < kFar ? c2 : above;
    const float mx = fmaxf(top * st.c2, kLowest);
    const float f = raise ? __builtin_amdgcn_exp2f(st.m - mx) : 1.f;
    st.m = raise ? mx : st.m;
    st.l *= f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[i][e] *= f;
  }
  const float m = st.m == neg_inf() ? 0.f : st.m;
  bf16x8_t p;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4], st.c2, -m));
    if (MASK && !seen(i / 4, i % 4)) e = 0.f;
    p[i] = static_cast<__bf16>(e);
  }
  const bf16x2_t ones = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
#pragma unroll
  for (int i = 0; i < 8; i += 2) st.l = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{p[i], p[i + 1]}, ones, st.l, false);
  return p;
}

// What the wave's lane l knows of block 2 (first + kWaves (l / 2)) + l % 2: its place in the pool
// (-1: no row of it is read) and its scales.
struct Blocks {
  int at;
  float ks, vs;
};
__device__ __forceinline__ Blocks blocks_from(const PagedPool& p, int b, int j, int first, int end) {
  const int lane = threadIdx.x & 63;
  const int block = 2 * (first + kWaves * (lane >> 1)) + (lane & 1);
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

// Grid: kv head (fastest), request, 16 NT query rows.
template <int NT>
__global__ __launch_bounds__(kThreads) void paged_attention_kernel(PagedAttentionArgs a) {
  __shared__ float os[kWaves][16][D + 4];
  __shared__ float ms[kWaves][16], ls[kWaves][16];
  const PagedPool& p = a.pool;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = blockIdx.x;
  const int j = id % p.n_kv;
  id /= p.n_kv;
  const int b = id % a.B;
  const int r0 = id / a.B * 16 * NT;
  const int rows = a.T * a.G;

  const int len = max(a.lens[b], 0);
  const int count = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  // Rows that query t sees (those behind the last real one: as many as that).
  auto visible = [&](int t) { return min(max(len - max(count - 1 - t, 0), 0), 16 * p.blocks); };
  const int t_first = r0 / a.G, t_last = min(r0 + 16 * NT, rows) - 1;
  const int least = count > t_first ? visible(t_first) : 0;
  const int most = count > t_first ? visible(t_last / a.G) : 0;
  const int end_block = (most + 15) / 16, steps = (end_block + 1) / 2;

  bf16x8_t q[NT][4];
  int limit[NT];
  State st[NT];
  const float c2 = fabsf(a.scale) * 1.44269504088896341f;
  const unsigned flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = min(r0 + 16 * n + c, rows - 1);
    const int t = r / a.G, h = j * a.G + r % a.G;
    limit[n] = visible(t);
    st[n] = empty_state(c2);
    const __bf16* from = a.q + (size_t)b * a.q_b + (size_t)h * a.q_h + (size_t)t * a.q_t + 16 * g;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u32x4_t w = *reinterpret_cast<const u32x4_t*>(from + 64 * (k >> 1) + 8 * (k & 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] ^= flip;
      q[n][k] = __builtin_bit_cast(bf16x8_t, w);
    }
  }

  for (int first = wave; first < steps; first += 32 * kWaves) {
    const Blocks blocks = blocks_from(p, b, j, first, end_block);
    const int here = min(32, (steps - first + kWaves - 1) / kWaves);
    for (int i = 0; i < here; ++i) {
      const int row0 = 32 * (first + kWaves * i);
      int at[2];
      float ks[2], vs[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        at[m] = __builtin_amdgcn_readlane(blocks.at, 2 * i + m);
        ks[m] = row_lane(blocks.ks, 2 * i + m);
        vs[m] = row_lane(blocks.vs, 2 * i + m);
      }
      u32x4_t kq[2][2], vq[2][2];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) kq[m][h] = load_1k(p.k, at[m], h);
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) vq[m][h] = load_1k(p.v, at[m], h);

      f32x4_t s[NT][2];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bf16x8_t key = eight(kq[m][k >> 1][2 * (k & 1)], kq[m][k >> 1][2 * (k & 1) + 1], ks[m], ks[m]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            s[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key, q[n][k], k ? s[n][m] : f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
        }
      const bool masked = row0 + 32 > least || at[0] < 0 || at[1] < 0;
      bf16x8_t w[NT];
      if (!masked) {
#pragma unroll
        for (int n = 0; n < NT; ++n) w[n] = step_weights<false>(s[n], c2, st[n], [](int, int) { return true; });
      } else {
        // (a weight of zero does not take a NaN out of a product: those become zero here
        // and come back for the query rows that see them)
        unsigned found = 0;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) found |= nan_bytes(vq[m][h][e]);
        const bool special = __ballot(found != 0) != 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          auto seen = [&](int m, int e) { return row0 + 16 * m + 4 * g + e < limit[n] && at[m] >= 0; };
          w[n] = step_weights<true>(s[n], c2, st[n], seen);
          if (special) {
            bf16x8_t sees;
#pragma unroll
            for (int e = 0; e < 8; ++e) sees[e] = static_cast<__bf16>(seen(e / 4, e % 4) ? 1.f : 0.f);
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              const bf16x8_t nans = eight(nan_bytes(vq[0][d & 1][d >> 1]) & 0x38383838u,
                                          nan_bytes(vq[1][d & 1][d >> 1]) & 0x38383838u, 1.f, 1.f);
              const f32x4_t met =
                  __builtin_amdgcn_mfma_f32_16x16x32_bf16(nans, sees, f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (met[e] > 0.f) st[n].o[d][e] = __builtin_nanf("");
            }
          }
        }
        if (special) {
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
        for (int n = 0; n < NT; ++n)
          st[n].o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value, w[n], st[n].o[d], 0, 0, 0);
      }
    }
  }

#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (n) __syncthreads();
    const float l = rows_sum(st[n].l);
#pragma unroll
    for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4_t*>(&os[wave][c][16 * d + 4 * g]) = st[n].o[d];
    if (g == 0) {
      ms[wave][c] = st[n].m;
      ls[wave][c] = l;
    }
    __syncthreads();
    // 16 lanes to a query row, 8 dims each
    const int r = threadIdx.x >> 4;
    const int row = r0 + 16 * n + r;
    if (row < rows) {
      const int t = row / a.G, h = j * a.G + row % a.G;
      float m = neg_inf(), sum = 0.f, w[kWaves];
#pragma unroll
      for (int i = 0; i < kWaves; ++i) m = fmaxf(m, ms[i][r]);
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        w[i] = ms[i][r] == m ? 1.f : __builtin_amdgcn_exp2f(ms[i][r] - m);
        sum += w[i] * ls[i][r];
      }
      const bool none = t >= count || m == neg_inf();
      bf16x8_t o;
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kWaves; ++i) x += w[i] * *reinterpret_cast<const f32x4_t*>(&os[i][r][8 * (threadIdx.x & 15) + e]);
#pragma unroll
        for (int u = 0; u < 4; ++u) o[e + u] = static_cast<__bf16>(none ? 0.f : x[u] / sum);
      }
      *reinterpret_cast<bf16x8_t*>(a.out + (((size_t)b * a.T + t) * a.n_q + h) * D + 8 * (threadIdx.x & 15)) = o;
    }
  }
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t stream) {
  const int rows = a.T * a.G;
  const int nt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const dim3 grid((unsigned)a.pool.n_kv * a.B * ceil_div(rows, 16 * nt));
  if (nt == 1) launch_kernel(paged_attention_kernel<1>, grid, dim3(kThreads), 0, stream, a);
  if (nt == 2) launch_kernel(paged_attention_kernel<2>, grid, dim3(kThreads), 0, stream, a);
  if (nt == 4) launch_kernel(paged_attention_kernel<4>, grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace lsk
