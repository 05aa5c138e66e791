// Pages of an 8-bit key/value cache for gfx950: new rows in, rows out, pages copied.
//
// 16 rows of a kv head are a block of 16 x 128 e4m3 bytes with one exponent e,
//   value = byte 2^e,  e the least with |x| <= 448 2^e over the block's rows,
// for keys and values apart.  With a power of two as scale a stored value is exact
// in bf16 (one conversion instruction), e comes from the exponent bits of the largest
// |x|, and rows that are rounded again because a later row of their block is larger
// lose bits only where they fall below e4m3's normal range.
//
// A block's bytes are in the order in which the attention's lanes take them (a page is
// its blocks one behind the other):
//   K: row t, dim d at (d / 64) 1024 + ((d / 16) % 4 * 16 + t) 16 + d % 16
//   V: row t, dim d at (d / 16 % 2) 1024 + (t / 4 * 16 + d % 16) 16 + d / 32 * 4 + t % 4
// so that 16 bytes a lane are 1 KB in a row, K by rows and V by dims.
//
// All three are bound by their bytes, the small calls by one chain of latencies
// (lens, table, rows, store): appends of 32 x 2000 rows 81 us and reads of them 82, 4.8 TB/s, single
// rows of 64 requests 5.4 and 4.3 us; 50 pages of 64 rows in 36 layers copied in 99 us, 4.8 TB/s.
// Appends and reads of a row touch what holds it, not its block: 256 single rows all over a pool
// 11.0 us for 13.8.

#include <hip/hip_runtime.h>

#include "lsk_internal.h"

namespace lsk {
namespace {

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr unsigned kNaN = 0x7fu;

// 2^n; 0 below the normal range.
__device__ __forceinline__ float power_of_two(int n) {
  return n < -126 ? 0.f : __builtin_bit_cast(float, (unsigned)(n + 127) << 23);
}

// Four floats within +-448 as e4m3 bytes.
__device__ __forceinline__ unsigned four_bytes(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Which bytes of a word are NaN, as 0xff each.
__device__ __forceinline__ unsigned nan_bytes(unsigned w) {
  const unsigned t = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // 0x7f + 1: no carry beyond a byte
  return (t >> 7) * 0xffu;
}

// Four stored bytes rounded again with `factor` (a power of two below 1).
__device__ __forceinline__ unsigned again(unsigned w, float factor) {
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  const unsigned nan = nan_bytes(w);
  return (four_bytes(lo[0] * factor, lo[1] * factor, hi[0] * factor, hi[1] * factor) & ~nan) | (nan & 0x7f7f7f7fu);
}

// Four bf16 values (two words) in units of 1 / factor.
__device__ __forceinline__ unsigned rounded(unsigned w0, unsigned w1, float factor) {
  const unsigned bits[4] = {w0 << 16, w0 & 0xffff0000u, w1 << 16, w1 & 0xffff0000u};
  float f[4];
  unsigned nan = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool fine = (bits[e] & 0x7f800000u) != 0x7f800000u;
    f[e] = fine ? __builtin_amdgcn_fmed3f(__builtin_bit_cast(float, bits[e]) * factor, -448.f, 448.f) : 0.f;
    nan |= fine ? 0u : 0xffu << (8 * e);
  }
  return (four_bytes(f[0], f[1], f[2], f[3]) & ~nan) | (nan & 0x7f7f7f7fu);
}

// Larger of the finite |x| in both halves of a word of bf16, as bits.
__device__ __forceinline__ unsigned top_of(unsigned w, unsigned top) {
  const unsigned lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
  if (lo < 0x7f80u && lo > top) top = lo;
  if (hi < 0x7f80u && hi > top) top = hi;
  return top;
}

// The least e with x <= 448 2^e for a bf16's bits (448 = 1.75 * 2^8).
__device__ __forceinline__ int exponent_of(unsigned top) {
  const int e = (int)(top >> 7) - 127 - 8 + ((top & 0x7fu) > 0x60u ? 1 : 0);
  return min(max(e, kPagedLeastExponent), kPagedMostExponent);
}

// Where block `block` of request b lies: its number in the pool for kv head j, or -1.
__device__ __forceinline__ long long block_in_pool(const PagedPool& p, int b, int j, int block) {
  const int page = p.table[(size_t)b * p.table_ld + (block >> p.page_shift)];
  if ((unsigned)page >= (unsigned)p.pages) return -1;
  return (((long long)page * p.n_kv + j) << p.page_shift) | (block & ((1 << p.page_shift) - 1));
}

// One wave per block that new rows fall into, K or V of one kv head.
__global__ __launch_bounds__(kThreads) void append_kernel(PagedAppendArgs a) {
  __shared__ unsigned rows[kWaves][16][33];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const PagedPool& p = a.pool;
  const long long unit = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * kWaves + wave));
  const int kv = (int)(unit & 1), j = (int)(unit / 2 % p.n_kv);
  const int w = (int)(unit / 2 / p.n_kv % a.windows), b = (int)(unit / 2 / p.n_kv / a.windows);
  if (b >= a.B) return;
  const int len = max(a.lens[b], 0);
  const int count = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  const int start = len - count;  // of the new rows; those before row 0 are dropped
  const int block = max(start, 0) / 16 + w;
  if (block >= p.blocks) return;
  const int row0 = block * 16;
  const int first = max(start, row0), end = min(len, row0 + 16);
  if (first >= end) return;
  const long long at = block_in_pool(p, b, j, block);
  if (at < 0) return;
  const int begun = first - row0;
  unsigned char* out = (kv ? p.v : p.k) + at * kPagedBlockBytes;
  unsigned char* exponent = (kv ? p.v_exp : p.k_exp) + at;

  // Row c of the block, dims 64 h + 16 g .. + 15.
  u32x4_t x[2][2] = {};
  const bool fresh = row0 + c >= first && row0 + c < end;
  if (fresh) {
    const __bf16* src = kv ? a.v + (size_t)b * a.v_b + (size_t)j * a.v_h + (size_t)(row0 + c - start) * a.v_t
                           : a.k + (size_t)b * a.k_b + (size_t)j * a.k_h + (size_t)(row0 + c - start) * a.k_t;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i) x[h][i] = *reinterpret_cast<const u32x4_t*>(src + 64 * h + 16 * g + 8 * i);
  }
  // What the block holds, of V, whose words hold four rows, next to the new ones.
  const int new_of_four = min(end, row0 + 4 * g + 4) - max(first, row0 + 4 * g);
  u32x4_t old[2] = {};
  if (kv && new_of_four > 0 && new_of_four < 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) old[h] = *reinterpret_cast<const u32x4_t*>(out + h * 1024 + lane * 16);
  }
  const int was = begun > 0 ? (int)*exponent - 127 : 0;

  unsigned top = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = top_of(x[h][i][e], top);
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, s));
  int e = exponent_of(top);
  if (begun > 0) e = max(e, was);
  const float factor = power_of_two(-e);
  const bool move = begun > 0 && e != was;
  const float less = power_of_two(was - e);
  if (move) {  // (seldom: then all in front of the new rows is rounded again)
#pragma unroll
    for (int h = 0; h < 2; ++h) old[h] = *reinterpret_cast<const u32x4_t*>(out + h * 1024 + lane * 16);
  }

  u32x4_t q[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) q[h][i] = rounded(x[h][i >> 1][2 * (i & 1)], x[h][i >> 1][2 * (i & 1) + 1], factor);

  if (kv == 0) {
    const bool moved = move && row0 + c < first;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (moved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) q[h][i] = again(old[h][i], less);
      }
      if (fresh || moved) *reinterpret_cast<u32x4_t*>(out + h * 1024 + lane * 16) = q[h];
    }
  } else {
    // Rows to columns: lane (c, g) gets rows 4 g .. + 3 of dims 32 i + 16 h + c.
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) rows[wave][c][16 * h + 4 * g + i] = q[h][i];
    wave_lds_order();
    const auto* bytes = reinterpret_cast<const unsigned char*>(&rows[wave][0][0]);
    unsigned is_new = 0, is_old = 0;  // bytes of a word
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = row0 + 4 * g + r;
      if (row >= first && row < end) is_new |= 0xffu << (8 * r);
      if (row < first) is_old |= 0xffu << (8 * r);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4_t o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned t = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) t |= (unsigned)bytes[(4 * g + r) * 132 + 32 * i + 16 * h + c] << (8 * r);
        unsigned before = old[h][i];
        if (move) before = (again(before, less) & is_old) | (before & ~is_old);
        o[i] = (t & is_new) | (before & ~is_new);
      }
      if (new_of_four > 0 || move) *reinterpret_cast<u32x4_t*>(out + h * 1024 + lane * 16) = o;
    }
  }
  if (lane == 0) *exponent = (unsigned char)(e + 127);
}

// One wave per block of a request's rows start .. start + rows - 1, K or V of one kv head.
__global__ __launch_bounds__(kThreads) void read_kernel(PagedReadArgs a) {
  __shared__ unsigned rows[kWaves][16][33];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const PagedPool& p = a.pool;
  const long long unit = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * kWaves + wave));
  const int kv = (int)(unit & 1), j = (int)(unit / 2 % p.n_kv);
  const int w = (int)(unit / 2 / p.n_kv % a.windows), b = (int)(unit / 2 / p.n_kv / a.windows);
  if (b >= a.B) return;
  const int start = max(a.starts[b], 0);
  const long long row0 = ((long long)start / 16 + w) * 16;
  const long long row = row0 + c;  // the lane's row
  const bool wanted = row >= start && row < (long long)start + a.rows;
  const int len = a.lens ? max(a.lens[b], 0) : 0x7fffffff;
  u32x4_t q[2] = {};
  float scale = 1.f;
  long long at = -1;
  if (row0 < len && row0 / 16 < p.blocks) at = block_in_pool(p, b, j, (int)(row0 / 16));
  if (at >= 0) {
    const unsigned char* from = (kv ? p.v : p.k) + at * kPagedBlockBytes;
    // the lane's row of K, four rows of V: if one is wanted
    const long long low = row0 + (kv ? 4 * g : c), high = low + (kv ? 4 : 1);
    if (high > start && low < (long long)start + a.rows && low < len) {
#pragma unroll
      for (int h = 0; h < 2; ++h) q[h] = *reinterpret_cast<const u32x4_t*>(from + h * 1024 + lane * 16);
    }
    scale = power_of_two((int)(kv ? p.v_exp : p.k_exp)[at] - 127);
    if (kv) {
      auto* bytes = reinterpret_cast<unsigned char*>(&rows[wave][0][0]);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) bytes[(4 * g + r) * 132 + 32 * i + 16 * h + c] = (unsigned char)(q[h][i] >> (8 * r));
      wave_lds_order();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) q[h][i] = rows[wave][c][16 * h + 4 * g + i];
    }
  }
  if (!wanted) return;
  const bool there = at >= 0 && row < len;
  __bf16* out = (kv ? a.v : a.k) + (((size_t)b * p.n_kv + j) * a.rows + (size_t)(row - start)) * kAttnHeadDim;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      u32x4_t o;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned word = there ? q[h][2 * i + u] : 0u;
        o[2 * u] = __builtin_bit_cast(unsigned, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, false));
        o[2 * u + 1] = __builtin_bit_cast(unsigned, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, true));
      }
      *reinterpret_cast<u32x4_t*>(out + 64 * h + 16 * g + 8 * i) = o;
    }
}

// A part of one page of one layer's K or V per workgroup; the first part's moves the exponents too.
constexpr int kCopyAhead = 4;
__global__ __launch_bounds__(kThreads) void copy_kernel(PagedCopyArgs a) {
  int id = blockIdx.x;
  const int part = id % a.parts;
  id /= a.parts;
  const int plane = id % a.planes, n = id / a.planes;
  const int src = a.src[n], dst = a.dst[n];
  if ((unsigned)src >= (unsigned)a.pages || (unsigned)dst >= (unsigned)a.pages || src == dst) return;
  const size_t blocks = (size_t)a.page_blocks;
  const size_t from = ((size_t)plane * a.pages + src) * blocks, to = ((size_t)plane * a.pages + dst) * blocks;
  const auto* x = reinterpret_cast<const u32x4_t*>(a.storage + from * kPagedBlockBytes);
  auto* y = reinterpret_cast<u32x4_t*>(a.storage + to * kPagedBlockBytes);
  const int units = a.page_blocks * (kPagedBlockBytes / 16);  // (at most 2^27)
  const int u0 = part * kThreads * kCopyAhead + threadIdx.x;
  u32x4_t held[kCopyAhead];
#pragma unroll
  for (int i = 0; i < kCopyAhead; ++i)
    if (u0 + i * kThreads < units) held[i] = x[u0 + i * kThreads];
#pragma unroll
  for (int i = 0; i < kCopyAhead; ++i)
    if (u0 + i * kThreads < units) y[u0 + i * kThreads] = held[i];
  if (part == 0)
    for (int i = threadIdx.x; i < a.page_blocks; i += kThreads) a.exponents[to + i] = a.exponents[from + i];
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t stream) {
  const long long units = 2ll * a.B * a.windows * a.pool.n_kv;
  launch_kernel(append_kernel, dim3((unsigned)((units + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_paged_read(const PagedReadArgs& a, hipStream_t stream) {
  const long long units = 2ll * a.B * a.windows * a.pool.n_kv;
  launch_kernel(read_kernel, dim3((unsigned)((units + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_paged_copy(PagedCopyArgs a, hipStream_t stream) {
  a.parts = ceil_div((long long)a.page_blocks * (kPagedBlockBytes / 16), kThreads * kCopyAhead);
  launch_kernel(copy_kernel, dim3((unsigned)a.n * a.planes * a.parts), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace lsk
