// Host-side rules of the C ABI (declared in lsk_host.h): the packers, the
// argument validators and the thread-local message of lsk_last_error().
// Plain C++ with no HIP dependency, so the sanitizer test builds and runs it
// with g++ -fsanitize=address.  The Python layer turns LSK_ERR_INVALID /
// LSK_ERR_LAYOUT into ValueError, the way
// src/leanstack/runtime/cutile_logits.py:44-53 rejects bad input before
// launching.

#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <string>

#include "leanstack_amd.h"
#include "lsk_host.h"

namespace lsk {
namespace {

thread_local std::string g_last_error;

bool packed_layout(int layout_id) {
  return layout_id == LSK_LAYOUT_MFMA16X32 || layout_id == LSK_LAYOUT_MFMA16X32_GATEUP;
}

// Row of the row-major source matrix stored in packed row `pr`.
inline int source_row(int layout_id, int N, int pr) {
  if (layout_id != LSK_LAYOUT_MFMA16X32_GATEUP) return pr;
  const int half = N / 2;
  const int pair = pr / (2 * kTileRows);
  const int within = pr % (2 * kTileRows);
  return within < kTileRows ? pair * kTileRows + within : half + pair * kTileRows + (within - kTileRows);
}

// Byte offset (in 16-byte units) of W[packed row pr][k8 * 8 .. +8] in the tiles.
inline size_t packed_unit(int K, int pr, int k8) {
  const int KT = K / kTileK;
  const int rb = pr / kTileRows;
  const int r = pr % kTileRows;
  const int kt = k8 / 4;
  const int gq = k8 % 4;
  return ((size_t)rb * KT + kt) * 64 + (size_t)gq * 16 + r;
}

}  // namespace

int fail(int status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return status;
}

void clear_error() { g_last_error.clear(); }

const char* error_message() { return g_last_error.c_str(); }

bool attention_group_supported(int group) { return group == 1 || group == 2 || group == 4 || group == 8; }

int check_shape(int layout_id, int N, int K) {
  if (!packed_layout(layout_id)) return fail(LSK_ERR_LAYOUT, "unsupported weight layout id %d", layout_id);
  if (N <= 0 || K <= 0) return fail(LSK_ERR_INVALID, "N=%d and K=%d must be positive", N, K);
  if (N % kTileRows != 0) return fail(LSK_ERR_INVALID, "N=%d must be divisible by %d", N, kTileRows);
  if (K % kTileK != 0) return fail(LSK_ERR_INVALID, "K=%d must be divisible by %d", K, kTileK);
  if (layout_id == LSK_LAYOUT_MFMA16X32_GATEUP && N % (2 * kTileRows) != 0)
    return fail(LSK_ERR_INVALID, "fused gate_up N=%d must be divisible by %d", N, 2 * kTileRows);
  return LSK_OK;
}

int check_linear_args(const void* w_packed, int layout_id, int N, int K, const void* x, int M, int ldx,
                      const void* y, int ldy, int epilogue, const void* residual, int ldr) {
  if (int st = check_shape(layout_id, N, K)) return st;
  if (epilogue != LSK_EPI_NONE && epilogue != LSK_EPI_SILU_MUL && epilogue != LSK_EPI_RESIDUAL_ADD)
    return fail(LSK_ERR_INVALID, "unknown epilogue %d", epilogue);
  if ((epilogue == LSK_EPI_SILU_MUL) != (layout_id == LSK_LAYOUT_MFMA16X32_GATEUP))
    return fail(LSK_ERR_INVALID, "the SiLU*up epilogue requires the interleaved gate_up layout and vice versa");
  if (M < 1) return fail(LSK_ERR_INVALID, "M=%d must be >= 1", M);
  if (w_packed == nullptr || x == nullptr || y == nullptr) return fail(LSK_ERR_INVALID, "null device pointer");
  if (!aligned(w_packed, 16)) return fail(LSK_ERR_INVALID, "packed weights must be 16-byte aligned");
  if (ldx < K || ldx % 8 != 0 || !aligned(x, 16))
    return fail(LSK_ERR_INVALID, "x needs ldx >= K, ldx %% 8 == 0 and 16-byte alignment (ldx=%d, K=%d)", ldx, K);
  if (ldx > kMaxActivationStride)
    return fail(LSK_ERR_INVALID, "ldx=%d exceeds the largest activation row stride, %d", ldx, kMaxActivationStride);
  const int n_out = epilogue == LSK_EPI_SILU_MUL ? N / 2 : N;
  if (ldy < n_out || ldy % 4 != 0 || !aligned(y, 8))
    return fail(LSK_ERR_INVALID, "y needs ldy >= %d, ldy %% 4 == 0 and 8-byte alignment (ldy=%d)", n_out, ldy);
  if (epilogue == LSK_EPI_RESIDUAL_ADD) {
    if (residual == nullptr || ldr < N || !aligned(residual, 2))
      return fail(LSK_ERR_INVALID, "residual add needs a residual [M][N] with ldr >= N (ldr=%d)", ldr);
  } else if (residual != nullptr) {
    return fail(LSK_ERR_INVALID, "residual given without the residual-add epilogue");
  }
  return LSK_OK;
}

int check_rmsnorm_args(const void* x, int M, int K, int ldx, const void* norm_weight, float eps, const void* y) {
  if (M < 1) return fail(LSK_ERR_INVALID, "M=%d must be positive", M);
  if (K < 512 || K > 4096 || K % 512 != 0) return fail(LSK_ERR_INVALID, "K=%d must be a multiple of 512 up to 4096", K);
  if (ldx < K || ldx % 8 != 0) return fail(LSK_ERR_INVALID, "ldx=%d must be a multiple of 8, at least K=%d", ldx, K);
  if (x == nullptr || norm_weight == nullptr || y == nullptr) return fail(LSK_ERR_INVALID, "null device pointer");
  if (!aligned(x, 16) || !aligned(norm_weight, 16) || !aligned(y, 16))
    return fail(LSK_ERR_INVALID, "x, norm_weight and y must be 16-byte aligned");
  if (!std::isfinite(eps) || eps < 0.f) return fail(LSK_ERR_INVALID, "eps=%g must be finite and >= 0", (double)eps);
  return LSK_OK;
}

int check_qk_rope_args(const void* qkv, int B, int T, int ld, int n_q, int n_kv, int head_dim,
                       const void* q_norm_weight, const void* k_norm_weight, float eps, const void* cos,
                       const void* sin, long long rope_batch_stride, long long rope_row_stride, const void* q_out,
                       const void* k_out) {
  if (head_dim != kAttnHeadDim)
    return fail(LSK_ERR_INVALID, "head_dim=%d: the row kernel is built for %d", head_dim, kAttnHeadDim);
  if (n_q < 1 || n_kv < 1 || n_q > 4096 || n_kv > 4096)
    return fail(LSK_ERR_INVALID, "n_q=%d, n_kv=%d must be 1..4096", n_q, n_kv);
  if (B < 1 || T < 1 || (long long)B * T > 0x7fffffffLL) return fail(LSK_ERR_INVALID, "B=%d, T=%d rows", B, T);
  if (ld < (n_q + n_kv) * head_dim || ld % 8 != 0)
    return fail(LSK_ERR_INVALID, "ld=%d must be a multiple of 8, at least %d", ld, (n_q + n_kv) * head_dim);
  if (rope_batch_stride < 0 || rope_row_stride < 0 || rope_batch_stride % 8 != 0 || rope_row_stride % 8 != 0)
    return fail(LSK_ERR_INVALID, "the cos / sin strides must be multiples of 8, not negative");
  const void* all[] = {qkv, q_norm_weight, k_norm_weight, cos, sin, q_out, k_out};
  for (const void* p : all) {
    if (p == nullptr) return fail(LSK_ERR_INVALID, "null device pointer");
    if (!aligned(p, 16)) return fail(LSK_ERR_INVALID, "device pointers must be 16-byte aligned");
  }
  if (!std::isfinite(eps) || eps < 0.f) return fail(LSK_ERR_INVALID, "eps=%g must be finite and >= 0", (double)eps);
  return LSK_OK;
}

int check_attention_args(const void* qkv, int n_q, int n_kv, int head_dim, const void* q_norm_weight,
                         const void* k_norm_weight, float eps, const void* cos, const void* sin, const void* k_cache,
                         const void* v_cache, int max_seq_len, float scale, const void* out) {
  if (head_dim != kAttnHeadDim)
    return fail(LSK_ERR_INVALID, "head_dim=%d: the attention kernel is built for %d", head_dim, kAttnHeadDim);
  if (n_kv < 1 || n_kv > kAttnMaxKvHeads || n_q < n_kv || n_q % n_kv != 0 || !attention_group_supported(n_q / n_kv))
    return fail(LSK_ERR_INVALID, "n_q=%d, n_kv=%d: n_kv must be 1..%d and n_q 1, 2, 4 or 8 times n_kv", n_q, n_kv,
                kAttnMaxKvHeads);
  if (qkv == nullptr || q_norm_weight == nullptr || k_norm_weight == nullptr || cos == nullptr || sin == nullptr ||
      k_cache == nullptr || v_cache == nullptr || out == nullptr)
    return fail(LSK_ERR_INVALID, "null device pointer");
  if (!aligned(qkv, 2) || !aligned(q_norm_weight, 2) || !aligned(k_norm_weight, 2) || !aligned(cos, 2) ||
      !aligned(sin, 2) || !aligned(out, 2))
    return fail(LSK_ERR_INVALID, "bf16 arguments must be 2-byte aligned");
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16))
    return fail(LSK_ERR_INVALID, "the key and value caches must be 16-byte aligned");
  if (max_seq_len < 1 || max_seq_len > kAttnMaxRows)
    return fail(LSK_ERR_INVALID, "max_seq_len=%d: need 1 <= max_seq_len <= %d", max_seq_len, kAttnMaxRows);
  if (!std::isfinite(eps) || eps < 0.f) return fail(LSK_ERR_INVALID, "eps=%g must be finite and >= 0", (double)eps);
  if (!std::isfinite(scale)) return fail(LSK_ERR_INVALID, "scale must be finite");
  return LSK_OK;
}

int check_constrain_args(const void* logits, int logits_mode, int M, int V, long long logits_ld, const int* history,
                         long long history_ld, int history_len, const int* history_lens, const int* prompt_lens,
                         const float* repetition, const float* frequency, const float* presence, const int* bias_ids,
                         const float* bias_values, long long bias_ld, int bias_count, const int* allowed,
                         long long allowed_ld, const void* out, const long long* tokens) {
  if (logits_mode != LSK_LOGITS_FP32 && logits_mode != LSK_LOGITS_BF16)
    return fail(LSK_ERR_INVALID, "unknown logits mode %d", logits_mode);
  if (M < 1 || V < 1 || V > (1 << 30)) return fail(LSK_ERR_INVALID, "M=%d rows of V=%d values", M, V);
  if ((long long)M * constrain_slices(M, V) > 0xffffffffLL / kConstrainThreads)  // a grid's threads are counted in 32 bits
    return fail(LSK_ERR_INVALID, "M=%d rows of V=%d values are too many", M, V);
  if (logits == nullptr || out == nullptr || tokens == nullptr) return fail(LSK_ERR_INVALID, "null device pointer");
  const uintptr_t item = logits_mode == LSK_LOGITS_FP32 ? 4 : 2;
  if (!aligned(logits, item) || !aligned(out, item) || !aligned(tokens, 8))
    return fail(LSK_ERR_INVALID, "logits, out and tokens must be aligned to their values");
  if (logits_ld < V) return fail(LSK_ERR_INVALID, "logits_ld=%lld must be at least V=%d", logits_ld, V);
  if (logits == out && logits_ld != V) return fail(LSK_ERR_INVALID, "in place, the logits' rows must be contiguous");
  if (history != nullptr) {
    if (history_len < 1 || history_len > kConstrainMaxHistory || history_ld < history_len)
      return fail(LSK_ERR_INVALID, "history of %d tokens (1..%d) at stride %lld", history_len, kConstrainMaxHistory,
                  history_ld);
  } else if (history_lens || prompt_lens || repetition || frequency || presence) {
    return fail(LSK_ERR_INVALID, "lengths or penalties given without a history");
  }
  if (bias_count < 0 || bias_count > kConstrainMaxBias)
    return fail(LSK_ERR_INVALID, "bias_count=%d must be 0..%d", bias_count, kConstrainMaxBias);
  if (bias_count > 0 && (bias_ids == nullptr || bias_values == nullptr || bias_ld < bias_count))
    return fail(LSK_ERR_INVALID, "%d biases need their ids and values at a stride of at least that (%lld)", bias_count,
                bias_ld);
  if (allowed != nullptr && allowed_ld < (V + 31) / 32)
    return fail(LSK_ERR_INVALID, "allowed_ld=%lld must be at least %d words", allowed_ld, (V + 31) / 32);
  const void* words[] = {history,  history_lens, prompt_lens, repetition, frequency,
                         presence, bias_ids,     bias_values, allowed};
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(LSK_ERR_INVALID, "32-bit arguments must be 4-byte aligned");
  return LSK_OK;
}

int check_sample_sizes(int logits_mode, int M, int V) {
  if (logits_mode != LSK_LOGITS_FP32 && logits_mode != LSK_LOGITS_BF16)
    return fail(LSK_ERR_INVALID, "unknown logits mode %d", logits_mode);
  if (M < 1 || V < 1 || V > kSampleMaxVocab)
    return fail(LSK_ERR_INVALID, "M=%d rows of V=%d values (at most %d)", M, V, kSampleMaxVocab);
  if (M > (int)(0xffffffffLL / 1024)) return fail(LSK_ERR_INVALID, "M=%d rows are too many", M);
  return LSK_OK;
}

int check_sample_args(const void* logits, int logits_mode, int M, int V, long long logits_ld, const float* uniforms,
                      const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                      const long long* tokens, const float* logprobs) {
  if (int st = check_sample_sizes(logits_mode, M, V)) return st;
  if (logits_ld < V) return fail(LSK_ERR_INVALID, "logits_ld=%lld must be at least V=%d", logits_ld, V);
  if (logits == nullptr || uniforms == nullptr || tokens == nullptr || logprobs == nullptr)
    return fail(LSK_ERR_INVALID, "null device pointer");
  if (!aligned(logits, logits_mode == LSK_LOGITS_FP32 ? 4 : 2) || !aligned(tokens, 8))
    return fail(LSK_ERR_INVALID, "the logits must be aligned to their type, the tokens to 8 bytes");
  const void* words[] = {uniforms, temperature, top_k, top_p, min_p, logprobs};
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(LSK_ERR_INVALID, "32-bit arguments must be 4-byte aligned");
  return LSK_OK;
}

int check_prefix_sizes(int B, int T, int n_q, int n_kv, int P, int S) {
  if (n_kv < 1 || n_q < n_kv || n_q % n_kv != 0)
    return fail(LSK_ERR_INVALID, "n_q=%d must be a multiple of n_kv=%d", n_q, n_kv);
  if (B < 1 || T < 1 || P < 0 || S < 0) return fail(LSK_ERR_INVALID, "B=%d, T=%d, P=%d, S=%d rows", B, T, P, S);
  // Query rows and grids are counted in 32 bits, key rows addressed with 31 (the plan
  // is made of sizes that keep to both).
  const long long most = 0xffffffffLL / kPrefixThreads;
  if ((long long)B * T > most || (long long)B * T * n_q > most)
    return fail(LSK_ERR_INVALID, "B=%d, T=%d, n_q=%d: too many query rows", B, T, n_q);
  constexpr int most_rows = ((1 << 30) - 1) / kAttnHeadDim;
  if (P > most_rows || S > most_rows)
    return fail(LSK_ERR_INVALID, "%d and %d rows: a head's rows must stay below 2^31 bytes", P, S);
  const PrefixPlan p = prefix_plan(B, T, n_q, n_kv, P, S);
  const long long prefix_items = (long long)n_kv * p.prefix_tiles * p.prefix_parts;
  const long long own_items = (long long)n_kv * B * p.own_tiles;
  if (own_items > most || prefix_items > most || prefix_items + own_items * (p.joint ? 1 : p.own_parts) > most)
    return fail(LSK_ERR_INVALID, "B=%d, T=%d, n_q=%d over %d + %d rows: too many items", B, T, n_q, P, S);
  return LSK_OK;
}

int check_prefix_args(const void* q, long long q_batch, long long q_head, long long q_token, int B, int T, int n_q,
                      int n_kv, int head_dim, const void* prefix_k, const void* prefix_v, long long prefix_head,
                      int prefix_row, int P, const void* k, const void* v, long long batch, long long head, int row,
                      int S, const int* lens, float scale, const void* out) {
  if (head_dim != kAttnHeadDim)
    return fail(LSK_ERR_INVALID, "head_dim=%d: the attention kernel is built for %d", head_dim, kAttnHeadDim);
  if (int st = check_prefix_sizes(B, T, n_q, n_kv, P, S)) return st;
  // (a few steps past the last row are addressed, out of range: their offsets must not wrap)
  if (prefix_row < head_dim || row < head_dim || prefix_row % 8 != 0 || row % 8 != 0 ||
      prefix_row > kMaxActivationStride || row > kMaxActivationStride)
    return fail(LSK_ERR_INVALID, "row strides %d, %d must be multiples of 8, %d..%d", prefix_row, row, head_dim,
                kMaxActivationStride);
  if ((long long)P * prefix_row >= (1LL << 30) || (long long)S * row >= (1LL << 30))
    return fail(LSK_ERR_INVALID, "%d and %d rows at strides %d and %d: a head's rows must stay below 2^31 bytes", P, S,
                prefix_row, row);
  const long long strides[] = {q_batch, q_head, q_token, prefix_head, batch, head};
  for (long long s : strides)
    if (s < 0 || s % 8 != 0) return fail(LSK_ERR_INVALID, "strides must be multiples of 8, not negative (%lld)", s);
  if (q == nullptr || lens == nullptr || out == nullptr || (P > 0 && (prefix_k == nullptr || prefix_v == nullptr)) ||
      (S > 0 && (k == nullptr || v == nullptr)))
    return fail(LSK_ERR_INVALID, "null device pointer");
  const void* wide[] = {q, prefix_k, prefix_v, k, v, out};
  for (const void* w : wide)
    if (!aligned(w, 16)) return fail(LSK_ERR_INVALID, "q, the keys and values and out must be 16-byte aligned");
  if (!aligned(lens, 4)) return fail(LSK_ERR_INVALID, "lens must be 4-byte aligned");
  if (!std::isfinite(scale * 1.44269504088896341f))  // (scores are taken to base 2)
    return fail(LSK_ERR_INVALID, "scale=%g must be finite, also times log2(e)", (double)scale);
  return LSK_OK;
}

int check_paged_pool(const lsk_paged_pool* p) {
  if (p == nullptr) return fail(LSK_ERR_INVALID, "null pool");
  if (p->page_rows < kPagedBlockRows || p->page_rows > kPagedMostPageRows || (p->page_rows & (p->page_rows - 1)) != 0)
    return fail(LSK_ERR_INVALID, "page_rows=%d must be a power of two, %d..%d", p->page_rows, kPagedBlockRows,
                kPagedMostPageRows);
  if (p->pages < 1 || p->n_kv < 1 || p->table_pages < 1)
    return fail(LSK_ERR_INVALID, "pages=%d, n_kv=%d and table_pages=%d must be positive", p->pages, p->n_kv, p->table_pages);
  // Blocks are numbered in 31 bits, and so are a request's rows with some to spare.
  const long long page_blocks = p->page_rows / kPagedBlockRows;
  if ((long long)p->n_kv * page_blocks > INT_MAX / p->pages)
    return fail(LSK_ERR_INVALID, "%d pages of %d heads: a layer must hold fewer than 2^31 blocks", p->pages, p->n_kv);
  if ((long long)p->table_pages * p->page_rows > (1LL << 30))
    return fail(LSK_ERR_INVALID, "%d pages of %d rows: a request holds at most 2^30", p->table_pages, p->page_rows);
  if (p->table_stride < p->table_pages)
    return fail(LSK_ERR_INVALID, "table_stride=%lld must be at least %d", p->table_stride, p->table_pages);
  const void* wide[] = {p->k_blocks, p->v_blocks};
  for (const void* w : wide)
    if (w == nullptr || !aligned(w, 16)) return fail(LSK_ERR_INVALID, "the pool's blocks must be 16-byte aligned");
  if (p->k_exponents == nullptr || p->v_exponents == nullptr) return fail(LSK_ERR_INVALID, "null exponents");
  if (p->table == nullptr || !aligned(p->table, 4)) return fail(LSK_ERR_INVALID, "the table must be 4-byte aligned");
  return LSK_OK;
}

namespace {

// One wave per unit: a grid's threads are counted in 32 bits.
int check_units(long long a, long long b, long long c) {
  constexpr long long most = 0xffffffffLL / 64 - 4;
  if (a > most || b > most || a * b > most || c > most || a * b * c > most)
    return fail(LSK_ERR_INVALID, "%lld x %lld x %lld: too many blocks for one call", a, b, c);
  return LSK_OK;
}

}  // namespace

int check_paged_append(const lsk_paged_pool* pool, const void* k, long long k_batch, long long k_head, long long k_token,
                       const void* v, long long v_batch, long long v_head, long long v_token, int B, int T,
                       const int* lens, const int* counts) {
  if (int st = check_paged_pool(pool)) return st;
  if (B < 1 || T < 1) return fail(LSK_ERR_INVALID, "B=%d requests of T=%d rows must be positive", B, T);
  if (int st = check_units(B, paged_windows(T), 2LL * pool->n_kv)) return st;
  const long long strides[] = {k_batch, k_head, k_token, v_batch, v_head, v_token};
  for (long long s : strides)
    if (s < 0 || s % 8 != 0) return fail(LSK_ERR_INVALID, "strides must be multiples of 8, not negative (%lld)", s);
  if (k == nullptr || v == nullptr || lens == nullptr) return fail(LSK_ERR_INVALID, "null device pointer");
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(LSK_ERR_INVALID, "k and v must be 16-byte aligned");
  if (!aligned(lens, 4) || !aligned(counts, 4)) return fail(LSK_ERR_INVALID, "lens and counts must be 4-byte aligned");
  return LSK_OK;
}

int check_paged_read(const lsk_paged_pool* pool, const int* starts, const int* lens, int B, int rows, const void* k,
                     const void* v) {
  if (int st = check_paged_pool(pool)) return st;
  if (B < 1 || rows < 1) return fail(LSK_ERR_INVALID, "B=%d requests of %d rows must be positive", B, rows);
  if (int st = check_units(B, paged_windows(rows), 2LL * pool->n_kv)) return st;
  if (starts == nullptr || k == nullptr || v == nullptr) return fail(LSK_ERR_INVALID, "null device pointer");
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(LSK_ERR_INVALID, "the outputs must be 16-byte aligned");
  if (!aligned(starts, 4) || !aligned(lens, 4)) return fail(LSK_ERR_INVALID, "starts and lens must be 4-byte aligned");
  return LSK_OK;
}

int check_paged_copy(const void* storage, const void* exponents, int planes, int pages, int page_blocks, const int* src,
                     const int* dst, int n) {
  if (planes < 1 || pages < 1 || page_blocks < 1 || n < 1)
    return fail(LSK_ERR_INVALID, "planes=%d, pages=%d, page_blocks=%d and n=%d must be positive", planes, pages,
                page_blocks, n);
  if (page_blocks > (1 << 20)) return fail(LSK_ERR_INVALID, "page_blocks=%d must be at most 2^20", page_blocks);
  // (16 KB to a workgroup of 4 waves)
  if (int st = check_units(n, planes, 4LL * ((page_blocks + 7) / 8))) return st;
  if (storage == nullptr || exponents == nullptr || src == nullptr || dst == nullptr)
    return fail(LSK_ERR_INVALID, "null device pointer");
  if (!aligned(storage, 16)) return fail(LSK_ERR_INVALID, "storage must be 16-byte aligned");
  if (!aligned(src, 4) || !aligned(dst, 4)) return fail(LSK_ERR_INVALID, "src and dst must be 4-byte aligned");
  return LSK_OK;
}

int check_paged_attention_sizes(int B, int T, int n_q, int n_kv, int capacity) {
  if (n_kv < 1 || n_q < n_kv || n_q % n_kv != 0)
    return fail(LSK_ERR_INVALID, "n_q=%d must be a multiple of n_kv=%d", n_q, n_kv);
  if (B < 1 || T < 1 || capacity < kPagedBlockRows || capacity % kPagedBlockRows != 0 || capacity > (1 << 30))
    return fail(LSK_ERR_INVALID, "B=%d, T=%d, %d rows", B, T, capacity);
  // Query rows and grids (of 512 threads a workgroup at most) are counted in 32 bits, units of
  // all a head's items in 31.
  const long long most = 0xffffffffLL / 512;
  if ((long long)B * T > most || (long long)B * T * n_q > most)
    return fail(LSK_ERR_INVALID, "B=%d, T=%d, n_q=%d: too many query rows", B, T, n_q);
  const PagedPlan p = paged_plan(B, T, n_q, n_kv, capacity);
  if (p.items * n_kv * (p.rows / 16) > most || p.workers * n_kv > most ||
      p.items * ((capacity + p.unit - 1) / p.unit + kPagedManyStart) > INT_MAX)
    return fail(LSK_ERR_INVALID, "B=%d, T=%d, n_q=%d over %d rows: too many items", B, T, n_q, capacity);
  return LSK_OK;
}

int check_paged_attention(const lsk_paged_pool* pool, const void* q, long long q_batch, long long q_head,
                          long long q_token, int B, int T, int n_q, int head_dim, const int* lens, const int* counts,
                          float scale, const void* out) {
  if (head_dim != kAttnHeadDim)
    return fail(LSK_ERR_INVALID, "head_dim=%d: the attention kernel is built for %d", head_dim, kAttnHeadDim);
  if (int st = check_paged_pool(pool)) return st;
  if (int st = check_paged_attention_sizes(B, T, n_q, pool->n_kv, pool->table_pages * pool->page_rows)) return st;
  const long long strides[] = {q_batch, q_head, q_token};
  for (long long s : strides)
    if (s < 0 || s % 8 != 0) return fail(LSK_ERR_INVALID, "strides must be multiples of 8, not negative (%lld)", s);
  if (q == nullptr || lens == nullptr || out == nullptr) return fail(LSK_ERR_INVALID, "null device pointer");
  if (!aligned(q, 16) || !aligned(out, 16)) return fail(LSK_ERR_INVALID, "q and out must be 16-byte aligned");
  if (!aligned(lens, 4) || !aligned(counts, 4)) return fail(LSK_ERR_INVALID, "lens and counts must be 4-byte aligned");
  if (!(std::fabs(scale) <= 0x1p120f)) return fail(LSK_ERR_INVALID, "scale=%g must be at most 2^120", (double)scale);
  return LSK_OK;
}

int check_lora_sizes(int M, int N, int K, int rank_tiles, int count, int epilogue) {
  if (epilogue != LSK_EPI_NONE && epilogue != LSK_EPI_SILU_MUL)
    return fail(LSK_ERR_INVALID, "epilogue %d: the adapters take none or SiLU*up", epilogue);
  if (int st = check_shape(epilogue == LSK_EPI_SILU_MUL ? LSK_LAYOUT_MFMA16X32_GATEUP : LSK_LAYOUT_MFMA16X32, N, K))
    return st;
  if (M < 1 || count < 1) return fail(LSK_ERR_INVALID, "M=%d rows and %d adapters must be positive", M, count);
  if (!adapter_rank_supported(rank_tiles))
    return fail(LSK_ERR_INVALID, "rank_tiles=%d: the rank must be 16, 32, 48, 64, 96 or 128", rank_tiles);
  if (N > kMaxActivationStride || K > kMaxActivationStride)
    return fail(LSK_ERR_INVALID, "N=%d and K=%d must be at most %d", N, K, kMaxActivationStride);
  const AdapterPlan p = adapter_plan(M, N, K, rank_tiles, count, epilogue == LSK_EPI_SILU_MUL);
  const long long groups = (long long)p.tiles * p.slots;
  if (groups * (p.ranges > p.splits ? p.ranges : p.splits) > 0xffffffffLL / kAdapterThreads)
    return fail(LSK_ERR_INVALID, "M=%d rows are too many", M);  // a grid's threads are counted in 32 bits
  return LSK_OK;
}

int check_lora_args(const void* y, int M, int N, int ldy, const void* x, int K, int ldx, const void* a_tiles,
                    const void* b_tiles, const float* scale, const int* ranks, int count, int rank_tiles,
                    const int* index, int epilogue, const void* out) {
  if (int st = check_lora_sizes(M, N, K, rank_tiles, count, epilogue)) return st;
  if (ldx < K || ldx % 8 != 0 || ldx > kMaxActivationStride)
    return fail(LSK_ERR_INVALID, "ldx=%d must be a multiple of 8, K=%d..%d", ldx, K, kMaxActivationStride);
  if (ldy < N || ldy % 8 != 0 || ldy > kMaxActivationStride)
    return fail(LSK_ERR_INVALID, "ldy=%d must be a multiple of 8, N=%d..%d", ldy, N, kMaxActivationStride);
  const void* wide[] = {y, x, a_tiles, b_tiles, out};
  for (const void* q : wide)
    if (q == nullptr || !aligned(q, 16)) return fail(LSK_ERR_INVALID, "y, x, the tiles and out must be 16-byte aligned device pointers");
  const void* words[] = {scale, ranks, index};
  for (const void* q : words)
    if (q == nullptr || !aligned(q, 4)) return fail(LSK_ERR_INVALID, "scale, ranks and index must be 4-byte aligned device pointers");
  if (out == y && (epilogue != LSK_EPI_NONE || ldy != N))
    return fail(LSK_ERR_INVALID, "in place, y's rows must be contiguous and the epilogue none");
  return LSK_OK;
}

int check_lm_head(const void* w_packed, int layout_id, int V, int K, const void* x, int M, int ldx,
                  const float* logits_opt, int logits_mode, const long long* out_idx) {
  if (layout_id != LSK_LAYOUT_MFMA16X32)
    return fail(LSK_ERR_LAYOUT, "lm_head needs layout %d, got %d", LSK_LAYOUT_MFMA16X32, layout_id);
  if (int st = check_shape(layout_id, V, K)) return st;  // V % 16 == 0: whole row-blocks, any count
  if (M < 1 || M > kDecodeMaxM) return fail(LSK_ERR_INVALID, "M=%d must be in 1..%d", M, kDecodeMaxM);
  if (logits_mode != LSK_LOGITS_FP32 && logits_mode != LSK_LOGITS_BF16)
    return fail(LSK_ERR_INVALID, "unknown logits mode %d", logits_mode);
  if (w_packed == nullptr || x == nullptr || out_idx == nullptr) return fail(LSK_ERR_INVALID, "null device pointer");
  if (!aligned(w_packed, 16)) return fail(LSK_ERR_INVALID, "packed weights must be 16-byte aligned");
  if (ldx < K || ldx % 8 != 0 || !aligned(x, 16))
    return fail(LSK_ERR_INVALID, "x needs ldx >= K, ldx %% 8 == 0 and 16-byte alignment (ldx=%d, K=%d)", ldx, K);
  if (logits_opt != nullptr && !aligned(logits_opt, 16))
    return fail(LSK_ERR_INVALID, "logits buffer must be 16-byte aligned");
  if (!aligned(out_idx, 8)) return fail(LSK_ERR_INVALID, "out_idx must be 8-byte aligned");
  return LSK_OK;
}

int check_lm_head_call(const void* w_packed, int layout_id, int V, int K, const void* x, int M, int ldx,
                       const float* logits_opt, int logits_mode, const long long* out_idx) {
  clear_error();
  return check_lm_head(w_packed, layout_id, V, K, x, M, ldx, logits_opt, logits_mode, out_idx);
}

}  // namespace lsk

extern "C" {

const char* lsk_last_error(void) { return lsk::error_message(); }

size_t lsk_packed_bytes(int layout_id, int N, int K) {
  if (lsk::check_shape(layout_id, N, K) != LSK_OK) return 0;
  return (size_t)N * (size_t)K * 2;
}

int lsk_pack_bf16(const void* w_rowmajor_host, int N, int K, int layout_id, void* out_host) {
  lsk::clear_error();
  if (int st = lsk::check_shape(layout_id, N, K)) return st;
  if (w_rowmajor_host == nullptr || out_host == nullptr) return lsk::fail(LSK_ERR_INVALID, "null buffer");
  const auto* src = static_cast<const unsigned char*>(w_rowmajor_host);
  auto* dst = static_cast<unsigned char*>(out_host);
  const int k8s = K / 8;
  for (int pr = 0; pr < N; ++pr) {
    const unsigned char* row = src + (size_t)lsk::source_row(layout_id, N, pr) * K * 2;
    for (int k8 = 0; k8 < k8s; ++k8) std::memcpy(dst + lsk::packed_unit(K, pr, k8) * 16, row + (size_t)k8 * 16, 16);
  }
  return LSK_OK;
}

int lsk_unpack_bf16(const void* packed_host, int N, int K, int layout_id, void* out_rowmajor_host) {
  lsk::clear_error();
  if (int st = lsk::check_shape(layout_id, N, K)) return st;
  if (packed_host == nullptr || out_rowmajor_host == nullptr) return lsk::fail(LSK_ERR_INVALID, "null buffer");
  const auto* src = static_cast<const unsigned char*>(packed_host);
  auto* dst = static_cast<unsigned char*>(out_rowmajor_host);
  const int k8s = K / 8;
  for (int pr = 0; pr < N; ++pr) {
    unsigned char* row = dst + (size_t)lsk::source_row(layout_id, N, pr) * K * 2;
    for (int k8 = 0; k8 < k8s; ++k8) std::memcpy(row + (size_t)k8 * 16, src + lsk::packed_unit(K, pr, k8) * 16, 16);
  }
  return LSK_OK;
}

}  // extern "C"
