// Host-side rules of the C ABI that need no HIP: tile geometry, the packed
// layouts' index arithmetic, argument validation and the thread-local error
// message of lsk_last_error().  Defined in host_rules.cpp, which builds with a
// plain C++ compiler (the sanitizer test builds it with g++
// -fsanitize=address).  Not part of the ABI.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "leanstack_amd.h"

namespace lsk {

// Tile geometry of LSK_LAYOUT_MFMA16X32: 16 rows x 32 K of bf16 = 1024 bytes,
// one v_mfma_f32_16x16x32_bf16 operand per 64-lane wavefront.
constexpr int kTileRows = 16;
constexpr int kTileK = 32;
constexpr int kTileBytes = kTileRows * kTileK * 2;

// Largest M served by the decode/verify kernel (the MFMA column count).
constexpr int kDecodeMaxM = 16;

// Largest activation row stride (elements) of a projection: the prefill
// kernel reads a 256-row block of x through a buffer descriptor whose byte
// offsets are 32-bit, so 256 * ldx * 2 must stay below 2^31 (and ldx is a
// multiple of 8).
constexpr int kMaxActivationStride = (1 << 22) - 8;

// Decode attention geometry (attention.hip): up to kAttnMinChunkRows rows
// attended run as one chunk (one workgroup per kv head, no combine); up to
// 8 * kAttnSplitRows rows as at most 8 chunks of kAttnSplitRows rows (one
// combine round); beyond that, at most kAttnMaxChunks chunks of the smallest
// multiple of kAttnMinChunkRows rows that allows it.
constexpr int kAttnHeadDim = 128;
constexpr int kAttnMinChunkRows = 128;
constexpr int kAttnSplitRows = 64;
constexpr int kAttnMaxChunkRows = 512;
constexpr int kAttnMaxChunks = 32;
constexpr int kAttnMaxRows = kAttnMaxChunks * kAttnMaxChunkRows;  // 16384
constexpr int kAttnMaxKvHeads = 64;
static_assert(kAttnSplitRows % 16 == 0 && kAttnSplitRows >= 16 && kAttnSplitRows <= kAttnMinChunkRows,
              "chunks are whole 16-row MFMA groups, at most one workgroup's 128");

// Rows per chunk when `rows` rows (1..kAttnMaxRows) are attended; the host
// and the kernel share it.
constexpr int attention_rows_per_chunk(int rows) {
  if (rows <= kAttnMinChunkRows) return kAttnMinChunkRows;
  if (rows <= 8 * kAttnSplitRows) return kAttnSplitRows;
  const int units = (rows + kAttnMinChunkRows - 1) / kAttnMinChunkRows;
  return kAttnMinChunkRows * ((units + kAttnMaxChunks - 1) / kAttnMaxChunks);
}

// Chunk slots per kv head that a position below max_seq_len can need.
constexpr int attention_most_chunks(int max_seq_len) {
  if (max_seq_len <= kAttnMinChunkRows) return 1;
  if (max_seq_len <= 8 * kAttnSplitRows) return (max_seq_len + kAttnSplitRows - 1) / kAttnSplitRows;
  const int units = (max_seq_len + kAttnMinChunkRows - 1) / kAttnMinChunkRows;
  const int most = units > 8 ? units : 8;
  return most < kAttnMaxChunks ? most : kAttnMaxChunks;
}

// Attention over a shared prefix (prefix_attention.hip).
constexpr int kPrefixThreads = 512;     // the most of a workgroup
constexpr int kPrefixSharedRows = 128;  // query rows of an item whose waves share key rows

// How a call runs.  joint: one launch, an item per 32 query rows of one request
// and kv head.  Else prefix_parts ranges of prefix_chunk prefix rows per kv head and
// prefix_tiles of 32 (shared: 128) query rows, and own_parts ranges of own_chunk own
// rows per kv head, request and own_tiles of 32 query rows.
struct PrefixPlan {
  bool joint, shared;
  int prefix_tiles, prefix_chunk, prefix_parts, own_tiles, own_chunk, own_parts;
};
constexpr int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Measured with 32 q and 8 kv heads, B x T tokens, P + S rows:
// - One launch while the rows are few and its items, one per CU, run at once:
//   12x1 500+128 8.5 us in one, 9.7 in two; 1x1 900+64 10.0 in one, 9.1 in two; with
//   three rounds of items (81x1 187+9) 17.4 in one, 14.8 in two.
// - Waves that share query rows read the prefix rows once per 32 of them, waves that
//   share key rows once per 128, and have a barrier per step and fewer items: up to 192
//   query rows per kv head the first are faster (32x1 4096+1024 19.6 against 24.3 us; 8x5
//   12000+64 22.5 against 30.5), with 256 the second (64x1 8191+1088 47 against 55).
// - A part more costs every query row 520 bytes written and read, so items are as many as
//   the chip runs of them at once and no more: two per CU of items that share key
//   rows, one of those that do not and are bound by memory (8x1 9000+128 14.9 us,
//   17.6 with two), and half a CU's worth of own items.
// - Of the 512 places of shared items the prefix gets its share of all key rows to be
//   read, so that it does not finish long before the own rows do, whose reads bound
//   them: 64x1 8191+1088 47 us with 7 parts, 48 with 12, 52 with 16; 48x4 16000+320, where it
//   is most of the work, 82 us with 10 parts, 88 with 5.  But not fewer than 192: how
//   many of the S rows are written only the device knows (64x1 8191+4096 of which 100
//   29 us, with the share alone 87; the same with 1088 of 1088 61, 59).
constexpr int kPrefixJointRows = 768;
constexpr int kPrefixJointItems = 256;
constexpr int kPrefixSplitRows = 192;
constexpr int kPrefixLeastPlaces = 192;
constexpr PrefixPlan prefix_plan(int B, int T, int n_q, int n_kv, int P, int S) {
  PrefixPlan p = {false, false, 0, 128, 0, ceil_div((long long)T * (n_q / n_kv), 32), 128, 0};
  const long long rows = (long long)B * T * (n_q / n_kv);
  const long long own_items = (long long)n_kv * B * p.own_tiles;
  // (with no key row at all there are no parts to add up)
  if (((long long)P + S <= kPrefixJointRows && own_items <= kPrefixJointItems) || (P == 0 && S == 0)) {
    p.joint = true;
    return p;
  }
  p.shared = rows > kPrefixSplitRows;
  if (P > 0) {
    const int unit = p.shared ? 32 : 128, least = p.shared ? 384 : 256;  // rows of a chunk
    p.prefix_tiles = ceil_div(rows, p.shared ? kPrefixSharedRows : 32);
    const long long items = (long long)n_kv * p.prefix_tiles;
    const long long prefix = (long long)p.prefix_tiles * P, own = (long long)B * S;
    const long long most = (p.shared ? 512 : 256) / items;
    const long long even = p.shared ? ceil_div(512 * prefix, (prefix + own) * items) : most;
    const long long share = even * items < kPrefixLeastPlaces ? ceil_div(kPrefixLeastPlaces, items) : even;
    const long long wanted = share < most ? share : most;
    const int chunk = ceil_div(ceil_div(P, wanted > 1 ? wanted : 1), unit) * unit;
    p.prefix_chunk = chunk < least ? least : chunk;
    p.prefix_parts = ceil_div(P, p.prefix_chunk);
  }
  if (S > 0) {
    const long long wanted = own_items < 512 ? 512 / own_items : 1;
    const int chunk = ceil_div(ceil_div(S, wanted), 128) * 128;
    p.own_chunk = chunk < 256 ? 256 : chunk;
    p.own_parts = ceil_div(S, p.own_chunk);
  }
  return p;
}
// fp32 (m, l) and O of every query row and part.
constexpr unsigned long long prefix_workspace_bytes(const PrefixPlan& p, int B, int T, int n_q) {
  return (unsigned long long)(p.prefix_parts + p.own_parts) * B * T * n_q * (kAttnHeadDim + 2) * 4ull;
}

// The sizes that prefix_plan takes, and argument rules of lsk_prefix_attention_bf16
// (all but the workspace's size).
int check_prefix_sizes(int B, int T, int n_q, int n_kv, int P, int S);
int check_prefix_args(const void* q, long long q_batch, long long q_head, long long q_token, int B, int T, int n_q,
                      int n_kv, int head_dim, const void* prefix_k, const void* prefix_v, long long prefix_head,
                      int prefix_row, int P, const void* k, const void* v, long long batch, long long head, int row,
                      int S, const int* lens, float scale, const void* out);

// Pages of an 8-bit key/value cache (paged_cache.hip, paged_attention.hip): blocks of
// kPagedBlockRows rows of one kv head with an exponent, a power of two of blocks to a page.
constexpr int kPagedBlockRows = 16;
constexpr int kPagedBlockBytes = kPagedBlockRows * kAttnHeadDim;
constexpr int kPagedLeastExponent = -100;  // of a block: 2^-100 .. 2^119, so that 448 times it is finite
constexpr int kPagedMostExponent = 119;
constexpr int kPagedMostPageRows = 1024;

// Blocks that `rows` rows from any row on can touch.
constexpr int paged_windows(int rows) { return (int)(((long long)rows + 2 * kPagedBlockRows - 2) / kPagedBlockRows); }

// How an attention call runs.  An item is `rows` query rows of one request and kv head.
// - Up to 64 rows over a context that is short for certain run in one launch, a workgroup per
//   item, while the chip holds all the workgroups: 24 requests over 2048 rows 21 us, 26 in two
//   launches; 1 request 14 us for 13, so few workgroups have the lower limit.  From
//   kPagedShortGroups workgroups on (64 requests of 8 kv heads) two launches take as long (20 us
//   over 512 rows), with 128 requests 29 us for 39.
// - Else up to 32 rows are cut into chunks of at least `least_units` units of key rows, a wave
//   each, at most `places` per kv head and one more per item.  2048 waves in all for up to 16
//   rows (64 requests over 4096 rows: 95 us, with 1024 waves 115), 1024 for 32, whose waves do
//   more with a row (24 x 5 tokens over 2000 rows: 24 us, with 2048 waves 26, with 512 37).
//   Chunks of 4 units: 1 request over 8192 rows 13.5 us, of 2 15.3, of 8 15.6.
// - More are taken 128 at a time by workgroups of which `workers` per kv head share all units,
//   512 in all (256 were 313 us for 260 in 2 x 1500 tokens over 5500 rows).  Also 33..64 rows: 8 x 16
//   tokens over 8192 rows 59 us, 71 by waves of 64 rows.
// The second launch adds up parts, 2^join_shift query rows to a workgroup; with more parts than
// its threads can take at once it has fewer rows (1 request over 32768 rows, 256 parts: 6.4 us, 39
// with 16 rows); with many query rows more of them, `join_passes` times, so that fewer
// workgroups wait for their first loads (2 x 1500 tokens behind 4000 and 7001 rows: 13 us, 14 with
// one pass or four), and of more items than workers those that a share's beginning cuts (64 prompts
// of 200 tokens, few of them cut: 4 us, 15 by items).
constexpr int kPagedFewUnit = 32;
constexpr int kPagedManyUnit = 64;
constexpr int kPagedManyRows = 128;
// Units that an item's beginning (lens, table, exponents, first rows, one behind the other) and end
// take as long as: 4 prompts of 2000 tokens, whose first items are short, 184 us, 253 counting none.
constexpr int kPagedManyStart = 6;
constexpr int kPagedShortRows = 2048, kPagedShortFewRows = 1536, kPagedShortFewGroups = 128, kPagedShortGroups = 512;
constexpr int kPagedJoinGroups = 2048, kPagedJoinPasses = 2;
struct PagedPlan {
  bool one_launch;
  int rows, slot_rows, unit, least_units, tiles;
  int join_shift;   // a workgroup of the second launch adds up the parts of 2^join_shift query rows
  int join_passes;  // .. times this many, one behind the other
  bool join_wide;   // .. with 1024 threads, not 256
  long long items, places, workers, slots, joins;  // slots: of parts, per kv head; joins: items that may have been cut
};
constexpr PagedPlan paged_plan(int B, int T, int n_q, int n_kv, int capacity) {
  const long long rows = (long long)T * (n_q / n_kv);
  PagedPlan p = {false, rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : kPagedManyRows, 0, kPagedFewUnit, 4, 0, 0, 1, false, 0, 0, 0, 0, 0};
  const long long groups = (long long)B * n_kv;
  p.one_launch = rows <= 64 && groups < kPagedShortGroups &&
                 capacity <= (groups < kPagedShortFewGroups ? kPagedShortFewRows : kPagedShortRows);
  if (rows > 32 && !p.one_launch) p.rows = kPagedManyRows;
  const bool many = p.rows == kPagedManyRows;
  if (many) p.unit = kPagedManyUnit;
  p.slot_rows = rows < p.rows ? (int)rows : p.rows;
  p.tiles = (int)((rows + p.rows - 1) / p.rows);
  p.items = (long long)B * p.tiles;
  const int all = many ? 512 : p.rows == 32 ? 1024 : 2048;
  const long long most = p.items * ((capacity + p.unit - 1) / p.unit);
  p.places = all / n_kv > 1 ? all / n_kv : 1;
  // (an item more or less than a chunk adds one: all chunks are to run at once)
  if (!many && p.places > 1) p.places = p.items < p.places / 2 ? p.places - p.items : p.places / 2;
  if (p.places > most) p.places = most;
  p.workers = many ? p.places : p.places + p.items;
  p.slots = many ? 2 * p.workers : p.workers;
  const long long shortest = many ? p.unit : p.unit * p.least_units, longest = (capacity + shortest - 1) / shortest;
  const long long parts = p.workers / p.items < longest ? p.workers / p.items : longest;
  p.join_shift = 4;
  while (p.join_shift > 0 && (p.slot_rows <= 1 << (p.join_shift - 1) || (64 >> p.join_shift) < parts)) --p.join_shift;
  p.join_wide = parts >= 128;
  p.joins = many && p.items > p.workers ? p.workers : p.items;
  p.join_passes = many && p.join_shift == 4 && p.joins * n_kv * ((p.slot_rows + 15) / 16) > kPagedJoinGroups ? kPagedJoinPasses : 1;
  return p;
}
static_assert(paged_plan(1, 64, 1, 1, 64).tiles == 1 && paged_plan(600, 16, 4, 1, 64).tiles == 1 && paged_plan(1, 17, 1, 1, 1 << 20).tiles == 1,
              "up to 64 query rows are one item: the kernels for few have no tiles");
// (m, l) and O of every slot, and where the items begin and which of 128 rows are cut.
constexpr unsigned long long paged_begins_bytes(const PagedPlan& p) {
  const unsigned long long words = (unsigned long long)p.items + 1 + (p.rows == kPagedManyRows ? (unsigned long long)p.workers : 0);
  return (words * 4 + 15) / 16 * 16;
}
constexpr unsigned long long paged_workspace_bytes(const PagedPlan& p, int n_kv) {
  return p.one_launch ? 0
                      : paged_begins_bytes(p) + (unsigned long long)p.slots * (unsigned long long)n_kv *
                                                    (unsigned long long)p.slot_rows * (kAttnHeadDim + 2) * 4ull;
}

// Argument rules of the lsk_paged entry points (all but workspaces' sizes).
int check_paged_pool(const lsk_paged_pool* pool);
int check_paged_append(const lsk_paged_pool* pool, const void* k, long long k_batch, long long k_head, long long k_token,
                       const void* v, long long v_batch, long long v_head, long long v_token, int B, int T,
                       const int* lens, const int* counts);
int check_paged_read(const lsk_paged_pool* pool, const int* starts, const int* lens, int B, int rows, const void* k,
                     const void* v);
int check_paged_copy(const void* storage, const void* exponents, int planes, int pages, int page_blocks, const int* src,
                     const int* dst, int n);
int check_paged_attention_sizes(int B, int T, int n_q, int n_kv, int capacity);
int check_paged_attention(const lsk_paged_pool* pool, const void* q, long long q_batch, long long q_head,
                          long long q_token, int B, int T, int n_q, int head_dim, const int* lens, const int* counts,
                          float scale, const void* out);

// Constrained logits (constrain.hip): a row's vocabulary is cut into slices, one
// workgroup each; a slice's counts are one LDS word per entry.
constexpr int kConstrainMaxHistory = 1 << 20;
constexpr int kConstrainMaxBias = 1023;
constexpr int kConstrainMaxSlice = 10176;
constexpr int kConstrainThreads = 512;
constexpr int kConstrainCounterWords = 16;  // a row's counter has 64 bytes to itself

// Vocabulary entries per slice: the most that a quarter of a CU's LDS counts while the rows
// alone fill the chip, fewer when there are few rows (a multiple of 64, so that a
// slice starts at an aligned value where its row does).
constexpr int constrain_slice(int M, int V) {
  const int least = (V + kConstrainMaxSlice - 1) / kConstrainMaxSlice;
  const int most = V / 2048 < 32 ? V / 2048 + 1 : 32;
  const int wanted = M >= 1024 ? 1 : (1024 + M - 1) / M;
  const int some = wanted > most ? most : wanted;
  const int slices = some < least ? least : some;
  const int slice = ((V + slices - 1) / slices + 63) / 64 * 64;
  return slice < kConstrainMaxSlice ? slice : kConstrainMaxSlice;
}
constexpr int constrain_slices(int M, int V) {
  const int slice = constrain_slice(M, V);
  return (V + slice - 1) / slice;
}

// Sampled tokens (sample.hip): a row's weights, whole numbers up to 2^44, add up in 63 bits.
constexpr int kSampleMaxVocab = 1 << 19;

// Rows are cut into three slices or more while the chip has room for all, of at least
// kSampleLeastSlice values.  16 rows of 151936 fp32 values without top-k and min-p 18 us for 75 (top-p 0.9 over flat
// ones 44 for 283, over peaked ones 36 for 97), of 32000 16 for 22; with two slices some are slower
// (256 rows 89 for 107, peaked with top-p 146 for 123).  With top-k or min-p (`ranked`) a second
// launch costs more than the sweeps of a row that is not kSampleRankedBytes long: 16 rows of 151936
// fp32 values 17 us for 28, of bf16 16 for 22; of 50257 fp32 values 16 either way, of 32000 15 for 13.
constexpr int kSampleMaxSlices = 16, kSampleLeastSlice = 8192, kSamplePlaces = 512, kSampleRankedBytes = 1 << 18;
constexpr int kSampleBins = 2048, kSampleSliceListed = 512, kSampleRankListed = 2048, kSampleRowBytes = 256;
constexpr int sample_slices(int M, int V, int value_bytes, bool ranked) {
  const int room = kSamplePlaces / M, most = V / kSampleLeastSlice;
  const int slices = room < most ? room : most;
  if (slices < 3 || (ranked && V < kSampleRankedBytes / value_bytes)) return 1;
  return slices < kSampleMaxSlices ? slices : kSampleMaxSlices;
}
// (parts of 64 accesses of 16 bytes; an even number keeps what follows them at 16 bytes)
constexpr int sample_max_parts(int V) { return (V / 256 + 4) / 2 * 2; }
constexpr unsigned long long sample_row_bytes(int slices, int V, bool by_p, bool ranked) {
  const unsigned long long each = ranked ? kSampleRankListed : by_p ? kSampleSliceListed + kSampleBins : 0;
  const unsigned long long words = slices * each + (ranked ? 0 : sample_max_parts(V));
  return slices < 2 ? 0 : (kSampleRowBytes + words * 8 + 255) / 256 * 256;
}
int check_sample_sizes(int logits_mode, int M, int V);
int check_sample_args(const void* logits, int logits_mode, int M, int V, long long logits_ld, const float* uniforms,
                      const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                      const long long* tokens, const float* logprobs);

// Low-rank adapters (adapters.hip): a tile of rows of x, an adapter that they name
// (slot) and a range of output columns per workgroup.
constexpr int kAdapterThreads = 512;
constexpr int kAdapterMaxSplits = 8;

// 16-row tiles of the adapters' rank that the kernels are built for.
constexpr bool adapter_rank_supported(int rank_tiles) {
  return rank_tiles >= 1 && rank_tiles <= 8 && rank_tiles != 5 && rank_tiles != 7;
}

// How a call runs: tiles of `rows` rows, slots per tile, ranges of output columns, and
// K ranges of the first of two launches (0: one launch).
//
// Up to 128 rows a decode batch is expected, whose rows each name an adapter of
// their own: tiles of 16 rows and a workgroup per (adapter named, column range), in
// one launch unless reading A anew for every range (from L2) costs more than a
// launch.  In one and in two launches, us:
//   1 tile (its ranges share an L2): QKV (K = 2560) 16 rows, rank 16 6.7, 8.6; o (4096), rank 32 7.7, 8.5;
//     1 row 6.7, 6.8; QKV, rank 64 14.3, 11.2
//   several: QKV, 64 rows, rank 16 9.8, 10.2; rank 32 12.8, 11.7; o, rank 16 11.3, 10.1;
//     rank 32 15.8, 11.1
// Above, prompts, whose neighbouring rows mostly name the same: 64 rows share an adapter's
// tiles, and the second launch takes y once whatever its rows name.  Slots beyond
// the first few would be workgroups that find nothing to do (2000 rows of gate_up
// with 4 slots per tile instead of 1: 14.9 instead of 7.6 us for the first launch).
// Each form is the slower one for the other's rows; all launches of a call, us, in
// tiles of 16 rows and of 64, where the rows name one adapter of the store and where
// each row names its own:
//                                128 rows: one        own      256 rows: one        own
//   o, 48 adapters of rank 16       9.7, 10.5  11.1, 35.4    15.1, 11.8  12.9, 43.5
//   o, 48 of rank 128              17.6, 18.3  21.5, 77.9    28.1, 19.8  28.9, 98.5
//   QKV, 48 of rank 16             14.3, 10.9  10.4, 35.5    22.0, 11.2  12.8, 43.8
//   gate_up, 8 of rank 32          16.7, 14.1  15.6, 23.7    26.4, 15.4  23.2, 25.4
// The host knows the store's count and not what the rows name: slots go by the count, so
// that one adapter out of a store of many has fewer workgroups than out of a store of one
// (gate_up, rank 16, 128 rows: 23.1 us of 32 adapters, 11.3 of one).
struct AdapterPlan {
  int rows, tiles, slots, ranges, splits;
};
constexpr int adapter_blocks(int N, bool silu) { return silu ? (N + 63) / 64 : (N + 31) / 32; }
// Column ranges of `tiles` 64-row tiles in the second launch.  A workgroup takes some 4 us
// until y streams, then about 13 bytes a nanosecond (a CU's share of 3.3 TB/s), a
// block per wave at a time; a CU runs one (of plain rank 16, whose registers allow two, it is
// taken to run one as well), so a few workgroups more than CUs would cost a whole round: gate_up, rank 32, with one round and with two: 512 rows 13.2, 20.5
// us, 1024 rows 18.2, 23.9; o, 2000 rows 9.5, 12.0.
constexpr int adapter_rows_ranges(int tiles, int N, bool silu) {
  const int blocks = adapter_blocks(N, silu), most = (blocks + 7) / 8;
  const long long pass_ns = 8 * 64 * (silu ? 192 : 128) / 13;
  int best = 1;
  long long least = 0;
  for (int r = 1; r <= most; ++r) {
    const long long rounds = ((long long)tiles * r + 255) / 256, passes = ((blocks + r - 1) / r + 7) / 8;
    const long long cost = rounds * (4000 + passes * pass_ns);
    if (r == 1 || cost <= least) best = r, least = cost;
    if (rounds > 4) break;
  }
  return best;
}
constexpr AdapterPlan adapter_plan(int M, int N, int K, int rank_tiles, int count, bool silu) {
  const bool decode = M <= 128;
  AdapterPlan p = {decode ? 16 : 64, 0, 0, 1, 0};
  p.tiles = (M - 1) / p.rows + 1;
  const int named = count < M ? count : M;
  const int share = 32 / p.tiles;
  const int most_slots = decode ? 16 : share < 1 ? 1 : share > 16 ? 16 : share;
  p.slots = named < most_slots ? named : most_slots;
  // Two workgroups per CU, each with a block of columns (a k-tile) for every wave.
  const int busy = p.tiles * (decode ? p.slots : 1);
  const int wanted = (512 + busy - 1) / busy;
  const int most = (adapter_blocks(N, silu) + 7) / 8;
  p.ranges = !decode ? adapter_rows_ranges(p.tiles, N, silu) : wanted > most ? most : wanted;
  const long long again = (long long)K * rank_tiles * 32;  // bytes of A per workgroup
  if (!decode || (p.ranges > 1 && again > (p.tiles == 1 ? 256 : 96) * 1024)) {
    const int most_splits = (K / kTileK + 7) / 8;
    p.splits = wanted > most_splits ? most_splits : wanted;
    if (p.splits > kAdapterMaxSplits) p.splits = kAdapterMaxSplits;
  }
  return p;
}
constexpr unsigned long long adapter_workspace_bytes(const AdapterPlan& p, int rank_tiles) {
  return (unsigned long long)p.splits * (unsigned long long)p.tiles * (unsigned long long)(rank_tiles * p.rows) * 64;
}

// The sizes that adapter_plan takes, and argument rules of lsk_lora_add_bf16 (all but the
// workspace's size).
int check_lora_sizes(int M, int N, int K, int rank_tiles, int count, int epilogue);
int check_lora_args(const void* y, int M, int N, int ldy, const void* x, int K, int ldx, const void* a_tiles,
                    const void* b_tiles, const float* scale, const int* ranks, int count, int rank_tiles,
                    const int* index, int epilogue, const void* out);

// Record `fmt` as this thread's lsk_last_error() message; returns `status`.
int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();
const char* error_message();

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// q heads per kv head the attention kernel is built for.
bool attention_group_supported(int group);

// Shape rules of the packed layouts (whole 16x32 tiles, whole gate/up pairs).
int check_shape(int layout_id, int N, int K);

// Argument rules of the projection entry points (see lsk_linear_bf16).
int check_linear_args(const void* w_packed, int layout_id, int N, int K, const void* x, int M, int ldx,
                      const void* y, int ldy, int epilogue, const void* residual, int ldr);

// Argument rules of lsk_rmsnorm_bf16 and lsk_qk_norm_rope_bf16.
int check_rmsnorm_args(const void* x, int M, int K, int ldx, const void* norm_weight, float eps, const void* y);
int check_qk_rope_args(const void* qkv, int B, int T, int ld, int n_q, int n_kv, int head_dim,
                       const void* q_norm_weight, const void* k_norm_weight, float eps, const void* cos,
                       const void* sin, long long rope_batch_stride, long long rope_row_stride, const void* q_out,
                       const void* k_out);

// Argument rules of lsk_constrain_logits (all but the workspace's size).
int check_constrain_args(const void* logits, int logits_mode, int M, int V, long long logits_ld, const int* history,
                         long long history_ld, int history_len, const int* history_lens, const int* prompt_lens,
                         const float* repetition, const float* frequency, const float* presence, const int* bias_ids,
                         const float* bias_values, long long bias_ld, int bias_count, const int* allowed,
                         long long allowed_ld, const void* out, const long long* tokens);

// Argument rules shared by both decode attention entry points (all but pos
// and the workspace).
int check_attention_args(const void* qkv, int n_q, int n_kv, int head_dim, const void* q_norm_weight,
                         const void* k_norm_weight, float eps, const void* cos, const void* sin, const void* k_cache,
                         const void* v_cache, int max_seq_len, float scale, const void* out);

// Every lm_head argument rule but the workspace's.
int check_lm_head(const void* w_packed, int layout_id, int V, int K, const void* x, int M, int ldx,
                  const float* logits_opt, int logits_mode, const long long* out_idx);

// check_lm_head after clearing the error message (for entry points defined
// outside abi.cpp).
int check_lm_head_call(const void* w_packed, int layout_id, int V, int K, const void* x, int M, int ldx,
                       const float* logits_opt, int logits_mode, const long long* out_idx);

}  // namespace lsk
