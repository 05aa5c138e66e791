// Drives the size and argument rules of the paged 8-bit cache and of sampled tokens
// (leanstack_amd/csrc/host_rules.cpp and lsk_host.h) at the ends of their arguments'
// ranges under AddressSanitizer and UndefinedBehaviorSanitizer: an overflow or a
// division by zero is a report.  Built and run by tests/test_paged_sizes.py with g++;
// prints "ok" and exits 0 when every check holds.

#include <climits>
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "leanstack_amd.h"
#include "lsk_host.h"

namespace {

int g_failures = 0;

void expect(bool cond, const char* what) {
  if (!cond) {
    std::printf("FAILED: %s (last error: %s)\n", what, lsk_last_error());
    ++g_failures;
  }
}

const int kEnds[] = {INT_MIN, -1, 0, 1, 2, 7, 16, 64, 100, 128, 129, 1024, 1 << 16, 1 << 20, 1 << 23, 1 << 26, 1 << 30, INT_MAX - 64, INT_MAX};

}  // namespace

int main() {
  void* p = reinterpret_cast<void*>(uintptr_t(0x10000));
  const int* i32 = static_cast<const int*>(p);
  const float* f32 = static_cast<const float*>(p);
  const long long* tokens = static_cast<const long long*>(p);
  lsk_paged_pool pool = {};
  pool.k_blocks = pool.v_blocks = p;
  pool.k_exponents = pool.v_exponents = static_cast<unsigned char*>(p);
  pool.table = i32;
  int pools = 0, appends = 0, reads = 0, copies = 0, plans = 0, calls = 0, samples = 0;
  for (int pages : kEnds)
    for (int n_kv : {INT_MIN, 0, 1, 8, 1 << 16, INT_MAX})
      for (int page_rows : kEnds)
        for (int table_pages : kEnds) {
          pool.pages = pages;
          pool.n_kv = n_kv;
          pool.page_rows = page_rows;
          pool.table_pages = table_pages;
          pool.table_stride = table_pages;
          if (lsk::check_paged_pool(&pool) != LSK_OK) continue;
          ++pools;
          for (int b : kEnds)
            for (int t : kEnds) {
              appends += lsk::check_paged_append(&pool, p, 128, 128, 128, p, 128, 128, 128, b, t, i32, i32) == LSK_OK;
              reads += lsk::check_paged_read(&pool, i32, i32, b, t, p, p) == LSK_OK;
              for (int g : {1, 4, 24}) {
                if ((long long)n_kv * g > INT_MAX) continue;
                calls += lsk::check_paged_attention(&pool, p, 128, 128, 128, b, t, n_kv * g, 128, i32, i32, 0.1f, p) == LSK_OK;
              }
            }
        }
  for (int b : kEnds)
    for (int t : kEnds)
      for (int n_kv : {0, 1, 3, 8, 1 << 12, 1 << 23, INT_MAX})
        for (int g : {0, 1, 4, 24})
          for (int capacity : kEnds) {
            if ((long long)n_kv * g > INT_MAX) continue;
            if (lsk::check_paged_attention_sizes(b, t, n_kv * g, n_kv, capacity) != LSK_OK) continue;
            ++plans;
            const lsk::PagedPlan plan = lsk::paged_plan(b, t, n_kv * g, n_kv, capacity);
            const long long rows = (long long)t * g;
            expect((long long)plan.tiles * plan.rows >= rows && (long long)(plan.tiles - 1) * plan.rows < rows,
                   "the tiles cover every query row");
            expect(plan.slot_rows >= 1 && plan.slot_rows <= plan.rows && plan.places >= 1 && plan.workers >= 1 &&
                       plan.slots >= plan.workers && plan.least_units >= 1,
                   "a plan has places, workers and slots");
            const unsigned long long bytes = lsk::paged_workspace_bytes(plan, n_kv);
            expect(plan.one_launch ? bytes == 0 : bytes / 520 >= (unsigned long long)plan.slots, "a workspace holds all slots");
          }
  for (int planes : kEnds)
    for (int pages : kEnds)
      for (int page_blocks : kEnds)
        for (int n : kEnds) copies += lsk::check_paged_copy(p, p, planes, pages, page_blocks, i32, i32, n) == LSK_OK;
  for (int mode : {-1, 0, 1, 2})
    for (int m : kEnds)
      for (int v : kEnds)
        samples += lsk::check_sample_args(p, mode, m, v, v, f32, f32, i32, f32, f32, tokens, f32) == LSK_OK;
  for (int m : kEnds)
    for (int v : kEnds) {
      if (lsk::check_sample_sizes(0, m, v) != LSK_OK) continue;
      for (int bytes : {2, 4})
        for (bool ranked : {false, true})
          for (bool by_p : {false, true}) {
            const int slices = lsk::sample_slices(m, v, bytes, ranked);
            const unsigned long long row = lsk::sample_row_bytes(slices, v, by_p, ranked);
            expect(slices >= 1 && slices <= lsk::kSampleMaxSlices && (long long)m * slices <= (m > 512 ? m : 512) &&
                       (slices == 1 || v / slices >= lsk::kSampleLeastSlice),
                   "slices fit the chip and hold values");
            expect((row == 0) == (slices == 1) && row % 256 == 0 && row < (1u << 20), "a row's sums are less than 1 MB");
          }
    }
  expect(pools > 0 && appends > 0 && reads > 0 && copies > 0 && plans > 0 && calls > 0 && samples > 0,
         "some sizes of every kind are served");

  if (g_failures) {
    std::printf("%d checks failed\n", g_failures);
    return 1;
  }
  std::printf("ok\n");
  return 0;
}
