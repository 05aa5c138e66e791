// Drives the size rules of the operators for a batch of requests (attention over
// a shared prefix, adapters, constrained logits; leanstack_amd/csrc/host_rules.cpp
// and lsk_host.h) at the ends of their arguments' ranges under AddressSanitizer and
// UndefinedBehaviorSanitizer: an overflow or a division by zero is a report.
// Built and run by tests/test_batch_sizes.py with g++; prints "ok" and exits 0
// when every check holds.

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

const int kEnds[] = {INT_MIN, -1, 0, 1, 2, 7, 128, 129, 1 << 16, 1 << 20, 1 << 22, 1 << 23, 1 << 30, INT_MAX - 64, INT_MAX};

}  // namespace

int main() {
  const void* p = reinterpret_cast<const void*>(uintptr_t(0x10000));
  const int* i32 = static_cast<const int*>(p);
  const float* f32 = static_cast<const float*>(p);
  const void* out = reinterpret_cast<const void*>(uintptr_t(0x20000));
  const long long* tokens = reinterpret_cast<const long long*>(uintptr_t(0x30000));
  int good = 0;
  for (int b : kEnds)
    for (int t : kEnds)
      for (int n_kv : {0, 1, 8, 1 << 16, 1 << 23, INT_MAX})
        for (int g : {1, 4})
          for (int P : kEnds)
            for (int S : kEnds) {
              const long long n_q = (long long)n_kv * g;
              if (n_q > INT_MAX) continue;
              good += lsk::check_prefix_args(p, 128, 128, 128, b, t, (int)n_q, n_kv, 128, p, p, 128, 128, P, p, p, 128, 128,
                                             128, S, i32, 0.1f, out) == LSK_OK;
              if (lsk::check_prefix_sizes(b, t, (int)n_q, n_kv, P, S) != LSK_OK) continue;
              const lsk::PrefixPlan plan = lsk::prefix_plan(b, t, (int)n_q, n_kv, P, S);
              const bool covered = plan.joint || ((long long)plan.prefix_chunk * plan.prefix_parts >= P &&
                                                  (long long)plan.own_chunk * plan.own_parts >= S &&
                                                  plan.prefix_parts + plan.own_parts > 0);
              expect(covered, "the parts cover every key row");
            }
  expect(good > 0, "some attention sizes are served");
  good = 0;
  for (int m : kEnds)
    for (int n : {INT_MIN, 0, 16, 32, 2560, (1 << 22) - 32, 1 << 22, INT_MAX - 31, INT_MAX})
      for (int k : {INT_MIN, 0, 32, 2560, (1 << 22) - 32, 1 << 22, INT_MAX - 31, INT_MAX})
        for (int count : kEnds)
          for (int rank_tiles : {INT_MIN, 0, 1, 8, INT_MAX})
            for (int epilogue : {0, 1})
              good += lsk::check_lora_args(p, m, n, n, p, k, k, p, p, f32, i32, count, rank_tiles, i32, epilogue, out) ==
                      LSK_OK;
  expect(good > 0, "some adapter sizes are served");
  good = 0;
  for (int m : kEnds)
    for (int v : kEnds)
      good += lsk::check_constrain_args(p, 0, m, v, v, nullptr, 0, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr,
                                        nullptr, 0, 0, nullptr, 0, out, tokens) == LSK_OK;
  expect(good > 0, "some logits are served");

  if (g_failures) {
    std::printf("%d checks failed\n", g_failures);
    return 1;
  }
  std::printf("ok\n");
  return 0;
}
