// key_weights_plan (paged.h), host code of the built library: what the GPU tests of few rows rely on, that
// their workgroups walk more tiles than the ring in LDS holds; few and many rows; sizes at their limits.
#include <cstdio>

#include "paged.h"

using arthip::key_weights_plan;

static arthip_key_weights_args args(int batch, int tokens, int k_heads, int q_heads, int slots) {
  arthip_key_weights_args a{};
  a.p.batch = batch;
  a.p.tokens = tokens;
  a.p.k_heads = k_heads;
  a.q_heads = q_heads;
  a.slots = slots;
  return a;
}

static int expect(const char* what, int64_t got, int64_t want) {
  if (got == want) return 0;
  std::printf("%s: %lld, not %lld\n", what, (long long)got, (long long)want);
  return 1;
}

int main() {
  int bad = 0;
  // tests/test_paged_gpu.py, few rows over a ring of tiles: six tiles of 32 slots.
  for (int q_heads : {32, 64}) {
    const arthip::KeyWeightsPlan p = key_weights_plan(args(6, 46, 32, q_heads, 5120));
    bad += expect("slots of a workgroup", p.stream, 192) + expect("workgroups a head", p.tiles, 27) +
           expect("workspace", (int64_t)p.workspace, 0);
  }
  // One tile where there are few slots, 1024 slots at most.
  bad += expect("short", key_weights_plan(args(1, 1, 16, 16, 777)).stream, 32);
  bad += expect("long", key_weights_plan(args(8192, 8192, 8, 8, 16384)).stream, 1024);
  bad += expect("longest", key_weights_plan(args(1, 1, 1, 1, 1 << 30)).stream, 1024);
  // Many rows: no ring; ranges of rows where there are few workgroups, whose sums are kept.
  const arthip::KeyWeightsPlan many = key_weights_plan(args(1, 10000, 1, 4, 4096));
  bad += expect("many", many.stream, 0) + expect("tiles", many.tiles, 16) + expect("ranges", many.splits, 64) +
         expect("sums", (int64_t)many.workspace, (int64_t)64 * 4096 * 4);
  bad += expect("nothing", key_weights_plan(args(0, 0, 1, 1, 100)).tiles, 1);
  return bad;
}
