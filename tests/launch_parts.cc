// launch_parts (transformer.h): every workgroup is launched once, in order, in launches
// whose threads number fewer than 2^32, as HIP's launch asks; no launch after one that fails.
#include <cstdio>

#include "transformer.h"

using arthip::launch_parts;

static int check(int64_t blocks, int threads, int64_t launches) {
  int64_t next = 0, n = 0;
  bool ok = true;
  const hipError_t e = launch_parts(blocks, threads, [&](int64_t first, unsigned count) {
    ok = ok && first == next && count > 0 && (uint64_t)count * threads < (uint64_t{1} << 32);
    next = first + count;
    ++n;
    return hipSuccess;
  });
  if (e == hipSuccess && ok && next == blocks && n == launches) return 0;
  std::printf("%lld workgroups of %d: %lld launches up to %lld\n", (long long)blocks, threads, (long long)n, (long long)next);
  return 1;
}

int main() {
  int bad = 0;
  for (int threads : {64, 256, 1024}) {
    const int64_t most = ((int64_t{1} << 32) - 1) / threads;
    bad += check(0, threads, 0) + check(1, threads, 1) + check(most, threads, 1) + check(most + 1, threads, 2) +
           check(2 * most, threads, 2) + check(INT32_MAX, threads, (INT32_MAX + most - 1) / most);
  }
  int calls = 0;
  const hipError_t e = launch_parts(int64_t{1} << 31, 256, [&](int64_t, unsigned) {
    ++calls;
    return hipErrorOutOfMemory;
  });
  return bad != 0 || calls != 1 || e != hipErrorOutOfMemory;
}
