// The cut of the keys by the attention of several query tokens over the 4-bit cache
// (csrc/kv4_cut.h), built with UndefinedBehaviorSanitizer by tests/test_kv4_cut.py.
#include <cstdint>
#include <cstdio>
#include <cstdlib>

#include "../../aegaeon_amd/csrc/kv4_cut.h"

using namespace aegkv;

#define CHECK(ok, ...)                 \
  do {                                 \
    if (!(ok)) {                       \
      std::printf(__VA_ARGS__);        \
      std::printf(" (%s)\n", #ok);     \
      std::exit(1);                    \
    }                                  \
  } while (0)

static void ranges() {
  const int steps[] = {0, 1, 2, 3, 15, 16, 17, 1000, 65536, 1 << 25};
  const int spans[] = {1, 2, 4, 16, 17, 999, 1 << 25, INT32_MAX - 1, INT32_MAX};
  for (const int n : steps)
    for (const int span : spans) {
      const int r = ranges_of(n, span);
      const int64_t want = n == 0 ? 1 : ((int64_t)n + span - 1) / span;
      CHECK(r == want, "ranges_of(%d, %d) = %d, %lld wanted", n, span, r, (long long)want);
    }
}

int main() {
  ranges();
  std::printf("ok\n");
  return 0;
}
