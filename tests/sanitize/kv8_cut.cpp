// The uneven cut of eight-wave tiles by the attention of several query tokens over the
// 8-bit cache (csrc/kv4_cut.h), built with UndefinedBehaviorSanitizer by
// tests/test_kv8_cut.py.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

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

// The pieces of any tile cover its steps once, in order; only the last one differs
// from the span, and a tile of fewer steps has no more pieces.
static void ranges() {
  const int steps[] = {0, 1, 7, 8, 9, 10, 16, 17, 250, 1000, 65536, 1 << 25};
  const int spans[] = {1, 2, 8, 9, 16, 200, 999, 1 << 25, INT32_MAX - 1, INT32_MAX};
  for (const int span : spans) {
    int before = 1;
    for (const int n : steps) {
      const int r = uneven_ranges(n, span);
      const int64_t last = n - (int64_t)(r - 1) * span;
      CHECK(r >= before, "%d steps by %d: %d pieces, fewer steps %d", n, span, r, before);
      CHECK(r == 1 || (last > kLeastRest && last <= (int64_t)span + kLeastRest),
            "%d steps by %d: %d pieces, the last of %lld", n, span, r, (long long)last);
      CHECK(r > 1 || n <= (int64_t)span + kLeastRest, "%d steps by %d: whole", n, span);
      before = r;
    }
  }
}

// Random batches, as the device finds their cut, against what the host gives them by
// their bounds alone.
static void batches() {
  std::mt19937_64 rng(5);
  auto upto = [&](double hi) {  // 1 .. hi, evenly over the logarithm
    return (int)std::exp(std::uniform_real_distribution<double>(0, std::log(hi + 0.999))(rng));
  };
  int64_t uneven = 0, cut_calls = 0, many = 0;
  for (int n = 0; n < 200000; ++n) {
    const int cus = n % 3 ? 256 : upto(304), batch = upto(40), hkv = upto(40), group = upto(40);
    const int top_q = upto(3000), top_len = upto(n % 7 ? 30000 : 3e5), causal = n & 1;
    struct Seq {
      int64_t tiles;
      int n0, n_kt;  // steps of the first tile and of the last one
    };
    std::vector<Seq> seqs;
    int64_t total = 0;
    int max_q = 0, max_len = 0;
    for (int b = 0; b < batch; ++b) {
      const int m = n % 11 ? upto(top_q + 1) - 1 : top_q, len = n % 13 ? upto(top_len + 1) - 1 : top_len;
      const int64_t rows = (int64_t)m * group, tiles = (rows + 255) / 256 * hkv;
      auto steps = [&](int keys) { return (std::max(keys, 0) + 63) / 64; };
      const int off = len - m, q0 = m > 0 ? (int)((std::min<int64_t>(rows, 256) - 1) / group) : 0;
      seqs.push_back({tiles, steps(causal ? std::min(off + q0 + 1, len) : len), m > 0 ? steps(len) : 0});
      total += m;
      max_q = std::max(max_q, m);
      max_len = std::max(max_len, len);
    }
    VarlenShape s, even;
    if (total == 0 ||
        !varlen_shape(cus, batch, total, max_q, max_len, hkv * group, hkv, 128, &s, true) ||
        !varlen_shape(cus, batch, total, max_q, max_len, hkv * group, hkv, 128, &even))
      continue;
    CHECK(!even.uneven && (!s.uneven || s.long_rows), "batch %d: an uneven cut", n);
    if (!s.uneven) {
      CHECK(s.pieces == even.pieces && s.target == even.target && s.workspace() == even.workspace(),
            "batch %d: another even cut", n);
      continue;
    }
    ++uneven;
    int64_t cost = 0, tiles = 0, cut = 0, more = 0;
    for (const Seq& q : seqs) {
      cost += q.tiles * ((q.n0 + q.n_kt + 1) / 2);
      tiles += q.tiles;
    }
    const int span = uneven_span(cost, tiles, s.target, s.least);
    CHECK(span > 0, "batch %d: a span of %d", n, span);
    for (const Seq& q : seqs) {
      const int r = uneven_ranges(q.n_kt, span);
      cut += r > 1 ? q.tiles : 0;
      more += q.tiles * (r - 1);
      many += r > 2;
    }
    CHECK(tiles + more <= s.pieces, "batch %d: %lld pieces, a grid of %lld", n,
          (long long)(tiles + more), (long long)s.pieces);
    CHECK(cut <= s.cut, "batch %d: %lld tiles cut, room for %lld", n, (long long)cut, (long long)s.cut);
    CHECK(s.workspace() == s.pieces * 256 * (4 * 128 + 8) + 256 + 24 * s.cut,
          "batch %d: a workspace of %lld", n, (long long)s.workspace());
    CHECK(s.merge_rows == 4 || s.merge_rows == 16, "batch %d: %d rows of a merge workgroup", n,
          s.merge_rows);
    cut_calls += cut > 0;
  }
  CHECK(uneven > 1000 && cut_calls > 500 && many > 100, "%lld uneven, %lld cut, %lld of three pieces",
        (long long)uneven, (long long)cut_calls, (long long)many);
}

int main() {
  ranges();
  batches();
  std::printf("ok\n");
  return 0;
}
