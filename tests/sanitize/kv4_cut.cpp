// The cut of the keys by the attention of several query tokens over the 4-bit cache
// (csrc/kv4_cut.h), built with UndefinedBehaviorSanitizer by tests/test_kv4_cut.py.
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

// Random batches against the shape that the host gives them by their bounds alone:
// as many pieces, cut tiles and merge workgroups as the device can find, and a
// merge kernel that exists.
static void batches() {
  std::mt19937_64 rng(7);
  auto upto = [&](double hi) {  // 1 .. hi, evenly over the logarithm
    return (int)std::exp(std::uniform_real_distribution<double>(0, std::log(hi + 0.999))(rng));
  };
  int64_t eight = 0, rows[3] = {}, cut_calls = 0;
  for (int n = 0; n < 60000; ++n) {
    const int cus = n % 3 ? 256 : upto(304), batch = upto(300), hkv = upto(40), group = upto(40);
    const int dim = n & 1 ? 128 : 64;
    const int top_q = upto(n % 5 ? 600 : 20000), top_len = upto(n % 7 ? 20000 : 3e5);
    struct Seq {
      int m, len;
    };
    std::vector<Seq> seqs(batch);
    int64_t total = 0;
    int max_q = 0, max_len = 0;
    for (Seq& s : seqs) {
      s.m = n % 11 ? upto(top_q + 1) - 1 : top_q;
      s.len = n % 13 ? upto(top_len + 1) - 1 : top_len;
      total += s.m;
      max_q = std::max(max_q, s.m);
      max_len = std::max(max_len, s.len);
    }
    if (total == 0) continue;
    VarlenShape s;
    if (!varlen_shape(cus, batch, total, max_q, max_len, hkv * group, hkv, dim, &s)) continue;
    const int tile_rows = 32 * (s.long_rows ? 8 : 4 / s.key_tiles), step = 64 * s.key_tiles;
    auto tiles_of = [&](const Seq& q) {
      return ((int64_t)q.m * group + tile_rows - 1) / tile_rows * hkv;
    };
    auto steps_of = [&](const Seq& q) {  // (the last query sees every key)
      return q.m > 0 ? (q.len + step - 1) / step : 0;
    };
    int64_t cost = 0, pieces = 0, cut = 0;
    for (const Seq& q : seqs) cost += tiles_of(q) * steps_of(q);
    const int span = s.target > 0 ? span_of(cost, s.target, s.least) : INT32_MAX;
    for (const Seq& q : seqs) {
      const int r = ranges_of(steps_of(q), span);
      pieces += tiles_of(q) * r;
      cut += r > 1 ? tiles_of(q) : 0;
    }
    CHECK(pieces <= s.pieces, "batch %d: %lld pieces, a grid of %lld", n, (long long)pieces,
          (long long)s.pieces);
    CHECK(cut <= s.cut, "batch %d: %lld tiles cut, room for %lld", n, (long long)cut, (long long)s.cut);
    CHECK(s.workspace() == (s.target > 0 ? s.pieces * tile_rows * (4ll * dim + 8) + 256 + 24 * s.cut : 0),
          "batch %d: a workspace of %lld", n, (long long)s.workspace());
    eight += s.long_rows;
    if (s.target == 0) continue;
    cut_calls += cut > 0;
    CHECK(s.merge_rows == 4 || s.merge_rows == 16 || (s.merge_rows == 32 && !s.long_rows),
          "batch %d: %d rows of a merge workgroup", n, s.merge_rows);
    CHECK(s.merge_rows * s.merge_per_tile >= std::min<int64_t>((int64_t)max_q * group, tile_rows),
          "batch %d: %lld merge workgroups of %d rows", n, (long long)s.merge_per_tile, s.merge_rows);
    ++rows[s.merge_rows == 4 ? 0 : s.merge_rows == 16 ? 1 : 2];
  }
  // the run took every form
  CHECK(eight > 100 && cut_calls > 1000 && rows[0] > 100 && rows[1] > 100 && rows[2] > 100,
        "%lld of eight waves, %lld cut, merges of 4 / 16 / 32 rows: %lld %lld %lld", (long long)eight,
        (long long)cut_calls, (long long)rows[0], (long long)rows[1], (long long)rows[2]);
}

// Sequences of one length under eight waves: their pieces fit the CUs at once wherever
// the row tiles do twice.
static void equal_lengths() {
  int64_t cut = 0;
  for (const int cus : {256, 304, 80})
    for (const int heads : {1, 2, 4, 8, 5})
      for (const int group : {1, 7, 8, 20})
        for (int batch = 1; batch <= 8; batch *= 2)
          for (const int len : {700, 4000, 16000, 60000, 131072})
            for (int m = 1; m <= 1200; m += m < 40 ? 1 : 7) {
              VarlenShape s;
              if (m > len ||
                  !varlen_shape(cus, batch, (int64_t)batch * m, m, len, heads * group, heads, 128, &s))
                continue;
              const int64_t tiles = (int64_t)(m * group + 255) / 256 * heads * batch;
              if (!s.long_rows || s.target == 0 || tiles > cus / 2) continue;
              const int steps = (len + 63) / 64;
              const int64_t pieces = tiles * ranges_of(steps, span_of(tiles * steps, s.target, s.least));
              CHECK(pieces <= cus, "%d x %d queries over %d, %d x %d heads: %lld pieces of %lld tiles, "
                    "%d CUs", batch, m, len, heads, group, (long long)pieces, (long long)tiles, cus);
              cut += pieces > tiles;
            }
  CHECK(cut > 1000, "%lld cut", (long long)cut);
}

// The largest arguments that the entry points let through: no product wraps, and a
// grid that fits or a refusal.
static void extremes() {
  const int32_t big = INT32_MAX;
  for (const int32_t batch : {1, 1000, big})
    for (const int64_t total : {(int64_t)1, (int64_t)big, (int64_t)1 << 40, INT64_MAX})
      for (const int32_t hkv : {1, 255, 65535})
        for (const int32_t group : {1, 257, 65535})
          for (const int32_t max_len : {0, 4096, big - 256})
            for (const int32_t max_q : {1, 64, 4096, big / 2 / group}) {
              if ((int64_t)hkv * group > 65535 || (int64_t)max_q * group > big / 2) continue;
              for (const int dim : {64, 128}) {
                VarlenShape s;
                if (!varlen_shape(256, batch, total, max_q, max_len, hkv * group, hkv, dim, &s)) continue;
                CHECK(s.pieces > 0 && s.pieces <= big / 2 && s.workspace() >= 0 && s.cut >= 0,
                      "batch %d, %lld tokens, %d x %d heads: %lld pieces", batch, (long long)total, hkv,
                      group, (long long)s.pieces);
              }
            }
}

int main() {
  equal_lengths();
  extremes();
  ranges();
  batches();
  std::printf("ok\n");
  return 0;
}
