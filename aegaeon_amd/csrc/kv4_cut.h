// How the attention of several query tokens over the 4- and the 8-bit
// cache cuts its work into workgroups: arithmetic alone, without device code.
#pragma once

#include <algorithm>
#include <cstdint>

namespace aegkv {

constexpr int kUnitRows = 32;    // rows of a wave
constexpr int kKeyTile = 64;     // keys of a tile
constexpr int kShortWaves4 = 4;
constexpr int kLongWaves4 = 8;

// A row tile whose keys are cut: its rows [row0, row1) of kv head `head`, the first
// of its pieces, which follow each other.
struct CutTile {
  int32_t t0, head, row0, row1, piece0, pieces;
};

// Key steps of a piece at most, for `target` pieces of a batch of `cost` (key steps
// times row tiles).
constexpr int span_of(int64_t cost, int64_t target, int least) {
  const int64_t span = (cost + target - 1) / target;
  return span > INT32_MAX ? INT32_MAX : span > least ? (int)span : least;
}

// The ranges into which n_kt key steps are cut at a span of at most `span` each (one
// without any step; INT32_MAX: uncut).
constexpr int ranges_of(int n_kt, int span) {
  const uint32_t r = ((uint32_t)n_kt + (uint32_t)span - 1) / (uint32_t)span;  // < 2^32
  return r > 1 ? (int)r : 1;
}

// The other cut, of eight-wave tiles (one workgroup per CU) that are fewer than the
// CUs but more than half of them: a tile's first piece has `span` key steps, and what
// is left of the tiles goes to the CUs that have none or are done.  Workgroups are dealt
// to groups of 8 CUs in turn and stay there: of T tiles on P places a group has up to
// m = ceil(8 T / P) first pieces, and its 8 - m other CUs take m remainders in
// ceil(m / (8 - m)) rounds, so a span is rounds / (rounds + 1) of a tile (m = 8: a whole
// one of average length, so that only longer ones are cut), and the average work of a
// place at least; a piece costs kPieceStart steps beside its own (its start, its
// partials).  Sequences of more steps get more pieces of `span`.  `cost`: key steps of
// all tiles.  Us a pass of the 8-bit cache, uncut and so (bf16, D = 128; one session):
// 28/4 heads, 1250 queries over 16000 tokens (140 tiles) 470 and 342, 1500 (168) 471 and
// 379, 2048 (224) 473 and 450 (a step takes 2.1 us with every CU at work, 1.85 with 224),
// 3 x 700 over 4100 to 7400 (240) 229 and 215; 8/8 heads, 14 x 512 over 4258 to 7471 (224)
// 228 and 200, over 8000 each 245 and 251.  So tiles of one length on 7/8 of the CUs gain
// nothing and pay the merge; they are cut all the same, as the host does not know the
// lengths and uneven ones gain more than that.
constexpr int kPieceStart = 8;
constexpr int uneven_span(int64_t cost, int64_t tiles, int64_t places, int least) {
  if (tiles <= 0 || places <= 0) return INT32_MAX;
  if (2 * tiles <= places) return span_of(2 * cost, places, least);
  const int64_t whole = cost + kPieceStart * tiles, each = whole / tiles + 1;
  const int64_t m = (8 * tiles + places - 1) / places, rounds = m < 8 ? 7 / (8 - m) : 0;
  const int64_t even = (whole + places - 1) / places;
  const int64_t part = m < 8 ? each * rounds / (rounds + 1) : each;
  const int64_t span = even > part ? even : part;
  return span > INT32_MAX ? INT32_MAX : (int)span;
}
// The pieces of n_kt key steps then; all have `span` steps but the last one, which has
// more than kLeastRest, and up to as many more than `span`.
constexpr int kLeastRest = 8;
constexpr int uneven_ranges(int n_kt, int span) {
  return n_kt - kLeastRest > span ? (n_kt - kLeastRest - 1) / span + 1 : 1;
}

// The launch of a call: which kernel, how many pieces at most, and whether
// sequences are cut.
struct VarlenShape {
  bool long_rows;
  bool uneven;      // cut by uneven_span
  int key_tiles;    // of a step
  int64_t pieces;   // bound of the pieces (the main grid)
  int64_t target;   // pieces wanted (0: uncut)
  int32_t least;    // key steps of a piece at least
  int64_t cut;      // bound of the row tiles that are cut
  int merge_rows;   // rows of a merge workgroup
  int64_t merge_per_tile;  // merge workgroups of a row tile
  int64_t o_bytes, ml_bytes, cut_bytes;
  int64_t workspace() const { return o_bytes + ml_bytes + cut_bytes; }
};
// The ping-pong kernel takes rows past the four-wave kernel's two tiles when its row
// tiles fit the CUs at once and leave each 32 key steps or more (head_dim 128, 28/4
// heads, equal lengths, us, against four waves: 4 x 512 over 8000 tokens 239 and 259,
// 1 x 1024 over 16000 247 and 270, 8/8 heads 14 x 512 over 8000 240 and 262).
// Shorter or more numerous tiles do better with two workgroups per CU, which
// overlap one's start and end with the other's steps (4 x 64 over 4000 51 and 40,
// 18 x 128 over 1000 83 and 54, 48 prompts of 220 tokens 93 and 71), and so does
// head_dim 64 always (8/8, 14 x 512 over 8000: 229 and 207, 16/1, 24 x 512 over 2000:
// 217 and 148).
constexpr int kLongRows = 256, kLongSteps = 32;
// A piece's key steps at least: its partials cost about what half of these do
// (48 x 5 drafted tokens over 1000 each: 31 us, with 8 steps 35, with 2 still 31).
constexpr int kLeastLong = 16, kLeastShort = 4;

// False: more pieces than a grid.  (Heads of up to 65535 and rows of a sequence of up
// to 2^30: no product passes 64 bits.)  uneven: the cache's kernels take that cut.
inline bool varlen_shape(int64_t cus, int32_t batch, int64_t total_q, int32_t max_q,
                         int32_t max_len, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                         VarlenShape* out, bool uneven = false) {
  const int64_t group = n_q_heads / n_kv_heads, max_rows = (int64_t)max_q * group;
  total_q = std::min<int64_t>(total_q, INT32_MAX);  // (cu_seqlens end there)
  VarlenShape s{};
  // row tiles: those that the tokens fill, and a part-filled one per sequence
  auto jobs_of = [&](int64_t rows) {
    return n_kv_heads * std::min(batch * ((max_rows + rows - 1) / rows),
                                 total_q * group / rows + batch);
  };
  const int64_t long_jobs = jobs_of(kLongWaves4 * kUnitRows);
  s.long_rows = head_dim == 128 && max_rows > kLongRows && long_jobs <= cus &&
                long_jobs * ((max_len + kKeyTile - 1) / kKeyTile) >= kLongSteps * cus;
  s.key_tiles = max_rows <= kShortWaves4 / 2 * kUnitRows ? 2 : 1;
  const int64_t tile_rows =
      (s.long_rows ? kLongWaves4 : kShortWaves4 / s.key_tiles) * kUnitRows;
  const int64_t jobs = s.long_rows ? long_jobs : jobs_of(tile_rows);
  const int64_t step = (int64_t)s.key_tiles * kKeyTile;
  const int64_t max_kt = (max_len + step - 1) / step;
  s.pieces = jobs;
  s.least = s.long_rows ? kLeastLong : kLeastShort;
  // Workgroups that run at once.  With half as many row tiles or fewer, their keys
  // are cut into about as many pieces, but not more where a second round costs much:
  // a tile's ranges are rounded up, so 7/8 of a piece a tile less (2 x 256 queries
  // over 4000, 112 tiles: 53 us, of as many pieces as places and more 66; of up to 64
  // rows the work is as uneven anyway: 48 x 5 over 1000, 192 tiles: 26.9, so 28.4).
  // Eight waves have their CU to themselves, and a second round of them costs a whole
  // one: no more pieces a tile than go into the places as a whole number (1 x 448 over
  // 16001, 28/4 heads, 52 tiles of four pieces: 132 us, of five 201; four waves, whose
  // second round overlaps the first, take the piece more: 2 x 698 over 12000, 16/1
  // heads of 64, 176 tiles of three 140, of two 161).  With more tiles only sequences
  // of twice the average work of a place are cut, as partials cost more than an uneven
  // last round (2048 queries over 16001 tokens, 224 tiles: whole 460 us, cut in two
  // 498).  Four times as many tiles even out by themselves.
  const int64_t slots = cus * (s.long_rows ? 1 : 2);
  if (jobs < 4 * slots && max_kt > s.least) {
    s.target = jobs > slots / 2 ? slots / 2 : s.key_tiles > 1 ? slots : slots - jobs * 7 / 8;
    if (s.long_rows && jobs <= slots / 2) s.target = std::min(s.target, slots / jobs * jobs);
    // a sequence of cost x has at most x / span + its tiles
    s.pieces = std::min(s.target + jobs, jobs * ((max_kt + s.least - 1) / s.least));
    s.uneven = uneven && s.long_rows && jobs > slots / 2;
    if (s.uneven) {
      // (its cost is of the tiles' own steps, half of the sequences' at least; the span
      // is a place's share of it at least)
      s.target = slots;
      s.pieces = jobs + 2 * slots;
    }
    s.cut = jobs;
    auto per_tile = [&](int64_t r) { return (std::min(max_rows, tile_rows) + r - 1) / r; };
    // Rows of a merge workgroup.  4 where a tile has 16 pieces or more (28/4 heads over
    // 16000 tokens, us with 4 and with 16 rows: 2 / 4 / 8 / 12 / 16 x 4 queries, of 64,
    // 32, 16, 11, 8 pieces a tile, 21.3 and 24.5, 25.2 and 28.3, 33.4 and 34.6, 55.7 and
    // 56.2, 51.4 and 50.9; 2 / 4 / 8 / 12 x 16, of 63, 31, 15, 10: 31.3 and 38.4, 39.3
    // and 40.0, 54.5 and 53.6, 71.0 and 69.3), 16 where it has fewer, 32 where those
    // would be more than 4096 workgroups, of tiles mostly uncut (16 and 32 rows: 100 x 64
    // over 1500 on average, 12800: 227 and 225; 400 x 9 over 1000, 6400: 144 and 141;
    // 256 x 9, 4096: 91.3 and 91.5).
    s.merge_rows = s.target >= 16 * jobs ? 4
                   : s.long_rows || jobs * per_tile(16) <= 4096 ? 16 : 32;
    s.merge_per_tile = per_tile(s.merge_rows);
    s.ml_bytes = s.pieces * tile_rows * 8;
    s.cut_bytes = 256 + s.cut * (int64_t)sizeof(CutTile);
    s.o_bytes = s.pieces * tile_rows * head_dim * 4;
  }
  *out = s;
  return s.pieces <= INT32_MAX / 2 && s.cut * s.merge_per_tile <= INT32_MAX / 2;
}

}  // namespace aegkv
