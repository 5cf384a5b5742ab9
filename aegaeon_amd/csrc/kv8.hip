// Writing and de-paging the 8-bit KV cache (kv8_format.h) on gfx950:
//  - kv8_append: slot-mapped write of new 16-bit K/V rows, one layer or every
//    layer of a step in one launch, or one layer's rows turned by their positions
//    on the way, with the queries turned beside them (rotary_rows.h);
//  - kv8_gather: block-table-driven de-page of sequences into contiguous 16-bit
//    [sum(len), Hkv, D] buffers.
// A wave takes one block of one head and side, a lane the 8 dims 8 c .. of the
// tokens 4 g .. 4 g + 3 (lane = 16 g + c; D = 64: c < 8; D = 256: and dims 128
// further): a block's maximum is a reduction within the wave, and V's words, four
// tokens of a dim, come together in one lane's registers.
//   Both are bound by memory once they are large.  4 kv heads of 128, bf16:
//   append    28 layers of a decode step of 128 tokens 10.9 us: latency of the chain
//             slot, scale byte, new scale, and lines written in part.  Of 256 tokens 15.9:
//             a token's K is 16 bytes in each of eight lines per head and layer, its V
//             one byte in four of another four, so 128 tokens touch 24 MB of lines for
//             3.7 MB of codes, beside 7.3 MB of rows.  8 layers of 4 x 1024 tokens 21.2 us
//             (100 MB, 4.7 TB/s).
//   rotating  one layer beside 28 query heads: 128 tokens 5.0 us, 4000 of four prompts
//             18.3 (71 MB, 3.9 TB/s: the keys' waves load partners and angles too).
//   gather    128 sequences of 400 tokens on average 25.4 us (155 MB, 6.1 TB/s).
#include <algorithm>

#include "aegkv_internal.h"
#include "kv8_format.h"
#include "rotary_rows.h"
#include "wave_scan.h"

namespace aegkv {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kAppend8Threads = 256;
// How a call turns its keys and queries: not at all, pairs half a row apart, neighbours.
constexpr int kStill = 0, kHalves = 1, kNeighbours = 2;

struct Append8Args {
  HeadRows k, v;             // sources (dst unused)
  int64_t k_layer_b, v_layer_b;
  const int64_t* slots;
  uint8_t* cache;
  int64_t blk_b, layer_b;    // cache byte strides
  int64_t n_slots;           // n_blocks * 16
  int64_t scales_at;         // kv8_scales_at
  uint32_t n_tokens, n_heads;
  uint32_t window;           // tokens whose runs a wave takes, 1 .. 16
  uint32_t n_windows;
  uint32_t n_waves;          // that write the cache: layers * windows * heads * 2
  // a rotating call (q.src != nullptr): then the tasks of the queries, and of the
  // keys to out_key
  RotaryTable r;
  HeadRows q, ok;
  uint32_t q_tasks, ok_tasks;  // per token
  uint32_t n_tasks;            // waves in all
};

// The largest value of the lane's 16, and of the wave, in every lane.
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true));   // lane ^ 1
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true));   // lane ^ 2
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x124, 0xf, 0xf, true));  // row_ror 4
  return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xf, 0xf, true));  // row_ror 8
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = row_max(x);
  const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return max(b[0], b[1]);
}

// Four floats to a word of codes.  clamp: |x| may exceed 448 only where the exponent
// is held at its top; NaN stays NaN (the comparisons keep it).
__device__ __forceinline__ float code_range(float x) {
  x = x > kKv8Largest ? kKv8Largest : x;
  return x < -kKv8Largest ? -kKv8Largest : x;
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(code_range(a), code_range(b), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(code_range(c), code_range(d), w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ void floats4(uint32_t w, float (&f)[4]) {
  const f32x2 a = __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false));
  const f32x2 b = __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true));
  f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
}
// The wave's part of a call: a head and side of a layer.
struct Side {
  const uint8_t* rows;  // of token 0
  int64_t tok_b;
  uint8_t* layer;       // the layer's part of block 0
  int64_t codes, scale; // offsets there
  bool value;
};
__device__ __forceinline__ Side side_of(const Append8Args& a, uint32_t layer, uint32_t head,
                                        bool value, int dim) {
  const HeadRows& h = value ? a.v : a.k;
  return {h.src + layer * (value ? a.v_layer_b : a.k_layer_b) + (int64_t)head * dim * 2,
          h.src_tok_b, a.cache + layer * a.layer_b,
          (int64_t)(2 * head + (value ? 1 : 0)) * kv8_side_bytes(dim), a.scales_at + 4 * head,
          value};
}

// Chunk c of four tokens' rows (tok < 0: none, zeros) in 32 bits, turned if they are
// keys: the loads of all four are in flight together.  top: the largest of the
// finite magnitudes' bits; bad: there are others, which become NaN.
template <int DT, int TURN>
__device__ __forceinline__ void load_rows(const Append8Args& a, const Side& s, const int (&tok)[4],
                                          int c, float (&f)[4][8], uint32_t (&top)[4],
                                          bool (&bad)[4]) {
  constexpr bool INTER = TURN == kNeighbours;
  const bool turns = TURN != kStill && !s.value && chunk_turns(a.r, c);
  u32x4 x[4], y[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[k] = y[k] = u32x4{0u, 0u, 0u, 0u};
    if (tok[k] >= 0) {
      const uint8_t* p = s.rows + (int64_t)tok[k] * s.tok_b;
      x[k] = *reinterpret_cast<const u32x4*>(p + 16 * c);
      if (turns) y[k] = *reinterpret_cast<const u32x4*>(p + 16 * partner_chunk<INTER>(a.r, c));
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (TURN != kStill && turns && tok[k] >= 0)
      turn_chunk<DT, INTER>(x[k], y[k], load_angles<INTER>(a.r, a.r.positions[tok[k]], c), f[k]);
    else
      unpack8<DT>(x[k], f[k]);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const uint32_t u = __float_as_uint(f[k][d]) & 0x7fffffffu;
      const bool odd = u >= 0x7f800000u;
      bad[k] |= odd;
      top[k] = max(top[k], odd ? 0u : u);
      f[k][d] = odd ? __builtin_nanf("") : f[k][d];
    }
  }
}
// A held scale byte within the type's bounds.
template <int DT>
__device__ __forceinline__ int held_scale(int byte) {
  return min(max(byte, Kv8Elem<DT>::kLow), Kv8Elem<DT>::kTop);
}
// A word of codes under an exponent that is larger by the factor's inverse.
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float down) {
  float t[4];
  floats4(w, t);
  return codes4(t[0] * down, t[1] * down, t[2] * down, t[3] * down);
}
__device__ __forceinline__ float down_factor(int from, int to) {
  return kv8_scale((uint32_t)max(127 + from - to, 0));
}

// One run: tokens of block blk; tok[k]: the one for place 4 g + k.
template <int DT, int D, int TURN>
__device__ __forceinline__ void append_run(const Append8Args& a, const Side& s, int64_t blk,
                                           int (&tok)[4], bool anew) {
  constexpr int NC = D > 128 ? D / 128 : 1;  // chunks of a lane
  const int lane = threadIdx.x & 63, g = lane >> 4, c0 = lane & 15;
  const bool idle = D < 128 && c0 >= D / 8;
  bool here[4];  // places that get a token
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (idle) tok[k] = -1;
    here[k] = tok[k] >= 0;
  }
  uint8_t* rec = s.layer + blk * a.blk_b;
  uint8_t* scale = rec + s.scale;
  rec += s.codes;
  int held = Kv8Elem<DT>::kLow;
  if (!anew) held = scale[s.value ? 1 : 0];
  float f[NC][4][8];
  uint32_t top[4] = {};
  bool bad[4] = {};
#pragma unroll
  for (int q = 0; q < NC; ++q) load_rows<DT, TURN>(a, s, tok, c0 + 16 * q, f[q], top, bad);
  const bool nan = __builtin_amdgcn_ballot_w64(bad[0] || bad[1] || bad[2] || bad[3]) != 0;
  const int own =
      kv8_scale_byte<DT>(wave_max(max(max(top[0], top[1]), max(top[2], top[3]))));
  held = __builtin_amdgcn_readfirstlane(held);  // (0 in a cache never written)
  const int old = held_scale<DT>(held);
  const int now = anew ? own : max(old, own);
  const float inv = kv8_scale((uint32_t)(254 - now));  // 2^-e
  const bool rescale = !anew && now > old;             // uniform
  const float down = down_factor(old, now);
  if (!idle) {
#pragma unroll
    for (int q = 0; q < NC; ++q) {
      const int c = c0 + 16 * q;
      // new codes, of places without a new token 0
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int d = 0; d < 8; ++d) f[q][k][d] *= inv;
      if (!s.value) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          u32x2* p = reinterpret_cast<u32x2*>(rec + kv8_k_byte(4 * g + k, c));
          u32x2 w = {codes4(f[q][k][0], f[q][k][1], f[q][k][2], f[q][k][3]),
                     codes4(f[q][k][4], f[q][k][5], f[q][k][6], f[q][k][7])};
          if (rescale && !here[k]) {
            const u32x2 o = *p;
            w = u32x2{rescaled(o[0], down), rescaled(o[1], down)};
          }
          if (anew || rescale || here[k]) *p = w;
        }
      } else {
        uint32_t mine = 0;  // bytes of a word that get a token
#pragma unroll
        for (int k = 0; k < 4; ++k) mine |= here[k] ? 0xffu << (8 * k) : 0u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint8_t* p = rec + kv8_v_byte<D>(g, 2 * c + i);
          u32x4 w;
#pragma unroll
          for (int d = 0; d < 4; ++d)
            w[d] = codes4(f[q][0][4 * i + d], f[q][1][4 * i + d], f[q][2][4 * i + d],
                          f[q][3][4 * i + d]);
          if (rescale) {
            const u32x4 o = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int d = 0; d < 4; ++d) w[d] = (w[d] & mine) | (rescaled(o[d], down) & ~mine);
          }
          if (anew || rescale || mine == 0xffffffffu) {
            *reinterpret_cast<u32x4*>(p) = w;
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (here[k]) {
#pragma unroll
                for (int d = 0; d < 4; ++d) p[4 * d + k] = (uint8_t)(w[d] >> (8 * k));
              }
          }
        }
      }
    }
  }
  if (lane == 0) {
    if (anew || now != held) scale[s.value ? 1 : 0] = (uint8_t)now;
    if (s.value && (anew || nan)) scale[2] = nan ? 1 : 0;
  }
}

// Up to 16 runs of one token each, as a decode step's: the lanes 16 g .. take the
// window's tokens 4 k + g, every load of the four in flight together (28 layers of
// 128 tokens of 4 heads of 128, of the same first form of the kernel: 12.6 us, one run
// after the other 27.4; V's words read and written whole instead of their bytes 12.1, but
// prompts, whose waves it leaves fewer registers, 5-15% slower).  tok[k] (-1: none) goes to place off[k] of block
// blk[k].
template <int DT, int D, int TURN>
__device__ __forceinline__ void append_singles(const Append8Args& a, const Side& s,
                                               int (&tok)[4], const int (&blk)[4],
                                               const int (&off)[4]) {
  constexpr int NC = D > 128 ? D / 128 : 1;
  const int lane = threadIdx.x & 63, c0 = lane & 15;
  const bool idle = D < 128 && c0 >= D / 8;
  bool run[4];
  uint8_t* rec[4];
  int held[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    run[k] = tok[k] >= 0;
    if (idle) tok[k] = -1;
    rec[k] = s.layer + (int64_t)(run[k] ? blk[k] : 0) * a.blk_b;
    held[k] = Kv8Elem<DT>::kLow;
    if (run[k] && off[k] > 0) held[k] = rec[k][s.scale + (s.value ? 1 : 0)];
  }
  float f[NC][4][8];
  uint32_t top[4] = {};
  bool bad[4] = {};
#pragma unroll
  for (int q = 0; q < NC; ++q) load_rows<DT, TURN>(a, s, tok, c0 + 16 * q, f[q], top, bad);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const bool nan = (__builtin_amdgcn_ballot_w64(bad[k]) >> (lane & 48) & 0xffffu) != 0;
    const int own = kv8_scale_byte<DT>(row_max(top[k]));
    const bool anew = off[k] == 0;
    const int old = held_scale<DT>(held[k]);
    const int now = anew ? own : max(old, own);
    const float inv = kv8_scale((uint32_t)(254 - now));
    const float down = down_factor(old, now);
    uint8_t* scale = rec[k] + s.scale;
    uint8_t* side = rec[k] + s.codes;
    if (run[k] && !idle) {
#pragma unroll
      for (int q = 0; q < NC; ++q) {
        const int c = c0 + 16 * q;
        uint32_t w[2];  // the token's codes, a byte a dim
#pragma unroll
        for (int i = 0; i < 2; ++i)
          w[i] = codes4(f[q][k][4 * i] * inv, f[q][k][4 * i + 1] * inv, f[q][k][4 * i + 2] * inv,
                        f[q][k][4 * i + 3] * inv);
        if (anew || now > old) {  // the whole block: zeros, or what it holds rounded once more
          if (!s.value) {
#pragma unroll 1
            for (int r = 0; r < kKv8Tokens; ++r) {
              u32x2* p = reinterpret_cast<u32x2*>(side + kv8_k_byte(r, c));
              u32x2 o = {0u, 0u};
              if (!anew) {
                o = *p;
                o = u32x2{rescaled(o[0], down), rescaled(o[1], down)};
              }
              *p = r == off[k] ? u32x2{w[0], w[1]} : o;
            }
          } else {
#pragma unroll 1
            for (int g = 0; g < 4; ++g) {
              const uint32_t sh = 8 * (off[k] & 3), mine = g == off[k] >> 2 ? 0xffu << sh : 0u;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                u32x4* p = reinterpret_cast<u32x4*>(side + kv8_v_byte<D>(g, 2 * c + i));
                u32x4 o = {0u, 0u, 0u, 0u};
                if (!anew) o = *p;
#pragma unroll
                for (int d = 0; d < 4; ++d)
                  o[d] = ((w[i] >> (8 * d) << sh) & mine) |
                         ((anew ? 0u : rescaled(o[d], down)) & ~mine);
                *p = o;
              }
            }
          }
        } else if (!s.value) {
          *reinterpret_cast<u32x2*>(side + kv8_k_byte(off[k], c)) = u32x2{w[0], w[1]};
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint8_t* p = side + kv8_v_byte<D>(off[k] >> 2, 2 * c + i) + (off[k] & 3);
#pragma unroll
            for (int d = 0; d < 4; ++d) p[4 * d] = (uint8_t)(w[i] >> (8 * d));
          }
        }
      }
    }
    if (run[k] && c0 == 0) {
      if (anew || now != held[k]) scale[s.value ? 1 : 0] = (uint8_t)now;
      if (s.value && (anew || nan)) scale[2] = nan ? 1 : 0;
    }
  }
}

// Skipped rows (slots outside the cache) do not part a run: what lies behind them or
// before them may be any number of rows away.  Both searches are uniform, 512 rows a
// round trip, and rare: a wave makes one where the rows next to its own, up to the end of
// its 64, are all skipped (a rotating call of 1000 tokens and 3096 skipped rows behind
// them 16.1 us, 13.7 without the search; 100 single tokens and 156 such rows 5.7 for 5.1).
constexpr int kSearchLoads = 8;
// The first token at or past `from` that is not skipped (n_tokens: none).
__device__ __forceinline__ int token_from(const Append8Args& a, int from) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (; from < (int)a.n_tokens; from += 64 * kSearchLoads) {
    int64_t s[kSearchLoads];
#pragma unroll
    for (int k = 0; k < kSearchLoads; ++k)
      s[k] = a.slots[min(from + 64 * k + lane, (int)a.n_tokens - 1)];
#pragma unroll
    for (int k = 0; k < kSearchLoads; ++k) {
      const int t = from + 64 * k;
      const uint64_t in = __builtin_amdgcn_ballot_w64(t + lane < (int)a.n_tokens && s[k] >= 0 &&
                                                      s[k] < a.n_slots);
      if (in) return t + __builtin_ctzll(in);
    }
  }
  return (int)a.n_tokens;
}
// The block of the last token before `end` that is not skipped (-1: none).
__device__ __forceinline__ int block_before(const Append8Args& a, int end) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (; end > 0; end -= 64 * kSearchLoads) {
    int64_t s[kSearchLoads];
#pragma unroll
    for (int k = 0; k < kSearchLoads; ++k) s[k] = a.slots[max(end - 64 * (k + 1) + lane, 0)];
#pragma unroll
    for (int k = 0; k < kSearchLoads; ++k) {
      const uint64_t in = __builtin_amdgcn_ballot_w64(end - 64 * (k + 1) + lane >= 0 && s[k] >= 0 &&
                                                      s[k] < a.n_slots);
      if (in)
        return __builtin_amdgcn_readlane((int)(s[k] / kKv8Tokens), 63 - __builtin_clzll(in));
    }
  }
  return -1;
}
// The bits of `mine` below the first one of `others`.
__device__ __forceinline__ uint64_t up_to(uint64_t mine, uint64_t others) {
  return mine & ((others & -others) - 1);  // (no others: all of them)
}

// A wave of the cache's writers: a head and side of the runs that begin in its
// window of tokens.  A run is tokens of one block with no other block's between them in
// the call.
template <int DT, int D, int TURN>
__device__ __forceinline__ void append_window(const Append8Args& a, uint32_t id) {
  const bool value = id & 1;
  uint32_t rest = id >> 1;
  const uint32_t head = rest % a.n_heads;
  rest /= a.n_heads;
  const uint32_t win = rest % a.n_windows, layer = rest / a.n_windows;
  const int lane = threadIdx.x & 63, g = lane >> 4;
  // lane i: token `first` + i, the one before the window in lane 0
  const int first = (int)(win * a.window) - 1, tok = first + lane;  // (below 2^30: append_args)
  int64_t s = -1;
  if (tok >= 0 && tok < (int)a.n_tokens) s = a.slots[tok];
  const bool in = s >= 0 && s < a.n_slots;
  const int blk = in ? (int)(s / kKv8Tokens) : -1, off = (int)(s & (kKv8Tokens - 1));
  const uint64_t held = __builtin_amdgcn_ballot_w64(in);
  // the blocks of the nearest tokens before the lane's and behind it that are not skipped
  // (before: -1, none; behind: its own where it is not among the wave's)
  int before = __shfl_up(blk, 1), behind = __shfl_down(blk, 1);  // (every lane active)
  const bool whole = held == __builtin_amdgcn_ballot_w64(tok >= 0 && tok < (int)a.n_tokens);
  if (__builtin_expect(!whole, 0)) {  // uniform: some are skipped
    const uint64_t below = held & ((1ull << lane) - 1), above = held >> lane >> 1;
    before = __shfl(blk, below ? 63 - __builtin_clzll(below) : lane);
    behind = __shfl(blk, above ? lane + 1 + __builtin_ctzll(above) : lane);
    int back = -1;
    if (!(held & 1) && held & 0x1fffe && first > 0) back = block_before(a, first);  // uniform
    if (!below) before = back;
    if (!above && first + 64 >= (int)a.n_tokens) behind = -1;
  }
  const bool begins = lane > 0 && lane <= (int)a.window && in && blk != before;
  uint32_t heads = (uint32_t)__builtin_amdgcn_ballot_w64(begins);  // (lanes 1 .. 16)
  if (!heads) return;  // uniform
  const Side side = side_of(a, layer, head, value, D);
  if (a.window > 1 && __builtin_amdgcn_ballot_w64(begins && blk == behind) == 0) {
    int at[4];
    int b[4], o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 1 + 4 * k + g;  // the token's lane, at most 16
      b[k] = __shfl(blk, i);
      o[k] = __shfl(off, i);
      at[k] = heads >> i & 1 ? first + i : -1;
    }
    append_singles<DT, D, TURN>(a, side, at, b, o);
    return;
  }
  const int step = whole ? off - lane : INT32_MAX;  // the same in places one after the other
  while (heads) {  // uniform
    const int i = __builtin_ctz(heads);
    heads &= heads - 1;
    const int b = __builtin_amdgcn_readlane(blk, i);
    const uint64_t same = __builtin_amdgcn_ballot_w64(blk == b) >> i;
    const int n = __builtin_ctzll(~same);  // neighbours of one block (i > 0: bit 63 is clear)
    const int off0 = __builtin_amdgcn_readlane(off, i);
    int at[4];
    bool anew;
    const uint64_t run = (1ull << n) - 1;
    const uint64_t in_order = __builtin_amdgcn_ballot_w64(step == off0 - i) >> i;
    if (__builtin_expect((in_order & run) == run, 1)) {  // one place after the other
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = 4 * g + k - off0;
        at[k] = r >= 0 && r < n ? first + i + r : -1;
      }
      anew = off0 == 0;
    } else {  // of two tokens for one place the later one
#pragma unroll
      for (int k = 0; k < 4; ++k) at[k] = -1;
      anew = false;
      int base = first;
      int place = off;
      uint64_t todo = same << i;
      uint64_t others = (__builtin_amdgcn_ballot_w64(blk >= 0) & ~todo) >> i << i;
      todo = up_to(todo, others);
      while (true) {  // uniform
        for (; todo; todo &= todo - 1) {
          const int x = __builtin_ctzll(todo), o = __builtin_amdgcn_readlane(place, x);
          anew |= o == 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) at[k] = o == 4 * g + k ? base + x : at[k];
        }
        if (others) break;
        // the run may go on past the wave's tokens: the next 64, from one not skipped
        base = token_from(a, base + 64);
        if (base >= (int)a.n_tokens) break;
        const int64_t next = base + lane < (int)a.n_tokens ? a.slots[base + lane] : -1;
        place = (int)(next & (kKv8Tokens - 1));
        const bool there = next >= 0 && next < a.n_slots;
        const uint64_t on = __builtin_amdgcn_ballot_w64(there && next / kKv8Tokens == b);
        others = __builtin_amdgcn_ballot_w64(there) & ~on;
        todo = up_to(on, others);
      }
    }
    append_run<DT, D, TURN>(a, side, b, at, anew);
  }
}

// (Four waves per SIMD asked for: a register too many left three, 15% slower for prompts
// of heads of 64; five made the loads wait for registers, 10% slower for 4 x 1000 tokens.
// Three for heads of 256, whose rotating form in fp16 needs all of those 168 registers.)
template <int DT, int D, int TURN>
__global__ __launch_bounds__(kAppend8Threads, D > 128 ? 3 : 4) void kv8_append_kernel(Append8Args a) {
  uint32_t id = __builtin_amdgcn_readfirstlane(blockIdx.x * (kAppend8Threads / 64) +
                                               (threadIdx.x >> 6));
  if (id >= a.n_tasks) return;
  if (id < a.n_waves) {
    append_window<DT, D, TURN>(a, id);
    return;
  }
  if constexpr (TURN != kStill) {
    id -= a.n_waves;
    const uint32_t per = a.q_tasks + a.ok_tasks, tok = id / per;
    const int part = (int)(id - tok * per);
    if (part < (int)a.q_tasks)
      turn_heads<DT, TURN == kNeighbours>(a.q, a.r, true, (int)tok, part, D / 8, nullptr);
    else
      turn_heads<DT, TURN == kNeighbours>(a.ok, a.r, true, (int)tok, part - (int)a.q_tasks, D / 8, nullptr);
  }
}

// De-page: a tile is one block of one sequence in a pass of 8 / (head, side) units,
// two per wave.  Each workgroup scans the batch's block counts into LDS and walks
// its layer's tiles round-robin; the next tile's block id and output row are fetched
// while the current one's loads are in flight.
constexpr int kGather8Threads = 256;
constexpr int kGather8MaxBatch = 1024;  // sequences per launch (LDS scan)
constexpr int kGather8PerWave = 2;      // units of a wave in a tile (D = 64: twice that)
constexpr int kGather8WorkgroupsPerCu = 16;

struct Gather8Args {
  const uint8_t* cache;
  int64_t blk_b, layer_b, scales_at;
  int64_t n_blocks;
  const int32_t* block_tables;
  int32_t max_blocks;
  const int32_t* seq_lens;
  const int32_t* cu_seqlens;
  uint8_t* out_k;
  uint8_t* out_v;
  int64_t out_tokens;   // capacity of the output in tokens
  int64_t out_layer_b;
  int32_t max_seq_len;
  int32_t batch;        // <= kGather8MaxBatch
  int32_t n_heads;
  int32_t passes;       // of a block
};

// The 8 dims of chunk c of tokens 4 g + k of K: eight bytes of each token.
__device__ __forceinline__ void load_k8(const uint8_t* side, int g, int c, u32x2 (&w)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    w[k] = *reinterpret_cast<const u32x2*>(side + kv8_k_byte(4 * g + k, c));
}
// Those of V, from words of one dim and four tokens.
template <int D>
__device__ __forceinline__ void load_v8(const uint8_t* side, int g, int c, u32x4 (&w)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = *reinterpret_cast<const u32x4*>(side + kv8_v_byte<D>(g, 2 * c + i));
}
__device__ __forceinline__ void by_token(const u32x4 (&w)[2], u32x2 (&t)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // (a.0 b.0 a.1 b.1) of two dims, then of four
    const uint32_t a = __builtin_amdgcn_perm(w[i][1], w[i][0], 0x05010400u);
    const uint32_t b = __builtin_amdgcn_perm(w[i][1], w[i][0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[i][3], w[i][2], 0x05010400u);
    const uint32_t d = __builtin_amdgcn_perm(w[i][3], w[i][2], 0x07030602u);
    t[0][i] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    t[1][i] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    t[2][i] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    t[3][i] = __builtin_amdgcn_perm(d, b, 0x07060302u);
  }
}

template <int DT, int D>
__global__ __launch_bounds__(kGather8Threads) void kv8_gather_kernel(Gather8Args a) {
  using E = Kv8Elem<DT>;
  __shared__ int32_t pre[kGather8MaxBatch + 1];  // first block of each sequence
  __shared__ int32_t lens[kGather8MaxBatch];
  __shared__ int32_t wsum[kGather8Threads / 64];
  constexpr int PER = kGather8MaxBatch / kGather8Threads;
  const int t = threadIdx.x, B = a.batch;
  int cnt[PER], run = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {  // loads issued together, clamped in bounds
    const int b = t * PER + k;
    const int raw = a.seq_lens[min(b, B - 1)];
    const int len = b < B ? min(max(raw, 0), a.max_seq_len) : 0;
    if (b < B) lens[b] = len;
    cnt[k] = (len + kKv8Tokens - 1) / kKv8Tokens;
    run += cnt[k];
  }
  const int incl = wave_prefix(run);
  if ((t & 63) == 63) wsum[t >> 6] = incl;
  __syncthreads();
  int excl = incl - run;
  for (int w = 0; w < (t >> 6); ++w) excl += wsum[w];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = t * PER + k;
    if (b <= B) pre[b] = excl;
    excl += cnt[k];
  }
  if (t == kGather8Threads - 1) pre[B] = excl;  // total (B may equal the capacity)
  __syncthreads();
  const uint32_t total = (uint32_t)pre[B] * a.passes;
  uint32_t at = blockIdx.x;
  if (at >= total) return;  // uniform

  auto locate = [&](uint32_t x, int& b, int& j, int& ps) {
    const int r = (int)(x / (uint32_t)a.passes);
    ps = (int)(x - (uint32_t)r * a.passes);
    int lo = 0, hi = B - 1;  // the last sequence whose first block is <= r
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] <= r) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    j = r - pre[lo];
  };
  // a wave's units: D = 64 two at once, of 32 lanes each; D = 256 in two halves
  constexpr int UW = D == 64 ? 2 : 1, NC = D == 256 ? 2 : 1, LC = D == 64 ? 8 : 16;
  const int lane = t & 63, wave = t >> 6;
  const int g = lane / LC & 3, c0 = lane % LC, sub = D == 64 ? lane >> 5 : 0;
  const int64_t row_b = (int64_t)a.n_heads * D * 2;
  const int layer = (int)blockIdx.y;
  int b, j, ps;
  locate(at, b, j, ps);
  int32_t id = a.block_tables[(int64_t)b * a.max_blocks + j];
  int64_t row0 = a.cu_seqlens[b];
  while (true) {
    const int64_t row = row0 + (int64_t)j * kKv8Tokens;
    int n_tok = min(kKv8Tokens, lens[b] - j * kKv8Tokens);
    if (row < 0 || row >= a.out_tokens || id < 0 || id >= a.n_blocks) n_tok = 0;
    else n_tok = (int)min((int64_t)n_tok, a.out_tokens - row);
    const uint8_t* blk = a.cache + (int64_t)max(id, 0) * a.blk_b + layer * a.layer_b;
    u32x2 kw[kGather8PerWave][NC][4];
    u32x4 vw[kGather8PerWave][NC][2];
    uint32_t sb[kGather8PerWave];
    bool have[kGather8PerWave];
    int unit[kGather8PerWave];
#pragma unroll
    for (int u = 0; u < kGather8PerWave; ++u) {
      // units: K of every head, then V of every head; a wave's follow each other
      const int x = ((ps * (kGather8Threads / 64) + wave) * kGather8PerWave + u) * UW + sub;
      unit[u] = x;
      have[u] = x < 2 * a.n_heads && 4 * g < n_tok;
      sb[u] = 0;
      if (have[u]) {
        const bool value = x >= a.n_heads;
        const int head = value ? x - a.n_heads : x;
        const uint8_t* side = blk + (int64_t)(2 * head + (value ? 1 : 0)) * kv8_side_bytes(D);
        sb[u] = blk[a.scales_at + 4 * head + (value ? 1 : 0)];
#pragma unroll
        for (int q = 0; q < NC; ++q) {
          if (value) load_v8<D>(side, g, c0 + 16 * q, vw[u][q]);
          else load_k8(side, g, c0 + 16 * q, kw[u][q]);
        }
      }
    }
    const uint32_t an = at + gridDim.x;
    const bool more = an < total;
    int nb, nj, nps;
    locate(more ? an : at, nb, nj, nps);
    const int32_t nid = a.block_tables[(int64_t)nb * a.max_blocks + nj];
    const int64_t nrow0 = a.cu_seqlens[nb];
#pragma unroll
    for (int u = 0; u < kGather8PerWave; ++u) {
      if (!have[u]) continue;
      const bool value = unit[u] >= a.n_heads;
      const int head = value ? unit[u] - a.n_heads : unit[u];
      const float s = kv8_scale(sb[u]);
      uint8_t* out = (value ? a.out_v : a.out_k) + layer * a.out_layer_b + (row + 4 * g) * row_b +
                     (int64_t)head * D * 2;
#pragma unroll
      for (int q = 0; q < NC; ++q) {
        u32x2 w[4];
        if (value) {
          by_token(vw[u][q], w);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = kw[u][q][k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const u32x4 x = {E::template dq<false>(w[k][0], s), E::template dq<true>(w[k][0], s),
                           E::template dq<false>(w[k][1], s), E::template dq<true>(w[k][1], s)};
          if (4 * g + k < n_tok)
            __builtin_nontemporal_store(
                x, reinterpret_cast<u32x4*>(out + k * row_b + 16 * (c0 + 16 * q)));
        }
      }
    }
    if (!more) break;
    at = an;
    b = nb;
    j = nj;
    ps = nps;
    id = nid;
    row0 = nrow0;
  }
}

bool head_dim_ok(int32_t d) { return d == 64 || d == 128 || d == 256; }
bool dtype_ok(int32_t t) { return t == AEGKV_DTYPE_BF16 || t == AEGKV_DTYPE_FP16; }

template <int DT, int TURN>
void launch_append(const Append8Args& a, int32_t head_dim, hipStream_t st) {
  constexpr uint32_t kWavesOf = kAppend8Threads / 64;
  const dim3 g((a.n_tasks + kWavesOf - 1) / kWavesOf), t(kAppend8Threads);
  if (head_dim == 64) hipLaunchKernelGGL((kv8_append_kernel<DT, 64, TURN>), g, t, 0, st, a);
  else if (head_dim == 128) hipLaunchKernelGGL((kv8_append_kernel<DT, 128, TURN>), g, t, 0, st, a);
  else hipLaunchKernelGGL((kv8_append_kernel<DT, 256, TURN>), g, t, 0, st, a);
}
template <int DT>
void launch_gather(const Gather8Args& a, int32_t head_dim, dim3 g, hipStream_t st) {
  const dim3 t(kGather8Threads);
  if (head_dim == 64) hipLaunchKernelGGL((kv8_gather_kernel<DT, 64>), g, t, 0, st, a);
  else if (head_dim == 128) hipLaunchKernelGGL((kv8_gather_kernel<DT, 128>), g, t, 0, st, a);
  else hipLaunchKernelGGL((kv8_gather_kernel<DT, 256>), g, t, 0, st, a);
}

// Tokens of a wave's window.  A wave looks for the runs that begin there and writes
// longer ones one after the other, so 1 is best while the waves fit the chip; of a
// prompt 15 of 16 tokens begin none.
constexpr uint64_t kAppend8Waves = 2048;
uint32_t window_of(uint64_t waves_of_one) {
  uint32_t w = 1;
  while (w < 16 && waves_of_one > kAppend8Waves * w) w *= 2;
  return w;
}

// The part of a call that both appends share: checks of the cache and the rows, and
// the waves that write.  A status; AEGKV_OK without tokens too, with `a` as it was.
int append_args(Append8Args& a, const void* key, const void* value, int64_t key_token_stride,
                int64_t value_token_stride, int64_t key_layer_stride, int64_t value_layer_stride,
                const int64_t* slot_mapping, int64_t n_tokens, void* cache,
                int64_t cache_block_stride, int64_t cache_layer_stride, int64_t n_blocks,
                int32_t n_layers, int32_t n_kv_heads, int32_t head_dim, int32_t dtype) {
  if (n_tokens < 0 || n_layers <= 0 || n_kv_heads <= 0 || head_dim <= 0 || n_blocks < 0)
    return AEGKV_ERR_INVALID_ARG;
  if (!head_dim_ok(head_dim) || !dtype_ok(dtype) || n_kv_heads > kKv8MaxHeads ||
      n_blocks > INT32_MAX)
    return AEGKV_ERR_UNSUPPORTED;
  if (n_tokens == 0) return AEGKV_OK;
  if (!key || !value || !slot_mapping || (!cache && n_blocks > 0)) return AEGKV_ERR_INVALID_ARG;
  if (!aligned16(key) || !aligned16(value) || !aligned16(cache) || key_token_stride % 8 ||
      value_token_stride % 8 || key_layer_stride % 8 || value_layer_stride % 8 ||
      cache_block_stride % 16 || cache_layer_stride % 16)
    return AEGKV_ERR_MISALIGNED;
  // waves of windows of one token, counted in 128 bits so that no product wraps
  const unsigned __int128 waves = (unsigned __int128)(uint64_t)n_layers * 2 *
                                  (uint64_t)n_kv_heads * (uint64_t)n_tokens;
  if (n_tokens > INT32_MAX || waves > INT32_MAX) return AEGKV_ERR_UNSUPPORTED;
  a.k = HeadRows{static_cast<const uint8_t*>(key), nullptr, key_token_stride * 2, 0, n_kv_heads};
  a.v = HeadRows{static_cast<const uint8_t*>(value), nullptr, value_token_stride * 2, 0,
                 n_kv_heads};
  a.k_layer_b = key_layer_stride * 2;
  a.v_layer_b = value_layer_stride * 2;
  a.slots = slot_mapping;
  a.cache = static_cast<uint8_t*>(cache);
  a.blk_b = cache_block_stride;
  a.layer_b = cache_layer_stride;
  a.n_slots = n_blocks * kKv8Tokens;
  a.scales_at = kv8_scales_at(n_kv_heads, head_dim);
  a.n_tokens = (uint32_t)n_tokens;
  a.n_heads = (uint32_t)n_kv_heads;
  a.window = window_of((uint64_t)waves);
  a.n_windows = (a.n_tokens + a.window - 1) / a.window;
  a.n_waves = n_blocks > 0 ? (uint32_t)n_layers * 2 * a.n_heads * a.n_windows : 0;
  a.r = RotaryTable{};
  a.q = a.ok = HeadRows{};
  a.q_tasks = a.ok_tasks = 0;
  a.n_tasks = a.n_waves;
  return AEGKV_OK;
}

}  // namespace
}  // namespace aegkv

using namespace aegkv;

extern "C" {

int64_t aegkv_kv8_block_bytes(int32_t n_kv_heads, int32_t head_dim) {
  if (n_kv_heads <= 0) return AEGKV_ERR_INVALID_ARG;
  if (!head_dim_ok(head_dim) || n_kv_heads > kKv8MaxHeads) return AEGKV_ERR_UNSUPPORTED;
  return kv8_layer_bytes(n_kv_heads, head_dim);
}

int aegkv_kv8_append(const void* key, const void* value, int64_t key_token_stride,
                     int64_t value_token_stride, int64_t key_layer_stride,
                     int64_t value_layer_stride, const int64_t* slot_mapping, int64_t n_tokens,
                     void* cache, int64_t cache_block_stride, int64_t cache_layer_stride,
                     int64_t n_blocks, int32_t n_layers, int32_t n_kv_heads, int32_t head_dim,
                     int32_t dtype, aegkv_stream_t stream) {
  Append8Args a{};
  const int rc = append_args(a, key, value, key_token_stride, value_token_stride, key_layer_stride,
                             value_layer_stride, slot_mapping, n_tokens, cache, cache_block_stride,
                             cache_layer_stride, n_blocks, n_layers, n_kv_heads, head_dim, dtype);
  if (rc) return rc;
  if (a.n_tasks == 0) return AEGKV_OK;
  if (dtype == AEGKV_DTYPE_BF16)
    launch_append<AEGKV_DTYPE_BF16, kStill>(a, head_dim, (hipStream_t)stream);
  else
    launch_append<AEGKV_DTYPE_FP16, kStill>(a, head_dim, (hipStream_t)stream);
  AEGKV_HIP_TRY(hipGetLastError());
  return AEGKV_OK;
}

int aegkv_kv8_rotary_append(const void* query, int64_t query_token_stride, void* out_query,
                            int64_t out_query_token_stride, int32_t n_q_heads, const void* key,
                            int64_t key_token_stride, const void* value,
                            int64_t value_token_stride, void* out_key,
                            int64_t out_key_token_stride, int32_t n_kv_heads, int32_t head_dim,
                            const int64_t* slot_mapping, const int64_t* positions,
                            int64_t n_tokens, const float* table, int64_t max_positions,
                            int32_t rotary_dim, int32_t interleaved, void* cache,
                            int64_t cache_block_stride, int64_t n_blocks, int32_t dtype,
                            aegkv_stream_t stream) {
  Append8Args a{};
  int rc = append_args(a, key, value, key_token_stride, value_token_stride, 0, 0, slot_mapping,
                       n_tokens, cache, cache_block_stride, 0, n_blocks, 1, n_kv_heads, head_dim,
                       dtype);
  if (rc) return rc;
  if (n_q_heads <= 0) return AEGKV_ERR_INVALID_ARG;
  a.r = RotaryTable{table, positions, max_positions, rotary_dim};
  rc = check_rotary(a.r, head_dim);
  if (rc) return rc;
  if (n_q_heads > 65535) return AEGKV_ERR_UNSUPPORTED;
  if (n_tokens == 0) return AEGKV_OK;
  if (!query || !out_query || !positions || !table || max_positions == 0)
    return AEGKV_ERR_INVALID_ARG;
  if (!aligned16(query) || !aligned16(out_query) || !aligned16(out_key) || !aligned16(table) ||
      query_token_stride % 8 || out_query_token_stride % 8 || out_key_token_stride % 8)
    return AEGKV_ERR_MISALIGNED;
  a.q = HeadRows{static_cast<const uint8_t*>(query), static_cast<uint8_t*>(out_query),
                 query_token_stride * 2, out_query_token_stride * 2, n_q_heads};
  a.ok = HeadRows{a.k.src, static_cast<uint8_t*>(out_key), a.k.src_tok_b,
                  out_key_token_stride * 2, n_kv_heads};
  a.q_tasks = (uint32_t)head_tasks(n_q_heads, head_dim / 8);
  a.ok_tasks = out_key ? (uint32_t)head_tasks(n_kv_heads, head_dim / 8) : 0;
  const uint64_t tasks = a.n_waves + (uint64_t)n_tokens * (a.q_tasks + a.ok_tasks);
  if (tasks > INT32_MAX) return AEGKV_ERR_UNSUPPORTED;
  a.n_tasks = (uint32_t)tasks;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == AEGKV_DTYPE_BF16)
    interleaved ? launch_append<AEGKV_DTYPE_BF16, kNeighbours>(a, head_dim, st)
                : launch_append<AEGKV_DTYPE_BF16, kHalves>(a, head_dim, st);
  else
    interleaved ? launch_append<AEGKV_DTYPE_FP16, kNeighbours>(a, head_dim, st)
                : launch_append<AEGKV_DTYPE_FP16, kHalves>(a, head_dim, st);
  AEGKV_HIP_TRY(hipGetLastError());
  return AEGKV_OK;
}

int aegkv_kv8_gather_tokens(const void* cache, int64_t cache_block_stride,
                            int64_t cache_layer_stride, int64_t n_blocks,
                            const int32_t* block_tables, int32_t max_blocks,
                            const int32_t* seq_lens, const int32_t* cu_seqlens, int32_t batch,
                            int32_t max_seq_len, void* out_key, void* out_value,
                            int64_t out_tokens, int64_t out_layer_stride, int32_t n_layers,
                            int32_t n_kv_heads, int32_t head_dim, int32_t dtype,
                            aegkv_stream_t stream) {
  if (batch < 0 || max_seq_len < 0 || n_layers <= 0 || n_kv_heads <= 0 || head_dim <= 0 ||
      max_blocks < 0 || n_blocks < 0 || out_tokens < 0)
    return AEGKV_ERR_INVALID_ARG;
  if (!head_dim_ok(head_dim) || !dtype_ok(dtype) || n_kv_heads > kKv8MaxHeads)
    return AEGKV_ERR_UNSUPPORTED;
  if (batch == 0 || max_seq_len == 0 || out_tokens == 0) return AEGKV_OK;
  if (!cache || !block_tables || !seq_lens || !cu_seqlens || !out_key || !out_value)
    return AEGKV_ERR_INVALID_ARG;
  if (!aligned16(cache) || !aligned16(out_key) || !aligned16(out_value) ||
      cache_block_stride % 16 || cache_layer_stride % 16 || out_layer_stride % 8)
    return AEGKV_ERR_MISALIGNED;
  const int64_t blocks_needed = ((int64_t)max_seq_len + kKv8Tokens - 1) / kKv8Tokens;
  if (blocks_needed > max_blocks) return AEGKV_ERR_INVALID_ARG;
  const int64_t per_tile = kGather8Threads / 64 * kGather8PerWave * (head_dim == 64 ? 2 : 1);
  const int64_t passes = (2 * (int64_t)n_kv_heads + per_tile - 1) / per_tile;
  if (n_layers > 65535 || blocks_needed * kGather8MaxBatch * passes > INT32_MAX)
    return AEGKV_ERR_UNSUPPORTED;
  DeviceState* ds = nullptr;
  const int rc = current_device_state(&ds);
  if (rc) return rc;
  Gather8Args a;
  a.cache = static_cast<const uint8_t*>(cache);
  a.blk_b = cache_block_stride;
  a.layer_b = cache_layer_stride;
  a.scales_at = kv8_scales_at(n_kv_heads, head_dim);
  a.n_blocks = n_blocks;
  a.max_blocks = max_blocks;
  a.out_k = static_cast<uint8_t*>(out_key);
  a.out_v = static_cast<uint8_t*>(out_value);
  a.out_tokens = out_tokens;
  a.out_layer_b = out_layer_stride * 2;
  a.max_seq_len = max_seq_len;
  a.n_heads = n_kv_heads;
  a.passes = (int32_t)passes;
  const int64_t max_grid = std::max<int64_t>(
      1, ((int64_t)std::max(ds->num_cu, 1) * kGather8WorkgroupsPerCu + n_layers - 1) / n_layers);
  for (int32_t b0 = 0; b0 < batch; b0 += kGather8MaxBatch) {
    const int32_t nb = std::min(kGather8MaxBatch, batch - b0);
    a.batch = nb;
    a.block_tables = block_tables + (int64_t)b0 * max_blocks;
    a.seq_lens = seq_lens + b0;
    a.cu_seqlens = cu_seqlens + b0;
    const int64_t tiles_max = blocks_needed * nb * passes;  // bound of a layer's tiles
    const dim3 grid((uint32_t)std::min(tiles_max, max_grid), (uint32_t)n_layers);
    if (dtype == AEGKV_DTYPE_BF16)
      launch_gather<AEGKV_DTYPE_BF16>(a, head_dim, grid, (hipStream_t)stream);
    else
      launch_gather<AEGKV_DTYPE_FP16>(a, head_dim, grid, (hipStream_t)stream);
    AEGKV_HIP_TRY(hipGetLastError());
  }
  return AEGKV_OK;
}

}  // extern "C"
