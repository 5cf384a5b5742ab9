// Attention of several query tokens per sequence over the paged 4-bit KV cache
// (kv4_format.h) on gfx950: a prompt's next chunk over what is cached of it, or
// drafted tokens.  Sequence b has queries [cu_seqlens[b], cu_seqlens[b + 1]),
// m of them, the last of its seq_lens[b] = n cached tokens; query i attends to
// keys j <= n - m + i (every key j < n when not causal).
//
// Rows.  The m queries of a sequence times the G query heads of one kv head
// are rows r = i * G + (head in the group) that share that head's K and V.  32
// consecutive rows are a wave's unit, W units a workgroup's tile.  A tile's
// workgroup walks the sequence's keys 64 at a time: a wave holds one 16-token
// block's codes in registers ahead of its tile, converts them to 16 bits, where
// they are exact, and stores them to LDS; every wave takes S = K.Q^T, the online
// softmax and O += V^T.P^T of its rows from there (prefill_wave.h, 32x32x16
// MFMA, fp32 sums; P rounded to 16 bits as in the prompt attention: a weight is off
// by half a step at most, as the output is by its own rounding, and P in two parts
// would take half as many products again; relative L2 error against 64 bits 0.0023 in
// bf16 and 0.00027 in fp16, 0.0017 and 0.00021 the output's rounding alone; the sum of
// the weights is of the unrounded ones).  The conversion, 190 instructions per 128 keys and
// wave, is shared by the tile's units, so few rows pay for it most.  By the rows
// of a sequence (varlen_shape):
//   up to 64      four waves, two units; two key tiles per step, one per pair of
//                 waves, joined at the end;
//   more          four waves, four units, two workgroups per CU;
//   past 256, few tiles of many keys, head_dim 128: eight waves in ping-pong, one
//                 workgroup per CU.
//
// Pieces.  When the batch has too few tiles to fill the chip, a tile's keys are
// cut into pieces of a workgroup each, which write fp32 partials (O, running
// maximum in log2 units, sum) that a second kernel merges.  The cut is the same
// for a sequence's tiles: `splits` ranges of ceil(n_kt / splits) key steps,
// splits = ceil(n_kt / C), with one C for the batch that every workgroup
// computes for itself: the batch's key steps times row tiles divided by the
// pieces wanted.
//
// Bounds and measured.  Per cached token and kv head 17 D / 16 bytes are read
// and 4 D G flops done per query, so past some 10 queries at G = 7 the products
// bound it: 2048 queries over 16001 tokens (28/4 heads, D = 128) 453 us, 972
// TFLOP/s (224 of 256 CUs hold a tile, at 92% of the rate of a large matrix
// product each); 4 x 512 over 3800 tokens each 137 us, the longest sequence's;
// two whole prompts of 2048 81 us, 747 TFLOP/s.  Few queries are bound by the latency
// of their steps, 1.7 us each of a lone workgroup (conversion, products and softmax
// of a wave follow each other): 48 x 5 over 1000 tokens each (32/4) 23.9 us a call,
// the main kernel 21.3 and the merge 4.4.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "aegkv_internal.h"
#include "kv4_cut.h"
#include "kv4_format.h"
#include "prefill_wave.h"

namespace aegkv {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kTileBlocks = kPfKTile / kKv4Tokens;
static_assert(kKeyTile == kPfKTile, "the key tiles of the cut");

struct VarlenArgs {
  const uint8_t* q;
  uint8_t* out;
  int64_t q_tok_b, o_tok_b;  // byte strides per token
  const uint8_t* cache;
  int64_t blk_b;             // byte stride per block
  int64_t n_blocks;
  const int32_t* tables;
  int32_t max_blocks;
  const int32_t* cu;         // [batch + 1]
  const int32_t* seq_lens;   // [batch]
  int32_t batch, n_kv_heads, group, max_q, max_len, causal;
  int32_t token_bound;       // min(total query tokens, INT32_MAX)
  FastDiv by_group;
  float scale_log2;          // |softmax scale| * log2(e), > 0 (1 for 0)
  int32_t scale_sign;        // of the scale: 1, -1 or 0
  int64_t target;            // pieces wanted (0: no sequence is cut)
  int32_t least;             // least key tiles of a piece
  int32_t n_pieces;          // bound of the pieces: the main grid, and the partials' slots
  float* part_o;             // [n_pieces][32 W][D]
  float2* part_ml;           // [n_pieces][32 W] (running max less kTop in log2 units, sum)
  int32_t* n_cut;            // row tiles that are cut, and one CutTile each: written
  CutTile* cut;              // by the main kernel (target > 0) for the merge
  int32_t max_cut;           // bound of them
  int32_t merge_per_tile;    // workgroups of the merge on a row tile
};

// What a sequence asks for, in row tiles of W units and steps of KS key tiles.
struct SeqWork {
  int t0, m;        // first query token, queries (at most max_q)
  int off;          // key position of query 0
  int len;          // keys
  int rows, tiles;  // rows of one kv head, row tiles
  int n_kt;         // key steps that its last row sees
};
template <int W, int KS>
__device__ __forceinline__ SeqWork seq_work(const VarlenArgs& a, int b) {
  SeqWork s;
  const int c0 = a.cu[b], c1 = a.cu[b + 1], n = max(a.seq_lens[b], 0);
  s.t0 = min(max(c0, 0), a.token_bound);
  const int m_all = min(max(c1, s.t0), a.token_bound) - s.t0;
  s.m = min(m_all, a.max_q);
  s.off = n - m_all;
  s.len = min(n, a.max_len);
  s.rows = s.m * a.group;
  s.tiles = (s.rows + kUnitRows * W - 1) / (kUnitRows * W);
  const int last = a.causal ? min(s.off + s.m, s.len) : s.len;  // keys of the last query
  s.n_kt = s.m > 0 ? (max(last, 0) + KS * kPfKTile - 1) / (KS * kPfKTile) : 0;
  return s;
}

// One piece of work: the sequence, its kv head, row tile and range of key steps;
// a cut row tile's number among those.
struct Piece {
  SeqWork s;
  int b, head, tile, split, splits, span, cut;
};

struct LocateLds {
  int64_t cost[16];
  int sum[16], cut[16];
  int found[11];
};
// The piece numbered blockIdx.x, found by all NT threads, each summing its own
// sequences.  False: there are fewer.  The first workgroup writes n_cut.
template <int W, int KS, int NT>
__device__ __forceinline__ bool locate(const VarlenArgs& a, LocateLds& x, Piece& p) {
  constexpr int NW = NT / 64;
  const int index = (int)blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int per = (a.batch + NT - 1) / NT, b0 = min(t * per, a.batch), b1 = min(b0 + per, a.batch);
  // the thread's first sequence, its only one in batches of up to NT
  const SeqWork mine = seq_work<W, KS>(a, min(b0, a.batch - 1));
  auto work = [&](int b) { return b == b0 ? mine : seq_work<W, KS>(a, b); };
  int span = INT32_MAX;
  if (a.target > 0) {  // uniform
    int64_t cost = 0;
    for (int b = b0; b < b1; ++b) {
      const SeqWork s = work(b);
      cost += (int64_t)s.tiles * s.n_kt;
    }
    // (the wave's sum in 25-bit digits, as 64 of them stay in 31 bits)
    constexpr int kDigit = (1 << 25) - 1;
    const int d0 = wave_prefix((int)cost & kDigit), d1 = wave_prefix((int)(cost >> 25) & kDigit),
              d2 = wave_prefix((int)(cost >> 50));
    if (lane == 63) x.cost[wave] = ((int64_t)d2 << 50) + ((int64_t)d1 << 25) + d0;
    __syncthreads();
    cost = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) cost += x.cost[w];
    cost *= a.n_kv_heads;
    span = span_of(cost, a.target, a.least);
  }
  int count = 0, cuts = 0;  // this thread's pieces and cut row tiles
  auto add = [&](const SeqWork& s, int& pieces, int& cut) {
    const int n = s.tiles * a.n_kv_heads, r = ranges_of(s.n_kt, span);
    pieces += n * r;
    cut += r > 1 ? n : 0;
    return r;
  };
  for (int b = b0; b < b1; ++b) add(work(b), count, cuts);
  const int incl = wave_prefix(count), cincl = wave_prefix(cuts);
  if (lane == 63) {
    x.sum[wave] = incl;
    x.cut[wave] = cincl;
  }
  if (t == 0) x.found[0] = -1;
  __syncthreads();
  int excl = incl - count, cexcl = cincl - cuts;
  for (int w = 0; w < wave; ++w) {
    excl += x.sum[w];
    cexcl += x.cut[w];
  }
  // (none if there are pieces past the grid: of overlapping sequences)
  if (a.target > 0 && index == 0 && t == NT - 1)
    *a.n_cut = excl + count <= a.n_pieces ? min(cexcl + cuts, a.max_cut) : 0;
  if (index >= excl && index < excl + count) {  // one thread
    for (int b = b0; b < b1; ++b) {
      const SeqWork s = work(b);
      int pieces = 0, cut = 0;
      const int r = add(s, pieces, cut);
      if (index < excl + pieces) {
        const int f[11] = {b,   index - excl, r,      (s.n_kt + r - 1) / r, cexcl, s.t0,
                           s.m, s.off,        s.len, s.rows,               s.tiles};
#pragma unroll
        for (int i = 0; i < 11; ++i) x.found[i] = f[i];
        break;
      }
      excl += pieces;
      cexcl += cut;
    }
  }
  __syncthreads();
  int f[11];
#pragma unroll
  for (int i = 0; i < 11; ++i) f[i] = __builtin_amdgcn_readfirstlane(x.found[i]);
  p.b = f[0];
  if (p.b < 0) return false;
  p.splits = f[2];
  p.span = f[3];
  p.s.t0 = f[5];
  p.s.m = f[6];
  p.s.off = f[7];
  p.s.len = f[8];
  p.s.rows = f[9];
  p.s.tiles = f[10];
  // row tiles from the last (the most keys) to the first, kv heads within
  const int q = f[1] / p.splits;
  p.split = f[1] - q * p.splits;
  p.cut = f[4] + q;
  p.tile = q / a.n_kv_heads;
  p.head = q - p.tile * a.n_kv_heads;
  p.tile = p.s.tiles - 1 - p.tile;
  return true;
}
// A cut row tile's entry for the merge, by one thread of its first piece.
template <int W>
__device__ __forceinline__ void put_cut(const VarlenArgs& a, const Piece& p) {
  if (p.splits == 1 || p.split || threadIdx.x || p.cut >= a.max_cut) return;
  const int row0 = p.tile * W * kUnitRows;
  a.cut[p.cut] = {p.s.t0, p.head, row0, min(row0 + W * kUnitRows, p.s.rows), (int)blockIdx.x,
                  p.splits};
}

// Nothing is scheduled across: the softmax would otherwise sink into the next
// matrix phase.
#define KV4_BARRIER()                                  \
  do {                                                 \
    __builtin_amdgcn_sched_barrier(0);                 \
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); \
    __builtin_amdgcn_s_barrier();                      \
    asm volatile("" ::: "memory");                     \
    __builtin_amdgcn_sched_barrier(0);                 \
  } while (0)

// The K or V codes of one block for one lane, as in the decode attention:
// words and scale byte(s).
template <int D>
struct CodeRegs {
  uint32_t w[D / 32], s;
};
template <int D>
__device__ __forceinline__ void load_words4(CodeRegs<D>& c, __amdgpu_buffer_rsrc_t r, int at,
                                            int lane) {
  if constexpr (D == 64) {
    const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, at + 8 * lane, 0, 0);
    c.w[0] = x.x; c.w[1] = x.y;
  } else {
    const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, at + 16 * lane, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) c.w[i] = x[i];
  }
}
template <int D>
__device__ __forceinline__ void load_k(CodeRegs<D>& c, __amdgpu_buffer_rsrc_t r, int lane) {
  const int j = lane & 15, g = lane >> 4;
  load_words4<D>(c, r, 0, lane);
  c.s = __builtin_amdgcn_raw_buffer_load_b8(
      r, kv4_code_bytes(D) + (D == 64 ? g >> 1 : g) * kKv4Tokens + j, 0, 0);
}
template <int D>
__device__ __forceinline__ void load_v(CodeRegs<D>& c, __amdgpu_buffer_rsrc_t r, int lane) {
  constexpr int REC = kv4_record_bytes(D);
  const int j = lane & 15, g = lane >> 4;
  load_words4<D>(c, r, REC, lane);
  c.s = __builtin_amdgcn_raw_buffer_load_b32(
      r, REC + kv4_code_bytes(D) + (j * (D / 16) / kKv4Group) * kKv4Tokens + 4 * g, 0, 0);
}

// Rows of 2 D bytes in LDS, their 16-byte chunks permuted by the row so that the
// operand reads hit distinct banks (as the prompt attention stores them).
template <int D>
__device__ __forceinline__ int k_chunk(int row, int c) {
  return D == 128 ? c ^ (row & 15) : c ^ ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_chunk(int row, int c) {
  return D == 128 ? c ^ ((row & 3) << 2) : c ^ (((row >> 1) & 1) << 2);
}

template <int DT, int D>
__device__ __forceinline__ void put_k(uint8_t* lds, const CodeRegs<D>& c, int u, int lane) {
  using C = Kv4Elem<DT>;
  constexpr int NW = D / 32;
  const int j = lane & 15, g = lane >> 4, row = kKv4Tokens * u + j;
  const float s = kv4_scale(c.s);
#pragma unroll
  for (int i = 0; i < NW; ++i)
    *reinterpret_cast<u32x4*>(lds + row * 2 * D + k_chunk<D>(row, NW * g + i) * 16) =
        u32x4{C::template dq<0>(c.w[i], s), C::template dq<1>(c.w[i], s),
              C::template dq<2>(c.w[i], s), C::template dq<3>(c.w[i], s)};
}
// V's tokens at or past `left` (of the block's 16) and its NaN groups are stored
// as zeros, as a weight of zero does not undo a NaN.  True when there was such a
// group (uniform): its rows are found at the end (RowUnit::find_nan).
template <int DT, int D>
__device__ __forceinline__ bool put_v(uint8_t* lds, CodeRegs<D>& c, int u, int left, int lane) {
  using C = Kv4Elem<DT>;
  const int j = lane & 15, g = lane >> 4;
  uint32_t e[4];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e[i] = (c.s >> (8 * i)) & 0xffu;
    const bool past = 4 * g + i >= left, nan = e[i] == kKv4ScaleNan;
    bad |= nan && !past;
    e[i] = past || nan ? 0u : e[i];  // scale byte 0: finite whatever the codes
    if constexpr (D == 64) c.w[i >> 1] = past ? c.w[i >> 1] & (i & 1 ? 0x0000ffffu : 0xffff0000u) : c.w[i >> 1];
    else c.w[i] = past ? 0u : c.w[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = kKv4Tokens * u + 4 * g + i;
    const float s = kv4_scale(e[i]);
    if constexpr (D == 64) {
      const uint32_t w = c.w[i >> 1];
      const u32x2 x = i & 1 ? u32x2{C::template dq<2>(w, s), C::template dq<3>(w, s)}
                            : u32x2{C::template dq<0>(w, s), C::template dq<1>(w, s)};
      *reinterpret_cast<u32x2*>(lds + row * 2 * D + v_chunk<D>(row, j >> 1) * 16 + 8 * (j & 1)) = x;
    } else {
      const uint32_t w = c.w[i];
      *reinterpret_cast<u32x4*>(lds + row * 2 * D + v_chunk<D>(row, j) * 16) =
          u32x4{C::template dq<0>(w, s), C::template dq<1>(w, s), C::template dq<2>(w, s),
                C::template dq<3>(w, s)};
    }
  }
  return __builtin_amdgcn_ballot_w64(bad) != 0;
}

// The block ids of a piece's key tiles, 16 tiles at a time, one id per lane, with
// the next 16 tiles' loaded ahead.  Tiles are asked for in order.
struct TileIds {
  const int32_t* table;  // the sequence's, n_blk > 0 entries
  int n_blk, n_blocks;   // (pools are below 2^31 blocks, as ids are int32)
  int base, cur, next;   // first tile at hand
  __device__ __forceinline__ int from(int tile) const {
    return table[min(tile * kTileBlocks + (int)(threadIdx.x & 63), n_blk - 1)];
  }
  __device__ __forceinline__ void start(int tile) {
    base = tile;
    cur = from(tile);
    next = from(tile + 16);
  }
  __device__ __forceinline__ void reach(int tile) {
    if (tile - base == 16) {
      cur = next;
      base += 16;
      next = from(base + 16);
    }
  }
  // the id of block u of the tile, -1 when it is none of the sequence's or unreadable
  __device__ __forceinline__ int id(int tile, int u) const {
    const int x = __builtin_amdgcn_readlane(cur, ((tile - base) * kTileBlocks + u) & 63);
    return tile * kTileBlocks + u < n_blk && x >= 0 && x < n_blocks ? x : -1;
  }
  // the tile's blocks that are the sequence's and unreadable
  __device__ __forceinline__ uint32_t unreadable(int tile) const {
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < kTileBlocks; ++u)
      if (tile * kTileBlocks + u < n_blk && id(tile, u) < 0) m |= 1u << u;
    return m;
  }
};

// A wave's unit of 32 rows.
template <int DT, int D>
struct RowUnit : WaveSoftmax<DT, D, true> {
  using Base = WaveSoftmax<DT, D, true>;
  using Base::DB;
  using Base::KS;
  using Base::lsum;
  using Base::m;
  using Base::o;
  using Base::qv;
  int r0, rows;     // first row; the sequence's rows
  int limit;        // last key of this lane's row (-1: none)
  int lim_lo;       // of the unit's first row
  uint32_t spoiled;    // bit: dims 32 db .. of this lane's row are NaN

  __device__ __forceinline__ void init(const VarlenArgs& a, const SeqWork& s, int head, int unit) {
    const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
    r0 = unit * kUnitRows;
    rows = s.rows;
    const int r = min(r0 + col, rows - 1);
    const int i = a.by_group.div(r), h = head * a.group + r - i * a.group;
    auto last_of = [&](int row) {
      const int q = a.by_group.div(min(row, rows - 1));
      return max(-1, a.causal ? min(s.off + q, s.len - 1) : s.len - 1);
    };
    limit = last_of(r);
    lim_lo = last_of(r0);
    const uint8_t* qp = a.q + (int64_t)(s.t0 + i) * a.q_tok_b + ((int64_t)h * D + 8 * hh) * 2;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qv[ks] = *reinterpret_cast<const u32x4*>(qp + 32 * ks);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] = 0.f;
    m = -INFINITY;
    lsum = 0.f;
    spoiled = 0;
  }
  // the softmax's scale is positive: another one's sign goes into the queries
  // (0: no query, every score 0)
  __device__ __forceinline__ void sign_queries(int sign) {
    if (sign > 0) return;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) qv[ks][e] = sign < 0 ? qv[ks][e] ^ 0x80008000u : 0u;
  }

  // LDS reads stay two MFMAs ahead of their use (pv: four), as the long prompts'
  // kernel orders them
  __device__ __forceinline__ void qk(const uint8_t* lds, f32x16 (&s)[2]) const {
    const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
    const uint8_t* kp = lds + col * 2 * D;
    const int kx = k_chunk<D>(col, hh) * 16;
#pragma unroll
    for (int sb = 0; sb < 2; ++sb)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[sb][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int sb = 0; sb < 2; ++sb)
        s[sb] = PfOps<DT>::mfma(
            *reinterpret_cast<const u32x4*>(kp + (kx ^ (32 * ks)) + 32 * sb * 2 * D), qv[ks], s[sb]);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
#pragma unroll
    for (int i = 0; i < 2 * KS - 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // the next read
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
  }
  // -inf for keys past a row's last one and for unreadable blocks (bit u)
  __device__ __forceinline__ void mask(f32x16 (&s)[2], int k0, uint32_t unreadable) const {
    if (k0 + kPfKTile - 1 > lim_lo || unreadable) {
      asm volatile("");  // a branch, not selects on every tile
      const int hh = (threadIdx.x & 63) >> 5, last = limit - k0 - 4 * hh;
#pragma unroll
      for (int u = 0; u < kTileBlocks; ++u) {
        const int l = unreadable >> u & 1 ? -1 : last;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = 8 * (u & 1) + e;
          s[u >> 1][i] = l >= 16 * u + 8 * (e >> 2) + (e & 3) ? s[u >> 1][i] : -INFINITY;
        }
      }
    }
  }
  __device__ __forceinline__ void pv(const uint8_t* lds, const u32x4 (&pb)[4]) {
    constexpr int RB = 2 * D;
    const int lane = threadIdx.x & 63, G = lane >> 4, x = lane & 15;
    const int key = 4 * (G >> 1) + (x >> 2);
    const int vx = v_chunk<D>(key, 0) * 16;
    const uint8_t* vp = lds + key * RB + (2 * (G & 1) + ((x & 3) >> 1)) * 16 + 8 * (x & 1);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const uint8_t* y = vp + (vx ^ (64 * db)) + 16 * kk * RB;
        const u32x2 lo = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)y));
        const u32x2 hi = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(y + 8 * RB)));
        o[db] = PfOps<DT>::mfma(u32x4{lo[0], lo[1], hi[0], hi[1]}, pb[kk], o[db]);
      }
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < 4 * DB - 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
  }
  // Key tiles [kt0, kt1) hold V groups of NaN (rare): the rows that see one's
  // token get NaN in its dims when they are stored.  Visible keys are a prefix, so
  // each group's first such key decides.
  __device__ void find_nan(const VarlenArgs& a, const int32_t* table, int64_t head_off, int len,
                           int kt0, int kt1) {
    const int lane = threadIdx.x & 63;
    const int n_blk = min(kt1 * kTileBlocks, (len + kKv4Tokens - 1) / kKv4Tokens);
    uint32_t found = 0;  // groups whose first key is known
    for (int blk = kt0 * kTileBlocks; blk < n_blk; ++blk) {
      const int id = __builtin_amdgcn_readfirstlane(table[blk]);
      if (id < 0 || id >= a.n_blocks) continue;
      uint32_t e = 0;  // lane: group lane / 16, token lane % 16
      if (lane < D / 2 && blk * kKv4Tokens + (lane & 15) < len)
        e = a.cache[(int64_t)id * a.blk_b + head_off + kv4_record_bytes(D) + kv4_code_bytes(D) + lane];
      const uint64_t at = __builtin_amdgcn_ballot_w64(e == kKv4ScaleNan);
      for (int db = 0; db < DB; ++db) {
        const uint32_t t = (uint32_t)(at >> (16 * db)) & 0xffffu;
        if (!t || (found >> db & 1)) continue;
        found |= 1u << db;
        if (blk * kKv4Tokens + __builtin_ctz(t) <= limit) spoiled |= 1u << db;
      }
    }
  }
  __device__ __forceinline__ float finite_or_nan(int db) const {
    return spoiled >> db & 1 ? __builtin_nanf("") : 1.f;
  }
  // The sums to and from LDS, one float per lane and register (no key: -inf, 0, 0).
  __device__ __forceinline__ void put_sums(uint8_t* x) const {
    float* f = reinterpret_cast<float*>(x) + (threadIdx.x & 63);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) f[64 * (16 * db + e)] = o[db][e];
    f[64 * 16 * DB] = m;
    f[64 * (16 * DB + 1)] = lsum;
  }
  __device__ __forceinline__ void add_sums(const uint8_t* x) {
    const float* f = reinterpret_cast<const float*>(x) + (threadIdx.x & 63);
    const float m2 = f[64 * 16 * DB], mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.f : mn;
    const float w1 = __builtin_amdgcn_exp2f(m - ref), w2 = __builtin_amdgcn_exp2f(m2 - ref);
    lsum = lsum * w1 + f[64 * (16 * DB + 1)] * w2;
    m = mn;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] = o[db][e] * w1 + f[64 * (16 * db + e)] * w2;
  }
  __device__ __forceinline__ float total() const { return lsum + __shfl_xor(lsum, 32); }

  // normalise and store the rows (x: 32 rows of LDS of the wave's own), as the
  // prompt attention does; rows without a key get zeros
  __device__ __forceinline__ void store(const VarlenArgs& a, const SeqWork& s, uint8_t* x,
                                        int head) const {
    constexpr int RB = D * 2, CPR = D / 8, RPI = 64 / CPR;
    const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
    const float lt = total();
    uint8_t* xw = x + col * RB + 8 * hh;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x16& v = o[db];
        const float inv = (lt == 0.f ? 0.f : 1.f / lt) * finite_or_nan(db);
        *reinterpret_cast<u32x2*>(xw + ((4 * db + g) ^ (col % CPR)) * 16) =
            u32x2{PfOps<DT>::pack(v[4 * g] * inv, v[4 * g + 1] * inv),
                  PfOps<DT>::pack(v[4 * g + 2] * inv, v[4 * g + 3] * inv)};
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own writes
    const int row = lane / CPR, pos = lane % CPR;
#pragma unroll
    for (int n = 0; n < 32 / RPI; ++n) {
      const int r = RPI * n + row;
      const u32x4 v = *reinterpret_cast<const u32x4*>(x + 1024 * n + 16 * lane);
      if (r0 + r < rows) {
        const int i = a.by_group.div(r0 + r), h = head * a.group + r0 + r - i * a.group;
        *reinterpret_cast<u32x4*>(a.out + (int64_t)(s.t0 + i) * a.o_tok_b + (int64_t)h * RB +
                                  (pos ^ (r % CPR)) * 16) = v;
      }
    }
  }
  __device__ __forceinline__ void store_partial(const VarlenArgs& a, int64_t slot_row) const {
    const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
    const float lt = total();
    if (r0 + col >= rows) return;
    float* po = a.part_o + (slot_row + col) * D + 4 * hh;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(po + 32 * db + 8 * g) =
            f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]} *
            finite_or_nan(db);
    if (hh == 0) a.part_ml[slot_row + col] = make_float2(m, lt);
  }
};

// Four waves.  KS = 1: four units, and wave w converts block w of each key tile.
// KS = 2, for row tiles of up to two units: waves 2 and 3 take the units of waves 0
// and 1 over the second of two key tiles per step, and the pairs are joined at the
// end.  (Two waves converting only: 48 x 5 drafted tokens over 1000 each of 32/4
// heads 49.7 us, so 31.1.)
template <int DT, int D, int KS>
__global__ __launch_bounds__(64 * kShortWaves4, 2) void kv4_varlen_kernel(VarlenArgs a) {
  constexpr int NW = kShortWaves4, W = NW / KS;  // waves, units of a row tile
  constexpr int T_BYTES = kPfKTile * D * 2;
  static_assert(NW == kTileBlocks, "a block of each key tile per wave");
  static_assert(W * kUnitRows * D * 2 <= 2 * T_BYTES, "the outputs fit the tiles");
  static_assert(KS == 1 || W * 64 * (D / 2 + 3) * 4 <= KS * 2 * T_BYTES, "the joined halves fit");
  __shared__ __align__(16) uint8_t lds[KS * 2 * T_BYTES];  // K and V of each key tile
  __shared__ uint32_t s_nan[NW];
  __shared__ LocateLds s_loc;
  Piece p;
  if (!locate<W, KS, 64 * NW>(a, s_loc, p)) return;  // uniform
  put_cut<W>(a, p);
  const SeqWork& s = p.s;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = w / W;  // the key tile of a step that the wave attends to
  const int n_blk = (s.len + kKv4Tokens - 1) / kKv4Tokens;
  // the key steps of this piece that the tile's last row sees
  const int last_q = a.by_group.div(min(s.rows, (p.tile + 1) * W * kUnitRows) - 1);
  const int keys = a.causal ? min(s.off + last_q + 1, s.len) : s.len;
  const int kt0 = p.split * p.span;
  const int kt1 =
      min(kt0 + p.span, (max(keys, 0) + KS * kPfKTile - 1) / (KS * kPfKTile));

  RowUnit<DT, D> unit;
  unit.init(a, s, p.head, p.tile * W + w % W);
  unit.sign_queries(a.scale_sign);

  const int32_t* table = a.tables + (int64_t)p.b * a.max_blocks;
  const int64_t head_off = (int64_t)p.head * 17 * D;
  bool nan = false;
  if (kt0 < kt1) {  // uniform
    TileIds ids{table, n_blk, (int)min(a.n_blocks, (int64_t)INT32_MAX)};
    ids.start(kt0 * KS);
    // this wave's codes of the next step (tiles past the piece: nothing)
    struct {
      CodeRegs<D> k, v;
    } next[KS];
    uint32_t unreadable_next = 0;  // of the wave's key tile
    auto load = [&](int kt) {
      ids.reach(kt * KS);
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const int id = kt < kt1 ? ids.id(kt * KS + t, w) : -1;
        const auto r = byte_range(a.cache + (int64_t)max(id, 0) * a.blk_b + head_off,
                                  id >= 0 ? 17 * D : 0u);
        load_k<D>(next[t].k, r, lane);
        load_v<D>(next[t].v, r, lane);
      }
      unreadable_next = kt < kt1 ? ids.unreadable(kt * KS + part) : 0u;
    };
    uint8_t* mine = lds + part * 2 * T_BYTES;
    // No step is skipped for rows that do not see it: branches around the products
    // had their accumulators copied.  A wave without rows only converts.
    auto step = [&](auto with_rows, int kt) {
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        uint8_t* tile = lds + t * 2 * T_BYTES;
        put_k<DT, D>(tile, next[t].k, w, lane);
        nan |= put_v<DT, D>(tile + T_BYTES, next[t].v, w,
                            s.len - ((kt * KS + t) * kTileBlocks + w) * kKv4Tokens, lane);
      }
      const uint32_t unreadable = unreadable_next;
      load(kt + 1);
      KV4_BARRIER();
      if constexpr (decltype(with_rows)::value) {
        f32x16 sc[2];
        u32x4 pb[4];
        unit.qk(mine, sc);
        unit.mask(sc, (kt * KS + part) * kPfKTile, unreadable);
        unit.softmax(sc, pb, a.scale_log2, kt == kt0);
        __builtin_amdgcn_sched_barrier(0);  // V's reads stay behind the softmax: registers
        unit.pv(mine + T_BYTES, pb);
      }
      KV4_BARRIER();  // every wave's reads of the tiles
    };
    load(kt0);
    if (unit.r0 < s.rows) {
      for (int kt = kt0; kt < kt1; ++kt) step(std::true_type{}, kt);
    } else {
      for (int kt = kt0; kt < kt1; ++kt) step(std::false_type{}, kt);
    }
  }
  if constexpr (KS > 1) {  // the second key tiles' sums to the waves of the first
    uint8_t* x = lds + w % W * (64 * (D / 2 + 3) * 4);
    if (part > 0) unit.put_sums(x);
    if (lane == 0) s_nan[w] = nan;
    KV4_BARRIER();
    if (part == 0) unit.add_sums(x);
  } else {
    if (lane == 0) s_nan[w] = nan;
  }
  KV4_BARRIER();
  nan = false;
#pragma unroll
  for (int i = 0; i < NW; ++i) nan |= s_nan[i] != 0;
  if (part > 0) return;
  if (__builtin_amdgcn_readfirstlane(nan))
    unit.find_nan(a, table, head_off, s.len, kt0 * KS, kt1 * KS);
  if (p.splits > 1) unit.store_partial(a, ((int64_t)blockIdx.x * W + w) * kUnitRows);
  else unit.store(a, s, lds + w * (kUnitRows * D * 2), p.head);
}

// Long rows: eight units in ping-pong, as the long prompts' kernel runs them.
// Waves w and w + 4 share a SIMD and run opposite phases between workgroup
// barriers: in a matrix phase a wave takes S_j and O += V_{j-1}^T.P_{j-1}, in the
// next its softmax, waves 4-7 one phase later than waves 0-3.  The conversions
// go with the softmax: in slot 2j + 1 waves 0-3 convert a block of K_{j+1} each,
// in slot 2j waves 4-7 one of V_j.  K_{j+1}'s stage was last read (as K_{j-1})
// in slot 2j - 1 and is read from slot 2j + 2 on, V_j's as well.
template <int DT, int D>
__global__ __launch_bounds__(64 * kLongWaves4) void kv4_varlen_long_kernel(VarlenArgs a) {
  constexpr int W = kLongWaves4;
  constexpr int T_BYTES = kPfKTile * D * 2;
  static_assert(W / 2 * kUnitRows * D * 2 <= 2 * T_BYTES, "a half's outputs fit its stages");
  __shared__ __align__(16) uint8_t lds[4 * T_BYTES];  // two K stages, two V stages
  __shared__ uint32_t s_nan[W / 2];
  __shared__ LocateLds s_loc;
  Piece p;
  if (!locate<W, 1, 64 * W>(a, s_loc, p)) return;  // uniform
  const SeqWork& s = p.s;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = w >> 2, u = w & 3;  // and the block of each tile that the wave converts
  const int n_blk = (s.len + kKv4Tokens - 1) / kKv4Tokens;
  const int last_q = a.by_group.div(min(s.rows, (p.tile + 1) * W * kUnitRows) - 1);
  const int keys = a.causal ? min(s.off + last_q + 1, s.len) : s.len;
  const int kt0 = p.split * p.span;
  const int n_kt = max(min(p.span, (max(keys, 0) + kPfKTile - 1) / kPfKTile - kt0), 0);

  RowUnit<DT, D> unit;
  unit.init(a, s, p.head, p.tile * W + w);
  unit.sign_queries(a.scale_sign);

  const int32_t* table = a.tables + (int64_t)p.b * a.max_blocks;
  const int64_t head_off = (int64_t)p.head * 17 * D;
  TileIds ids{table, n_blk, (int)min(a.n_blocks, (int64_t)INT32_MAX)};
  // this wave's codes of two key tiles (K of block u, or V), loaded two tiles
  // ahead of their conversion (tiles past the piece: nothing), and the unreadable
  // blocks of three tiles: of the one computed and the two loaded
  CodeRegs<D> c[2];
  uint32_t bad[3] = {};
  auto load = [&](CodeRegs<D>& r, int j) {
    ids.reach(kt0 + j);
    const int id = j < n_kt ? ids.id(kt0 + j, u) : -1;
    bad[2] = j < n_kt ? ids.unreadable(kt0 + j) : ~0u;
    const auto range = byte_range(a.cache + (int64_t)max(id, 0) * a.blk_b + head_off,
                                  id >= 0 ? 17 * D : 0u);
    if (half == 0) load_k<D>(r, range, lane);
    else load_v<D>(r, range, lane);
  };
  bool nan = false;
  auto put = [&](CodeRegs<D>& r, int j) {  // and the loads of the tile two further on
    if (half == 0)
      put_k<DT, D>(lds + (j & 1) * T_BYTES, r, u, lane);
    else
      nan |= put_v<DT, D>(lds + (2 + (j & 1)) * T_BYTES, r, u,
                          s.len - ((kt0 + j) * kTileBlocks + u) * kKv4Tokens, lane);
    bad[0] = bad[1];
    bad[1] = bad[2];
    load(r, j + 2);
  };
  auto qk = [&](int j, f32x16 (&sc)[2]) { unit.qk(lds + (j & 1) * T_BYTES, sc); };
  auto softmax = [&](int j, f32x16 (&sc)[2], u32x4 (&pb)[4], uint32_t bad) {
    unit.mask(sc, (kt0 + j) * kPfKTile, bad);
    unit.softmax(sc, pb, a.scale_log2, j == 0);
  };
  auto pv = [&](int j, const u32x4 (&pb)[4]) {
    unit.pv(lds + (2 + (j & 1)) * T_BYTES, pb);
  };

  u32x4 pb[4];
  // Tile j: the matrix phase, then the softmax with the conversion of tile j + 1.
  // Tiles come in pairs behind the first, as the codes ahead have two sets of
  // registers; a tile past the piece is masked like an unreadable one, and none is
  // skipped for rows that do not see it (branches around the products had their
  // accumulators copied).
  auto tile = [&](auto first, int j, CodeRegs<D>& next) {
    f32x16 sc[2];
    qk(j, sc);
    if constexpr (!decltype(first)::value) pv(j - 1, pb);
    KV4_BARRIER();
    const uint32_t unreadable = bad[0];
    put(next, j + 1);
    softmax(j, sc, pb, unreadable);
    KV4_BARRIER();
  };
  if (n_kt > 0) {  // uniform: every wave passes 2 (n_kt rounded up to odd) + 3 barriers
    ids.start(kt0);
    load(c[0], 0);
    bad[1] = bad[2];
    load(c[1], 1);
    if (half == 0) put(c[0], 0);  // K_0
    KV4_BARRIER();
    if (half == 1) {
      put(c[0], 0);  // slot 0: V_0
      KV4_BARRIER();
    }
    tile(std::true_type{}, 0, c[1]);
    int j = 1;
    for (; j < n_kt; j += 2) {
      tile(std::false_type{}, j, c[0]);
      tile(std::false_type{}, j + 1, c[1]);
    }
    pv(j - 1, pb);  // slot 2 j, or 2 j + 1
    KV4_BARRIER();
    if (half == 0) KV4_BARRIER();
  }
  if (half == 1 && lane == 0) s_nan[u] = nan;
  KV4_BARRIER();  // and the stages: every wave is past its last read of them
  nan = false;
#pragma unroll
  for (int i = 0; i < W / 2; ++i) nan |= s_nan[i] != 0;
  if (__builtin_amdgcn_readfirstlane(nan))
    unit.find_nan(a, table, head_off, s.len, kt0, kt0 + n_kt);
  put_cut<W>(a, p);
  if (p.splits > 1) unit.store_partial(a, ((int64_t)blockIdx.x * W + w) * kUnitRows);
  else unit.store(a, s, lds + w * (kUnitRows * D * 2), p.head);
}

// Merges the pieces of R rows of a cut sequence's kv head:
//   out = sum_s w_s o_s / sum_s w_s l_s,  w_s = 2^(m_s - max m).
// Eight threads take a row's columns, and 32 / R slices of them the pieces in
// turn, which meet in LDS: with few rows each slice has few pieces and the loads
// of all are one round trip.  (One slice: a query over 60000 tokens in 235 pieces
// 62 us; 32 slices cost 10 us more than 8, by the 32 steps in which they meet.)
constexpr int kMerge4Threads = 256;
template <int DT, int D, int W, int R>
__global__ __launch_bounds__(kMerge4Threads) void kv4_varlen_merge_kernel(VarlenArgs a) {
  constexpr int SL = 32 / R, NV = D / 32;
  __shared__ f32x4 s_o[SL > 1 ? SL : 1][SL > 1 ? R : 1][SL > 1 ? D / 4 : 1];
  __shared__ float2 s_ml[SL][R];
  const int index = (int)blockIdx.x / a.merge_per_tile;
  const CutTile c = a.cut[index];
  if (index >= *a.n_cut) return;  // uniform; before c is looked at
  const int part = threadIdx.x & 7, row = ((int)threadIdx.x >> 3) % R, sl = ((int)threadIdx.x >> 3) / R;
  const int r = c.row0 + ((int)blockIdx.x - index * a.merge_per_tile) * R + row;
  const int n = r < c.row1 ? c.pieces : 0;
  constexpr int64_t kStep = (int64_t)W * kUnitRows;  // slot rows from piece to piece
  const int64_t row0 = (int64_t)c.piece0 * kStep + (r - c.row0);
  float mx = -INFINITY, lt = 0.f;
  f32x4 acc[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto add = [&](float m2, float l2, const f32x4 (&v)[NV]) {
    const float mn = fmaxf(mx, m2), ref = mn == -INFINITY ? 0.f : mn;
    const float w1 = __builtin_amdgcn_exp2f(mx - ref), w2 = __builtin_amdgcn_exp2f(m2 - ref);
    lt = lt * w1 + l2 * w2;
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = acc[i] * w1 + v[i] * w2;
    mx = mn;
  };
#pragma unroll 4
  for (int k = sl; k < n; k += SL) {
    const float2 ml = a.part_ml[row0 + k * kStep];
    const float* po = a.part_o + (row0 + k * kStep) * D + 4 * part;
    f32x4 v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = *reinterpret_cast<const f32x4*>(po + 32 * i);
    add(ml.x, ml.y, v);
  }
  if constexpr (SL > 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) s_o[sl][row][8 * i + part] = acc[i];
    if (part == 0) s_ml[sl][row] = make_float2(mx, lt);
    __syncthreads();
    if (sl > 0) return;
#pragma unroll
    for (int k = 1; k < SL; ++k) {
      f32x4 v[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = s_o[k][row][8 * i + part];
      add(s_ml[k][row].x, s_ml[k][row].y, v);
    }
  }
  if (r >= c.row1) return;
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  const int i = a.by_group.div(r), h = c.head * a.group + r - i * a.group;
  uint8_t* op = a.out + (int64_t)(c.t0 + i) * a.o_tok_b + ((int64_t)h * D + 4 * part) * 2;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    *reinterpret_cast<u32x2*>(op + 64 * k) =
        u32x2{PfOps<DT>::pack(acc[k][0] * inv, acc[k][1] * inv),
              PfOps<DT>::pack(acc[k][2] * inv, acc[k][3] * inv)};
}

int varlen_check(int32_t batch, int64_t total_q, int32_t max_q, int32_t max_len, int32_t n_q_heads,
                 int32_t n_kv_heads, int32_t head_dim, int32_t dtype) {
  if (batch < 0 || total_q < 0 || max_q < 0 || max_len < 0 || n_q_heads <= 0 || n_kv_heads <= 0 ||
      n_q_heads % n_kv_heads)
    return AEGKV_ERR_INVALID_ARG;
  if ((head_dim != 64 && head_dim != 128) ||
      (dtype != AEGKV_DTYPE_BF16 && dtype != AEGKV_DTYPE_FP16) || n_q_heads > 65535)
    return AEGKV_ERR_UNSUPPORTED;
  // in 32 bits: the rows of a sequence, a tile further; its keys, the end of a step of
  // two tiles and two tiles of loads ahead further
  if ((int64_t)max_q * (n_q_heads / n_kv_heads) > INT32_MAX / 2 ||
      max_len > INT32_MAX - 4 * kPfKTile)
    return AEGKV_ERR_UNSUPPORTED;
  return AEGKV_OK;
}

int shape_of(int32_t batch, int64_t total_q, int32_t max_q, int32_t max_len, int32_t n_q_heads,
             int32_t n_kv_heads, int32_t head_dim, VarlenShape* s) {
  DeviceState* ds = nullptr;
  const int rc = current_device_state(&ds);
  if (rc) return rc;
  return varlen_shape(std::max(1, ds->num_cu), batch, total_q, max_q, max_len, n_q_heads,
                      n_kv_heads, head_dim, s)
             ? AEGKV_OK
             : AEGKV_ERR_UNSUPPORTED;
}

template <int DT, int D, int W>
int launch_merge(const VarlenArgs& a, const VarlenShape& s, hipStream_t st) {
  const dim3 g((uint32_t)(s.cut * s.merge_per_tile)), t(kMerge4Threads);
  if (s.merge_rows == 4) {
    hipLaunchKernelGGL((kv4_varlen_merge_kernel<DT, D, W, 4>), g, t, 0, st, a);
  } else if (s.merge_rows == 16) {
    hipLaunchKernelGGL((kv4_varlen_merge_kernel<DT, D, W, 16>), g, t, 0, st, a);
  } else if constexpr (W < kLongWaves4) {
    hipLaunchKernelGGL((kv4_varlen_merge_kernel<DT, D, W, 32>), g, t, 0, st, a);
  } else {
    return AEGKV_ERR_UNSUPPORTED;  // not of eight waves' few tiles (varlen_shape)
  }
  AEGKV_HIP_TRY(hipGetLastError());
  return AEGKV_OK;
}
template <int DT, int D>
int launch_varlen(const VarlenArgs& a, const VarlenShape& s, hipStream_t st) {
  const dim3 g((uint32_t)s.pieces), four(64 * kShortWaves4), eight(64 * kLongWaves4);
  if (s.long_rows) hipLaunchKernelGGL((kv4_varlen_long_kernel<DT, 128>), g, eight, 0, st, a);
  else if (s.key_tiles == 2) hipLaunchKernelGGL((kv4_varlen_kernel<DT, D, 2>), g, four, 0, st, a);
  else hipLaunchKernelGGL((kv4_varlen_kernel<DT, D, 1>), g, four, 0, st, a);
  AEGKV_HIP_TRY(hipGetLastError());
  if (s.target > 0) {
    if (s.long_rows) return launch_merge<DT, 128, kLongWaves4>(a, s, st);
    if (s.key_tiles == 2) return launch_merge<DT, D, kShortWaves4 / 2>(a, s, st);
    return launch_merge<DT, D, kShortWaves4>(a, s, st);
  }
  return AEGKV_OK;
}

}  // namespace
}  // namespace aegkv

using namespace aegkv;

extern "C" {

int64_t aegkv_kv4_varlen_attention_workspace_size(int32_t batch, int64_t total_q,
                                                  int32_t max_seqlen_q, int32_t max_seq_len,
                                                  int32_t n_q_heads, int32_t n_kv_heads,
                                                  int32_t head_dim, int32_t dtype) {
  int rc = varlen_check(batch, total_q, max_seqlen_q, max_seq_len, n_q_heads, n_kv_heads, head_dim,
                        dtype);
  if (rc) return rc;
  if (batch == 0 || total_q == 0 || max_seqlen_q == 0) return 0;
  VarlenShape s;
  rc = shape_of(batch, total_q, max_seqlen_q, max_seq_len, n_q_heads, n_kv_heads, head_dim, &s);
  if (rc) return rc > 0 ? AEGKV_ERR_RUNTIME : rc;
  return s.workspace();
}

int aegkv_kv4_varlen_attention(void* out, int64_t out_token_stride, const void* q,
                               int64_t q_token_stride, const void* cache,
                               int64_t cache_block_stride, int64_t n_blocks,
                               const int32_t* block_tables, int32_t max_blocks,
                               const int32_t* cu_seqlens_q, const int32_t* seq_lens, int32_t batch,
                               int64_t total_q, int32_t max_seqlen_q, int32_t max_seq_len,
                               int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float scale,
                               int32_t causal, int32_t dtype, void* workspace,
                               uint64_t workspace_bytes, aegkv_stream_t stream) {
  int rc = varlen_check(batch, total_q, max_seqlen_q, max_seq_len, n_q_heads, n_kv_heads, head_dim,
                        dtype);
  if (rc) return rc;
  if (max_blocks < 0 || n_blocks < 0 || !std::isfinite(scale * 1.4426950408889634f))
    return AEGKV_ERR_INVALID_ARG;
  if (batch == 0 || total_q == 0 || max_seqlen_q == 0) return AEGKV_OK;
  if (!out || !q || !cache || !block_tables || !cu_seqlens_q || !seq_lens || n_blocks == 0)
    return AEGKV_ERR_INVALID_ARG;
  if (q_token_stride < (int64_t)n_q_heads * head_dim ||
      out_token_stride < (int64_t)n_q_heads * head_dim)
    return AEGKV_ERR_INVALID_ARG;
  if (!aligned16(out) || !aligned16(q) || !aligned16(cache) || q_token_stride % 8 ||
      out_token_stride % 8 || cache_block_stride % 16)
    return AEGKV_ERR_MISALIGNED;
  if (((int64_t)max_seq_len + kKv4Tokens - 1) / kKv4Tokens > max_blocks) return AEGKV_ERR_INVALID_ARG;
  VarlenShape s;
  rc = shape_of(batch, total_q, max_seqlen_q, max_seq_len, n_q_heads, n_kv_heads, head_dim, &s);
  if (rc) return rc;
  if (s.target > 0 && (!workspace || workspace_bytes < (uint64_t)s.workspace()))
    return AEGKV_ERR_WORKSPACE;
  if (s.target > 0 && !aligned16(workspace)) return AEGKV_ERR_MISALIGNED;
  VarlenArgs a;
  a.q = static_cast<const uint8_t*>(q);
  a.out = static_cast<uint8_t*>(out);
  a.q_tok_b = q_token_stride * 2;
  a.o_tok_b = out_token_stride * 2;
  a.cache = static_cast<const uint8_t*>(cache);
  a.blk_b = cache_block_stride;
  a.n_blocks = n_blocks;
  a.tables = block_tables;
  a.max_blocks = max_blocks;
  a.cu = cu_seqlens_q;
  a.seq_lens = seq_lens;
  a.batch = batch;
  a.n_kv_heads = n_kv_heads;
  a.group = n_q_heads / n_kv_heads;
  a.max_q = max_seqlen_q;
  a.max_len = max_seq_len;
  a.causal = causal ? 1 : 0;
  a.token_bound = (int32_t)std::min<int64_t>(total_q, INT32_MAX);
  a.by_group = fast_div(a.group);
  a.scale_sign = scale > 0 ? 1 : scale < 0 ? -1 : 0;
  a.scale_log2 = scale == 0 ? 1.f : std::fabs(scale) * 1.4426950408889634f;
  a.target = s.target;
  a.least = s.least;
  a.n_pieces = (int32_t)s.pieces;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + s.o_bytes);
  a.n_cut = reinterpret_cast<int32_t*>(ws + s.o_bytes + s.ml_bytes);
  a.cut = reinterpret_cast<CutTile*>(ws + s.o_bytes + s.ml_bytes + 256);
  a.max_cut = (int32_t)s.cut;
  a.merge_per_tile = (int32_t)s.merge_per_tile;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == AEGKV_DTYPE_BF16)
    return head_dim == 64 ? launch_varlen<AEGKV_DTYPE_BF16, 64>(a, s, st)
                          : launch_varlen<AEGKV_DTYPE_BF16, 128>(a, s, st);
  return head_dim == 64 ? launch_varlen<AEGKV_DTYPE_FP16, 64>(a, s, st)
                        : launch_varlen<AEGKV_DTYPE_FP16, 128>(a, s, st);
}

}  // extern "C"
