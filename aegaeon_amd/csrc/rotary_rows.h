// Rows of heads turned by their token's position: what the appends that rotate
// share.  Of a row's first `rot` dims, dims i and i + rot/2 (interleaved: 2 i and
// 2 i + 1) are a pair (x, y) that becomes (x cos - y sin, y cos + x sin) of the
// position's angle i; the dims past `rot` stay.  Each product and sum is rounded
// to 32 bits by itself (no fused multiply-add), so that the result is the one of
// the same formula in separate operations, bit for bit, and the rounding to
// 16 or 8 bits that follows is its only other one.
//
// A lane holds a chunk of 8 dims.  Its partner dims lie in the chunk rot/16
// further on or back (interleaved: in its own), which it loads too: a second
// load of the same lines.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/aegkv.h"

namespace aegkv {
namespace {

typedef unsigned int rr_u32x4 __attribute__((ext_vector_type(4)));
typedef float rr_f32x4 __attribute__((ext_vector_type(4)));
typedef float rr_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 rr_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 rr_f16x2 __attribute__((ext_vector_type(2)));

template <int DT>
struct RowElem;
template <>
struct RowElem<AEGKV_DTYPE_BF16> {
  static __device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float high(uint32_t w) {
    return __uint_as_float(w & 0xffff0000u);
  }
  // to nearest even
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(rr_f32x2{x, y}, rr_bf16x2));
  }
};
template <>
struct RowElem<AEGKV_DTYPE_FP16> {
  static __device__ __forceinline__ float low(uint32_t w) {
    return (float)__builtin_bit_cast(rr_f16x2, w)[0];
  }
  static __device__ __forceinline__ float high(uint32_t w) {
    return (float)__builtin_bit_cast(rr_f16x2, w)[1];
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(rr_f32x2{x, y}, rr_f16x2));
  }
};

template <int DT>
__device__ __forceinline__ void unpack8(rr_u32x4 x, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = RowElem<DT>::low(x[i]);
    f[2 * i + 1] = RowElem<DT>::high(x[i]);
  }
}
template <int DT>
__device__ __forceinline__ rr_u32x4 pack8(const float (&f)[8]) {
  return rr_u32x4{RowElem<DT>::pack(f[0], f[1]), RowElem<DT>::pack(f[2], f[3]),
                  RowElem<DT>::pack(f[4], f[5]), RowElem<DT>::pack(f[6], f[7])};
}

// The call's angles: cosines and sines of a position's rot / 2 angles, one after
// the other, [max_pos][rot] float.
struct RotaryTable {
  const float* table;
  const int64_t* positions;  // [n_tokens]
  int64_t max_pos;
  int32_t rot;
};

// What a lane's chunk takes of the table for one position: cosines and (signed)
// sines of its dims' angles, of an interleaved chunk (INTER) four of each.
template <bool INTER>
struct ChunkAngles {
  static constexpr int N = INTER ? 1 : 2;
  rr_f32x4 cos[N], sin[N];
};
__device__ __forceinline__ bool chunk_turns(const RotaryTable& r, int c) { return 8 * c < r.rot; }
// the chunk that holds c's partner dims
template <bool INTER>
__device__ __forceinline__ int partner_chunk(const RotaryTable& r, int c) {
  const int half = r.rot / 16;
  return INTER ? c : c < half ? c + half : c - half;
}
// A position outside the table turns its rows to NaN: nothing is read there, and
// the mistake shows.
template <bool INTER>
__device__ __forceinline__ ChunkAngles<INTER> load_angles(const RotaryTable& r, int64_t pos, int c) {
  ChunkAngles<INTER> a;
  const bool inside = pos >= 0 && pos < r.max_pos;
  const int half = r.rot / 2;
  const bool first = INTER || 8 * c < half;
  const float* p = r.table + (inside ? pos : 0) * (int64_t)r.rot +
                   (INTER ? 4 * c : first ? 8 * c : 8 * c - half);
  const float nan = __builtin_nanf("");
#pragma unroll
  for (int q = 0; q < ChunkAngles<INTER>::N; ++q) {
    const rr_f32x4 x = *reinterpret_cast<const rr_f32x4*>(p + 4 * q);
    const rr_f32x4 y = *reinterpret_cast<const rr_f32x4*>(p + half + 4 * q);
    a.cos[q] = inside ? x : rr_f32x4{nan, nan, nan, nan};
    a.sin[q] = !inside ? rr_f32x4{nan, nan, nan, nan} : INTER || !first ? y : -y;
  }
  return a;
}

// The chunk's dims x turned, y its partner chunk's.
template <int DT, bool INTER>
__device__ __forceinline__ void turn_chunk(rr_u32x4 x, rr_u32x4 y, const ChunkAngles<INTER>& a,
                                           float (&f)[8]) {
#pragma clang fp contract(off)
  float p[8];
  unpack8<DT>(x, p);
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = p[2 * i] * a.cos[0][i] - p[2 * i + 1] * a.sin[0][i];
      f[2 * i + 1] = p[2 * i + 1] * a.cos[0][i] + p[2 * i] * a.sin[0][i];
    }
  } else {
    float q[8];
    unpack8<DT>(y, q);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = p[i] * a.cos[i >> 2][i & 3] + q[i] * a.sin[i >> 2][i & 3];
  }
}

// A side of a call's rows: n_heads dense heads per token.
struct HeadRows {
  const uint8_t* src;
  uint8_t* dst;        // dense rows out (may be src; null: none)
  int64_t src_tok_b, dst_tok_b;
  int32_t n_heads;
};

constexpr int kHeadPasses = 4;  // heads per lane of a task: its loads are in flight together

// Tasks of a wave for one token's rows of `n_heads` heads of `chunks` 8-dim chunks.
__host__ __device__ inline int head_tasks(int n_heads, int chunks) {
  const int per = 64 / chunks * kHeadPasses;
  return (n_heads + per - 1) / per;
}

// Task `part` of token `tok`: up to kHeadPasses rounds of 64 / chunks heads, turned
// (or copied: !turn) to the dense rows out and, with `cache`, to the token's row in
// the 16-bit cache.  A wave reads all of a row before it writes any of it.
template <int DT, bool INTER>
__device__ __forceinline__ void turn_heads(const HeadRows& h, const RotaryTable& r, bool turn,
                                           int tok, int part, int chunks, uint8_t* cache) {
  const int lane = threadIdx.x & 63;
  const int per = 64 / chunks;  // heads per round
  const int hl = lane / chunks, c = lane - hl * chunks;
  const int head0 = part * per * kHeadPasses + hl;
  const bool turns = turn && chunk_turns(r, c);
  const int64_t row_b = (int64_t)chunks * 16;
  const uint8_t* row = h.src + (int64_t)tok * h.src_tok_b;
  const int64_t at = (int64_t)head0 * row_b + 16 * c;
  const int64_t other = turns ? (int64_t)(partner_chunk<INTER>(r, c) - c) * 16 : 0;
  rr_u32x4 x[kHeadPasses], y[kHeadPasses];
  bool ok[kHeadPasses];
#pragma unroll
  for (int i = 0; i < kHeadPasses; ++i) {
    ok[i] = hl < per && head0 + i * per < h.n_heads;
    if (ok[i]) {
      const uint8_t* p = row + at + (int64_t)i * per * row_b;
      x[i] = *reinterpret_cast<const rr_u32x4*>(p);
      y[i] = *reinterpret_cast<const rr_u32x4*>(p + other);
    } else {
      x[i] = y[i] = rr_u32x4{0u, 0u, 0u, 0u};
    }
  }
  ChunkAngles<INTER> a = {};
  if (turns) a = load_angles<INTER>(r, r.positions[tok], c);
#pragma unroll
  for (int i = 0; i < kHeadPasses; ++i) {
    if (turns) {
      float f[8];
      turn_chunk<DT, INTER>(x[i], y[i], a, f);
      x[i] = pack8<DT>(f);
    }
    if (ok[i]) {
      const int64_t o = at + (int64_t)i * per * row_b;
      if (h.dst) *reinterpret_cast<rr_u32x4*>(h.dst + (int64_t)tok * h.dst_tok_b + o) = x[i];
      if (cache) *reinterpret_cast<rr_u32x4*>(cache + o) = x[i];
    }
  }
}

// Host checks of a rotating call's table and rows (0 or a status).
inline int check_rotary(const RotaryTable& r, int32_t head_dim) {
  if (r.max_pos < 0 || r.rot <= 0 || r.rot > head_dim) return AEGKV_ERR_INVALID_ARG;
  if (r.rot % 16) return AEGKV_ERR_UNSUPPORTED;
  return AEGKV_OK;
}

}  // namespace
}  // namespace aegkv
