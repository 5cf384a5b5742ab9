// The 4-bit KV cache: what a value becomes and where its bits lie.
//
// Values.  A group is 32 consecutive dims of one token's K or V row of one
// head.  Its exponent e is the least integer with max|x| < 7 * 2^e, within
// [-125, 125] (bf16) or [-125, 13] (fp16); a value becomes its sign and
// |x| / 2^e rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the
// even code, at most 6): no element is off by more than half a step of the
// largest one's binade, as a maximum below 7 * 2^e rounds to 6 * 2^e at most.
// The group keeps the byte E = e + 127.  The bounds keep code * 2^e a normal
// (fp16: finite) number of the 16-bit type, so that every value the cache
// stands for is exact in the type it was written from.  A group that holds an
// infinity or a NaN keeps E = 255 and zero codes, and reads back as NaN.
// gfx950 converts both ways a pair at a time (v_cvt_scalef32_pk_*: round to
// nearest even, saturating; scale byte 255 reads as NaN).
//
// Bits.  A block's 16 tokens of one layer and kv head are 17 D consecutive
// bytes (D = 128: 17 lines of 128), a K record and a V record of 8 D bytes of
// codes and D/2 scale bytes [D/32 groups][16 tokens] each.  The codes lie as
// the lanes of the attention's matrix operands read them, 4 D (D <= 128: all 8
// D) consecutive bytes per wave-wide load; a pair's lower dim is in the low
// half of its byte:
//   K: [chunk][16 tokens][16 bytes], 32 consecutive dims per chunk (D = 64: 8
//      bytes, 16 dims), so a lane's load is one token's group;
//   V: [piece][4 token quads][16 lanes][4 tokens][4 bytes], lane j holding dims
//      D/16 j + 8 piece .. + 7 (D = 64: 2 bytes, 4 dims, one piece).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/aegkv.h"

namespace aegkv {

constexpr int kKv4Group = 32;        // dims per scale
constexpr int kKv4Tokens = 16;       // tokens per block
constexpr int kKv4ScaleMin = 2;      // e = -125
constexpr uint32_t kKv4ScaleNan = 255;

// Bytes of a K or V record, and of its codes.
__host__ __device__ constexpr int kv4_record_bytes(int head_dim) { return head_dim * 17 / 2; }
__host__ __device__ constexpr int kv4_code_bytes(int head_dim) { return head_dim * 8; }

// The byte, in a record, of the codes of dims 8 c .. 8 c + 7 of token r: four
// consecutive bytes, but for V at D = 64 two and two, 8 further on.
template <int D>
__device__ __forceinline__ int kv4_k_byte(int r, int c) {
  if constexpr (D == 64) return ((c >> 1) * kKv4Tokens + r) * 8 + (c & 1) * 4;
  else return ((c >> 2) * kKv4Tokens + r) * 16 + (c & 3) * 4;
}
template <int D>
__device__ __forceinline__ int kv4_v_byte(int r, int c) {
  if constexpr (D == 64) return ((r >> 2) * 16 + 2 * c) * 8 + (r & 3) * 2;
  else if constexpr (D == 128) return ((r >> 2) * 16 + c) * 16 + (r & 3) * 4;
  else return (((c & 1) * 4 + (r >> 2)) * 16 + (c >> 1)) * 16 + (r & 3) * 4;
}

// The conversions of a 16-bit type.  dq: byte SEL of a word of codes to two
// 16-bit values (the lower dim in the low half); q: two values to byte SEL of
// the word.  scale: 2^e.
template <int DT>
struct Kv4Elem;

template <>
struct Kv4Elem<AEGKV_DTYPE_BF16> {
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kNotFinite = 0x7f80u;  // magnitude bits of infinity
  static constexpr int kScaleMax = 252;            // e = 125: 6 * 2^125 is finite
  static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits << 16); }
  template <int SEL>
  static __device__ __forceinline__ uint32_t dq(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t q(uint32_t codes, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(x2, pair), scale, SEL);
  }
};

template <>
struct Kv4Elem<AEGKV_DTYPE_FP16> {
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kNotFinite = 0x7c00u;
  static constexpr int kScaleMax = 140;            // e = 13: 6 * 2^13 = 49152
  static __device__ __forceinline__ float value(uint32_t bits) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)bits);
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t dq(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t q(uint32_t codes, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(x2, pair), scale, SEL);
  }
};

// 2^e of a scale byte (255: an infinity, which the conversions read as NaN).
__device__ __forceinline__ float kv4_scale(uint32_t e) { return __uint_as_float(e << 23); }

// The scale byte of a group whose largest magnitude has the bits `top` of the
// 16-bit type: the carry of 1/4 into the exponent moves maxima of 7 * 2^k and
// above to the next one.
template <int DT>
__device__ __forceinline__ uint32_t kv4_scale_byte(uint32_t top) {
  const int e = (int)((__float_as_uint(Kv4Elem<DT>::value(top)) + 0x200000u) >> 23) - 2;
  const int c = min(max(e, kKv4ScaleMin), Kv4Elem<DT>::kScaleMax);
  return top >= Kv4Elem<DT>::kNotFinite ? kKv4ScaleNan : (uint32_t)c;
}

}  // namespace aegkv
