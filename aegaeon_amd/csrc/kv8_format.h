// The 8-bit KV cache: what a value becomes and where its byte lies.
//
// Values.  The 16 tokens of a block share, per layer, kv head and side (K or V),
// an exponent e: the least integer with max|x| <= 448 * 2^e over the block's finite
// values, within [-117, 119] (bf16) or [-15, 7] (fp16).  A value's code is the
// 8-bit float (four exponent and three mantissa bits, largest 448) nearest to
// x / 2^e, ties to even; an infinity or a NaN gets the code 0xff, a NaN.  An element
// rounded once is off by at most 2^-4 of itself or 2^-10 * 2^e, half a step of the
// codes or of the least of them, whichever is more.  The bounds keep code * 2^e
// exact in the rows' 16-bit type (2^TOP * 448 finite, its least step a number of
// the type), so that everything past the conversion is the 16-bit operators'
// arithmetic; values past 448 * 2^TOP are stored as that (fp16: 65504 as 57344).
//   Tokens that join a block in which earlier ones are (none of them at the block's
// first place) take e = max(the block's, their own).  When that rises, the earlier
// tokens' values are rounded once more, to the codes of the new exponent: as the
// scale is a power of two, only what falls below 2^-6 of it loses bits, and an element
// is off by less than 2^-9 * 2^e, or 2^-4 of itself, after any number of rises: each
// rounding there is off by 2^-10 of its own 2^e, at most half of the next one's, and the
// one before them by at most half of the first's.  No append lowers an exponent but
// at a block's first place: a token written over another leaves the block as coarse as
// that one made it.  A token at a block's first place begins the block anew, the tokens
// not written read as 0.
//
// Bytes.  A block of one layer: per kv head the 16 D codes of K, then V's; then 4
// bytes per head: K's e + 127, V's, 1 where V holds a NaN, 0; padded to a whole
// line of 128 bytes, so that every wave-wide load of codes is of whole lines.  The
// codes lie as the lanes of the attention's matrix operands read them, 1024
// consecutive bytes per wave-wide load:
//   K: [chunk of 16 dims][16 tokens][16 dims], a lane's 16 bytes one token's dims;
//   V: [D/64 pieces][4 token quads][16 lanes][4 dims][4 tokens], lane j holding
//      dims D/16 j .., piece i its dims 4 i .. 4 i + 3: a word is one dim of four
//      consecutive tokens, two conversions of two from the operand's registers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/aegkv.h"

namespace aegkv {

constexpr int kKv8Tokens = 16;  // tokens per block
constexpr int kKv8MaxHeads = 256;
constexpr float kKv8Largest = 448.f;

// Bytes of one kv head's K (or V) codes of a block.
__host__ __device__ constexpr int kv8_side_bytes(int head_dim) { return 16 * head_dim; }
// Where the heads' scale bytes begin in a layer's block, and its size.
__host__ __device__ constexpr int64_t kv8_scales_at(int64_t heads, int head_dim) {
  return heads * 2 * kv8_side_bytes(head_dim);
}
__host__ __device__ constexpr int64_t kv8_layer_bytes(int64_t heads, int head_dim) {
  return kv8_scales_at(heads, head_dim) + (4 * heads + 127) / 128 * 128;
}

// The byte, in a side's codes, of dims 8 c .. 8 c + 7 of token r of K (eight
// consecutive), and of dims 4 f .. 4 f + 3 of tokens 4 g .. 4 g + 3 of V (sixteen,
// [dim][token]).
__device__ __forceinline__ int kv8_k_byte(int r, int c) {
  return (c >> 1) * 256 + r * 16 + (c & 1) * 8;
}
template <int D>
__device__ __forceinline__ int kv8_v_byte(int g, int f) {
  constexpr int P = D / 64;  // pieces
  return ((f % P * 4 + g) * 16 + f / P) * 16;
}

// dq: two codes (HI: of the upper half) of a word to two 16-bit values times 2^e.
template <int DT>
struct Kv8Elem;
template <>
struct Kv8Elem<AEGKV_DTYPE_BF16> {
  static constexpr int kLow = 10, kTop = 246;  // scale bytes of e = -117, 119
  template <bool HI>
  static __device__ __forceinline__ uint32_t dq(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HI));
  }
};
template <>
struct Kv8Elem<AEGKV_DTYPE_FP16> {
  static constexpr int kLow = 112, kTop = 134;  // e = -15, 7
  template <bool HI>
  static __device__ __forceinline__ uint32_t dq(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HI));
  }
};

// 2^e of a scale byte.
__device__ __forceinline__ float kv8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The scale byte of finite values whose largest magnitude has the bits `top` of a
// float: the carry of 1/4 into the exponent moves maxima past 1.75 * 2^k to the next.
template <int DT>
__device__ __forceinline__ int kv8_scale_byte(uint32_t top) {
  return min(max((int)((top + 0x1fffffu) >> 23) - 8, Kv8Elem<DT>::kLow), Kv8Elem<DT>::kTop);
}

}  // namespace aegkv
