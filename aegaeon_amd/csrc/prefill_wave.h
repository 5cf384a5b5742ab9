// What the prompt attention kernels share: the 16-bit matrix products, divisions
// by a launch's constants, and a wave's online softmax over tiles of 64 keys.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/aegkv.h"
#include "wave_scan.h"

namespace aegkv {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kPfKTile = 64;                 // keys per step
constexpr float kPfRescaleSlack = 8.f;

// kTop: log2 of the weight of a row's largest score (where nothing was rescaled
// lately up to kPfRescaleSlack more).  fp16 holds weights up to 2^15, so that its
// subnormals, off by 2^-25 at most, begin 2^21 below the largest weight: with 2^0 for
// it thousands of keys of 2^-25 each were rounded away beside one key, while the sum
// of the weights counted them.
template <int DT>
struct PfOps;

template <>
struct PfOps<AEGKV_DTYPE_BF16> {
  static constexpr float kTop = 0.f;
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  // two floats to two 16-bit values, round to nearest even (one instruction)
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
  }
};

template <>
struct PfOps<AEGKV_DTYPE_FP16> {
  static constexpr float kTop = 7.f;
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, f16x2));
  }
};

// max(a, b, c) through the compiler's own max, never inline asm.  The
// scores are MFMA results, and a VALU read of an MFMA result needs wait states
// that only the compiler's hazard tracking inserts: it does not see the
// operands of an inline-asm v_max3_f32.  That form read unfinished scores on
// unmasked key tiles whenever the matrix core ran late, which showed as
// run-to-run output differences (one ulp, in ~7% of rows) once the four-wave
// kernel's workgroups were dealt to CUs in another order.  The compiler's max
// costs a few canonicalising v_max_f32 (0-3% per call).
__device__ __forceinline__ float max3(float a, float b, float c) {
  return __builtin_fmaxf(__builtin_fmaxf(a, b), c);
}

// floor(n / d) for 0 <= n < 2^31 by a multiplication (mul = floor(2^(31 + shift)
// / d) + 1, shift = ceil(log2 d): 2^(31 + shift) < mul * d <= 2^(31 + shift) +
// 2^shift).  A division by a number the compiler does not know is some twenty
// vector instructions; a workgroup's start has half a dozen of them.
struct FastDiv {
  uint32_t mul, shift;
  __device__ __forceinline__ int div(int n) const {
    return (int)(__umulhi(2u * (uint32_t)n, mul) >> shift);
  }
};
inline FastDiv fast_div(int32_t d) {  // 1 <= d < 2^31
  FastDiv f;
  f.shift = 0;
  while ((1ll << f.shift) < d) ++f.shift;
  f.mul = (uint32_t)((((uint64_t)1 << (31 + f.shift)) / (uint64_t)d) + 1);
  return f;
}

// A wave's 32 query rows: the Q^T operand, the O^T accumulators and the online
// softmax.  Lane (col = l & 31, hh = l / 32) belongs to row col; it holds of
// S^T's 32-key block sb the keys 32 sb + 8 (i / 4) + 4 hh + i % 4 (element i),
// and of O^T head dims 32 db + 8 g + 4 hh .. + 3 in element 4 g .. 4 g + 3 of
// o[db].  KEYLESS: a row may have seen no key beside one that has (in a prompt each
// row sees its first tile's first).
template <int DT, int D, bool KEYLESS>
struct WaveSoftmax {
  static constexpr int KS = D / 16;  // k-steps of K.Q^T
  static constexpr int DB = D / 32;  // 32-row blocks of O^T
  u32x4 qv[KS];                      // Q^T operand: dims 16 ks + 8 hh .. +7
  f32x16 o[DB];
  float m, lsum;  // m: the running maximum less kTop (log2 units); lsum: of this lane's keys

  // online softmax of a masked S^T tile into the P^T operands of its four
  // 16-key steps
  // (`first`: the wave's first tile, whose sums are still zero)
  __device__ __forceinline__ void softmax(f32x16 (&s)[2], u32x4 (&pb)[4], float scale_log2,
                                          bool first) {
    // raw-score max (the scale is positive) over four chains of triples: a lone
    // pair of scores would be canonicalised first (28 instructions, now 16:
    // 1 x 8192 435.5 -> 427.0 us, 4 x 2048 131.3 -> 128.9)
    float c4[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const f32x16& x = s[c >> 1];
      const int e = 8 * (c & 1);
      c4[c] = max3(x[e], x[e + 1], x[e + 2]);
    }
#pragma unroll
    for (int k = 3; k < 7; k += 2)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        c4[c] = max3(c4[c], s[c >> 1][8 * (c & 1) + k], s[c >> 1][8 * (c & 1) + k + 1]);
    const float d0 = max3(c4[0], s[0][7], s[0][15]), d1 = max3(c4[1], s[1][7], s[1][15]);
    float bm = fmaxf(max3(d0, c4[2], c4[3]), d1);
    // the partner lane's max (same query), exchanged between the wave's
    // halves in registers: one v_permlane32_swap instead of the LDS round trip
    // of a shuffle.  (Both kernels, 20 repeated calls each, also with two
    // unsynchronised workgroups per CU: bit-identical outputs, and bit-identical
    // to the shuffle; the four-wave kernel 0-2% faster with it.)
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(bm), __float_as_uint(bm),
                                                     false, false);
    bm = fmaxf(fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])), bm);
    if constexpr (PfOps<DT>::kTop == 0.f) bm *= scale_log2;
    else bm = __builtin_fmaf(bm, scale_log2, -PfOps<DT>::kTop);
    if (first) {
      m = fmaxf(m, bm);
    } else if (__builtin_amdgcn_ballot_w64(bm > m + kPfRescaleSlack)) {
      const float mn = fmaxf(m, bm);
      // 0 while m = -inf (a row without a key: of sums that are 0)
      const float alpha = __builtin_amdgcn_exp2f(m - (KEYLESS && mn == -INFINITY ? 0.f : mn));
      lsum *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
      m = mn;
    }
    const float nms = m == -INFINITY ? 0.f : -m;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const int sb = kk >> 1, base = 8 * (kk & 1);
      uint32_t pw[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p0 =
            __builtin_amdgcn_exp2f(__builtin_fmaf(s[sb][base + 2 * j], scale_log2, nms));
        const float p1 =
            __builtin_amdgcn_exp2f(__builtin_fmaf(s[sb][base + 2 * j + 1], scale_log2, nms));
        lsum += p0 + p1;
        pw[j] = PfOps<DT>::pack(p0, p1);
      }
      pb[kk] = u32x4{pw[0], pw[1], pw[2], pw[3]};
    }
  }
};

}  // namespace
}  // namespace aegkv
