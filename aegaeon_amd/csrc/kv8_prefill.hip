// Attention of several query tokens per sequence over the paged 8-bit KV cache
// (kv8_format.h) on gfx950: varlen_cache.h's kernels with this cache's loads and
// conversions.  K's codes become rows of 16-bit values in LDS as the 4-bit cache's do.
// V's lie four tokens of a dim to a word, so they become V^T: a word converts to the
// 8 bytes of a dim's four tokens, and the operand V^T[32 dims x 16 keys] is one
// ordinary 16-byte read per lane, without a transposing read.
//   Bound by the products where rows are many (2048 queries over 16001 tokens, 28/4
// heads, bf16: 450 to 464 us a pass by the session, 977 to 948 TFLOP/s) and by the latency of a piece's start and
// steps where they are few (48 x 5 over 1000 tokens, 32/4 heads: 22.4 us and the merge's
// 4.4; 52 MB).  Measured and no better: V^T's rows permuted by
// one more bit (0 to +1.5%), reads four ahead (0), left to the compiler's order (+2%),
// four key tiles a step for up to 32 rows (28.5 -> 39.0 us).
#include "kv8_format.h"
#include "varlen_cache.h"

namespace aegkv {
namespace {

// The K or V codes of one block for one lane and the head's scale bytes, as in the
// decode attention.
template <int D>
struct CodeRegs8 {
  uint32_t w[D / 16], s;
};

// V^T in LDS: rows of a dim's 64 keys, 128 bytes, their 16-byte chunks permuted by
// the dim so that both the stores (dims D/16 apart in neighbouring lanes) and the
// operand reads (neighbouring dims) hit distinct banks.  Chunk 2 u + (q & 1) holds
// the quads q and q + 2 (q < 2) of block u: a lane's half of the operand, whose keys
// are 4 hh .. + 3 and 8 + 4 hh .. + 3 (WaveSoftmax).
__device__ __forceinline__ int vt_chunk(int dim, int c) { return c ^ ((dim ^ dim >> 3) & 7); }

struct Codes8 {
  static constexpr bool kUneven = true;
  template <int D>
  using Regs = CodeRegs8<D>;
  template <int D>
  static __device__ __forceinline__ HeadPart head(const VarlenArgs& a, int h) {
    const int codes = h * 2 * kv8_side_bytes(D);
    const int scale = (int)kv8_scales_at(a.n_kv_heads, D) + 4 * h - codes;
    return {codes, (uint32_t)scale + 4, scale};
  }
  template <int D>
  static __device__ __forceinline__ void load(Regs<D>& c, __amdgpu_buffer_rsrc_t r, int at,
                                              int scale, int lane) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, at + 1024 * i + 16 * lane, 0, 0);
#pragma unroll
      for (int k = 0; k < 4; ++k) c.w[4 * i + k] = x[k];
    }
    c.s = __builtin_amdgcn_raw_buffer_load_b32(r, scale, 0, 0);
  }
  template <int D>
  static __device__ __forceinline__ void load_k(Regs<D>& c, __amdgpu_buffer_rsrc_t r,
                                                const HeadPart& h, int lane) {
    load<D>(c, r, 0, h.scale, lane);
  }
  template <int D>
  static __device__ __forceinline__ void load_v(Regs<D>& c, __amdgpu_buffer_rsrc_t r,
                                                const HeadPart& h, int lane) {
    load<D>(c, r, kv8_side_bytes(D), h.scale, lane);
  }

  template <int DT, int D>
  static __device__ __forceinline__ void put_k(uint8_t* lds, const Regs<D>& c, int u, int lane) {
    using C = Kv8Elem<DT>;
    const int j = lane & 15, g = lane >> 4, row = kKv8Tokens * u + j;
    const float s = kv8_scale(__builtin_amdgcn_readfirstlane(c.s) & 0xffu);
    uint8_t* p = lds + row * 2 * D;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // dims 64 i + 16 g + 8 e ..
        const uint32_t x = c.w[4 * i + 2 * e], y = c.w[4 * i + 2 * e + 1];
        *reinterpret_cast<u32x4*>(p + k_chunk<D>(row, 8 * i + 2 * g + e) * 16) =
            u32x4{C::template dq<false>(x, s), C::template dq<true>(x, s),
                  C::template dq<false>(y, s), C::template dq<true>(y, s)};
      }
  }
  // V's tokens at or past `left` (of the block's 16) and NaN codes are stored as
  // zeros.  True when there was a NaN (uniform; the block says whether to look).
  template <int DT, int D>
  static __device__ __forceinline__ bool put_v(uint8_t* lds, Regs<D>& c, int u, int left,
                                               int lane) {
    using C = Kv8Elem<DT>;
    const int j = lane & 15, g = lane >> 4;
    const uint32_t bytes = __builtin_amdgcn_readfirstlane(c.s);
    bool nan = false;
    if (left < kKv8Tokens) {  // uniform
      uint32_t keep = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) keep |= 4 * g + i < left ? 0xffu << (8 * i) : 0u;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) c.w[t] &= keep;
    }
    if (bytes >> 16 & 0xffu) {  // rare
      bool bad = false;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        const uint32_t at = ((c.w[t] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        bad |= at != 0;
        c.w[t] &= ~((at >> 7) * 0xffu);
      }
      nan = __builtin_amdgcn_ballot_w64(bad) != 0;
    }
    const float s = kv8_scale(bytes >> 8 & 0xffu);
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      const int dim = D / 16 * j + t;
      *reinterpret_cast<u32x2*>(lds + dim * 128 + vt_chunk(dim, 2 * u + (g & 1)) * 16 +
                                8 * (g >> 1)) =
          u32x2{C::template dq<false>(c.w[t], s), C::template dq<true>(c.w[t], s)};
    }
    return nan;
  }
  // O^T += V^T.P^T of a tile; LDS reads stay two MFMAs ahead of their use
  template <int DT, int D>
  static __device__ __forceinline__ void pv(f32x16 (&o)[D / 32], const uint8_t* lds,
                                            const u32x4 (&pb)[4]) {
    constexpr int DB = D / 32;
    const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
    const uint8_t* row = lds + col * 128;
    const int x = vt_chunk(col, hh) * 16;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        // vt_chunk(32 db + col, 2 kk + hh): dim / 8 grows by 4 db
        const uint8_t* p = row + (x ^ (32 * kk) ^ (64 * (db & 1))) + 4096 * db;
        o[db] = PfOps<DT>::mfma(*reinterpret_cast<const u32x4*>(p), pb[kk], o[db]);
      }
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
#pragma unroll
    for (int i = 0; i < 4 * DB - 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // the next read
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
  }
  static __device__ __host__ constexpr int nan_entry(int dim) { return dim; }
  // Whether the lane's block (ok: it is one), of the 64 from b0 on, has a NaN in V; then
  // the wave takes such blocks one by one, a lane 4 dims of 4 tokens.
  template <int D>
  static __device__ void find_nan(const uint8_t* part, const HeadPart& h, bool ok, int b0,
                                  int32_t* first) {
    const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
    uint64_t bad = __builtin_amdgcn_ballot_w64(ok && part[h.scale + 2] != 0);
    for (; bad; bad &= bad - 1) {  // uniform
      const int u = __builtin_ctzll(bad);
      const uint64_t p = (uint64_t)part;
      const uint8_t* v = reinterpret_cast<const uint8_t*>(
                             (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(p >> 32), u) << 32 |
                             (uint32_t)__builtin_amdgcn_readlane((int)p, u)) +
                         kv8_side_bytes(D) + 16 * lane;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(v + 1024 * i);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const uint32_t at = ((x[d] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          if (at)
            first_key(first + D / 16 * j + 4 * i + d,
                      (b0 + u) * kKv8Tokens + 4 * g + (__builtin_ctz(at) >> 3));
        }
      }
    }
  }
};

}  // namespace
}  // namespace aegkv

using namespace aegkv;

extern "C" {

int64_t aegkv_kv8_varlen_attention_workspace_size(int32_t batch, int64_t total_q,
                                                  int32_t max_seqlen_q, int32_t max_seq_len,
                                                  int32_t n_q_heads, int32_t n_kv_heads,
                                                  int32_t head_dim, int32_t dtype) {
  if (n_kv_heads > kKv8MaxHeads) return AEGKV_ERR_UNSUPPORTED;
  return varlen_workspace<Codes8>(batch, total_q, max_seqlen_q, max_seq_len, n_q_heads, n_kv_heads,
                          head_dim, dtype);
}

int aegkv_kv8_varlen_attention(void* out, int64_t out_token_stride, const void* q,
                               int64_t q_token_stride, const void* cache,
                               int64_t cache_block_stride, int64_t n_blocks,
                               const int32_t* block_tables, int32_t max_blocks,
                               const int32_t* cu_seqlens_q, const int32_t* seq_lens, int32_t batch,
                               int64_t total_q, int32_t max_seqlen_q, int32_t max_seq_len,
                               int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float scale,
                               int32_t causal, int32_t dtype, void* workspace,
                               uint64_t workspace_bytes, aegkv_stream_t stream) {
  if (n_kv_heads > kKv8MaxHeads) return AEGKV_ERR_UNSUPPORTED;
  return run_varlen<Codes8>(out, out_token_stride, q, q_token_stride, cache, cache_block_stride,
                            n_blocks, block_tables, max_blocks, cu_seqlens_q, seq_lens, batch,
                            total_q, max_seqlen_q, max_seq_len, n_q_heads, n_kv_heads, head_dim,
                            scale, causal, dtype, workspace, workspace_bytes, stream);
}

}  // extern "C"
