// Attention of several query tokens per sequence over the paged 4-bit KV cache
// (kv4_format.h) on gfx950: varlen_cache.h's kernels with this cache's loads and
// conversions (190 instructions per 128 keys and wave).
//
// Bounds and measured.  Per cached token and kv head 17 D / 16 bytes are read
// and 4 D G flops done per query, so past some 10 queries at G = 7 the products
// bound it: 2048 queries over 16001 tokens (28/4 heads, D = 128) 453 to 462 us by the
// session, 972 to 952 TFLOP/s (224 of 256 CUs hold a tile, at 92% of the rate of a large matrix
// product each); 4 x 512 over 3800 tokens each 137 us, the longest sequence's;
// two whole prompts of 2048 81 us, 747 TFLOP/s.  Few queries are bound by the latency
// of their steps, 1.7 us each of a lone workgroup (conversion, products and softmax
// of a wave follow each other): 48 x 5 over 1000 tokens each (32/4) 23.9 us a call,
// the main kernel 21.3 and the merge 4.4.
#include "kv4_format.h"
#include "varlen_cache.h"

namespace aegkv {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// The K or V codes of one block for one lane, as in the decode attention:
// words and scale byte(s).
template <int D>
struct CodeRegs {
  uint32_t w[D / 32], s;
};

// V's rows of 2 D bytes in LDS, their 16-byte chunks permuted by the row.
template <int D>
__device__ __forceinline__ int v_chunk(int row, int c) {
  return D == 128 ? c ^ ((row & 3) << 2) : c ^ (((row >> 1) & 1) << 2);
}

struct Codes4 {
  static constexpr bool kUneven = false;
  template <int D>
  using Regs = CodeRegs<D>;
  template <int D>
  static __device__ __forceinline__ HeadPart head(const VarlenArgs&, int h) {
    return {(int64_t)h * 17 * D, 17 * D, 0};
  }
  template <int D>
  static __device__ __forceinline__ void load_words4(CodeRegs<D>& c, __amdgpu_buffer_rsrc_t r, int at,
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
  static __device__ __forceinline__ void load_k(CodeRegs<D>& c, __amdgpu_buffer_rsrc_t r, const HeadPart&,
                                              int lane) {
    const int j = lane & 15, g = lane >> 4;
    load_words4<D>(c, r, 0, lane);
    c.s = __builtin_amdgcn_raw_buffer_load_b8(
        r, kv4_code_bytes(D) + (D == 64 ? g >> 1 : g) * kKv4Tokens + j, 0, 0);
  }
  template <int D>
  static __device__ __forceinline__ void load_v(CodeRegs<D>& c, __amdgpu_buffer_rsrc_t r, const HeadPart&,
                                              int lane) {
    constexpr int REC = kv4_record_bytes(D);
    const int j = lane & 15, g = lane >> 4;
    load_words4<D>(c, r, REC, lane);
    c.s = __builtin_amdgcn_raw_buffer_load_b32(
        r, REC + kv4_code_bytes(D) + (j * (D / 16) / kKv4Group) * kKv4Tokens + 4 * g, 0, 0);
  }

  template <int DT, int D>
  static __device__ __forceinline__ void put_k(uint8_t* lds, const CodeRegs<D>& c, int u, int lane) {
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
  // group (uniform): its rows are found at the end (find_nan).
  template <int DT, int D>
  static __device__ __forceinline__ bool put_v(uint8_t* lds, CodeRegs<D>& c, int u, int left, int lane) {
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
  // O^T += V^T.P^T of a tile: V's rows through transposing reads, four ahead of their
  // use (see RowUnit::qk)
  template <int DT, int D>
  static __device__ __forceinline__ void pv(f32x16 (&o)[D / 32], const uint8_t* lds,
                                            const u32x4 (&pb)[4]) {
    constexpr int RB = 2 * D, DB = D / 32;
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
  // NaN comes by groups of V's dims.
  static __device__ __host__ constexpr int nan_entry(int dim) { return dim / kKv4Group * kKv4Group; }
  // The lane's block (ok: it is one), of the 64 from b0 on: its groups' scale bytes, a
  // group's 16 tokens in one load, and the first NaN of each.  (Group after group: with
  // all of them in flight the eight-wave kernel is 2% slower where there is no NaN.)
  template <int D>
  static __device__ void find_nan(const uint8_t* part, const HeadPart&, bool ok, int b0,
                                  int32_t* first) {
    if (!ok) return;
    const u32x4* e = reinterpret_cast<const u32x4*>(part + kv4_record_bytes(D) + kv4_code_bytes(D));
#pragma unroll 1
    for (int g = 0; g < D / kKv4Group; ++g) {
      const u32x4 x = ~e[g];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // a byte of zero (255 was there): the lowest one's bit 7 is exact
        const uint32_t at = (x[i] - 0x01010101u) & ~x[i] & 0x80808080u;
        if (at)
          first_key(first + kKv4Group * g, (b0 + (int)(threadIdx.x & 63)) * kKv4Tokens + 4 * i +
                                   (__builtin_ctz(at) >> 3));
      }
    }
  }
};

}  // namespace
}  // namespace aegkv

using namespace aegkv;

extern "C" {

int64_t aegkv_kv4_varlen_attention_workspace_size(int32_t batch, int64_t total_q,
                                                  int32_t max_seqlen_q, int32_t max_seq_len,
                                                  int32_t n_q_heads, int32_t n_kv_heads,
                                                  int32_t head_dim, int32_t dtype) {
  return varlen_workspace<Codes4>(batch, total_q, max_seqlen_q, max_seq_len, n_q_heads, n_kv_heads,
                          head_dim, dtype);
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
  return run_varlen<Codes4>(out, out_token_stride, q, q_token_stride, cache, cache_block_stride,
                            n_blocks, block_tables, max_blocks, cu_seqlens_q, seq_lens, batch,
                            total_q, max_seqlen_q, max_seq_len, n_q_heads, n_kv_heads, head_dim,
                            scale, causal, dtype, workspace, workspace_bytes, stream);
}

}  // extern "C"
