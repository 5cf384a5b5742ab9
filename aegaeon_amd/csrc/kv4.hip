// Writing and de-paging the 4-bit KV cache (kv4_format.h) on gfx950:
//  - kv4_append: slot-mapped write of new 16-bit K/V rows, one layer or every
//    layer of a step in one launch;
//  - kv4_gather: block-table-driven de-page of sequences into contiguous 16-bit
//    [sum(len), Hkv, D] buffers.
// A thread converts 8 dims of one token and head: 16 bytes of the 16-bit side,
// 4 bytes of codes; the four threads of a group share its scale byte.
#include <algorithm>

#include "aegkv_internal.h"
#include "kv4_format.h"
#include "wave_scan.h"

namespace aegkv {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr int kAppend4Threads = 256;

struct Append4Args {
  const uint8_t* key;
  const uint8_t* value;
  int64_t key_tok_b, val_tok_b, key_layer_b, val_layer_b;  // byte strides
  const int64_t* slots;
  uint8_t* cache;
  int64_t blk_b, layer_b;  // cache byte strides
  int64_t n_slots;         // n_blocks * 16
  uint32_t n_tokens;
  uint32_t n_heads;
  uint32_t total;          // threads: n_layers * 2 * n_heads * n_tokens * D / 8
};

// Thread order: dims fastest, then tokens, heads, K/V, layers, so a workgroup
// covers 2048 / D consecutive tokens of one head and side: of a prompt, whole
// records, whose scattered 4-byte stores its XCD's L2 merges into lines.  Bound by
// the rows read: 8 layers of 4 x 1024 tokens, 4 heads of 128 (85 MB moved) 20.4
// us, 4.2 TB/s of the 5.1 of a large copy; a step of 128 tokens, 28 layers, 5 us.
template <int DT, int D>
__global__ __launch_bounds__(kAppend4Threads) void kv4_append_kernel(Append4Args a) {
  using E = Kv4Elem<DT>;
  const uint32_t gid = blockIdx.x * kAppend4Threads + threadIdx.x;
  if (gid >= a.total) return;  // whole groups of four: total is a multiple of 8
  const uint32_t c = gid % (D / 8);
  uint32_t rest = gid / (D / 8);
  const uint32_t tok = rest % a.n_tokens;
  rest /= a.n_tokens;
  const uint32_t head = rest % a.n_heads;
  rest /= a.n_heads;
  const uint32_t kv = rest & 1, layer = rest >> 1;
  const uint8_t* src = kv ? a.value + layer * a.val_layer_b + tok * a.val_tok_b
                          : a.key + layer * a.key_layer_b + tok * a.key_tok_b;
  const int64_t s = a.slots[tok];
  const u32x4 x = __builtin_nontemporal_load(
      reinterpret_cast<const u32x4*>(src + ((int64_t)head * D + 8 * c) * 2));
  // the group's largest magnitude: the magnitude bits of either type order as
  // the numbers do, NaN above infinity above the rest
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[i] & 0x7fff7fffu));
  uint32_t top = max((uint32_t)m.x, (uint32_t)m.y);
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true));  // lane ^ 1
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4e, 0xf, 0xf, true));  // lane ^ 2
  const uint32_t e = kv4_scale_byte<DT>(top);
  const float scale = kv4_scale(e);
  uint32_t codes = E::template q<0>(0u, x[0], scale);
  codes = E::template q<1>(codes, x[1], scale);
  codes = E::template q<2>(codes, x[2], scale);
  codes = E::template q<3>(codes, x[3], scale);
  if (e == kKv4ScaleNan) codes = 0;
  if (s < 0 || s >= a.n_slots) return;
  const int64_t blk = s / kKv4Tokens;
  const int r = (int)(s - blk * kKv4Tokens);
  uint8_t* rec = a.cache + blk * a.blk_b + layer * a.layer_b +
                 (int64_t)(head * 2 + kv) * kv4_record_bytes(D);
  if (kv && D == 64) {
    uint8_t* p = rec + kv4_v_byte<D>(r, c);
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)codes;
    *reinterpret_cast<uint16_t*>(p + 8) = (uint16_t)(codes >> 16);
  } else {
    *reinterpret_cast<uint32_t*>(rec + (kv ? kv4_v_byte<D>(r, c) : kv4_k_byte<D>(r, c))) = codes;
  }
  if ((c & 3) == 0) rec[kv4_code_bytes(D) + (c >> 2) * kKv4Tokens + r] = (uint8_t)e;
}

// De-page: a tile is one pass of one block of one sequence, 1024 chunks of 8
// dims of the block's [K/V][head][token] rows.  Each workgroup scans the batch's
// block counts into LDS and walks its layer's tiles round-robin; the next tile's
// block id and output row are fetched while the current one's loads are in
// flight.  Of a block that its sequence fills in part only the tokens are
// chunks: the open blocks of 128 sequences, 28 layers of 4 heads of 128 (71 MB
// needed) take 22.8 us, 26.4 with a thread per token of every block.  Bound by
// the 16-bit rows written: 128 sequences of 400 tokens, one layer (131 MB) 24.3
// us, 5.4 TB/s.
constexpr int kGather4Threads = 256;
constexpr int kGather4MaxBatch = 1024;    // sequences per launch (LDS scan)
constexpr int kGather4PerThread = 4;      // chunks of a thread in a tile
constexpr int kGather4WorkgroupsPerCu = 16;  // (8: 25.1 us for 24.3 and 41.7 for 36.5 of
                                             // 256 x 8 tokens, 28 layers; 32: 25.3 and 40.1)

struct Gather4Args {
  const uint8_t* cache;
  int64_t blk_b, layer_b;
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
  int32_t batch;        // <= kGather4MaxBatch
  int32_t n_heads;
  int32_t passes;       // of a block
};

template <int DT, int D>
__global__ __launch_bounds__(kGather4Threads) void kv4_gather_kernel(Gather4Args a) {
  using E = Kv4Elem<DT>;
  __shared__ int32_t pre[kGather4MaxBatch + 1];  // first block of each sequence
  __shared__ int32_t lens[kGather4MaxBatch];
  __shared__ int32_t wsum[kGather4Threads / 64];
  constexpr int PER = kGather4MaxBatch / kGather4Threads;
  const int t = threadIdx.x, B = a.batch;
  int cnt[PER], run = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {  // loads issued together, clamped in bounds
    const int b = t * PER + k;
    const int raw = a.seq_lens[min(b, B - 1)];
    const int len = b < B ? min(max(raw, 0), a.max_seq_len) : 0;
    if (b < B) lens[b] = len;
    cnt[k] = (len + kKv4Tokens - 1) / kKv4Tokens;
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
  if (t == kGather4Threads - 1) pre[B] = excl;  // total (B may equal the capacity)
  __syncthreads();
  const uint32_t total = (uint32_t)pre[B] * a.passes;
  uint32_t g = blockIdx.x;
  if (g >= total) return;  // uniform

  auto locate = [&](uint32_t gg, int& b, int& j, int& ps) {
    const int r = (int)(gg / (uint32_t)a.passes);
    ps = (int)(gg - (uint32_t)r * a.passes);
    int lo = 0, hi = B - 1;  // the last sequence whose first block is <= r
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] <= r) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    j = r - pre[lo];
  };
  constexpr int CPR = D / 8;                    // chunks per head's row
  const int64_t row_b = (int64_t)a.n_heads * D * 2;
  const int layer = (int)blockIdx.y;
  int b, j, ps;
  locate(g, b, j, ps);
  int32_t id = a.block_tables[(int64_t)b * a.max_blocks + j];
  int64_t row0 = a.cu_seqlens[b];
  while (true) {
    const int64_t row = row0 + (int64_t)j * kKv4Tokens;
    int n_tok = min(kKv4Tokens, lens[b] - j * kKv4Tokens);
    if (row < 0 || row >= a.out_tokens || id < 0 || id >= a.n_blocks) n_tok = 0;
    else n_tok = (int)min((int64_t)n_tok, a.out_tokens - row);
    const uint8_t* blk = a.cache + (int64_t)max(id, 0) * a.blk_b + layer * a.layer_b;
    // 2^32 / n_tok rounded up: rows below 2^28 divide exactly
    const uint32_t magic = n_tok > 1 ? 0xffffffffu / (uint32_t)n_tok + 1 : 0;
    const uint32_t n_rows = 2u * a.n_heads * n_tok;
    uint32_t codes[kGather4PerThread], sb[kGather4PerThread];
    uint8_t* dst[kGather4PerThread];
#pragma unroll
    for (int k = 0; k < kGather4PerThread; ++k) {
      const int ch = (ps * kGather4PerThread + k) * kGather4Threads + t;
      const uint32_t c = ch % CPR, row_at = ch / CPR;
      const int side = n_tok > 1 ? __umulhi(row_at, magic) : row_at, r = row_at - side * n_tok;
      const int kv = side >= a.n_heads, head = side - kv * a.n_heads;
      dst[k] = nullptr;
      codes[k] = sb[k] = 0;
      if (row_at < n_rows) {
        const uint8_t* rec = blk + (int64_t)(head * 2 + kv) * kv4_record_bytes(D);
        if (kv && D == 64) {
          const uint8_t* p = rec + kv4_v_byte<D>(r, c);
          codes[k] = *reinterpret_cast<const uint16_t*>(p) |
                     ((uint32_t)*reinterpret_cast<const uint16_t*>(p + 8) << 16);
        } else {
          codes[k] = *reinterpret_cast<const uint32_t*>(
              rec + (kv ? kv4_v_byte<D>(r, c) : kv4_k_byte<D>(r, c)));
        }
        sb[k] = rec[kv4_code_bytes(D) + (c >> 2) * kKv4Tokens + r];
        dst[k] = (kv ? a.out_v : a.out_k) + layer * a.out_layer_b + (row + r) * row_b +
                 ((int64_t)head * D + 8 * c) * 2;
      }
    }
    const uint32_t gn = g + gridDim.x;
    const bool more = gn < total;
    int nb, nj, nps;
    locate(more ? gn : g, nb, nj, nps);
    const int32_t nid = a.block_tables[(int64_t)nb * a.max_blocks + nj];
    const int64_t nrow0 = a.cu_seqlens[nb];
#pragma unroll
    for (int k = 0; k < kGather4PerThread; ++k) {
      const float s = kv4_scale(sb[k]);
      const u32x4 v = {E::template dq<0>(codes[k], s), E::template dq<1>(codes[k], s),
                       E::template dq<2>(codes[k], s), E::template dq<3>(codes[k], s)};
      if (dst[k]) __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(dst[k]));
    }
    if (!more) break;
    g = gn;
    b = nb;
    j = nj;
    ps = nps;
    id = nid;
    row0 = nrow0;
  }
}

bool head_dim_ok(int32_t d) { return d == 64 || d == 128 || d == 256; }
bool dtype_ok(int32_t t) { return t == AEGKV_DTYPE_BF16 || t == AEGKV_DTYPE_FP16; }

template <int DT>
void launch_append(const Append4Args& a, int32_t head_dim, uint32_t grid, hipStream_t st) {
  const dim3 g(grid), t(kAppend4Threads);
  if (head_dim == 64) hipLaunchKernelGGL((kv4_append_kernel<DT, 64>), g, t, 0, st, a);
  else if (head_dim == 128) hipLaunchKernelGGL((kv4_append_kernel<DT, 128>), g, t, 0, st, a);
  else hipLaunchKernelGGL((kv4_append_kernel<DT, 256>), g, t, 0, st, a);
}
template <int DT>
void launch_gather(const Gather4Args& a, int32_t head_dim, dim3 g, hipStream_t st) {
  const dim3 t(kGather4Threads);
  if (head_dim == 64) hipLaunchKernelGGL((kv4_gather_kernel<DT, 64>), g, t, 0, st, a);
  else if (head_dim == 128) hipLaunchKernelGGL((kv4_gather_kernel<DT, 128>), g, t, 0, st, a);
  else hipLaunchKernelGGL((kv4_gather_kernel<DT, 256>), g, t, 0, st, a);
}

}  // namespace
}  // namespace aegkv

using namespace aegkv;

extern "C" {

int64_t aegkv_kv4_block_bytes(int32_t n_kv_heads, int32_t head_dim) {
  if (n_kv_heads <= 0) return AEGKV_ERR_INVALID_ARG;
  if (!head_dim_ok(head_dim)) return AEGKV_ERR_UNSUPPORTED;
  return 2 * (int64_t)n_kv_heads * kv4_record_bytes(head_dim);
}

int aegkv_kv4_append(const void* key, const void* value, int64_t key_token_stride,
                     int64_t value_token_stride, int64_t key_layer_stride,
                     int64_t value_layer_stride, const int64_t* slot_mapping, int64_t n_tokens,
                     void* cache, int64_t cache_block_stride, int64_t cache_layer_stride,
                     int64_t n_blocks, int32_t n_layers, int32_t n_kv_heads, int32_t head_dim,
                     int32_t dtype, aegkv_stream_t stream) {
  if (n_tokens < 0 || n_layers <= 0 || n_kv_heads <= 0 || head_dim <= 0 || n_blocks < 0)
    return AEGKV_ERR_INVALID_ARG;
  if (!head_dim_ok(head_dim) || !dtype_ok(dtype)) return AEGKV_ERR_UNSUPPORTED;
  if (n_tokens == 0 || n_blocks == 0) return AEGKV_OK;
  if (!key || !value || !slot_mapping || !cache) return AEGKV_ERR_INVALID_ARG;
  if (!aligned16(key) || !aligned16(value) || !aligned16(cache) || key_token_stride % 8 ||
      value_token_stride % 8 || key_layer_stride % 8 || value_layer_stride % 8 ||
      cache_block_stride % 16 || cache_layer_stride % 16)
    return AEGKV_ERR_MISALIGNED;
  // threads of the launch, counted in 128 bits so that no product wraps
  const unsigned __int128 total = (unsigned __int128)(uint64_t)n_layers * 2 * (uint64_t)n_kv_heads *
                                  (uint64_t)n_tokens * (uint64_t)(head_dim / 8);
  if (total >= ((unsigned __int128)1 << 32) - kAppend4Threads) return AEGKV_ERR_UNSUPPORTED;
  Append4Args a;
  a.key = static_cast<const uint8_t*>(key);
  a.value = static_cast<const uint8_t*>(value);
  a.key_tok_b = key_token_stride * 2;
  a.val_tok_b = value_token_stride * 2;
  a.key_layer_b = key_layer_stride * 2;
  a.val_layer_b = value_layer_stride * 2;
  a.slots = slot_mapping;
  a.cache = static_cast<uint8_t*>(cache);
  a.blk_b = cache_block_stride;
  a.layer_b = cache_layer_stride;
  a.n_slots = n_blocks * kKv4Tokens;
  a.n_tokens = (uint32_t)n_tokens;
  a.n_heads = (uint32_t)n_kv_heads;
  a.total = (uint32_t)total;
  const uint32_t grid = (a.total + kAppend4Threads - 1) / kAppend4Threads;
  if (dtype == AEGKV_DTYPE_BF16) launch_append<AEGKV_DTYPE_BF16>(a, head_dim, grid, (hipStream_t)stream);
  else launch_append<AEGKV_DTYPE_FP16>(a, head_dim, grid, (hipStream_t)stream);
  AEGKV_HIP_TRY(hipGetLastError());
  return AEGKV_OK;
}

int aegkv_kv4_gather_tokens(const void* cache, int64_t cache_block_stride,
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
  if (!head_dim_ok(head_dim) || !dtype_ok(dtype)) return AEGKV_ERR_UNSUPPORTED;
  if (batch == 0 || max_seq_len == 0 || out_tokens == 0) return AEGKV_OK;
  if (!cache || !block_tables || !seq_lens || !cu_seqlens || !out_key || !out_value)
    return AEGKV_ERR_INVALID_ARG;
  if (!aligned16(cache) || !aligned16(out_key) || !aligned16(out_value) ||
      cache_block_stride % 16 || cache_layer_stride % 16 || out_layer_stride % 8)
    return AEGKV_ERR_MISALIGNED;
  const int64_t blocks_needed = ((int64_t)max_seq_len + kKv4Tokens - 1) / kKv4Tokens;
  if (blocks_needed > max_blocks) return AEGKV_ERR_INVALID_ARG;
  const int64_t chunks = 2 * (int64_t)n_kv_heads * kKv4Tokens * (head_dim / 8);
  const int64_t per_tile = kGather4Threads * kGather4PerThread;
  const int64_t passes = (chunks + per_tile - 1) / per_tile;
  if (n_layers > 65535 || chunks > INT32_MAX - per_tile || blocks_needed * kGather4MaxBatch * passes > INT32_MAX)
    return AEGKV_ERR_UNSUPPORTED;
  DeviceState* ds = nullptr;
  int rc = current_device_state(&ds);
  if (rc) return rc;
  Gather4Args a;
  a.cache = static_cast<const uint8_t*>(cache);
  a.blk_b = cache_block_stride;
  a.layer_b = cache_layer_stride;
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
      1, ((int64_t)std::max(ds->num_cu, 1) * kGather4WorkgroupsPerCu + n_layers - 1) / n_layers);
  for (int32_t b0 = 0; b0 < batch; b0 += kGather4MaxBatch) {
    const int32_t nb = std::min(kGather4MaxBatch, batch - b0);
    a.batch = nb;
    a.block_tables = block_tables + (int64_t)b0 * max_blocks;
    a.seq_lens = seq_lens + b0;
    a.cu_seqlens = cu_seqlens + b0;
    const int64_t tiles_max = blocks_needed * nb * passes;  // bound of a layer's tiles
    const dim3 grid((uint32_t)std::min(tiles_max, max_grid), (uint32_t)n_layers);
    if (dtype == AEGKV_DTYPE_BF16) launch_gather<AEGKV_DTYPE_BF16>(a, head_dim, grid, (hipStream_t)stream);
    else launch_gather<AEGKV_DTYPE_FP16>(a, head_dim, grid, (hipStream_t)stream);
    AEGKV_HIP_TRY(hipGetLastError());
  }
  return AEGKV_OK;
}

}  // extern "C"
