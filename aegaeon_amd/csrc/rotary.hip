// Appending K/V rows to the paged 16-bit cache with the position rotation applied
// on the way, and the queries rotated beside them (rotary_rows.h): one launch per
// layer where the rotation of queries and keys and the append would be three.
//
// A wave takes up to 4 x (64 / (D / 8)) heads of one token's queries, keys or
// values, every load of a task in flight at once, the position's angles loaded
// once for the task's heads.  Bound by memory, each row read and written once: 4057
// tokens of 32 query and 4 kv heads of 128 in fp16, half of each row turned, the turned
// keys kept, 88 MB in 15.6 us (5.6 TB/s; a copy of 1 GiB reaches 5.0).  A decode step's
// layer (128 tokens, 28 and 4 heads) 4.3 us, about what any launch takes.
#include <algorithm>

#include "aegkv_internal.h"
#include "rotary_rows.h"

namespace aegkv {
namespace {

constexpr int kRotaryThreads = 256;

struct RotaryArgs {
  HeadRows q, k, v;
  RotaryTable r;
  const int64_t* slots;
  uint8_t* kc;
  uint8_t* vc;
  int64_t blk_b;        // byte stride of the caches' blocks
  int64_t n_slots;      // n_blocks * block_size
  int32_t block_size;
  int32_t chunks;       // head_dim / 8
  int32_t q_tasks, kv_tasks;  // of a token: q_tasks + 2 kv_tasks
  uint32_t n_tasks;
};

template <int DT, bool INTER>
__global__ __launch_bounds__(kRotaryThreads) void rotary_append_kernel(RotaryArgs a) {
  const uint32_t id = __builtin_amdgcn_readfirstlane(
      blockIdx.x * (kRotaryThreads / 64) + (threadIdx.x >> 6));
  if (id >= a.n_tasks) return;
  const uint32_t per = a.q_tasks + 2 * a.kv_tasks;
  const int tok = (int)(id / per);
  int part = (int)(id - (uint32_t)tok * per);
  if (part < a.q_tasks) {
    turn_heads<DT, INTER>(a.q, a.r, true, tok, part, a.chunks, nullptr);
    return;
  }
  part -= a.q_tasks;
  const bool value = part >= a.kv_tasks;
  if (value) part -= a.kv_tasks;
  const int64_t s = a.slots[tok];
  uint8_t* cache = nullptr;
  if (s >= 0 && s < a.n_slots) {
    const int64_t blk = s / a.block_size;
    cache = (value ? a.vc : a.kc) + blk * a.blk_b +
            (s - blk * a.block_size) * ((int64_t)a.k.n_heads * a.chunks * 16);
  }
  if (value) {
    if (cache) turn_heads<DT, INTER>(a.v, a.r, false, tok, part, a.chunks, cache);
  } else if (cache || a.k.dst) {
    turn_heads<DT, INTER>(a.k, a.r, true, tok, part, a.chunks, cache);
  }
}

}  // namespace
}  // namespace aegkv

using namespace aegkv;

extern "C" {

int aegkv_rotary_append(const void* query, int64_t query_token_stride, void* out_query,
                        int64_t out_query_token_stride, int32_t n_q_heads, const void* key,
                        int64_t key_token_stride, const void* value, int64_t value_token_stride,
                        void* out_key, int64_t out_key_token_stride, int32_t n_kv_heads,
                        int32_t head_dim, const int64_t* slot_mapping, const int64_t* positions,
                        int64_t n_tokens, const float* table, int64_t max_positions,
                        int32_t rotary_dim, int32_t interleaved, void* key_cache,
                        void* value_cache, int64_t cache_block_stride, int64_t n_blocks,
                        int32_t block_size, int32_t dtype, aegkv_stream_t stream) {
  if (n_tokens < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || n_blocks < 0 ||
      block_size <= 0)
    return AEGKV_ERR_INVALID_ARG;
  RotaryArgs a;
  a.r = RotaryTable{table, positions, max_positions, rotary_dim};
  const int rc = check_rotary(a.r, head_dim);
  if (rc) return rc;
  if (head_dim % 8 || head_dim > 512 || n_q_heads > 65535 || n_kv_heads > 65535 ||
      (dtype != AEGKV_DTYPE_BF16 && dtype != AEGKV_DTYPE_FP16))
    return AEGKV_ERR_UNSUPPORTED;
  if (n_tokens == 0) return AEGKV_OK;
  if (!query || !out_query || !key || !value || !slot_mapping || !positions || !table ||
      (n_blocks > 0 && (!key_cache || !value_cache)))
    return AEGKV_ERR_INVALID_ARG;
  if (max_positions == 0) return AEGKV_ERR_INVALID_ARG;
  if (!aligned16(query) || !aligned16(out_query) || !aligned16(key) || !aligned16(value) ||
      !aligned16(out_key) || !aligned16(table) || !aligned16(key_cache) ||
      !aligned16(value_cache) || query_token_stride % 8 || out_query_token_stride % 8 ||
      key_token_stride % 8 || value_token_stride % 8 || out_key_token_stride % 8 ||
      cache_block_stride % 8)
    return AEGKV_ERR_MISALIGNED;
  a.q = HeadRows{static_cast<const uint8_t*>(query), static_cast<uint8_t*>(out_query),
                 query_token_stride * 2, out_query_token_stride * 2, n_q_heads};
  a.k = HeadRows{static_cast<const uint8_t*>(key), static_cast<uint8_t*>(out_key),
                 key_token_stride * 2, out_key_token_stride * 2, n_kv_heads};
  a.v = HeadRows{static_cast<const uint8_t*>(value), nullptr, value_token_stride * 2, 0,
                 n_kv_heads};
  a.slots = slot_mapping;
  a.kc = static_cast<uint8_t*>(key_cache);
  a.vc = static_cast<uint8_t*>(value_cache);
  a.blk_b = cache_block_stride * 2;
  a.n_slots = n_blocks > INT64_MAX / block_size ? INT64_MAX : n_blocks * block_size;
  a.block_size = block_size;
  a.chunks = head_dim / 8;
  a.q_tasks = head_tasks(n_q_heads, a.chunks);
  a.kv_tasks = head_tasks(n_kv_heads, a.chunks);
  // wave tasks, counted in 128 bits so that no product wraps
  const unsigned __int128 tasks = (unsigned __int128)(uint64_t)n_tokens *
                                  ((uint64_t)a.q_tasks + 2 * (uint64_t)a.kv_tasks);
  if (tasks > INT32_MAX) return AEGKV_ERR_UNSUPPORTED;
  a.n_tasks = (uint32_t)tasks;
  constexpr uint32_t kWavesOf = kRotaryThreads / 64;
  const dim3 grid((a.n_tasks + kWavesOf - 1) / kWavesOf);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kRotaryThreads), 0, (hipStream_t)stream, a);
  };
  if (dtype == AEGKV_DTYPE_BF16)
    interleaved ? launch(rotary_append_kernel<AEGKV_DTYPE_BF16, true>)
                : launch(rotary_append_kernel<AEGKV_DTYPE_BF16, false>);
  else
    interleaved ? launch(rotary_append_kernel<AEGKV_DTYPE_FP16, true>)
                : launch(rotary_append_kernel<AEGKV_DTYPE_FP16, false>);
  AEGKV_HIP_TRY(hipGetLastError());
  return AEGKV_OK;
}

}  // extern "C"
