// Attention over the paged cache of 16-bit rows: csrc/attention_core.h over the pool's rows as they are.
#include "attention_core.h"

using namespace mlora;

extern "C" int mlora_paged_attention(void *stream, const mlora_attention_plan *plan, void *workspace, size_t workspace_bytes,
                                     void *out, int64_t out_stride, const void *q, int64_t q_stride, const void *key_buffer,
                                     int64_t key_stride, const void *value_buffer, int64_t value_stride, int64_t n_rows,
                                     const int32_t *table, int64_t table_stride, int64_t table_width, float scale, float *weights,
                                     int64_t weights_stride, mlora_dtype dtype) {
  const char *who = "paged_attention";
  const auto pool = [&](AttnArgs &a, int64_t &n_pages, bool &there) {
    const int64_t kw = (int64_t)plan->kv_heads * plan->head_dim;
    if (key_stride < kw || value_stride < kw) return fail(MLORA_ERR_INVALID, "%s: a row of q, out or the pool is shorter than its heads", who);
    if ((key_stride | value_stride) & 7 || ((reinterpret_cast<uintptr_t>(key_buffer) | reinterpret_cast<uintptr_t>(value_buffer)) & 15))
      return fail(MLORA_ERR_INVALID, "%s: rows of q, out and the pool must be multiples of 16 bytes and 16-byte aligned", who);
    if (key_stride > 0x3fffffff || value_stride > 0x3fffffff) return fail(MLORA_ERR_NO_KERNEL, "%s: pool rows above 2 GB", who);
    if (n_rows < 0 || n_rows > 0x7fffffff) return fail(MLORA_ERR_NO_KERNEL, "%s: more than 2^31 - 1 pool rows", who);
    a.k = static_cast<const uint16_t *>(key_buffer);
    a.v = static_cast<const uint16_t *>(value_buffer);
    a.k_stride = (uint32_t)key_stride * 2;
    a.v_stride = (uint32_t)value_stride * 2;
    n_pages = n_rows / plan->page_size;
    there = key_buffer && value_buffer;
    return (int)MLORA_OK;
  };
  return attention_call<false>(who, stream, plan, workspace, workspace_bytes, out, out_stride, q, q_stride, table, table_stride, table_width,
                               scale, weights, weights_stride, dtype, pool);
}
