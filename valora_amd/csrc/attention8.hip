// Attention over the paged cache of 8-bit codes: csrc/attention_core.h, with the codes turned into 16-bit values on their way to the
// matrix instructions (csrc/codes8.h: exact, so a row's result is that of the 16-bit kernels over the values that are read back).
#include "attention_core.h"

using namespace mlora;

extern "C" int mlora_paged_attention_codes(void *stream, const mlora_attention_plan *plan, void *workspace, size_t workspace_bytes,
                                      void *out, int64_t out_stride, const void *q, int64_t q_stride, const mlora_cache8 *cache,
                                      const int32_t *table, int64_t table_stride, int64_t table_width, float scale, float *weights,
                                      int64_t weights_stride, mlora_dtype dtype) {
  const char *who = "paged_attention8";
  const auto pool = [&](AttnArgs &a, int64_t &n_pages, bool &there) {
    if (int rc = check_cache8(cache, plan->kv_heads, plan->head_dim, plan->page_size, who)) return rc;
    a.k = static_cast<const uint16_t *>(cache->key_codes);
    a.v = static_cast<const uint16_t *>(cache->value_codes);
    a.e = static_cast<const uint8_t *>(cache->powers);
    a.k_stride = (uint32_t)cache->key_stride;
    a.v_stride = (uint32_t)cache->value_stride;
    a.e_stride = (uint32_t)cache->powers_stride;
    n_pages = cache->n_pages;
    there = cache->key_codes && cache->value_codes && cache->powers;
    return (int)MLORA_OK;
  };
  return attention_call<true>(who, stream, plan, workspace, workspace_bytes, out, out_stride, q, q_stride, table, table_stride, table_width,
                              scale, weights, weights_stride, dtype, pool);
}
