// Attention over the paged cache of 16-bit rows: csrc/attention_core.h over the pool's rows as they are.
#include "attention_core.h"

namespace mlora {

namespace {

// Weights without scores: a wave owns 64 cached tokens and goes over all key heads and rows (csrc/attention8.hip shares them out).
constexpr int WEIGHT_WAVES = WEIGHT_TOKENS / 64;

template <typename T, int D>
__global__ __launch_bounds__(WEIGHT_WAVES * 64, 2) void attend_weights_kernel(AttnArgs a) {
  constexpr int CH = D / 32;
  using vec8 = typename Traits<T>::vec8;
  __shared__ int found;
  const int lane = threadIdx.x & 63, wave = (int)uniform(threadIdx.x >> 6), lrow = lane & 15, kg = lane >> 4;
  const int total = a.plan[AH_BLOCKS];
  for (int item = blockIdx.x; item < total; item += gridDim.x) {
    const int b = request_of(a, item, &found);
    const int32_t *record = a.plan + a.off_requests + (int64_t)b * AT_REC;
    const Weighed rq(a, record);
    if (rq.has_scores(a)) {
      sum_scores(a, record, rq, b, item);
      continue;
    }
    const int base = rq.begin + (item - rq.first_block) * WEIGHT_TOKENS + wave * 64;
    if (base >= rq.kv) continue;
    const Seeing rows(a, rq, base);
    const int32_t *table = a.table + (int64_t)b * a.table_stride;
    int64_t at[4];                                              // this lane's token of each 16: pool row
    uint64_t bad = 0;                                           // tokens whose page is none of the pool
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      const int j = min(base + tt * 16 + lrow, rq.kv - 1);
      const int32_t page = table[j >> a.page_shift];
      const bool none = (uint32_t)page >= (uint32_t)a.n_pages;
      at[tt] = none ? 0 : ((int64_t)page << a.page_shift) + (j & ((1 << a.page_shift) - 1));
      bad |= (uint64_t)(__ballot(none) & 0xffffu) << tt * 16;
    }
    float w[4][4] = {};
    for (int head = 0; head < a.kv_heads; ++head) {
      const char *kp = reinterpret_cast<const char *>(a.k) + head * D * 2 + kg * 16;
      vec8 kf[4][CH];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < CH; ++i) kf[tt][i] = as<vec8>(*reinterpret_cast<const u32x4 *>(kp + at[tt] * a.k_stride + i * 64));
      sum_rows<T, D>(a, rq, kf, head, rows.lo, rows.hi, base, bad, w);
    }
    over_rows(w, [&](int token, float x) {
      if (base + token < rq.kv) a.weights[(int64_t)b * a.weights_stride + base + token] += x;
    });
  }
}

template <typename T, int D>
int sum_weights(hipStream_t st, const AttnLayout &, const AttnArgs &a, int64_t most) {
  hipLaunchKernelGGL((attend_weights_kernel<T, D>), dim3((unsigned)(most < 1024 ? most : 1024)), dim3(WEIGHT_WAVES * 64), 0, st, a);
  return check_launch("attend_weights_kernel");
}

}  // namespace

}  // namespace mlora

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
