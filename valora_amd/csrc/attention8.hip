// Attention over the paged cache of 8-bit codes: csrc/attention_core.h, with the codes turned into 16-bit values on their way to the
// matrix instructions (csrc/codes8.h: exact, so a row's result is that of the 16-bit kernels over the values that are read back).
#include "attention_core.h"

namespace mlora {

namespace {

// Weights are summed by two kernels.  Where the scores are there, a thread sums a token's, as over 16 bits; where they are not, 64 tokens are a
// workgroup's, whose waves share out heads, and their rows where heads are few, and add up their parts in order.  (A wave alone with 64
// tokens leaves most of the device idle where few are cached.  us in all, alone / shared: a prompt of 2048, 32 heads of 128, 3070 / 633;
// 500 tokens over 11500 among 31 decoding requests, 8 key heads, 900 / 286.  64 decoding requests of 1000 to 4100: 99 either way.)
__global__ __launch_bounds__(WEIGHT_TOKENS) void attend_scores_kernel(AttnArgs a) {
  __shared__ int found;
  const int total = a.plan[AH_BLOCKS];
  for (int block = blockIdx.x; block < total; block += gridDim.x) {
    const int b = request_of(a, block, &found);
    const int32_t *record = a.plan + a.off_requests + (int64_t)b * AT_REC;
    const Weighed rq(a, record);
    if (rq.has_scores(a)) sum_scores(a, record, rq, b, block);
  }
}

constexpr int SHARED_WAVES = 8;
template <typename T, int D>
__global__ __launch_bounds__(SHARED_WAVES * 64) void attend_weights_codes_kernel(AttnArgs a) {
  constexpr int CH = D / 32, PARTS = WEIGHT_TOKENS / 64;
  using vec8 = typename Traits<T>::vec8;
  __shared__ int found;
  __shared__ float parts[SHARED_WAVES][64];
  const int lane = threadIdx.x & 63, wave = (int)uniform(threadIdx.x >> 6), lrow = lane & 15, kg = lane >> 4;
  const int total = a.plan[AH_BLOCKS] * PARTS;
  for (int item = blockIdx.x; item < total; item += gridDim.x) {
    const int b = request_of(a, item / PARTS, &found);
    const Weighed rq(a, a.plan + a.off_requests + (int64_t)b * AT_REC);
    if (rq.has_scores(a)) continue;
    const int base = rq.begin + (item - rq.first_block * PARTS) * 64;
    if (base >= rq.kv) continue;
    const Seeing rows(a, rq, base);
    const int32_t *table = a.table + (int64_t)b * a.table_stride;
    const char *kc[4], *ke[4];                                  // this lane's token of each 16: where its codes and powers are
    uint64_t bad = 0;                                           // tokens whose page is none of the pool
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      const int j = min(base + tt * 16 + lrow, rq.kv - 1);
      const int32_t page = table[j >> a.page_shift];
      const bool none = (uint32_t)page >= (uint32_t)a.n_pages;
      const int64_t at = none ? 0 : page, off = j & ((1 << a.page_shift) - 1);
      kc[tt] = reinterpret_cast<const char *>(a.k) + at * a.k_stride + off * D + kg * 8;
      ke[tt] = reinterpret_cast<const char *>(a.e) + at * a.e_stride + off * 2;
      bad |= (uint64_t)(__ballot(none) & 0xffffu) << tt * 16;
    }
    // heads, and where they are fewer than waves runs of their rows
    const int runs = (SHARED_WAVES + a.kv_heads - 1) / a.kv_heads;
    const int each = ((rows.hi - rows.lo + 15) / 16 + runs - 1) / runs * 16;
    float w[4][4] = {};
    for (int pair = wave; pair < a.kv_heads * runs; pair += SHARED_WAVES) {
      const int head = pair / runs, first = rows.lo + (pair - head * runs) * each, last_row = min(first + each, rows.hi);
      if (first >= last_row) continue;
      vec8 kf[4][CH];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const int64_t slots = (int64_t)head << a.page_shift;
        const float power = k_power(*reinterpret_cast<const uint8_t *>(ke[tt] + slots * 2));
#pragma unroll
        for (int i = 0; i < CH; ++i) kf[tt][i] = values_of<T>(*reinterpret_cast<const u32x2 *>(kc[tt] + slots * D + i * 32), power);
      }
      sum_rows<T, D>(a, rq, kf, head, first, last_row, base, bad, w);
    }
    over_rows(w, [&](int token, float x) { parts[wave][token] = x; });
    __syncthreads();
    if (threadIdx.x < 64 && base + lane < rq.kv) {
      float x = 0.0f;
#pragma unroll
      for (int i = 0; i < SHARED_WAVES; ++i) x += parts[i][lane];
      a.weights[(int64_t)b * a.weights_stride + base + lane] += x;
    }
  }
}

template <typename T, int D>
int sum_weights(hipStream_t st, const AttnLayout &L, const AttnArgs &a, int64_t most) {
  hipLaunchKernelGGL(attend_scores_kernel, dim3((unsigned)(most < 1024 ? most : 1024)), dim3(WEIGHT_TOKENS), 0, st, a);
  if (int rc = check_launch("attend_scores_kernel")) return rc;
  // requests without scores: those of more rows, and all where their room is bounded and may not do
  if (L.max_shares <= 0 && L.scores < MAX_SCORES) return MLORA_OK;
  const int64_t items = most * (WEIGHT_TOKENS / 64);
  hipLaunchKernelGGL((attend_weights_codes_kernel<T, D>), dim3((unsigned)(items < 1024 ? items : 1024)), dim3(SHARED_WAVES * 64), 0, st, a);
  return check_launch("attend_weights_codes_kernel");
}

}  // namespace

}  // namespace mlora

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
