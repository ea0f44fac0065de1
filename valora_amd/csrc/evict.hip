// Eviction from the paged cache: a request that holds more than `budget` pages keeps its first `sinks`, its last `recent` and,
// of those between, the pages whose tokens got the most attention (the sum of their accumulated weights; ties to the page that
// comes first), in their order.  Pages stay where they are: what changes is the table, the weights that go with it and the
// length, and the pages given up are listed.
//
// One workgroup per request.  A page's weight becomes a 32-bit key that orders as the weight does; the key of the last page that
// stays is found digit by digit (four histograms of 256), and one pass in page order writes everything out: a wave owns a
// run of pages, so that their places follow from ballots and one sum over the waves.  Keys stay in LDS (read again from
// the weights where a request holds more than LDS does).  Bound by the latency of these steps for few requests, by the bytes
// of the three output arrays for many.
#include "kernel_common.h"

namespace mlora {

namespace {

constexpr int EV_THREADS = 1024, EV_WAVES = EV_THREADS / 64;
constexpr int EV_MAX_KEYS = 36864;     // 144 of 160 KB

struct EvictArgs {
  const int32_t *table, *len;
  const float *weights;
  int64_t table_stride, weights_stride;
  int32_t *new_table, *new_len, *freed;
  float *new_weights;
  int width, page_shift, budget, recent, sinks, lds_keys;
};

// Orders as the value does; what is not a number comes first, both zeros are one value
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0;
  const uint32_t b = as<uint32_t>(x + 0.0f);     // (-0 + 0 is +0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ uint32_t page_key(const float *w, int page, int shift) {
  if (shift == 0) return order_key(w[page]);
  double sum = 0;      // 64 bits: the order of up to 256 terms does not show in the 32-bit sum
  for (int i = 0; i < 1 << shift; ++i) sum += (double)w[((int64_t)page << shift) + i];
  return order_key((float)sum);
}

__global__ __launch_bounds__(EV_THREADS) void evict_kernel(EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t hist[256];
  __shared__ uint32_t found[2];                  // digit, pages still to take
  __shared__ int sure_w[EV_WAVES], ties_w[EV_WAVES];
  const int req = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int shift = a.page_shift, ps = 1 << shift;
  const int32_t *table = a.table + (int64_t)req * a.table_stride;
  const float *w = a.weights + (int64_t)req * a.weights_stride;
  int32_t *new_table = a.new_table + (int64_t)req * a.width, *freed = a.freed + (int64_t)req * a.width;
  float *new_w = a.new_weights + ((int64_t)req * a.width << shift);
  const int64_t cap = (int64_t)a.width << shift;
  const int64_t raw = a.len[req];
  const int64_t len = raw < 0 ? 0 : raw > cap ? cap : raw;
  const int pages = (int)((len + ps - 1) >> shift);
  const bool over = pages > a.budget;
  const int first = a.sinks, last = pages - a.recent;          // the pages that compete: [first, last)
  const int need = a.budget - a.sinks - a.recent;              // how many of them stay (host: >= 0)
  const int kept = over ? a.budget : pages;

  uint32_t prefix = 0;
  int take = 0;                                                // of the pages with the last key, how many stay
  auto key_of = [&](int i) { return a.lds_keys ? keys[i - first] : page_key(w, i, shift); };
  if (over) {
    if (a.lds_keys)
      for (int i = first + tid; i < last; i += EV_THREADS) keys[i - first] = page_key(w, i, shift);
    uint32_t want = (uint32_t)need;
    for (int digit = 24; digit >= 0 && need > 0; digit -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = first + tid; i < last; i += EV_THREADS) {
        const uint32_t k = key_of(i);
        if (digit == 24 || (k >> (digit + 8)) == (prefix >> (digit + 8))) atomicAdd(&hist[(k >> digit) & 255], 1u);
      }
      __syncthreads();
      if (wave == 0) {
        // the digit d with sum(hist above d) < want <= sum(hist from d on): lane l holds bins 255 - 4 l downwards
        uint32_t h[4], mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += h[i] = hist[255 - 4 * lane - i];
        uint32_t above = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const uint32_t up = __shfl_up(above, d);
          if (lane >= d) above += up;
        }
        above -= mine;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (above < want && want <= above + h[i]) {
            found[0] = 255 - 4 * lane - i;
            found[1] = want - above;
          }
          above += h[i];
        }
      }
      __syncthreads();
      prefix |= found[0] << digit;
      want = found[1];
    }
    take = need > 0 ? (int)want : 0;
    if (need == 0) prefix = 0xffffffffu;                       // (no key is above it, and no tie is taken)
  }
  __syncthreads();

  // page order: wave w owns pages [w * run, (w + 1) * run)
  const int run = ((pages + EV_WAVES - 1) / EV_WAVES + 63) & ~63;
  const int lo = wave * run, hi = min(lo + run, pages);
  int sure = 0, ties = 0;
  if (over)
    for (int i0 = lo; i0 < hi; i0 += 64) {
      const int i = i0 + lane;
      const bool compete = i < hi && i >= first && i < last;
      const uint32_t k = compete ? key_of(i) : 0;
      sure += __popcll(__ballot(i < hi && (!compete || k > prefix)));
      ties += __popcll(__ballot(compete && k == prefix));
    }
  if (lane == 0) {
    sure_w[wave] = sure;
    ties_w[wave] = ties;
  }
  __syncthreads();
  int at = 0, tied = 0;                                        // pages that stay, ties, before this wave's run
  for (int i = 0; i < wave; ++i) {
    at += sure_w[i];
    tied += ties_w[i];
  }
  at += min(tied, take);
  const uint64_t below = (1ull << lane) - 1;
  for (int i0 = lo; i0 < hi; i0 += 64) {
    const int i = i0 + lane;
    bool stay = i < hi;
    int to = i;
    if (over) {
      const bool compete = i < hi && i >= first && i < last;
      const uint32_t k = compete ? key_of(i) : 0;
      const uint64_t tie = __ballot(compete && k == prefix);
      stay = i < hi && (!compete || k > prefix || (k == prefix && tied + __popcll(tie & below) < take));
      const uint64_t staying = __ballot(stay);
      to = at + __popcll(staying & below);
      at += __popcll(staying);
      tied += __popcll(tie);
    }
    if (i < hi) {
      const int32_t page = table[i];
      if (stay) new_table[to] = page;
      else freed[i - to] = page;
      if (stay)
        for (int j = 0; j < ps; ++j) {
          const int64_t t = ((int64_t)i << shift) + j;
          new_w[((int64_t)to << shift) + j] = t < len ? w[t] : 0.0f;
        }
    }
  }
  // what is behind
  for (int i = kept + tid; i < a.width; i += EV_THREADS) new_table[i] = -1;
  for (int i = pages - kept + tid; i < a.width; i += EV_THREADS) freed[i] = -1;
  for (int64_t i = ((int64_t)kept << shift) + tid; i < cap; i += EV_THREADS) new_w[i] = 0.0f;
  if (tid == 0) a.new_len[req] = (int32_t)(len - ((int64_t)(pages - kept) << shift));
}

}  // namespace

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_cache_evict(void *stream, const int32_t *table, int64_t table_stride, const int32_t *kv_len,
                                 const float *weights, int64_t weights_stride, int64_t n_req, int64_t width, int32_t page_size,
                                 int64_t budget, int64_t recent, int64_t sinks, int32_t *new_table, int32_t *new_kv_len,
                                 float *new_weights, int32_t *freed) {
  if (n_req < 0 || width < 0 || n_req > 0x7fffffff) return fail(MLORA_ERR_INVALID, "cache_evict: negative size");
  int shift = 0;
  while (shift < 8 && (1 << shift) < page_size) ++shift;
  if (page_size < 1 || (1 << shift) != page_size)
    return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. cache_evict: page_size=%d (a power of two up to 256)", page_size);
  if (width << shift > 0x7fffffff) return fail(MLORA_ERR_NO_KERNEL, "cache_evict: more than 2^31 - 1 tokens a request");
  if (recent < 1 || sinks < 0 || recent > 0x3fffffff || sinks > 0x3fffffff || budget > 0x7fffffff || budget < recent + sinks)
    return fail(MLORA_ERR_INVALID, "cache_evict: budget=%lld must hold recent=%lld (at least 1) and sinks=%lld pages",
                (long long)budget, (long long)recent, (long long)sinks);
  if (table_stride < width || weights_stride < width << shift)
    return fail(MLORA_ERR_INVALID, "cache_evict: a row of table or weights is shorter than %lld pages", (long long)width);
  if (n_req == 0) return MLORA_OK;
  if (!kv_len || !new_kv_len || (width > 0 && (!table || !weights || !new_table || !new_weights || !freed)))
    return fail(MLORA_ERR_INVALID, "cache_evict: null pointer");
  const bool lds = width <= EV_MAX_KEYS;
  EvictArgs a{table, kv_len, weights, table_stride, weights_stride, new_table, new_kv_len, freed, new_weights,
              (int)width, shift, (int)budget, (int)recent, (int)sinks, lds};
  hipLaunchKernelGGL(evict_kernel, dim3((unsigned)n_req), dim3(EV_THREADS), lds ? (size_t)width * 4 : 0, (hipStream_t)stream, a);
  return check_launch("evict_kernel");
}
