// Eviction from the paged cache: a request that holds more than `budget` pages keeps its first `sinks`, its last `recent` and,
// of those between, the pages whose tokens got the most attention (the sum of their accumulated weights; ties to the page that
// comes first), in their order.  Pages stay where they are: what changes is the table, the weights that go with it and the
// length, and the pages given up are listed.
//
// One workgroup per request.  A page's weight becomes a 32-bit key that orders as the weight does; the key of the last page that
// stays is found digit by digit (four histograms of 256), and one pass in page order writes everything out: a wave owns a
// run of pages, so that their places follow from ballots and one sum over the waves.  Up to 16384 pages a request are held in
// registers from the first load to the last store.  Bound by the latency of these steps for few requests, by the bytes of the
// three output arrays for many (8 requests of 900 to 1100 tokens 8 us; 256 of 300 to 16000, weights of 64 KB a request, 23: the
// workgroup with the longest request, four histograms and their scans, 2.4 TB/s over all).
#include "kernel_common.h"

namespace mlora {

namespace {

constexpr int EV_THREADS = 1024, EV_WAVES = EV_THREADS / 64;
constexpr int EV_MAX_KEYS = 32768;     // 128 KB beside the histograms
constexpr int EV_HELD = 16;            // pages a thread holds

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

// Histograms are kept EV_COPIES times, side by side: additions to one word wait for each other, and weights may well be alike (many
// are 0).  All 16000 pages of a request alike: 70 us with one copy, 21 with eight.
constexpr int EV_COPIES = 8;
static_assert(EV_MAX_KEYS * 4 + 2 * 256 * EV_COPIES * 4 + EV_WAVES * 8 + 64 <= 160 * 1024, "what a workgroup may have of LDS");

// n words of `value`, by all threads, 16 bytes at a time where they are aligned
__device__ __forceinline__ void fill(int32_t *p, int64_t n, int32_t value, int tid) {
  const int64_t head = min<int64_t>(n, (4 - (int64_t)((reinterpret_cast<uintptr_t>(p) >> 2) & 3)) & 3);
  if (tid < head) p[tid] = value;
  const int64_t quads = (n - head) / 4;
  typedef __attribute__((ext_vector_type(4))) int32_t i32x4;
  for (int64_t i = tid; i < quads; i += EV_THREADS) *reinterpret_cast<i32x4 *>(p + head + 4 * i) = i32x4{value, value, value, value};
  const int64_t done = head + 4 * quads;
  if (tid < n - done) p[done + tid] = value;
}

// HELD: the request's pages are held in registers, up to EV_HELD by a thread; otherwise keys stay in LDS where they fit, or are
// read again from the weights.
template <bool HELD>
__global__ __launch_bounds__(EV_THREADS) void evict_kernel(EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ __align__(16) uint32_t hist[2][256 * EV_COPIES];
  __shared__ uint32_t found[2];                  // digit, pages still to take
  __shared__ int sure_w[EV_WAVES], ties_w[EV_WAVES];
  const int req = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int shift = a.page_shift, ps = 1 << shift;
  const int32_t *__restrict__ table = a.table + (int64_t)req * a.table_stride;
  const float *__restrict__ w = a.weights + (int64_t)req * a.weights_stride;
  int32_t *__restrict__ new_table = a.new_table + (int64_t)req * a.width, *__restrict__ freed = a.freed + (int64_t)req * a.width;
  float *__restrict__ new_w = a.new_weights + ((int64_t)req * a.width << shift);
  const int64_t cap = (int64_t)a.width << shift;
  const int64_t raw = a.len[req];
  const int64_t len = raw < 0 ? 0 : raw > cap ? cap : raw;
  const int pages = (int)((len + ps - 1) >> shift);
  const bool over = pages > a.budget;
  const int kept = over ? a.budget : pages;

  // wave w owns pages [w * run, (w + 1) * run), lane l every 64th of them
  const int run = ((pages + EV_WAVES - 1) / EV_WAVES + 63) & ~63;
  const int lo = wave * run, hi = min(lo + run, pages);
  // What stays in any case has the highest key, which no weight has, and what is no page the lowest, behind all that are: so the
  // pages that stay are those of the `budget` highest keys.
  auto key_of = [&](int i, uint32_t k) { return i >= hi ? 0u : i < a.sinks || i >= pages - a.recent ? 0xffffffffu : k; };
  int32_t page[EV_HELD];
  float weight[EV_HELD];
  uint32_t key[EV_HELD];
  if constexpr (HELD) {
#pragma unroll
    for (int n = 0; n < EV_HELD; ++n) {
      if (n * 64 >= run) break;
      const int i = max(min(lo + n * 64 + lane, pages - 1), 0);
      page[n] = table[i];
      weight[n] = shift == 0 ? w[i] : 0.0f;
    }
  }
  // what is behind the results does not wait for them
  fill(new_table + kept, a.width - kept, -1, tid);
  fill(freed + (pages - kept), a.width - (pages - kept), -1, tid);
  fill(reinterpret_cast<int32_t *>(new_w) + ((int64_t)kept << shift), cap - ((int64_t)kept << shift), 0, tid);
  if (tid == 0) a.new_len[req] = (int32_t)(len - ((int64_t)(pages - kept) << shift));

  // f(n, i, key of page i) for this lane's pages, whole waves together
  auto each = [&](auto f) {
    if constexpr (HELD) {
#pragma unroll
      for (int n = 0; n < EV_HELD; ++n) {
        if (n * 64 >= run) break;
        f(n, lo + n * 64 + lane, key[n]);
      }
    } else {
      for (int i0 = lo; i0 < lo + run; i0 += 64) {
        const int i = i0 + lane;
        f(0, i, a.lds_keys ? (i < hi ? keys[i] : 0u) : key_of(i, i < hi ? page_key(w, i, shift) : 0u));
      }
    }
  };

  uint32_t prefix = 0;
  int take = 0;                                                // of the pages with the last key, how many stay
  if (over) {
    if constexpr (HELD) {
#pragma unroll
      for (int n = 0; n < EV_HELD; ++n) {
        if (n * 64 >= run) break;
        const int i = lo + n * 64 + lane;
        key[n] = key_of(i, shift == 0 ? order_key(weight[n]) : i < hi ? page_key(w, i, shift) : 0u);
      }
    } else if (a.lds_keys) {
      for (int i = lo + lane; i < hi; i += 64) keys[i] = key_of(i, page_key(w, i, shift));     // (the wave's own pages)
    }
    uint32_t want = (uint32_t)a.budget;
    for (int i = tid; i < 256 * EV_COPIES; i += EV_THREADS) hist[0][i] = 0;
    __syncthreads();
    for (int digit = 24; digit >= 0; digit -= 8) {
      uint32_t *h = hist[(digit >> 3 & 1) ^ 1];
      each([&](int, int, uint32_t k) {
        if (digit == 24 || (k >> (digit + 8)) == (prefix >> (digit + 8)))
          atomicAdd(&h[(k >> digit & 255) * EV_COPIES + (lane & (EV_COPIES - 1))], 1u);
      });
      __syncthreads();
      if (wave == 0) {
        // the digit d with sum(hist above d) < want <= sum(hist from d on): lane l holds bins 255 - 4 l downwards
        uint32_t bins[4], mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const u32x4 *copies = reinterpret_cast<const u32x4 *>(h + (255 - 4 * lane - i) * EV_COPIES);
          u32x4 sum = copies[0];
#pragma unroll
          for (int c = 1; c < EV_COPIES / 4; ++c) sum += copies[c];
          mine += bins[i] = sum[0] + sum[1] + sum[2] + sum[3];
        }
        uint32_t above = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const uint32_t up = __shfl_up(above, d);
          if (lane >= d) above += up;
        }
        above -= mine;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (above < want && want <= above + bins[i]) {
            found[0] = 255 - 4 * lane - i;
            found[1] = want - above;
          }
          above += bins[i];
        }
      } else {
        for (int i = tid - 64; i < 256 * EV_COPIES; i += EV_THREADS - 64) hist[digit >> 3 & 1][i] = 0;    // for the next digit
      }
      __syncthreads();
      prefix |= found[0] << digit;
      want = found[1];
    }
    take = (int)want;
  }

  // places follow from what the waves before keep
  int sure = 0, ties = 0;
  if (over)
    each([&](int, int, uint32_t k) {
      sure += __popcll(__ballot(k > prefix));
      ties += __popcll(__ballot(k == prefix));
    });
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
  each([&](int n, int i, uint32_t k) {
    bool stay = true;
    int to = i;
    if (over) {
      const uint64_t tie = __ballot(k == prefix);
      stay = k > prefix || (k == prefix && tied + __popcll(tie & below) < take);
      const uint64_t staying = __ballot(stay);
      to = at + __popcll(staying & below);
      at += __popcll(staying);
      tied += __popcll(tie);
    }
    if (i >= hi) return;
    const int32_t its = HELD ? page[n] : table[i];
    if (!stay) {
      freed[i - to] = its;
      return;
    }
    new_table[to] = its;
    if (shift == 0) {
      new_w[to] = HELD ? weight[n] : w[i];
      return;
    }
    const int64_t t0 = (int64_t)i << shift;
#pragma unroll 8
    for (int j = 0; j < ps; ++j) new_w[((int64_t)to << shift) + j] = t0 + j < len ? w[t0 + j] : 0.0f;
  });
}

}  // namespace

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_cache_evict(void *stream, const int32_t *table, int64_t table_stride, const int32_t *kv_len,
                                 const float *weights, int64_t weights_stride, int64_t n_req, int64_t width, int32_t page_size,
                                 int64_t budget, int64_t recent, int64_t sinks, int32_t *new_table, int32_t *new_kv_len,
                                 float *new_weights, int32_t *freed) {
  if (n_req < 0 || width < 0 || n_req > 0x7fffffff) return fail(MLORA_ERR_INVALID, "cache_evict: negative size");
  if (n_req > most_blocks(EV_THREADS)) return fail(MLORA_ERR_NO_KERNEL, "cache_evict: more than %lld requests", (long long)most_blocks(EV_THREADS));
  int shift = 0;
  while (shift < 8 && (1 << shift) < page_size) ++shift;
  if (page_size < 1 || (1 << shift) != page_size)
    return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. cache_evict: page_size=%d (a power of two up to 256)", page_size);
  if (width > 0x7fffffff || width << shift > 0x7fffffff) return fail(MLORA_ERR_NO_KERNEL, "cache_evict: more than 2^31 - 1 tokens a request");
  if (recent < 1 || sinks < 0 || recent > 0x3fffffff || sinks > 0x3fffffff || budget > 0x7fffffff || budget < recent + sinks)
    return fail(MLORA_ERR_INVALID, "cache_evict: budget=%lld must hold recent=%lld (at least 1) and sinks=%lld pages",
                (long long)budget, (long long)recent, (long long)sinks);
  if (table_stride < width || weights_stride < width << shift)
    return fail(MLORA_ERR_INVALID, "cache_evict: a row of table or weights is shorter than %lld pages", (long long)width);
  if (n_req == 0) return MLORA_OK;
  if (!kv_len || !new_kv_len || (width > 0 && (!table || !weights || !new_table || !new_weights || !freed)))
    return fail(MLORA_ERR_INVALID, "cache_evict: null pointer");
  const bool held = width <= EV_HELD * EV_THREADS, lds = !held && width <= EV_MAX_KEYS;
  EvictArgs a{table, kv_len, weights, table_stride, weights_stride, new_table, new_kv_len, freed, new_weights,
              (int)width, shift, (int)budget, (int)recent, (int)sinks, lds};
  hipLaunchKernelGGL((held ? evict_kernel<true> : evict_kernel<false>), dim3((unsigned)n_req), dim3(EV_THREADS), lds ? (size_t)width * 4 : 0,
                     (hipStream_t)stream, a);
  return check_launch("evict_kernel");
}
