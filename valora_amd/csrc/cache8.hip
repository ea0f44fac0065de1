// The 8-bit cache (csrc/codes8.h) written and read back.
//
// Writing: as csrc/rotary.hip, but k and v become codes on their way to their slots.  A lane owns eight elements of a head, so a head is up to
// 32 lanes of a wave, which find its largest element among themselves; a rotated element's partner is loaded a second time (it is in
// the L1).  k is rotated in 64 bits, sines and all, and rounded once, to its code: in 32 bits one code in some hundred thousand would be a
// neighbour of the nearest, a sixteenth off, and the vector units do 64 bits at the rate of 32.
#include "codes8.h"

namespace mlora {

namespace {

struct StoreArgs {
  mlora_rotary_part q;
  const uint16_t *k, *v;
  int64_t k_token, k_head, v_token, v_head;
  mlora_cache8 c;
  const int64_t *positions, *loc;
  const double *freqs;
  int64_t n_slots;
  float gain;
  int rotary_dim, page_shift;
  int heads, per_piece;                 // k's, v's and q's; of a workgroup
};

constexpr int ST_THREADS = 256;

// pairs of the lane's elements: element at + i is turned with `other` of a pair's sine and cosine
template <typename T, typename F, int D, bool INTERLEAVED, bool VEC, typename Table>
__device__ __forceinline__ void turn(const StoreArgs &a, const uint16_t *head, int at, const Table *cs, F (&out)[8], bool rotate) {
  const int R = rotate ? a.rotary_dim : 0;
  uint16_t x[8], y[8];
  if constexpr (VEC) {
    const bool turned = at < R;
    const u32x4 mine = load16(head + at), its = !INTERLEAVED && turned ? load16(head + (at < R / 2 ? at + R / 2 : at - R / 2)) : mine;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = (uint16_t)(mine[i / 2] >> i % 2 * 16);
      const int j = INTERLEAVED ? i ^ 1 : i;
      y[i] = (uint16_t)(its[j / 2] >> j % 2 * 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = at + i, o = e >= R ? e : INTERLEAVED ? e ^ 1 : e < R / 2 ? e + R / 2 : e - R / 2;
      x[i] = head[e];
      y[i] = head[o];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = at + i;
    const F f = (F)Traits<T>::to_float(x[i]), g = (F)Traits<T>::to_float(y[i]);
    if (e < R) {
      const bool second = INTERLEAVED ? e & 1 : e >= R / 2;
      const Table t = cs[INTERLEAVED ? e / 2 : second ? e - R / 2 : e];
      out[i] = second ? g * (F)t.y + f * (F)t.x : f * (F)t.x - g * (F)t.y;
    } else {
      out[i] = f;
    }
  }
}

template <typename T, int D, typename F>
__device__ __forceinline__ void keep(const StoreArgs &a, const F (&x)[8], bool mine, int64_t slot, int head, int at, int which) {
  constexpr int LANES = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32;
  float largest = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const F size = x[i] < 0 ? -x[i] : x[i];
    if (mine && size < (F)INFINITY) largest = fmaxf(largest, not_below(size));
  }
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
  if (!mine || slot < 0) return;
  const uint32_t byte = power_byte<T>(largest);
  const int64_t page = slot >> a.page_shift, off = slot & ((1 << a.page_shift) - 1);
  char *codes = static_cast<char *>(which ? a.c.value_codes : a.c.key_codes) + page * (which ? a.c.value_stride : a.c.key_stride);
  *reinterpret_cast<u32x2 *>(codes + (((int64_t)head << a.page_shift) + off) * D + at) = codes_of(x, byte);
  if (at == 0) (static_cast<uint8_t *>(a.c.powers) + page * a.c.powers_stride)[(((int64_t)head << a.page_shift) + off) * 2 + which] = (uint8_t)byte;
}

template <typename T, int D, bool INTERLEAVED, bool VEC>
__global__ __launch_bounds__(ST_THREADS) void store8_kernel(StoreArgs a) {
  constexpr int LANES = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32, HEADS = ST_THREADS / LANES;
  __shared__ double2 cs[D / 2];
  const int64_t token = blockIdx.x;
  int64_t slot = a.loc[token];
  if (slot >= a.n_slots) slot = -1;
  const int64_t pos = a.positions[token];
  for (int i = threadIdx.x; i < a.rotary_dim / 2; i += ST_THREADS) {
    const double turns = (double)pos * a.freqs[i];
    double s, c;
    sincospi(2.0 * (turns - rint(turns)), &s, &c);
    cs[i] = double2{c * (double)a.gain, s * (double)a.gain};
  }
  __syncthreads();
  const int lane = threadIdx.x & (LANES - 1), at = lane * 8, kv = a.c.kv_heads;
  const bool mine = at < D;                                      // (heads of 96 have twelve lanes of sixteen)
  const int lo = blockIdx.y * a.per_piece, hi = min(lo + a.per_piece, a.heads);
  for (int h0 = lo; h0 < hi; h0 += HEADS) {                      // (every lane goes round as often: they look at each other's)
    const int h = h0 + (int)threadIdx.x / LANES;
    const bool has = mine && h < hi;
    if (h < kv) {
      double x[8] = {};
      if (has) turn<T, double, D, INTERLEAVED, VEC>(a, a.k + token * a.k_token + h * a.k_head, at, cs, x, true);
      keep<T, D>(a, x, has, slot, h, at, 0);
    } else if (h < 2 * kv) {
      float x[8] = {};
      if (has) turn<T, float, D, INTERLEAVED, VEC>(a, a.v + token * a.v_token + (h - kv) * a.v_head, at, cs, x, false);
      keep<T, D>(a, x, has, slot, h - kv, at, 1);
    } else if (has) {
      const int64_t head = h - 2 * kv;
      float x[8];
      turn<T, float, D, INTERLEAVED, VEC>(a, static_cast<const uint16_t *>(a.q.src) + token * a.q.src_token_stride + head * a.q.src_head_stride, at, cs, x, true);
      uint16_t *dst = static_cast<uint16_t *>(a.q.dst) + token * a.q.dst_token_stride + head * a.q.dst_head_stride + at;
      if constexpr (VEC) {
        store16(dst, pack8<T>(x));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = Traits<T>::from_float(x[i]);
      }
    }
  }
}

template <typename T, int D>
void launch_store(hipStream_t st, dim3 grid, const StoreArgs &a, bool interleaved, bool vec) {
  auto *k = interleaved ? (vec ? store8_kernel<T, D, true, true> : store8_kernel<T, D, true, false>)
                        : (vec ? store8_kernel<T, D, false, true> : store8_kernel<T, D, false, false>);
  hipLaunchKernelGGL(k, grid, dim3(ST_THREADS), 0, st, a);
}

template <typename T>
void launch_store(hipStream_t st, dim3 grid, const StoreArgs &a, bool interleaved, bool vec) {
  switch (a.c.head_dim) {
    case 32: return launch_store<T, 32>(st, grid, a, interleaved, vec);
    case 64: return launch_store<T, 64>(st, grid, a, interleaved, vec);
    case 96: return launch_store<T, 96>(st, grid, a, interleaved, vec);
    case 128: return launch_store<T, 128>(st, grid, a, interleaved, vec);
    default: return launch_store<T, 256>(st, grid, a, interleaved, vec);
  }
}

// ---- reading back: a thread sixteen codes of k and of v --------------------------------------------------------------------------------
struct ReadArgs {
  mlora_cache8 c;
  const int64_t *loc;
  uint16_t *k, *v;
  int64_t n, k_stride, v_stride;
  int page_shift, pieces;               // of sixteen codes, of a token
};

template <typename T>
__global__ __launch_bounds__(256) void read8_kernel(ReadArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, token = unit / a.pieces;
  if (token >= a.n) return;
  const int part = (int)(unit - token * a.pieces), each = a.c.head_dim / 16;
  const int head = part / each, at = (part - head * each) * 16;
  const int64_t slot = a.loc[token], page = slot >> a.page_shift, row = ((int64_t)head << a.page_shift) + (slot & ((1 << a.page_shift) - 1));
  u32x4 k[2] = {}, v[2] = {};
  if (slot >= 0 && page < a.c.n_pages) {
    const u32x4 kc = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(a.c.key_codes) + page * a.c.key_stride + row * a.c.head_dim + at);
    const u32x4 vc = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(a.c.value_codes) + page * a.c.value_stride + row * a.c.head_dim + at);
    const uint32_t e = *reinterpret_cast<const uint16_t *>(static_cast<const char *>(a.c.powers) + page * a.c.powers_stride + row * 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      k[i] = as<u32x4>(values_of<T>(u32x2{kc[2 * i], kc[2 * i + 1]}, k_power(e)));
      v[i] = as<u32x4>(values_of<T>(u32x2{vc[2 * i], vc[2 * i + 1]}, v_power(e)));
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    store16(a.k + token * a.k_stride + part * 16 + i * 8, k[i]);
    store16(a.v + token * a.v_stride + part * 16 + i * 8, v[i]);
  }
}

int log2_of(int n) {
  int s = 0;
  while ((1 << s) < n) ++s;
  return s;
}

}  // namespace

int check_cache8(const mlora_cache8 *c, int kv_heads, int head_dim, int page_size, const char *who) {
  if (!c) return fail(MLORA_ERR_INVALID, "%s: cache is null", who);
  if (c->kv_heads != kv_heads || c->head_dim != head_dim || c->page_size != page_size)
    return fail(MLORA_ERR_INVALID, "%s: the cache has %d key heads of %d in pages of %d, not %d of %d in pages of %d", who, c->kv_heads, c->head_dim,
                c->page_size, kv_heads, head_dim, page_size);
  const int d = c->head_dim;
  if (d != 32 && d != 64 && d != 96 && d != 128 && d != 256)
    return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. %s: head_dim=%d (32, 64, 96, 128 or 256)", who, d);
  if (c->page_size < 1 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. %s: page_size=%d (a power of two up to 256)", who, c->page_size);
  if (c->kv_heads < 1 || c->kv_heads > 1024) return fail(MLORA_ERR_INVALID, "%s: kv_heads=%d out of range", who, c->kv_heads);
  if (c->n_pages < 0 || c->n_pages > 0x7fffffff) return fail(MLORA_ERR_NO_KERNEL, "%s: n_pages=%lld out of range", who, (long long)c->n_pages);
  const int64_t tokens = (int64_t)c->kv_heads * c->page_size, w = tokens * d;
  if (c->key_stride < w || c->value_stride < w || c->powers_stride < 2 * tokens)
    return fail(MLORA_ERR_INVALID, "%s: a page of the cache is shorter than its heads", who);
  if (c->key_stride > 0x7fffffff || c->value_stride > 0x7fffffff || c->powers_stride > 0x7fffffff)
    return fail(MLORA_ERR_NO_KERNEL, "%s: pages above 2 GB", who);
  if ((c->key_stride | c->value_stride | (int64_t)reinterpret_cast<uintptr_t>(c->key_codes) | (int64_t)reinterpret_cast<uintptr_t>(c->value_codes)) & 15)
    return fail(MLORA_ERR_INVALID, "%s: pages of codes must be multiples of 16 bytes and 16-byte aligned", who);
  if ((c->powers_stride | (int64_t)reinterpret_cast<uintptr_t>(c->powers)) & 1)
    return fail(MLORA_ERR_INVALID, "%s: powers must be 2-byte aligned", who);
  return MLORA_OK;
}

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_rotary_store_codes(void *stream, const mlora_rotary_part *q, const void *k, int64_t k_token_stride, int64_t k_head_stride,
                                   const void *v, int64_t v_token_stride, int64_t v_head_stride, const mlora_cache8 *cache,
                                   const int64_t *positions, const int64_t *loc, int64_t T, int32_t rotary_dim, int32_t interleaved,
                                   const double *freqs, float gain, mlora_dtype dtype) {
  const char *who = "rotary_store8";
  if (!cache) return fail(MLORA_ERR_INVALID, "%s: cache is null", who);
  if (int rc = check_cache8(cache, cache->kv_heads, cache->head_dim, cache->page_size, who)) return rc;
  if (dtype != MLORA_F16 && dtype != MLORA_BF16) return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. %s: dtype=%d", who, (int)dtype);
  if (T < 0) return fail(MLORA_ERR_INVALID, "%s: T=%lld out of range", who, (long long)T);
  if (T > 0x7fffffff) return fail(MLORA_ERR_NO_KERNEL, "%s: more than 2^31 - 1 tokens", who);
  const int d = cache->head_dim;
  if (rotary_dim < 2 || (rotary_dim & 1) || rotary_dim > d)
    return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. %s: head_dim=%d rotary_dim=%d (even, at most head_dim)", who, d, rotary_dim);
  const int q_heads = q ? q->heads : 0;
  if (q_heads < 0 || q_heads > 65536) return fail(MLORA_ERR_INVALID, "%s: heads=%d out of range", who, q_heads);
  if (q_heads > 0 && share_elements(T, q->dst_token_stride, q_heads, q->dst_head_stride, d))
    return fail(MLORA_ERR_INVALID, "%s: heads of a destination overlap", who);
  // k's codes and v's: apart, or each page's side by side
  const char *kc = static_cast<const char *>(cache->key_codes), *vc = static_cast<const char *>(cache->value_codes);
  const int64_t w = (int64_t)cache->kv_heads * cache->page_size * d;
  if (kc && vc && cache->n_pages > 0) {
    const int64_t apart = vc > kc ? vc - kc : kc - vc;
    const int64_t lower = (cache->n_pages - 1) * (vc > kc ? cache->key_stride : cache->value_stride) + w;
    const int64_t in_page = apart % cache->key_stride;
    if (apart < lower && (cache->key_stride != cache->value_stride || in_page < w || cache->key_stride - in_page < w))
      return fail(MLORA_ERR_INVALID, "%s: codes of keys and values overlap", who);
  }
  if (T == 0) return MLORA_OK;
  if (!k || !v || !positions || !loc || !freqs || (q_heads > 0 && (!q->src || !q->dst))) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  if (cache->n_pages > 0 && (!kc || !vc || !cache->powers)) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  StoreArgs a{};
  bool vec = rotary_dim % 16 == 0 && ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) == 0 &&
             ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  if (q_heads > 0) {
    a.q = *q;
    vec = vec && ((q->src_token_stride | q->src_head_stride | q->dst_token_stride | q->dst_head_stride) & 7) == 0 &&
          ((reinterpret_cast<uintptr_t>(q->src) | reinterpret_cast<uintptr_t>(q->dst)) & 15) == 0;
  }
  a.k = static_cast<const uint16_t *>(k);
  a.v = static_cast<const uint16_t *>(v);
  a.k_token = k_token_stride;
  a.k_head = k_head_stride;
  a.v_token = v_token_stride;
  a.v_head = v_head_stride;
  a.c = *cache;
  a.positions = positions;
  a.loc = loc;
  a.freqs = freqs;
  a.n_slots = cache->n_pages * cache->page_size;
  a.gain = gain;
  a.rotary_dim = rotary_dim;
  a.page_shift = log2_of(cache->page_size);
  a.heads = 2 * cache->kv_heads + q_heads;
  // Few tokens: a workgroup a round of heads, as in csrc/rotary.hip
  const int per_round = ST_THREADS / (d <= 32 ? 4 : d <= 64 ? 8 : d <= 128 ? 16 : 32);
  const int rounds = (a.heads + per_round - 1) / per_round, pieces = T >= 512 ? 1 : rounds;
  a.per_piece = (rounds + pieces - 1) / pieces * per_round;
  const dim3 grid((unsigned)T, (unsigned)((a.heads + a.per_piece - 1) / a.per_piece));
  if (dtype == MLORA_F16) launch_store<_Float16>((hipStream_t)stream, grid, a, interleaved != 0, vec);
  else launch_store<__bf16>((hipStream_t)stream, grid, a, interleaved != 0, vec);
  return check_launch("store8_kernel");
}

extern "C" int mlora_cache_read_codes(void *stream, const mlora_cache8 *cache, const int64_t *loc, int64_t n, void *k, int64_t k_stride, void *v,
                                 int64_t v_stride, mlora_dtype dtype) {
  const char *who = "cache8_read";
  if (!cache) return fail(MLORA_ERR_INVALID, "%s: cache is null", who);
  if (int rc = check_cache8(cache, cache->kv_heads, cache->head_dim, cache->page_size, who)) return rc;
  if (dtype != MLORA_F16 && dtype != MLORA_BF16) return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. %s: dtype=%d", who, (int)dtype);
  if (n < 0) return fail(MLORA_ERR_INVALID, "%s: n=%lld out of range", who, (long long)n);
  const int64_t w = (int64_t)cache->kv_heads * cache->head_dim;
  if (n > 1 && (k_stride < w || v_stride < w)) return fail(MLORA_ERR_INVALID, "%s: rows of k or v overlap", who);
  if ((k_stride | v_stride) & 7 || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15))
    return fail(MLORA_ERR_INVALID, "%s: rows of k and v must be multiples of 16 bytes and 16-byte aligned", who);
  if (n > 0x7fffffffll * 256 / (w / 16)) return fail(MLORA_ERR_NO_KERNEL, "%s: n=%lld too large", who, (long long)n);
  if (n == 0) return MLORA_OK;
  if (!loc || !k || !v) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  if (cache->n_pages > 0 && (!cache->key_codes || !cache->value_codes || !cache->powers)) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  ReadArgs a{*cache, loc, static_cast<uint16_t *>(k), static_cast<uint16_t *>(v), n, k_stride, v_stride, log2_of(cache->page_size), (int)(w / 16)};
  const dim3 grid((unsigned)((n * a.pieces + 255) / 256));
  if (dtype == MLORA_F16) hipLaunchKernelGGL((read8_kernel<_Float16>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL((read8_kernel<__bf16>), grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch("read8_kernel");
}
