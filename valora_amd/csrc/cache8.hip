// The 8-bit cache (csrc/codes8.h) written and read back.
//
// Writing: as csrc/rotary.hip, but k and v become codes on their way to their slots.  A lane owns eight pairs of a head (both halves of it, so
// nothing is loaded twice) or eight elements that pass through; a head's lanes are neighbours in a wave and find its largest element among
// themselves.  k is rotated in 64 bits, sines and all, and rounded once, to its code: in 32 bits one code in some hundred thousand would be a
// neighbour of the nearest, a sixteenth off, and the vector units do 64 bits at half the rate of 32.
//
// Bound by bytes (8191 tokens, 32 query and 8 key heads of 128, bf16: 185 MB in 40 us, 4.6 TB/s; a copy of as much takes 36).  Where tokens are many, four a
// workgroup share one wait for positions, frequencies and sines (a token a workgroup: 49 us; two and eight: 41), and a lane that owned eight
// elements and loaded their partners a second time took 55: half of it were the vector units.  Where rows or what is rotated of them are no whole runs
// of 16 bytes it goes by elements, a token a workgroup (120 of 128 rotated: 2048 tokens 30 us, 12.5 by runs, 8191 96 and 31 with part of it in the
// memory-side cache).
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
  int64_t n_slots, T;
  float gain;
  int rotary_dim, page_shift, lane_shift;
  int heads, per_piece;                 // k's, v's and q's; of a workgroup
  bool many;
};

constexpr int ST_THREADS = 256;
// A round is what a workgroup's threads take at once, some heads of a token.  From MANY on a workgroup has four tokens, whose heads are cut in pieces
// while there are fewer than FULL tokens; below it a round of one token, each of which works out the token's sines again (us of four tokens / of one,
// 32 query heads.  Heads of 128: 1024 and 2048 tokens of 8 key heads 9.7 / 8.3 and 12.5 / 14.8, 512 and 1024 of 32 9.8 / 7.6 and 11.1 / 13.5.  Of 256:
// 512 and 1024 of 8 10.1 / 7.7 and 11.4 / 12.9, 256 and 512 of 32 10.3 / 7.8 and 12.2 / 14.0.  Of 64: 1024, 1536 and 2048 of 8 6.3 / 6.0, 7.3 / 8.4 and
// 7.7 / 10.1, 1024 and 1536 of 32 9.5 / 8.7 and 11.4 / 12.1; the border of 8 key heads of 64 is set at 2731 tokens and lies near 1100).  FULL: 2048
// tokens of 32 key heads in pieces / whole 12.1 / 12.9 (heads of 64), 19.8 / 22.9 (128), 31.4 / 41.9 (256); 4096 in a piece a round / whole 19.5 / 18.2,
// 34.3 / 32.2, 84 / 77; 3000 the same within 4 % but for 32 heads of 256 (55 / 60).
constexpr int MANY = 2048, FULL = 4096;

// A lane's part of a head: n elements from a0 on and, where they are the first halves of pairs, as many from a1 on
struct Part {
  int a0, a1, n;
  __device__ __forceinline__ Part(int lane, int D, int R, bool interleaved) {
    const int turned = interleaved ? (R + 7) / 8 : (R / 2 + 7) / 8;         // parts that are rotated
    if (lane < turned) {
      a0 = lane * 8;
      a1 = interleaved ? -1 : a0 + R / 2;
      n = min(8, (interleaved ? R : R / 2) - a0);
    } else {
      a0 = R + (lane - turned) * 8;
      a1 = -1;
      n = min(8, D - a0);                                                    // (none, or less: a lane behind the head)
    }
  }
};

// (how many there are, as if it had just been found: comparisons kept from one use to the next would fill the scalar registers)
__device__ __forceinline__ int anew(int n) {
  asm volatile("" : "+v"(n));
  return n;
}
template <bool VEC>
__device__ __forceinline__ u32x4 load_eight(const uint16_t *p, int n) {
  if constexpr (VEC) return load16(p);
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (uint32_t)p[min(2 * i, n - 1)] | (uint32_t)p[min(2 * i + 1, n - 1)] << 16;
  return r;
}
template <bool VEC>
__device__ __forceinline__ void store_eight(uint16_t *p, int n, u32x4 x) {
  if constexpr (VEC) {
    store16(p, x);
  } else {
    n = anew(n);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint16_t)(x[i / 2] >> i % 2 * 16);
  }
}
template <bool VEC>
__device__ __forceinline__ void store_codes(char *p, int n, u32x2 x) {
  if constexpr (VEC) {
    *reinterpret_cast<u32x2 *>(p) = x;
  } else {
    n = anew(n);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (char)(x[i / 4] >> i % 4 * 8);
  }
}

struct Loaded {
  u32x4 a, b;
};

// Where the sine and cosine of a pair stand in LDS: those of eight lanes' pairs i, i + 1 side by side (lanes that read 8 of them in a row would
// meet in the banks)
template <int PAIRS>
__device__ __forceinline__ int place_of(int pair) { return (((pair & 7) >> 1) * (PAIRS / 8) + (pair >> 3)) * 2 + (pair & 1); }

// Rotates a lane's pairs: a (and b) in, out of them; in F, with sines of F
template <typename T, typename F, bool INTERLEAVED, typename Sines>
__device__ __forceinline__ void turn(const Loaded &p, Sines sines, F (&a)[8], F (&b)[8]) {
  float f[8], g[8];
  unpack8<T>(p.a, f);
  if constexpr (INTERLEAVED) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto t = sines(i);
      a[2 * i] = (F)f[2 * i] * t.x - (F)f[2 * i + 1] * t.y;
      a[2 * i + 1] = (F)f[2 * i] * t.y + (F)f[2 * i + 1] * t.x;
    }
  } else {
    unpack8<T>(p.b, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const auto t = sines(i);
      a[i] = (F)f[i] * t.x - (F)g[i] * t.y;
      b[i] = (F)f[i] * t.y + (F)g[i] * t.x;
    }
  }
}

// TOKENS of a workgroup: their sines are worked out together, a thread a pair, and their heads follow each other
template <typename T, int D, bool INTERLEAVED, bool VEC, int TOKENS>
__global__ __launch_bounds__(ST_THREADS) void store8_kernel(StoreArgs a) {
  constexpr int PAIRS = D / 2;
  __shared__ __align__(16) double2 cs[TOKENS * PAIRS];
  __shared__ __align__(16) float2 cs32[TOKENS * PAIRS];
  __shared__ int64_t slots[TOKENS];
  const int64_t first = (int64_t)blockIdx.x * TOKENS;
  const int tokens = (int)min<int64_t>(TOKENS, a.T - first);
  const int kv = a.c.kv_heads, R = a.rotary_dim, heads = ST_THREADS >> a.lane_shift, lanes = 1 << a.lane_shift;
  const Part part((int)threadIdx.x & (lanes - 1), D, R, INTERLEAVED);
  const bool rotates = part.a0 < R && part.n > 0, both = part.a1 >= 0;
  const int lo = blockIdx.y * a.per_piece, hi = min(lo + a.per_piece, a.heads);
  // heads in the order k's, v's, q's; a round's are asked for while those before are worked on, the first ones before the sines
  struct Item {
    int t, h;
  };
  auto load = [&](const Item &n) {
    Loaded p{};
    if (part.n > 0 && n.t < tokens) {
      const int64_t token = first + n.t;
      const uint16_t *src = n.h < kv ? a.k + token * a.k_token + n.h * a.k_head
                            : n.h < 2 * kv ? a.v + token * a.v_token + (n.h - kv) * a.v_head
                                           : static_cast<const uint16_t *>(a.q.src) + token * a.q.src_token_stride + (n.h - 2 * kv) * a.q.src_head_stride;
      p.a = load_eight<VEC>(src + part.a0, part.n);
      if (both) p.b = load_eight<VEC>(src + part.a1, part.n);
    }
    return p;
  };
  auto settle = [&](Item &n) {                                   // a head behind the last is one of the next token
    while (n.h >= hi && n.t < tokens) {
      n.h -= hi - lo;
      ++n.t;
    }
  };
  Item item{0, lo + ((int)threadIdx.x >> a.lane_shift)};
  settle(item);
  Loaded next = load(item);
  requested();
  for (int i = threadIdx.x; i < TOKENS * PAIRS; i += ST_THREADS) {
    const int t = i / PAIRS, pair = i - t * PAIRS;
    if (pair >= R / 2 || t >= tokens) continue;
    const double turns = (double)a.positions[first + t] * a.freqs[pair];
    double s, c;
    sincospi(2.0 * (turns - rint(turns)), &s, &c);
    const double2 v{c * (double)a.gain, s * (double)a.gain};
    const int at = t * PAIRS + place_of<PAIRS>(pair);
    cs[at] = v;
    cs32[at] = float2{(float)v.x, (float)v.y};
  }
  if (threadIdx.x < TOKENS && (int)threadIdx.x < tokens) {
    const int64_t slot = a.loc[first + threadIdx.x];
    slots[threadIdx.x] = slot < a.n_slots ? slot : -1;
  }
  __syncthreads();
  const int pair0 = rotates ? (INTERLEAVED ? part.a0 / 2 : part.a0) : 0;
  const int rounds = (tokens * (hi - lo) + heads - 1) / heads;
  for (int r = 0; r < rounds; ++r) {                             // (every lane goes round as often: they look at each other's)
    const Loaded p = next;
    const Item n = item;
    item.h += heads;
    settle(item);
    next = load(item);
    requested();
    const bool has = part.n > 0 && n.t < tokens;
    const int t = min(n.t, tokens - 1), h = n.h;
    float x[8], y[8];
    if (h >= 2 * kv) {
      if (!has) continue;                                        // (q's lanes look at no other's)
      u32x4 first8 = p.a, second8 = p.b;
      if (rotates) {
        turn<T, float, INTERLEAVED>(p, [&](int i) { return cs32[t * PAIRS + place_of<PAIRS>(pair0 + i)]; }, x, y);
        first8 = pack8<T>(x);
        if constexpr (!INTERLEAVED) second8 = pack8<T>(y);
      }
      uint16_t *dst = static_cast<uint16_t *>(a.q.dst) + (first + t) * a.q.dst_token_stride + (h - 2 * kv) * a.q.dst_head_stride;
      store_eight<VEC>(dst + part.a0, part.n, first8);
      if (both) store_eight<VEC>(dst + part.a1, part.n, second8);
      continue;
    }
    float largest = 0.0f;
    if (h < kv && rotates) {
      double u[8], w[8];
      const int some = VEC ? 8 : anew(part.n);
      turn<T, double, INTERLEAVED>(p, [&](int i) { return cs[t * PAIRS + place_of<PAIRS>(pair0 + i)]; }, u, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = sticky(u[i]);
        if (i < some && fabs(u[i]) < (double)INFINITY) largest = fmaxf(largest, fabsf(x[i]));      // (one beyond 32 bits counts, as the largest)
        if constexpr (!INTERLEAVED) {
          y[i] = sticky(w[i]);
          if (i < some && fabs(w[i]) < (double)INFINITY) largest = fmaxf(largest, fabsf(y[i]));
        }
      }
    } else {
      unpack8<T>(p.a, x);
      unpack8<T>(p.b, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (fabsf(x[i]) < INFINITY) largest = fmaxf(largest, fabsf(x[i]));
        if (fabsf(y[i]) < INFINITY) largest = fmaxf(largest, fabsf(y[i]));
      }
    }
    for (int d = 1; d < lanes; d <<= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
    const int64_t slot = slots[t];
    if (!has || slot < 0) continue;
    const uint32_t byte = power_byte<T>(largest);
    const int which = h >= kv;
    const int64_t page = slot >> a.page_shift, row = ((int64_t)(h - which * kv) << a.page_shift) + (slot & ((1 << a.page_shift) - 1));
    char *codes = static_cast<char *>(which ? a.c.value_codes : a.c.key_codes) + page * (which ? a.c.value_stride : a.c.key_stride) + row * D;
    store_codes<VEC>(codes + part.a0, part.n, codes_of(x, byte));
    if (both) store_codes<VEC>(codes + part.a1, part.n, codes_of(y, byte));
    if (part.a0 == 0) (static_cast<uint8_t *>(a.c.powers) + page * a.c.powers_stride)[row * 2 + which] = (uint8_t)byte;
  }
}

template <typename T, int D, int TOKENS>
void launch_store(hipStream_t st, dim3 grid, const StoreArgs &a, bool interleaved, bool vec) {
  auto *k = interleaved ? (vec ? store8_kernel<T, D, true, true, TOKENS> : store8_kernel<T, D, true, false, 1>)
                        : (vec ? store8_kernel<T, D, false, true, TOKENS> : store8_kernel<T, D, false, false, 1>);
  if (vec) grid.x = (grid.x + TOKENS - 1) / TOKENS;
  hipLaunchKernelGGL(k, grid, dim3(ST_THREADS), 0, st, a);
}

template <typename T, int D>
void launch_store(hipStream_t st, dim3 grid, const StoreArgs &a, bool interleaved, bool vec) {
  if (a.many) launch_store<T, D, 4>(st, grid, a, interleaved, vec);
  else launch_store<T, D, 1>(st, grid, a, interleaved, vec);
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

// ---- reading back: a thread eight codes of k and of v ----------------------------------------------------------------------------------
struct ReadArgs {
  mlora_cache8 c;
  const int64_t *loc;
  uint16_t *k, *v;
  int64_t n, k_stride, v_stride;
  int page_shift, pieces, tokens;       // of eight codes, of a token; of a workgroup
  float inv_pieces, inv_each;
};
constexpr int READ_THREADS = 256;

template <typename T>
__global__ __launch_bounds__(READ_THREADS) void read8_kernel(ReadArgs a) {
  uint32_t t, part, head, at;
  divmod24(threadIdx.x, (uint32_t)a.pieces, a.inv_pieces, t, part);      // (t is 0 where a token has more pieces than a workgroup threads)
  part += blockIdx.y * READ_THREADS;
  const int64_t token = (int64_t)blockIdx.x * a.tokens + t;
  if ((int)t >= a.tokens || token >= a.n || (int)part >= a.pieces) return;
  divmod24(part, (uint32_t)a.c.head_dim / 8, a.inv_each, head, at);
  at *= 8;
  const int64_t slot = a.loc[token], page = slot >> a.page_shift, row = ((int64_t)head << a.page_shift) + (slot & ((1 << a.page_shift) - 1));
  u32x4 k{}, v{};
  if (slot >= 0 && page < a.c.n_pages) {
    const u32x2 kc = *reinterpret_cast<const u32x2 *>(static_cast<const char *>(a.c.key_codes) + page * a.c.key_stride + row * a.c.head_dim + at);
    const u32x2 vc = *reinterpret_cast<const u32x2 *>(static_cast<const char *>(a.c.value_codes) + page * a.c.value_stride + row * a.c.head_dim + at);
    const uint32_t e = *reinterpret_cast<const uint16_t *>(static_cast<const char *>(a.c.powers) + page * a.c.powers_stride + row * 2);
    k = as<u32x4>(values_of<T>(kc, k_power(e)));
    v = as<u32x4>(values_of<T>(vc, v_power(e)));
  }
  store16(a.k + token * a.k_stride + part * 8, k);
  store16(a.v + token * a.v_stride + part * 8, v);
}

int log2_of(int n) {
  int s = 0;
  while ((1 << s) < n) ++s;
  return s;
}

// What the cache's pages take
Runs key_pages(const mlora_cache8 &c) { return {c.key_codes, c.n_pages, c.key_stride, 1, 0, (int64_t)c.kv_heads * c.page_size * c.head_dim}; }
Runs value_pages(const mlora_cache8 &c) { return {c.value_codes, c.n_pages, c.value_stride, 1, 0, (int64_t)c.kv_heads * c.page_size * c.head_dim}; }
Runs power_pages(const mlora_cache8 &c) { return {c.powers, c.n_pages, c.powers_stride, 1, 0, (int64_t)c.kv_heads * c.page_size * 2}; }

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
  // k's codes, v's and powers: apart, or each page's side by side
  if (share_memory(key_pages(*cache), value_pages(*cache))) return fail(MLORA_ERR_INVALID, "%s: codes of keys and values overlap", who);
  if (share_memory(power_pages(*cache), key_pages(*cache)) || share_memory(power_pages(*cache), value_pages(*cache)))
    return fail(MLORA_ERR_INVALID, "%s: powers overlap codes", who);
  if (T == 0) return MLORA_OK;
  if (q_heads > 0 && (!q->src || !q->dst)) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  // what other workgroups read may not be where q goes; q itself only in its own place
  if (q_heads > 0) {
    const auto heads = [&](const void *p, int n, int64_t token, int64_t head) { return Runs{p, T, token * 2, n, head * 2, (int64_t)d * 2}; };
    const Runs to = heads(q->dst, q_heads, q->dst_token_stride, q->dst_head_stride);
    const bool in_place = q->src == q->dst && (T == 1 || q->src_token_stride == q->dst_token_stride) &&
                          (q_heads == 1 || q->src_head_stride == q->dst_head_stride);
    if (!in_place && share_memory(to, heads(q->src, q_heads, q->src_token_stride, q->src_head_stride)))
      return fail(MLORA_ERR_INVALID, "%s: q's destination overlaps other heads of q", who);
    if (share_memory(to, heads(k, cache->kv_heads, k_token_stride, k_head_stride)) || share_memory(to, heads(v, cache->kv_heads, v_token_stride, v_head_stride)))
      return fail(MLORA_ERR_INVALID, "%s: q's destination overlaps k or v", who);
    if (share_memory(to, {positions, 1, 0, 1, 0, T * 8}) || share_memory(to, {loc, 1, 0, 1, 0, T * 8}))
      return fail(MLORA_ERR_INVALID, "%s: q's destination overlaps positions or loc", who);
  }
  if (!k || !v || !positions || !loc || !freqs) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  if (cache->n_pages > 0 && (!cache->key_codes || !cache->value_codes || !cache->powers)) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
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
  a.T = T;
  a.gain = gain;
  a.rotary_dim = rotary_dim;
  a.page_shift = log2_of(cache->page_size);
  a.heads = 2 * cache->kv_heads + q_heads;
  // lanes of a head: a power of two, so that they find each other by exchanging bits
  a.lane_shift = log2_of((interleaved ? (rotary_dim + 7) / 8 : (rotary_dim / 2 + 7) / 8) + (d - rotary_dim + 7) / 8);
  const int per_round = ST_THREADS >> a.lane_shift, rounds = (a.heads + per_round - 1) / per_round;
  a.many = T * a.heads >= (int64_t)MANY * per_round;
  const int64_t pieces = !a.many ? rounds : T >= FULL ? 1 : FULL / T < rounds ? FULL / T : rounds;
  a.per_piece = (int)((rounds + pieces - 1) / pieces) * per_round;
  for (int64_t at = 0; at < T; at += most_blocks(ST_THREADS)) {
    StoreArgs part = a;
    part.T = T - at < most_blocks(ST_THREADS) ? T - at : most_blocks(ST_THREADS);
    if (q_heads > 0) {
      part.q.src = static_cast<const uint16_t *>(a.q.src) + at * a.q.src_token_stride;
      part.q.dst = static_cast<uint16_t *>(a.q.dst) + at * a.q.dst_token_stride;
    }
    part.k += at * a.k_token;
    part.v += at * a.v_token;
    part.positions += at;
    part.loc += at;
    const dim3 grid((unsigned)part.T, (unsigned)((a.heads + a.per_piece - 1) / a.per_piece));
    if (dtype == MLORA_F16) launch_store<_Float16>((hipStream_t)stream, grid, part, interleaved != 0, vec);
    else launch_store<__bf16>((hipStream_t)stream, grid, part, interleaved != 0, vec);
  }
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
  const int pieces = (int)(w / 8), tokens = pieces >= READ_THREADS ? 1 : READ_THREADS / pieces;
  if (n > 0x7fffffffll * tokens) return fail(MLORA_ERR_NO_KERNEL, "%s: n=%lld too large", who, (long long)n);
  const Runs to_k{k, n, k_stride * 2, 1, 0, w * 2}, to_v{v, n, v_stride * 2, 1, 0, w * 2};
  if (share_memory(to_k, to_v)) return fail(MLORA_ERR_INVALID, "%s: k and v overlap", who);
  if (n == 0) return MLORA_OK;
  if (!loc || !k || !v) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  if (cache->n_pages > 0 && (!cache->key_codes || !cache->value_codes || !cache->powers)) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  for (const Runs &to : {to_k, to_v}) {
    if (share_memory(to, key_pages(*cache)) || share_memory(to, value_pages(*cache)) || share_memory(to, power_pages(*cache)))
      return fail(MLORA_ERR_INVALID, "%s: k or v overlaps the cache", who);
    if (share_memory(to, {loc, 1, 0, 1, 0, n * 8})) return fail(MLORA_ERR_INVALID, "%s: k or v overlaps loc", who);
  }
  ReadArgs a{*cache, loc, static_cast<uint16_t *>(k), static_cast<uint16_t *>(v), n, k_stride, v_stride, log2_of(cache->page_size), pieces, tokens,
             1.0f / (float)pieces, 8.0f / (float)cache->head_dim};
  const int64_t most = most_blocks(READ_THREADS) * tokens;
  for (int64_t at = 0; at < n; at += most) {
    ReadArgs part = a;
    part.n = n - at < most ? n - at : most;
    part.loc += at;
    part.k += at * k_stride;
    part.v += at * v_stride;
    const dim3 grid((unsigned)((part.n + tokens - 1) / tokens), (unsigned)((pieces + READ_THREADS - 1) / READ_THREADS));
    if (dtype == MLORA_F16) hipLaunchKernelGGL((read8_kernel<_Float16>), grid, dim3(READ_THREADS), 0, (hipStream_t)stream, part);
    else hipLaunchKernelGGL((read8_kernel<__bf16>), grid, dim3(READ_THREADS), 0, (hipStream_t)stream, part);
  }
  return check_launch("read8_kernel");
}
