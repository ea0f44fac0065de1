// Attention of new tokens over the paged cache.
//
// A row (new token i, query head h) of a request sees the cache indices j of [max(0, p - window + 1), p], p = kv_len - n + i:
//
//     out = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m)
//
// in one pass over the row's part of the cache, with the running maximum m and the running sum in 32 bits (csrc/attention.h
// says how the work is cut).  Rows that see nothing, and rows all of whose scores are -infinity, come out as zeros.
//
// Both matrix products keep the rows on the columns of the accumulators: S^T = K Q^T and O^T = V^T P^T.  A lane then holds scores
// of one row only, the running maximum and sum are one register each, and the exponentials are the second product's
// operand as they stand: its contraction may run over the cached tokens in any order, so it runs in the order in which the first
// product left them, and V^T is read from LDS to fit (ds_read_b64_tr_b16 hands a lane four tokens of one column).
// K and V go from memory into LDS without passing through registers, each 16 bytes to a place that keeps the reads free of bank
// conflicts.  The page numbers of a tile go ahead of it the same way, so the only waits of the loop are the counted ones
// written in it.
//
// The maximum is followed lazily: a row's scores are taken relative to a reference that stays as long as no score of the wave
// has grown 2^8 times above the maximum it was set by, and neither sums nor accumulators are scaled meanwhile.  The second product
// takes the weights in the tensors' 16-bit type, as its matrix instructions do (half a step off each, and so is what divides: their sum, in 32
// bits; a remainder in a product of its own would double that product).  In fp16 the reference lies 2^7 below the maximum: weights go up to
// 2^15 of the 65504 that fp16 holds, keep their eleven bits down to 2^-21 of the largest and are 0 below 2^-32 of it.  (With the
// maximum for a reference, tokens 18 below the highest score, in natural units, were lost: 60000 of them are 0.1 % of a row.)  In bf16,
// whose values may be as large as the accumulators hold, it lies 2^8 above: weights go up to 1.  Rows whose sums come near what those
// hold are done again with it 2^38 above: weights go up to 2^-30, and no sum over 2^30 tokens is larger than the values are.
#pragma once

#include <type_traits>

#include "attention.h"
#include "codes8.h"
#include "kernel_common.h"

namespace mlora {

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

constexpr float GROWTH = 8.0f;         // in powers of two

struct AttnArgs {
  const int32_t *plan;
  uint16_t *out;
  const uint16_t *q, *k, *v;
  const int32_t *table;
  float *few_o, *tall_o;               // sums of the pieces (csrc/attention.h)
  float4 *few_ml, *tall_ml;            // {reference, sum of the rounded weights, sum of the weights, -}
  float *lse;                          // null: not wanted
  float *scores;
  float *weights;
  int64_t out_stride, q_stride, table_stride, weights_stride;
  uint32_t k_stride, v_stride;         // bytes from a row of the pool to the next; of codes, from a page
  const uint8_t *e;                    // codes: powers, and bytes of a page of them
  uint32_t e_stride;
  float c;                             // scale * log2(e)
  int tall_blocks;                     // workgroups of the tall list; those of the other follow
  int max_few;                         // records that the other has room for
  int heads_together;                  // codes: a piece's key heads go to one XCD
  int q_heads, kv_heads, group, page_shift, window, n_req, n_pages;
  int off_few, off_tall, off_joins, off_tall_joins, off_arrive, off_requests, off_shares;      // of the plan, words
};

// The two 16-bit types as these kernels need them: the wide matrix product, the rounding of two values to one register, the sum of
// two rounded ones, the bits of the exponent
template <typename T>
struct Wide;
template <>
struct Wide<_Float16> {
  static __device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ float add2(uint32_t p, float l) { return __builtin_amdgcn_fdot2(as<f16x2>(p), f16x2{1, 1}, l, false); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return as<uint32_t>(__builtin_convertvector((f32x2{lo, hi}), f16x2)); }
  static constexpr uint32_t EXPONENT = 0x7c00;
  static constexpr float AHEAD = -7.0f, FAR = AHEAD;           // the reference above the maximum, and where values are large
};
template <>
struct Wide<__bf16> {
  static __device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ float add2(uint32_t p, float l) { return __builtin_amdgcn_fdot2_f32_bf16(as<bf16x2>(p), bf16x2{1, 1}, l, false); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return as<uint32_t>(__builtin_convertvector((f32x2{lo, hi}), bf16x2)); }
  static constexpr uint32_t EXPONENT = 0x7f80;
  static constexpr float AHEAD = GROWTH, FAR = GROWTH + 30.0f;
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// What is made of x below is made there
__device__ __forceinline__ void here(uint32_t &x) { asm volatile("" : "+v"(x)); }
// Bits lo to hi, of the 64 that there are
__device__ __forceinline__ uint64_t run(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 63);
  return lo <= hi ? (~0ull >> (63 - hi)) & (~0ull << lo) : 0;
}
// All ones where the bit is set.  (Flags kept as such would fill the scalar registers.)
__device__ __forceinline__ uint32_t bit(uint32_t bits, int at) { return (uint32_t)((int32_t)(bits << (31 - at)) >> 31); }
// x, or -infinity unless the bit is set
__device__ __forceinline__ float unless(float x, uint32_t ones) { return as<float>((as<uint32_t>(x) & ones) | (0xff800000u & ~ones)); }
template <typename T>
__device__ __forceinline__ uint32_t ones2(uint32_t lo, uint32_t hi) {
  const uint32_t one = Traits<T>::from_float(1.0f);
  return (lo & one) | (hi & one << 16);
}
// What is written below stays below, loads among it: the steps of the rare paths are not interleaved, which would take registers from
// the common one
__device__ __forceinline__ void one_by_one() {
  requested();
  __builtin_amdgcn_sched_barrier(0);
}

// ---- memory to LDS: lane l's 16 (4) bytes go to base + 16 l (4 l); base is the wave's --------------------------------------
// (M0 holds the base; nothing else here uses it.  Waits are the caller's: the compiler does not know of these loads.)
__device__ __forceinline__ void to_lds16(const void *p, uint32_t base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(base), "v"(p) : "memory");
}
__device__ __forceinline__ void to_lds4(const void *p, uint32_t base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(base), "v"(p) : "memory");
}
// The loads have arrived.  (Left to itself the compiler waits for them where they are first used, which is in the loop: every time round
// it would wait for what the loop has just asked for.)
template <typename V, int N>
__device__ __forceinline__ void arrived(V (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    u32x4 v = as<u32x4>(x[i]);
    asm volatile("" : "+v"(v));
    x[i] = as<V>(v);
  }
}
__device__ __forceinline__ uint32_t lds_offset(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

__device__ __forceinline__ u32x4 lds16(uint32_t at) { return *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)at; }
__device__ __forceinline__ int32_t lds_word(uint32_t at) { return *(const __attribute__((address_space(3))) int32_t *)(uintptr_t)at; }
__device__ __forceinline__ s16x4 lds_turned(uint32_t at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(uintptr_t)at);
}

// ---- a tile in LDS: rows of D elements, 16-byte pieces of a row exchanged so that what is read together lies in different banks --
// K is read 16 bytes of 16 or 32 rows at a time, V 64 bytes of 4 rows (tall tiles) or 32 bytes of 8.
template <int D>
struct Tile {
  static constexpr int P = D / 8, ROW = D * 2;
  static __device__ __forceinline__ int k_turn(int t) {
    return D >= 128 ? t & 15 : D == 64 ? (t >> 1) & 7 : D == 32 ? (t >> 2) & 3 : (t >> 2) & 3;
  }
  static __device__ __forceinline__ int v_turn(int t) {
    return D >= 128 ? (t & 3) << 2 | (t & 4) >> 1 : D == 64 ? (t & 2) << 1 | (t & 4) >> 1 : (t & 4) >> 1;
  }
  // 12 pieces (D = 96) are no power of two: they are rotated, where the others are exchanged
  static __device__ __forceinline__ int place(int piece, int turn) {
    if (D != 96) return piece ^ turn;
    const int s = piece + turn;
    return s >= P ? s - P : s;
  }
  static __device__ __forceinline__ int piece(int place, int turn) {
    if (D != 96) return place ^ turn;
    const int s = place - turn;
    return s < 0 ? s + P : s;
  }
  // Address of piece `low + high` of row t of a tile at `base`; `low` is the lane's, `high`, a multiple of a power of two above
  // it, the instruction's: one exchange of bits behind what a lane keeps for all of its reads.
  static __device__ __forceinline__ uint32_t at(uint32_t base, int t, int turn, int low, int high) {
    if (D != 96) return (base + t * ROW + (low ^ turn) * 16) ^ high * 16;
    return base + t * ROW + place(low + high, turn) * 16;
  }
  static __device__ __forceinline__ uint32_t k_at(uint32_t base, int t, int low, int high) { return at(base, t, k_turn(t), low, high); }
  static __device__ __forceinline__ uint32_t v_at(uint32_t base, int t, int low, int high) { return at(base, t, v_turn(t), low, high); }
};

// The request's pages and what a piece covers of its cache
struct Cache {
  const int32_t *table;
  const char *k, *v;          // of the key head
  uint32_t k_stride, v_stride;
  int begin, end, shift, n_pages;
  const uint8_t *e;           // codes: powers of the key head
  uint32_t e_stride;
};
template <int D, bool CODES>
__device__ __forceinline__ Cache cache_of(const AttnArgs &a, int req, int head, int begin, int end) {
  const int64_t ahead = CODES ? (int64_t)head * D << a.page_shift : head * D * 2;
  return {a.table + (int64_t)req * a.table_stride, reinterpret_cast<const char *>(a.k) + ahead, reinterpret_cast<const char *>(a.v) + ahead,
          a.k_stride, a.v_stride, begin, end, a.page_shift, a.n_pages, CODES ? a.e + ((int64_t)head * 2 << a.page_shift) : nullptr, a.e_stride};
}

// A record of the plan's lists, asked for at once and before it is known whether it is one (the lists have room for it either way)
struct Record {
  int w[AT_REC];
  __device__ __forceinline__ Record(const int32_t *plan, int64_t list, int i) {
    const int32_t *rec = plan + list + (int64_t)i * AT_REC;
#pragma unroll
    for (int n = 0; n < AT_REC; ++n) w[n] = rec[n];
    requested();
  }
};

// page numbers of tokens [base, base + 64), token base + l by lane l
__device__ __forceinline__ void load_pages(const Cache &c, int base, uint32_t slice, int lane) {
  const int t = min(base + lane, c.end - 1);
  to_lds4(c.table + (t >> c.shift), slice);
}

__device__ __forceinline__ bool bad_page(const Cache &c, int32_t page) { return (uint32_t)page >= (uint32_t)c.n_pages; }

// Pool row of token `at`, whose page number is given; row 0 where the page is none of the pool
__device__ __forceinline__ uint32_t row_of(const Cache &c, int at, int32_t page) {
  const int tok = min(at, c.end - 1);
  return bad_page(c, page) ? 0 : ((uint32_t)page << c.shift) + (tok & ((1 << c.shift) - 1));
}

// Where a token's codes and powers are; slot 0 of page 0 where its page is none of the pool
template <int D>
struct Slot {
  uint64_t page;
  uint32_t off;
  __device__ __forceinline__ Slot(const Cache &c, int at, int32_t page_) {
    const int tok = min(at, c.end - 1);
    page = bad_page(c, page_) ? 0 : (uint32_t)page_;
    off = (uint32_t)tok & ((1u << c.shift) - 1);
  }
  __device__ __forceinline__ const char *k(const Cache &c) const { return c.k + page * c.k_stride + off * D; }
  __device__ __forceinline__ const char *v(const Cache &c) const { return c.v + page * c.v_stride + off * D; }
  __device__ __forceinline__ uint32_t powers(const Cache &c) const { return *reinterpret_cast<const uint16_t *>(c.e + page * c.e_stride + off * 2); }
};

// K and V of tokens [base, base + N) into LDS, by WAVES waves together
template <int D, int N, int WAVES>
__device__ __forceinline__ void load_tile(const Cache &c, int base, uint32_t slice, uint32_t kt, uint32_t vt, int wave, int lane) {
  using L = Tile<D>;
  constexpr int EACH = N * L::P / 64 / WAVES;
  static_assert(EACH * 64 * WAVES == N * L::P, "whole loads");
  int32_t pages[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) pages[i] = lds_word(slice + ((i * WAVES + wave) * 64 + lane) / L::P * 4);
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int first = (i * WAVES + wave) * 64, unit = first + lane;
    const int t = unit / L::P, place = unit - t * L::P;
    const uint64_t row = row_of(c, base + t, pages[i]);
    to_lds16(c.k + row * c.k_stride + L::piece(place, L::k_turn(t)) * 16, uniform(kt + first * 16));
    to_lds16(c.v + row * c.v_stride + L::piece(place, L::v_turn(t)) * 16, uniform(vt + first * 16));
  }
}

// ---- 8-bit codes: through registers, where they become 16-bit values --------------------------------------------------------------------
template <typename V>
__device__ __forceinline__ void arrived(V &x) {
  asm volatile("" : "+v"(x));
}
// 16 codes of row t of a tile of D 16-bit elements at `base`
template <typename T, int D>
__device__ __forceinline__ void write_codes(uint32_t base, int t, int turn, int piece, u32x4 codes, float power) {
  using L = Tile<D>;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(base + t * L::ROW + L::place(2 * piece + h, turn) * 16) =
        as<u32x4>(values_of<T>(u32x2{codes[2 * h], codes[2 * h + 1]}, power));
}

// The part of a tile of N tokens that one of WAVES waves brings, K and V alike: a tile ahead, in registers.  (1000 tokens over 15000, 32 query and 8 key
// heads of 128, bf16: 272 us, 266 over 16 bits; heads of 256 782 and 744.  500 over 11500 among 31 decoding requests 143 and 161.)
template <int D, int N, int WAVES>
struct TileCodes {
  static constexpr int P = D / 16, ALL = N * P, EACH = (ALL + 64 * WAVES - 1) / (64 * WAVES);
  u32x4 k[EACH], v[EACH];
  uint32_t e[EACH];

  static __device__ __forceinline__ bool has(int unit) { return ALL % (64 * WAVES) == 0 || unit < ALL; }
  __device__ __forceinline__ void load(const Cache &c, int base, uint32_t slice, int wave, int lane) {
    int32_t pages[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int unit = min((i * WAVES + wave) * 64 + lane, ALL - 1);
      pages[i] = lds_word(slice + unit / P * 4);
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int unit = min((i * WAVES + wave) * 64 + lane, ALL - 1), t = unit / P, piece = unit - t * P;
      const Slot<D> s(c, base + t, pages[i]);
      k[i] = *reinterpret_cast<const u32x4 *>(s.k(c) + piece * 16);
      v[i] = *reinterpret_cast<const u32x4 *>(s.v(c) + piece * 16);
      e[i] = s.powers(c);
    }
    requested();
  }
  template <typename T>
  __device__ __forceinline__ void write(uint32_t kt, uint32_t vt, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      arrived(k[i]);
      arrived(v[i]);
      arrived(e[i]);
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int unit = (i * WAVES + wave) * 64 + lane, t = unit / P, piece = unit - t * P;
      if (!has(unit)) continue;
      write_codes<T, D>(kt, t, Tile<D>::k_turn(t), piece, k[i], k_power(e[i]));
      write_codes<T, D>(vt, t, Tile<D>::v_turn(t), piece, v[i], v_power(e[i]));
    }
  }
};

// A wave's tile of 32 tokens.  K goes into the first product as it comes: lane (row, kg) holds, of tokens `row` and 16 + row, the 16 elements
// from 16 kg on of each 64, and the 8 from 8 kg on of 32 that are left; q is read in that order too.  Powers are loaded once a token,
// by lane token and token + 32, and go round by ds_bpermute: loaded by each lane that needs one, they were 40 % of the look-ups
// in the L1 (256 requests of 200 to 2000 tokens, 32 heads, 344 us; then 326).  What was left of their cost is lines: 13 us of those 326 for the ones
// that hold the powers of a page of 2 tokens, which every XCD reads.  At that step, with two workgroups a CU, the loads of this loop took 319
// without its work, of 1.70 GB; with codes of two tiles on their way (at 234 registers) it was no faster.
template <int D>
struct WaveCodes {
  static constexpr int B = D / 64, REST = D % 64 / 32, P = D / 16, EACH = D / 32;
  u32x4 k[2][B + 1], v[EACH];
  u32x2 rest[2];
  uint32_t e;

  // first element of the lane's eight of chunk i
  static __device__ __forceinline__ int element(int i, int kg) { return i < 2 * B ? i / 2 * 64 + kg * 16 + i % 2 * 8 : B * 64 + kg * 8; }
  __device__ __forceinline__ void load(const Cache &c, int base, uint32_t slice, int lane) {
    const int lrow = lane & 15, kg = lane >> 4;
    int32_t pages[2], vpages[EACH];
    const int32_t its = lds_word(slice + (lane & 31) * 4);
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) pages[tt] = lds_word(slice + (tt * 16 + lrow) * 4);
#pragma unroll
    for (int i = 0; i < EACH; ++i) vpages[i] = lds_word(slice + (i * 64 + lane) / P * 4);
    e = Slot<D>(c, base + (lane & 31), its).powers(c);
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const char *p = Slot<D>(c, base + tt * 16 + lrow, pages[tt]).k(c);
#pragma unroll
      for (int b = 0; b < B; ++b) k[tt][b] = *reinterpret_cast<const u32x4 *>(p + b * 64 + kg * 16);
      if constexpr (REST) rest[tt] = *reinterpret_cast<const u32x2 *>(p + B * 64 + kg * 8);
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int unit = i * 64 + lane, t = unit / P, piece = unit - t * P;
      v[i] = *reinterpret_cast<const u32x4 *>(Slot<D>(c, base + t, vpages[i]).v(c) + piece * 16);
    }
    requested();
  }
  __device__ __forceinline__ uint32_t powers(int token) const { return (uint32_t)__builtin_amdgcn_ds_bpermute(token * 4, (int)e); }
  __device__ __forceinline__ void keys_arrived() {
    arrived(e);
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
      for (int b = 0; b < B; ++b) arrived(k[tt][b]);
      if constexpr (REST) arrived(rest[tt]);
    }
  }
  template <typename T>
  __device__ __forceinline__ typename Traits<T>::vec8 key(int tt, int i, float power) const {
    const u32x2 w = i < 2 * B ? u32x2{k[tt][i / 2][i % 2 * 2], k[tt][i / 2][i % 2 * 2 + 1]} : rest[tt];
    return values_of<T>(w, power);
  }
  template <typename T>
  __device__ __forceinline__ void write_values(uint32_t vt, int lane) {
    uint32_t ve[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) ve[i] = powers((i * 64 + lane) / P);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      arrived(v[i]);
      const int unit = i * 64 + lane, t = unit / P, piece = unit - t * P;
      write_codes<T, D>(vt, t, Tile<D>::v_turn(t), piece, v[i], v_power(ve[i]));
    }
  }
};

// ---- running maximum and sum of a lane's row ---------------------------------------------------------------------------------
// A weight is 2^(c x - m) of a score x.  Where scores are so large that c times the highest is off by more than 1 when it is rounded
// (2^25 and more), m does not fit it and weights could be infinite or 0: the row's sums are made no numbers, and the careful sweep does it
// again relative to the highest score itself, 2^(c (x - highest) - AHEAD), two instructions instead of one.
template <typename T>
struct Softmax {
  float m = -INFINITY;       // reference, in powers of two (in a careful sweep the highest score); -infinity: nothing seen yet
  float minus = 0.0f;        // -m, or 0
  float limit = -INFINITY;   // a score this much above m moves it
  float l = 0.0f;            // sum of the weights as the product takes them
  float sum = 0.0f;          // and of the weights before they are rounded (where the row's logarithm is wanted)

  // how far a score lies above the reference, in powers of two
  template <bool CAREFUL>
  __device__ __forceinline__ float above(float x, float c) const {
    return CAREFUL ? fmaf(x + minus, c, -Wide<T>::FAR) : fmaf(x, c, minus);
  }
  // the reference goes by the highest score seen; returns what accumulators are scaled by
  template <bool CAREFUL>
  __device__ __forceinline__ float move(float highest, float c) {
    constexpr float AHEAD = CAREFUL ? Wide<T>::FAR : Wide<T>::AHEAD;
    const float top = highest * c;
    const float to = fmaxf(m, CAREFUL ? highest : top + AHEAD);
    float alpha = m == -INFINITY ? 0.0f : exp2_(CAREFUL ? (m - to) * c : m - to);
    if (!CAREFUL && fabsf(fmaf(highest, c, -top)) > 1.0f) alpha = NAN;
    const bool none = to == -INFINITY;
    m = to;
    minus = none ? 0.0f : -to;
    limit = none ? -INFINITY : GROWTH - AHEAD;
    l *= alpha;
    sum *= alpha;
    return alpha;
  }
};

// Logarithm of a row's sum, in powers of two; -infinity: the row gives no weights, as it sees nothing, or as the logarithm is so large
// (2^22) that half of the sum and more is lost in its last bit
__device__ __forceinline__ float row_log(float m, float sum) {
  const float x = m + log2f(sum);
  return sum == 0.0f || fabsf(x) >= 0x1p22f ? -INFINITY : x;
}

// ---- V that is not finite, or as large as its type holds ----------------------------------------------------------------------
// A token that a row does not see has weight 0, and 0 times an infinity is not 0 but no number, which then stays in the row's sums
// whatever they are scaled by.  Rows whose sums are not finite at the end of a piece, or so large (2^61 and more) that those of several pieces
// might not be, are therefore done again the careful way (a loop of its own, which costs the common one no registers and no look at V):
// the product runs over the finite values alone, and a second one counts for each row and column the others that the row does see:
// +infinity as 1, -infinity as 128, not a number as 16384 (at most 64 tokens a sum).
template <typename V, int N, int W = sizeof(V) / 4>
__device__ __forceinline__ bool any_too_large(const V (&x)[N]) {
  float squares = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) squares = fmaf(x[i][j], x[i][j], squares);
  return __any(!(squares < INFINITY));
}
template <typename T>
__device__ __forceinline__ void split_not_finite(u32x4 &v, u32x4 &code) {
  constexpr uint32_t E = Wide<T>::EXPONENT;
  const uint32_t one = Traits<T>::from_float(1.0f), low = Traits<T>::from_float(128.0f), odd = Traits<T>::from_float(16384.0f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t fin = 0, cod = 0;
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      const uint32_t x = v[i] >> h & 0xffffu;
      const uint32_t which = x & (0x7fffu ^ E) ? odd : x & 0x8000u ? low : one;
      fin |= ((x & E) == E ? 0u : x) << h;
      cod |= ((x & E) == E ? which : 0u) << h;
    }
    v[i] = fin;
    code[i] = cod;
  }
}
__device__ __forceinline__ float not_finite(float code) {
  const int n = (int)code;
  const float plus = n & 127 ? INFINITY : 0.0f, minus = n & 16256 ? -INFINITY : 0.0f;
  return n >> 14 ? NAN : plus + minus;
}

// ---- few rows: up to 16, every wave on tokens of its own ------------------------------------------------------------------------
// Decoding: bound by the bytes of K and V.  Each wave streams tiles of 32 tokens through a K and a V buffer of its own, without
// barriers: K of the next tile is asked for as soon as the scores are there, V as soon as the product is, so one of the two is
// always on its way.  At the end the waves' sums are joined through LDS.  (D = 128, fp16: 256 requests of 200 to 2000 tokens, 32 key
// heads, 597 us, 5.6 TB/s; rows of 256 bytes scattered over memory are read at 5.8 by a kernel that does nothing else.  bf16,
// group 4: 5 of 30000 to 70000 tokens in pages of 16, 225 us, 5.2 TB/s.  One of 517 tokens 8.3 us: the launch, five round trips,
// the join.)
// Over codes K and V of a tile come into registers together, those of the next as soon as these have been used; V alone goes through LDS.  (The
// same requests, pages of 2 and of 16: 313 us, 5.4 TB/s; 117, 5.1, of which the loads alone take 112; 8.2.)
constexpr int FEW_TOKENS = 32, THREADS = 256;
template <int D, bool CODES>
struct Few {
  static constexpr int WAVES = D <= 128 || CODES ? 4 : 2;     // that have tokens (the buffers of two fill the room at 256)
  static constexpr uint32_t TILE = FEW_TOKENS * D * 2, SLICES = 4;
  static constexpr uint32_t WAVE = (CODES ? 1 : 2) * TILE + SLICES * 256, TOTAL = WAVES * WAVE;      // (codes: V alone)
  static constexpr int O_STRIDE = D + 4;                      // floats of a row of a wave's sums
  static_assert(WAVES * FEW_ROWS * (O_STRIDE + 4) * 4 <= TOTAL, "the sums fit where the tiles were");
};

// Sums of several pieces or waves: {reference, sum of the rounded weights, sum of the weights} and the lane's four columns
struct Joined {
  float m = -INFINITY, l = 0.0f, sum = 0.0f;
  f32x4 x{0, 0, 0, 0};

  __device__ __forceinline__ void add(float4 ml, f32x4 o) {
    if (ml.x == -INFINITY && ml.y == 0.0f) return;            // saw nothing (scores that are no numbers leave no reference, but a sum)
    const float to = fmaxf(m, ml.x), mine = m == -INFINITY ? 0.0f : exp2_(m - to), its = exp2_(ml.x - to);
    m = to;
    l = l * mine + ml.y * its;
    sum = sum * mine + ml.z * its;
    x = x * mine + o * its;
  }
};

template <typename T, int D>
__device__ __forceinline__ void write_row(const AttnArgs &a, int tok, int head, int d, const Joined &j) {
  const float inv = j.l == 0.0f ? 0.0f : 1.0f / j.l;
  const uint2 y{Wide<T>::pack(j.x[0] * inv, j.x[1] * inv), Wide<T>::pack(j.x[2] * inv, j.x[3] * inv)};
  *reinterpret_cast<uint2 *>(a.out + (int64_t)tok * a.out_stride + head * D + d) = y;
  if (a.lse && d == 0) a.lse[(int64_t)tok * a.q_heads + head] = row_log(j.m, j.sum);
}

// Stores and loads that other XCDs see and that see what they stored: past the L2, which the XCDs do not share
__device__ __forceinline__ void store_shared(void *p, f32x4 v) {
  typedef __attribute__((address_space(1))) u32x4 *GP;
  __builtin_amdgcn_global_store_b128((GP)(uintptr_t)p, as<u32x4>(v), "agent");
}
__device__ __forceinline__ f32x4 load_shared(const void *p) {
  typedef __attribute__((address_space(1))) u32x4 *GP;
  return as<f32x4>(__builtin_amdgcn_global_load_b128((GP)(uintptr_t)p, "agent"));
}

template <typename T, int D, bool SUMS, bool CODES>
__device__ __forceinline__ void few_tile(const AttnArgs &a, char *lds, int rec_i, int head) {
  using F = Few<D, CODES>;
  using L = Tile<D>;
  constexpr int WAVES = F::WAVES, CH = D / 32, DB = D / 16;
  using vec8 = typename Traits<T>::vec8;
  const Record rec(a.plan, a.off_few, rec_i);
  const int req = rec.w[0], row0 = rec.w[1], rows = rec.w[2] & 0xffff, join = rec.w[2] >> 16, slot = rec.w[5], tok0 = rec.w[6], pos0 = rec.w[7];
  if (rec_i >= a.plan[AH_FEW] || rows <= 0) return;
  const int lane = threadIdx.x & 63, wave = (int)uniform(threadIdx.x >> 6);
  const int lrow = lane & 15, kg = lane >> 4;
  const Cache c = cache_of<D, CODES>(a, req, head, rec.w[3], rec.w[4]);
  const uint32_t mem = lds_offset(lds) + wave * F::WAVE, kt = mem, vt = CODES ? mem : mem + F::TILE, slices = vt + F::TILE;

  const int tiles = (c.end - c.begin + FEW_TOKENS - 1) / FEW_TOKENS;
  const int mine = wave < WAVES && tiles > wave ? (tiles - wave + WAVES - 1) / WAVES : 0;
  auto base_of = [&](int k) { return c.begin + (wave + k * WAVES) * FEW_TOKENS; };

  // the lane's row: q, and what it sees
  const int row = row0 + min(lrow, rows - 1);
  const int tok = row / a.group, hq = head * a.group + row - tok * a.group;
  const int last = pos0 + tok, from = a.window > 0 ? last - a.window + 1 : 0;
  // with weights: where the lane's scores go, token 0 of the cache at 0 (null: nowhere)
  float *scores = nullptr;
  if constexpr (SUMS) {
    const int32_t *rq = a.plan + a.off_requests + (int64_t)req * AT_REC;
    const int64_t its = (int64_t)((uint64_t)(uint32_t)rq[5] | (uint64_t)(uint32_t)rq[6] << 32);
    const int first = a.window > 0 && pos0 + 1 > a.window ? pos0 + 1 - a.window : 0;
    if (a.plan[AH_SCORES] && lrow < rows) scores = a.scores + its + ((int64_t)head * rows + lrow) * rq[7] - first;
  }
  const int sure_from = a.window > 0 ? pos0 + (row0 + rows - 1) / a.group - a.window + 1 : 0, sure_last = pos0 + row0 / a.group;
  const uint16_t *qp = a.q + (int64_t)(tok0 + tok) * a.q_stride + hq * D;
  vec8 q[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) q[i] = as<vec8>(load16(qp + (CODES ? WaveCodes<D>::element(i, kg) : i * 32 + kg * 8)));
  arrived(q);

  f32x4 o[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) o[i] = f32x4{0, 0, 0, 0};        // (a wave may have no tile)
  Softmax<T> sm;

  constexpr int EACH = FEW_TOKENS * L::P / 64;                  // loads of a tile of K, as of V
  uint32_t rows_of[EACH];                                       // pool rows of the tile whose K was asked for last
  auto load_k = [&](int k) {
    int32_t pages[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) pages[i] = lds_word(slices + (k & 3) * 256 + (i * 64 + lane) / L::P * 4);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int unit = i * 64 + lane, t = unit / L::P, place = unit - t * L::P;
      rows_of[i] = row_of(c, base_of(k) + t, pages[i]);
      to_lds16(c.k + (uint64_t)rows_of[i] * c.k_stride + L::piece(place, L::k_turn(t)) * 16, uniform(kt + i * 1024));
    }
    load_pages(c, base_of(k + 2), slices + ((k + 2) & 3) * 256, lane & 31);
  };
  auto load_v = [&] {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int unit = i * 64 + lane, t = unit / L::P, place = unit - t * L::P;
      to_lds16(c.v + (uint64_t)rows_of[i] * c.v_stride + L::piece(place, L::v_turn(t)) * 16, uniform(vt + i * 1024));
    }
  };
  // (the page numbers that are asked for first have come when the codes have)
  [[maybe_unused]] WaveCodes<D> codes;
  auto load_codes = [&](int k) {
    load_pages(c, base_of(k + 1), slices + ((k + 1) & 3) * 256, lane & 31);
    codes.load(c, base_of(k), slices + (k & 3) * 256, lane);
  };
  auto step = [&](auto careful, int k) {
    constexpr bool CAREFUL = decltype(careful)::value;
    const bool more = k + 1 < mine;
    const int base = base_of(k);
    // K has come; V and the page numbers of a later tile are on their way
    if constexpr (CODES) {
      if constexpr (CAREFUL) load_codes(k);                     // (none ahead: the registers of this loop, the rare one, decide how many workgroups a CU holds)
      codes.keys_arrived();
    } else {
      wait_vmcnt<EACH + 1>();
    }
    f32x4 s[2];
    [[maybe_unused]] uint32_t powers[2];
    if constexpr (CODES)
      for (int tt = 0; tt < 2; ++tt) powers[tt] = codes.powers(tt * 16 + lrow);
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      s[tt] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if constexpr (CODES) s[tt] = Traits<T>::mfma(codes.template key<T>(tt, i, k_power(powers[tt])), q[i], s[tt]);
        else s[tt] = Traits<T>::mfma(as<vec8>(lds16(L::k_at(kt, lrow, kg, i * 4) + tt * 16 * L::ROW)), q[i], s[tt]);
      }
    }
    const uint32_t bad = (uint32_t)__ballot(bad_page(c, lds_word(slices + (k & 3) * 256 + (lane & 31) * 4)));
    if constexpr (CODES) {
      codes.template write_values<T>(vt, lane);
      if (!CAREFUL && more) load_codes(k + 1);
    } else {
      wait_lgkmcnt0();
      if (more) load_k(k + 1);
    }
    uint32_t seen = 0;                                          // bit tt * 16 + i: the lane's row sees token tt * 16 + kg * 4 + i
    const bool masked = CAREFUL || base < sure_from || base + FEW_TOKENS - 1 > sure_last || base + FEW_TOKENS > c.end || bad;
    if (masked) {
      seen = (uint32_t)(run(from - base, min(last, c.end - 1) - base) & ~(uint64_t)bad) >> kg * 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = unless(s[i >> 2][i & 3], bit(seen, (i >> 2) * 16 + (i & 3)));
    }
    float hi = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) hi = fmaxf(hi, s[i >> 2][i & 3]);
    if (__any(sm.template above<CAREFUL>(hi, a.c) > sm.limit)) {
      hi = fmaxf(hi, __shfl_xor(hi, 16));
      hi = fmaxf(hi, __shfl_xor(hi, 32));
      const float alpha = sm.template move<CAREFUL>(hi, a.c);
#pragma unroll
      for (int i = 0; i < DB; ++i) o[i] *= alpha;
    }
    u32x4 p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (the sum is that of the rounded weights, which the product takes: a row that looks at one token gets exactly its v)
      const float x = s[i >> 1][(i & 1) * 2], y = s[i >> 1][(i & 1) * 2 + 1];
      const float ex = exp2_(sm.template above<CAREFUL>(x, a.c)), ey = exp2_(sm.template above<CAREFUL>(y, a.c));
      p[i] = Wide<T>::pack(ex, ey);
      sm.l = Wide<T>::add2(p[i], sm.l);
      if constexpr (SUMS) sm.sum += ex + ey;
    }
    // (what is stored below is counted too, and only makes the waits stricter)
    if constexpr (!CODES) {
      if (more) wait_vmcnt<EACH + 1>();
      else wait_vmcnt<0>();
    }
    if constexpr (SUMS && !CAREFUL) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const int j = base + tt * 16 + kg * 4;
        if (scores && j < c.end) *reinterpret_cast<f32x4 *>(scores + j) = s[tt];
      }
    }
    const int vtok = kg * 4 + (lrow >> 2);
    auto values = [&](int db) {
      const uint32_t at = L::v_at(vt + (lane & 1) * 8, vtok, (lane & 3) >> 1, 2 * db);
      struct { s16x4 lo, hi; } v{lds_turned(at), lds_turned(at + 16 * L::ROW)};
      return as<u32x4>(v);
    };
    if constexpr (!CAREFUL) {
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = Traits<T>::mfma(as<vec8>(values(db)), as<vec8>(p), o[db]);
    } else {
      u32x4 ones;
#pragma unroll
      for (int i = 0; i < 4; ++i) ones[i] = ones2<T>(bit(seen, (i >> 1) * 16 + (i & 1) * 2), bit(seen, (i >> 1) * 16 + (i & 1) * 2 + 1));
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        u32x4 v = values(db), code;
        split_not_finite<T>(v, code);
        o[db] = Traits<T>::mfma(as<vec8>(v), as<vec8>(p), o[db]);
        const f32x4 n = Traits<T>::mfma(as<vec8>(code), as<vec8>(ones), f32x4{0, 0, 0, 0});
#pragma unroll
        for (int i = 0; i < 4; ++i) o[db][i] += not_finite(n[i]);
        one_by_one();
      }
    }
    if constexpr (!CODES) {
      wait_lgkmcnt0();
      if (more) load_v();
    }
  };
  auto sweep = [&](auto careful) {
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x4{0, 0, 0, 0};
    sm = Softmax<T>();
    load_pages(c, base_of(0), slices, lane & 31);
    load_pages(c, base_of(1), slices + 256, lane & 31);
    wait_vmcnt<0>();
    if constexpr (CODES) {
      if constexpr (!decltype(careful)::value) load_codes(0);
    } else {
      load_k(0);
      load_v();
    }
    for (int k = 0; k < mine; ++k) step(careful, k);
    if (decltype(careful)::value) sm.m = fmaf(sm.m, a.c, Wide<T>::FAR);
  };
  if (mine > 0) {
    sweep(std::false_type{});
    if (any_too_large(o)) sweep(std::true_type{});
  }

  // ---- the waves' sums
  sm.l += __shfl_xor(sm.l, 16);
  sm.l += __shfl_xor(sm.l, 32);
  if constexpr (SUMS) {
    sm.sum += __shfl_xor(sm.sum, 16);
    sm.sum += __shfl_xor(sm.sum, 32);
  }
  float *so = reinterpret_cast<float *>(lds);                   // [wave][row][O_STRIDE]
  float4 *ml = reinterpret_cast<float4 *>(so + WAVES * FEW_ROWS * F::O_STRIDE);
  __syncthreads();
  if (wave < WAVES) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
      *reinterpret_cast<f32x4 *>(so + (wave * FEW_ROWS + lrow) * F::O_STRIDE + db * 16 + kg * 4) = o[db];
    if (kg == 0) ml[wave * FEW_ROWS + lrow] = float4{sm.m, sm.l, sm.sum, 0.0f};
  }
  __syncthreads();
  constexpr int COLS = D / 4, SLOTS = THREADS / COLS;           // threads of a row, rows at a time
  const int ty = threadIdx.x / COLS, d = (threadIdx.x - ty * COLS) * 4;
  const int64_t step_ml = (int64_t)a.kv_heads * FEW_ROWS;       // rows from a slot to the next
  if (ty < SLOTS)
    for (int r = ty; r < rows; r += SLOTS) {
      Joined j;
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
        j.add(ml[w * FEW_ROWS + r], *reinterpret_cast<const f32x4 *>(so + (w * FEW_ROWS + r) * F::O_STRIDE + d));
      if (slot < 0) {
        const int t = (row0 + r) / a.group;
        write_row<T, D>(a, tok0 + t, head * a.group + row0 + r - t * a.group, d, j);
      } else {
        const int64_t at = slot * step_ml + head * FEW_ROWS + r;
        store_shared(a.few_o + at * D + d, j.x);
        if (d == 0) store_shared(a.few_ml + at, f32x4{j.m, j.l, j.sum, 0.0f});
      }
    }
  if (slot < 0) return;

  // ---- the pieces' sums: whoever of a tile's pieces comes last joins them, in their order
  const int32_t *jn = a.plan + a.off_joins + (int64_t)join * AT_REC;
  const int slot0 = jn[0], pieces = jn[1];
  uint32_t *arrive = reinterpret_cast<uint32_t *>(const_cast<int32_t *>(a.plan) + a.off_arrive) + (int64_t)join * a.kv_heads + head;
  int *flag = reinterpret_cast<int *>(lds);
  wait_vmcnt<0>();                                              // its sums are where the others see them
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t before = __hip_atomic_fetch_add(arrive, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before + 1 == (uint32_t)pieces) __hip_atomic_store(arrive, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next call
    *flag = before + 1 == (uint32_t)pieces;
  }
  __syncthreads();
  if (!*flag) return;
  __syncthreads();
  // Rows times COLS threads go over the pieces; where there are threads for it, several groups take turns, joined through LDS
  const int groups = rows < SLOTS ? SLOTS / rows : 1;
  const int grp = rows < SLOTS ? ty / rows : 0;
  const int64_t first = slot0 * step_ml + head * FEW_ROWS;
  for (int r = rows < SLOTS ? ty - grp * rows : ty; r < rows; r += SLOTS) {
    Joined j;
    if (ty < SLOTS && grp < groups) {
      constexpr int AHEAD = 4;
      for (int i = grp; i < pieces; i += AHEAD * groups) {
        f32x4 x[AHEAD], p[AHEAD];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) {
          const int64_t at = first + min(i + n * groups, pieces - 1) * step_ml + r;
          p[n] = load_shared(a.few_ml + at);
          x[n] = load_shared(a.few_o + at * D + d);
        }
#pragma unroll
        for (int n = 0; n < AHEAD; ++n)
          if (i + n * groups < pieces) j.add(as<float4>(p[n]), x[n]);
      }
    }
    if (groups > 1) {
      if (ty < SLOTS && grp < groups) {
        *reinterpret_cast<f32x4 *>(so + ty * F::O_STRIDE + d) = j.x;
        if (d == 0) *reinterpret_cast<float4 *>(so + ty * F::O_STRIDE + D) = float4{j.m, j.l, j.sum, 0.0f};
      }
      __syncthreads();
      if (ty >= rows) return;
      for (int g = 1; g < groups; ++g) {
        const float *other = so + (g * rows + r) * F::O_STRIDE;
        j.add(*reinterpret_cast<const float4 *>(other + D), *reinterpret_cast<const f32x4 *>(other + d));
      }
    }
    if (ty < SLOTS && grp == 0) {
      const int t = (row0 + r) / a.group;
      write_row<T, D>(a, tok0 + t, head * a.group + row0 + r - t * a.group, d, j);
    }
  }
}

// ---- tall tiles: 32 rows a wave, K and V shared by the workgroup ------------------------------------------------------------------
// Prompts.  K and V of 64 tokens (two buffers, 64 KB) come in while the 64 before are worked on; a wave keeps its q and its
// accumulators in registers, two waves a SIMD.  1000 tokens over 31000, 32 query and 8 key heads, D = 128, fp16, the whole call in a run of
// passes: 547 to 588 us by the card, 880 to 945 TFLOP/s; a large fp16 product of the library reaches 1180.  (The first passes after the
// device was idle are slower, up to 770 us, while its clock settles; the forty of a trace have a median of 598.)  The matrix units are busy
// for 48 % of the cycles (two products of 1024 cycles a SIMD against some 900 of exponentials and sums and 512 of loads into LDS, which
// overlap in part), at 1.8 GHz of the 2.4 that short launches run at.  16 prompts of 272 to 384 tokens, 32 key heads, bf16: 51 to 53 us for
// the 123 MB read and 41 written that it takes, 3.2 TB/s, the matrix units busy for 14 %: neither bounds it, but that a workgroup is
// short beside its start and end (record, page numbers, first tile, one after the other).
constexpr int TALL_WAVES = TALL_ROWS / 32;
template <int D>
struct Tall {
  static constexpr int TOKENS = D <= 128 ? 64 : 32;          // of a tile (scores and accumulators have to fit the registers)
  static constexpr uint32_t TILE = TOKENS * D * 2, BUFFER = 2 * TILE, SLICES = 4, TOTAL = 2 * BUFFER + TALL_WAVES * SLICES * 256;
};

template <typename T, int D, bool SUMS, bool CODES>
__device__ __forceinline__ void tall_tile(const AttnArgs &a, char *lds, int rec_i, int head) {
  using F = Tall<D>;
  using L = Tile<D>;
  constexpr int CH = D / 16, DB = D / 32, TOKENS = F::TOKENS, BL = TOKENS / 32, AHEAD = 4;
  using vec8 = typename Traits<T>::vec8;
  int *again = reinterpret_cast<int *>(lds + F::TOTAL);         // the tile's rows are done again the careful way
  const Record rec(a.plan, a.off_tall, rec_i);
  const int req = rec.w[0], row0 = rec.w[1], rows = rec.w[2], slot = rec.w[5], tok0 = rec.w[6], pos0 = rec.w[7];
  if (rows <= 0) return;
  const int lane = threadIdx.x & 63, wave = (int)uniform(threadIdx.x >> 6);
  const int lrow = lane & 31, half = lane >> 5;
  const Cache c = cache_of<D, CODES>(a, req, head, rec.w[3], rec.w[4]);
  const uint32_t mem = lds_offset(lds), slices = mem + 2 * F::BUFFER + wave * F::SLICES * 256;
  const int tiles = (c.end - c.begin + TOKENS - 1) / TOKENS;
  auto base_of = [&](int k) { return c.begin + k * TOKENS; };

  const int wrow = wave * 32;                                   // the wave's rows: [wrow, wrow + wrows) of the tile
  const int wrows = min(32, rows - wrow);
  const bool works = wrows > 0;
  const int row = row0 + (works ? wrow + min(lrow, wrows - 1) : 0);
  const int tok = row / a.group, hq = head * a.group + row - tok * a.group;
  const int last = pos0 + tok, from = a.window > 0 ? last - a.window + 1 : 0;
  const int first_tok = (row0 + wrow) / a.group, last_tok = (row0 + wrow + (works ? wrows : 1) - 1) / a.group;
  const int sure_from = a.window > 0 ? pos0 + last_tok - a.window + 1 : 0, sure_last = pos0 + first_tok;   // all its rows see these,
  const int any_from = a.window > 0 ? pos0 + first_tok - a.window + 1 : 0, any_last = pos0 + last_tok;     // and some row these
  const uint16_t *qp = a.q + (int64_t)(tok0 + tok) * a.q_stride + hq * D;
  vec8 q[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) q[i] = as<vec8>(load16(qp + i * 16 + half * 8));
  arrived(q);

  f32x16 o[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) o[i] = f32x16{};                 // (there may be no tile)
  Softmax<T> sm;

  auto compute = [&](auto careful, int k, uint64_t bad) {
    constexpr bool CAREFUL = decltype(careful)::value;
    const int base = base_of(k);
    const uint32_t kt = mem + (k & 1) * F::BUFFER, vt = kt + F::TILE;
    // Both products read LDS AHEAD steps before the matrix instruction that takes it, in an order of their own: left to itself the
    // compiler reads right before it, and waits.
    vec8 ks[AHEAD];
    auto key = [&](int n) { return as<vec8>(lds16(L::k_at(kt, lrow, half, n / BL * 2) + n % BL * 32 * L::ROW)); };
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) ks[n] = key(n);
    f32x16 s[BL];
#pragma unroll
    for (int b = 0; b < BL; ++b) s[b] = f32x16{};
#pragma unroll
    for (int n = 0; n < BL * CH; ++n) {
      s[n % BL] = Wide<T>::mfma(ks[n % AHEAD], q[n / BL], s[n % BL]);
      if (n + AHEAD < BL * CH) ks[n % AHEAD] = key(n + AHEAD);
      one_by_one();
    }
    // tokens 16 g + 4 half .. + 3 and 8 further, of the lane's column of 32 from 32 db on
    const int vtok = half * 4 + ((lane & 15) >> 2);
    auto values = [&](int g, int db) {
      const uint32_t at = L::v_at(vt + (lane & 1) * 8, vtok, (lane >> 4 & 1) * 2 + ((lane & 3) >> 1), 4 * db) + g * 16 * L::ROW;
      struct { s16x4 lo, hi; } v{lds_turned(at), lds_turned(at + 8 * L::ROW)};
      return as<u32x4>(v);
    };
    uint32_t seen[BL] = {};                                     // bit 8 x + i of b: the lane's row sees token 32 b + 8 x + 4 half + i
    // (one way for all tiles: two would keep the accumulators twice)
    if (CAREFUL || base < sure_from || base + TOKENS - 1 > sure_last || base + TOKENS > c.end || bad) {
      const uint64_t sees = (run(from - base, min(last, c.end - 1) - base) & ~bad) >> half * 4;
#pragma unroll
      for (int b = 0; b < BL; ++b) {
        seen[b] = (uint32_t)(sees >> 32 * b);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = unless(s[b][i], bit(seen[b], (i >> 2) * 8 + (i & 3)));
      }
    }
    float hi = s[0][0];
#pragma unroll
    for (int i = 1; i < 16 * BL; ++i) hi = fmaxf(hi, s[i >> 4][i & 15]);
    if (__any(sm.template above<CAREFUL>(hi, a.c) > sm.limit)) {
      hi = fmaxf(hi, __shfl_xor(hi, 32));
      const float alpha = sm.template move<CAREFUL>(hi, a.c);
#pragma unroll
      for (int i = 0; i < DB; ++i) o[i] *= alpha;
    }
    u32x4 p[2 * BL];
    auto weigh = [&](int g, int i) {
      const float x = s[g >> 1][(g & 1) * 8 + 2 * i], y = s[g >> 1][(g & 1) * 8 + 2 * i + 1];
      const float ex = exp2_(sm.template above<CAREFUL>(x, a.c)), ey = exp2_(sm.template above<CAREFUL>(y, a.c));
      p[g][i] = Wide<T>::pack(ex, ey);
      sm.l = Wide<T>::add2(p[g][i], sm.l);
      if constexpr (SUMS) sm.sum += ex + ey;
    };
    if constexpr (!CAREFUL) {
      // between the matrix instructions of a group of 16 tokens the weights of the next; ahead of the SIMD's other wave, so that the
      // two come to differ in what they do (563 us instead of 598 for 1000 tokens over 31000, D = 128, group 4)
      __builtin_amdgcn_s_setprio(1);
      u32x4 vs[AHEAD];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) vs[n] = values(n / DB, n % DB);
#pragma unroll
      for (int i = 0; i < 4; ++i) weigh(0, i);
      one_by_one();
#pragma unroll
      for (int n = 0; n < 2 * BL * DB; ++n) {
        const int g = n / DB, db = n % DB;
        o[db] = Wide<T>::mfma(as<vec8>(vs[n % AHEAD]), as<vec8>(p[g]), o[db]);
        if (n + AHEAD < 2 * BL * DB) vs[n % AHEAD] = values((n + AHEAD) / DB, (n + AHEAD) % DB);
        if (g + 1 < 2 * BL)
#pragma unroll
          for (int i = db * 4 / DB; i < (db + 1) * 4 / DB; ++i) weigh(g + 1, i);
        one_by_one();
      }
      __builtin_amdgcn_s_setprio(0);
    } else {
#pragma unroll
      for (int g = 0; g < 2 * BL; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) weigh(g, i);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        f32x16 n{};
#pragma unroll
        for (int g = 0; g < 2 * BL; ++g) {
          u32x4 ones, v = values(g, db), code;
          uint32_t sees = seen[g >> 1];
          here(sees);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = (g & 1) * 16 + (i >> 1) * 8 + (i & 1) * 2;
            ones[i] = ones2<T>(bit(sees, at), bit(sees, at + 1));
          }
          split_not_finite<T>(v, code);
          o[db] = Wide<T>::mfma(as<vec8>(v), as<vec8>(p[g]), o[db]);
          n = Wide<T>::mfma(as<vec8>(code), as<vec8>(ones), n);
          one_by_one();
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] += not_finite(n[i]);
        one_by_one();
      }
    }
  };
  auto sweep = [&](auto careful) {
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x16{};
    sm = Softmax<T>();
    load_pages(c, base_of(0), slices, lane);
    load_pages(c, base_of(1), slices + 256, lane);
    wait_vmcnt<0>();
    [[maybe_unused]] TileCodes<D, TOKENS, TALL_WAVES> codes;
    if constexpr (CODES) {
      codes.load(c, base_of(0), slices, wave, lane);
    } else {
      load_tile<D, TOKENS, TALL_WAVES>(c, base_of(0), slices, mem, mem + F::TILE, wave, lane);
      load_pages(c, base_of(2), slices + 2 * 256, lane);
    }
    for (int k = 0; k < tiles; ++k) {
      // tile k has come, and every wave is through with the other buffer (codes: with what was in this one)
      if constexpr (CODES) {
        const uint32_t kt = mem + (k & 1) * F::BUFFER;
        codes.template write<T>(kt, kt + F::TILE, wave, lane);
        if (k + 1 < tiles) {
          load_pages(c, base_of(k + 2), slices + ((k + 2) & 3) * 256, lane);
          codes.load(c, base_of(k + 1), slices + ((k + 1) & 3) * 256, wave, lane);
        }
      } else {
        wait_vmcnt<0>();
      }
      wait_lgkmcnt0();
      __syncthreads();
      if (!CODES && k + 1 < tiles) {
        const uint32_t kt = mem + ((k + 1) & 1) * F::BUFFER;
        load_tile<D, TOKENS, TALL_WAVES>(c, base_of(k + 1), slices + ((k + 1) & 3) * 256, kt, kt + F::TILE, wave, lane);
        load_pages(c, base_of(k + 3), slices + ((k + 3) & 3) * 256, lane);
      }
      const int base = base_of(k);
      if (!works || base > any_last || base + TOKENS <= any_from) continue;
      const uint64_t bad = __ballot(bad_page(c, lds_word(slices + (k & 3) * 256 + lane * 4)));   // (lanes behind the tile: of later tokens)
      compute(careful, k, bad);
    }
    if (decltype(careful)::value) sm.m = fmaf(sm.m, a.c, Wide<T>::FAR);
  };
  if (tiles > 0) {
    if (threadIdx.x == 0) *again = 0;
    sweep(std::false_type{});
    if (any_too_large(o) && lane == 0) *again = 1;
    wait_lgkmcnt0();
    __syncthreads();                                            // (also: the buffers have been read by everyone)
    if (*again) {
      sweep(std::true_type{});
      __syncthreads();
    }
  }

  if (!works) return;
  sm.l += __shfl_xor(sm.l, 32);
  if constexpr (SUMS) sm.sum += __shfl_xor(sm.sum, 32);
  const int first = (int)uniform((uint32_t)(row0 + wrow));
  if (slot >= 0) {
    if (lrow < wrows) {
      const int64_t at = ((int64_t)slot * a.kv_heads + head) * TALL_ROWS + wrow + lrow;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4 *>(a.tall_o + at * D + db * 32 + i * 8 + half * 4) =
              f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
      if (half == 0) a.tall_ml[at] = float4{sm.m, sm.l, sm.sum, 0.0f};
    }
  } else {
    // A lane holds 16 bytes of columns here and there of one row: through LDS, which the wave has a part of to itself now, the
    // rows go out whole.
    const float inv = sm.l == 0.0f ? 0.0f : 1.0f / sm.l;
    constexpr int STRIDE = L::ROW + 16;
    static_assert(TALL_WAVES * 32 * STRIDE <= (int)F::TOTAL, "a part for each wave");
    char *mine = lds + wave * 32 * STRIDE;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint2 *>(mine + lrow * STRIDE + (db * 32 + i * 8 + half * 4) * 2) =
            uint2{Wide<T>::pack(o[db][4 * i] * inv, o[db][4 * i + 1] * inv), Wide<T>::pack(o[db][4 * i + 2] * inv, o[db][4 * i + 3] * inv)};
#pragma unroll
    for (int i = 0; i < L::P / 2; ++i) {
      const int unit = i * 64 + lane, r = unit / L::P, piece = unit - r * L::P;
      const int t = (first + r) / a.group, h = head * a.group + first + r - t * a.group;
      if (r < wrows) store16(a.out + (int64_t)(tok0 + t) * a.out_stride + h * D + piece * 8, *reinterpret_cast<const u32x4 *>(mine + r * STRIDE + piece * 16));
    }
    if (SUMS && half == 0 && lrow < wrows) {
      const int t = (first + lrow) / a.group, h = head * a.group + first + lrow - t * a.group;
      a.lse[(int64_t)(tok0 + t) * a.q_heads + h] = row_log(sm.m, sm.sum);
    }
  }
}

// ---- the launch: tall tiles first, which take longest ---------------------------------------------------------------------------------
enum { TALL_LIST = 1, FEW_LIST = 2 };

template <typename T, int D, bool SUMS, int LISTS, bool CODES>
__global__ __launch_bounds__(THREADS, D <= 128 ? 2 : 1) void attend_kernel(AttnArgs a) {
  using F = Few<D, CODES>;
  constexpr uint32_t ROOM = (CODES && LISTS == FEW_LIST) || F::TOTAL > Tall<D>::TOTAL + 16 ? F::TOTAL : Tall<D>::TOTAL + 16;
  __shared__ __align__(256) char lds[ROOM];
  const bool tall = LISTS == TALL_LIST || (LISTS != FEW_LIST && (int)blockIdx.x < a.tall_blocks);
  const unsigned block = blockIdx.x - (tall ? 0 : a.tall_blocks);
  // the key heads of a piece follow each other: they read the same pages, and what reads the same head's rows again is eight, or a
  // multiple of it, further where kv_heads is: on the same XCD
  int i = (int)(block / (unsigned)a.kv_heads), head = (int)(block - (unsigned)i * a.kv_heads);
  if (!tall) {
    if (CODES && a.heads_together) {
      // eight pieces at a time, all of whose heads follow each other on an XCD
      const int in8 = (i & 7) * a.kv_heads + head;
      i = (i & ~7) + (in8 & 7);
      head = in8 >> 3;
      if (i >= a.max_few) return;
    } else if (CODES && (a.kv_heads & 7) == 0) {
      // heads that are neighbours go to one XCD, which then reads of a page what lies side by side (256 requests of 32 heads, pages of 2,
      // 326 -> 321 us, 128 of 40 heads 213 -> 202; pages of 16 and of 1, and 16 heads, the same either way.  The L2s ask for as many bytes,
      // so it is not a line that they share; what it is was not found.)
      head = (head & 7) * (a.kv_heads >> 3) + (head >> 3);
    }
    few_tile<T, D, SUMS, CODES>(a, lds, i, head);
    return;
  }
  const int32_t *shares = a.plan + a.off_shares;
  if (i >= a.plan[AH_SHARES]) return;
  const int last = min(shares[i + 1], a.plan[AH_TALL]);
  for (int rec = shares[i]; rec < last; ++rec) {
    tall_tile<T, D, SUMS, CODES>(a, lds, rec, head);
    __syncthreads();                                            // (what the next one loads goes where this one's was)
  }
}

template <typename T, int D, bool SUMS, bool CODES>
int launch_lists(hipStream_t st, const AttnLayout &L, AttnArgs a) {
  // A head's codes of a page that are no whole lines share one with the next head's: those heads' workgroups go to one XCD, whose L2
  // then has the line.  (64 requests of 2000 tokens, 8 key heads, pages of 2, us apart / together: heads of 32 30.4 / 20.6, of 96 58.7 / 55.2;
  // whole lines: 32 heads of 128, 256 requests 343 / 358, as a page is then read by one XCD alone.)
  a.heads_together = CODES && ((D << a.page_shift) & 127) != 0;
  const int64_t few = (a.heads_together ? align_up(L.max_few, 8) : L.max_few) * a.kv_heads, tall = L.max_shares * a.kv_heads;
  if (few + tall > most_blocks(THREADS)) return fail(MLORA_ERR_NO_KERNEL, "paged_attention: too many tiles");
  a.tall_blocks = (int)tall;
  a.max_few = (int)L.max_few;
  // both lists in one kernel do not fit the scalar registers at 256; decoding over codes has a kernel without the room that tall tiles take
  const bool together = D <= 128 && (!CODES || tall > 0);
  if constexpr (D <= 128) {
    if (together) {
      hipLaunchKernelGGL((attend_kernel<T, D, SUMS, TALL_LIST | FEW_LIST, CODES>), dim3((unsigned)(tall + few)), dim3(THREADS), 0, st, a);
      return check_launch("attend_kernel");
    }
  }
  if constexpr (D > 128) {
    if (tall > 0) {
      hipLaunchKernelGGL((attend_kernel<T, D, SUMS, TALL_LIST, CODES>), dim3((unsigned)tall), dim3(THREADS), 0, st, a);
      if (int rc = check_launch("attend_kernel")) return rc;
    }
  }
  if constexpr (D > 128 || CODES) {
    a.tall_blocks = 0;
    // Over codes of 128 three workgroups have the registers of a CU, and where requests are whole and a page's heads no long run the third
    // helps.  A cut list fills two a CU to the end, and of three it leaves a third idle in its last round; of long runs more at once
    // part more from each other.  There room that nobody uses keeps the third out.  (us with two / three.  Whole: 256 requests of 32 heads,
    // pages of 2, 322 / 313, 400 of 8, pages of 16, 131 / 128; 200 of 32, pages of 8 and 64, 230 / 234 and 223 / 231.  Cut: 5 long 117 / 127,
    // 64 of 8 heads 62 / 65, and a list cut for three 119 and 65.  Heads of 32, 64 and 96 have the registers of five, four and three, and take
    // them: 64 requests of 2000, 8 key heads, with two / so 23.9 / 19.6, 34.2 / 32.0, 39.2 / 38.8.)  Lengths are not known here: that requests are
    // whole goes by how many can have new tokens, as if their lengths were alike; slots of the plan that have none do not count (5 long ones in 256 slots,
    // pages of 2 and of 16, 125.5 and 116.1, and 134.3 and 127.6 as if each slot had some).
    constexpr uint32_t THIRD = 56 << 10;                       // more than a third of a CU's room, less than half
    const bool third = L.few_whole && (int64_t)a.kv_heads << a.page_shift <= 128;
    const uint32_t unused = CODES && D == 128 && !third ? THIRD - Few<D, CODES>::TOTAL : 0;
    hipLaunchKernelGGL((attend_kernel<T, D, SUMS, FEW_LIST, CODES>), dim3((unsigned)few), dim3(THREADS), unused, st, a);
    return check_launch("attend_kernel");
  }
  return MLORA_OK;
}

// ---- joining the pieces of tall tiles ---------------------------------------------------------------------------------------------
// One workgroup per tile, key head and 16 rows; always in the order of the pieces.  (A launch of its own: a tile's pieces are 64 KB
// each, which one workgroup would be long about.  256 tiles in 2 to 4 pieces, 64 MB: 12 us, bytes; none: 4, a launch.)
constexpr int JOIN_ROWS = 16;

template <typename T, int D>
__global__ __launch_bounds__(THREADS) void attend_join_kernel(AttnArgs a) {
  constexpr int COLS = D / 4, SLOTS = THREADS / COLS;
  const int join_i = (int)(blockIdx.x / (unsigned)a.kv_heads), head = (int)(blockIdx.x - (unsigned)join_i * a.kv_heads);
  if (join_i >= a.plan[AH_TALL_JOINS]) return;
  const int32_t *join = a.plan + a.off_tall_joins + (int64_t)join_i * AT_REC;
  const int slot0 = join[0], pieces = join[1], rows = join[2], row0 = join[3], tok0 = join[4];
  if (pieces <= 0) return;
  const int ty = threadIdx.x / COLS, d = (threadIdx.x - ty * COLS) * 4;
  if (ty >= SLOTS) return;
  const int64_t step = (int64_t)a.kv_heads * TALL_ROWS;
  const int end = min((int)(blockIdx.y + 1) * JOIN_ROWS, rows);
  for (int r = blockIdx.y * JOIN_ROWS + ty; r < end; r += SLOTS) {
    const int64_t at = slot0 * step + head * TALL_ROWS + r;
    Joined j;
#pragma unroll 4
    for (int i = 0; i < pieces; ++i)
      j.add(a.tall_ml[at + i * step], *reinterpret_cast<const f32x4 *>(a.tall_o + (at + i * step) * D + d));
    const int t = (row0 + r) / a.group;
    write_row<T, D>(a, tok0 + t, head * a.group + row0 + r - t * a.group, d, j);
  }
}

// ---- weights: how much attention each cached token got ---------------------------------------------------------------------------
//     weights[b][j] += sum over the call's rows of exp(scale q.k_j - log sum)
// The sum of a row is not known before its last token.  Decoding tiles therefore leave their scores, 4 bytes for the 512 of a token's
// K and V that each query head of a group shares, and a thread sums those of a token.  (K read a second time: 64 requests of
// 1000 to 4100 tokens, 8 key heads, 68 us of 194.)  For tall tiles, and where the scores have no room, the keys are read again, for 64
// cached tokens at a time.  A weight is one sum in a fixed order either way.  (The same requests over 16 bits now: 14 us for leaving the
// scores, 15 for this launch, 149 in all.)

// The request whose run of blocks of WEIGHT_TOKENS holds the block, for everyone
__device__ __forceinline__ int request_of(const AttnArgs &a, int block, int *found) {
  const int32_t *requests = a.plan + a.off_requests;
  __syncthreads();
  for (int b = threadIdx.x; b < a.n_req; b += blockDim.x)
    if (requests[(int64_t)b * AT_REC] <= block && (b + 1 == a.n_req || block < requests[(int64_t)(b + 1) * AT_REC])) *found = b;
  __syncthreads();
  return (int)uniform((uint32_t)*found);
}

// What the kernels below take of a request's record
struct Weighed {
  int first_block, tok0, n, kv, pos0, rows, begin;
  __device__ __forceinline__ Weighed(const AttnArgs &a, const int32_t *rq)
      : first_block(rq[0]), tok0(rq[1]), n(rq[2]), kv(rq[3]), pos0(kv - n), rows(n * a.group),
        begin(a.window > 0 && pos0 + 1 > a.window ? pos0 + 1 - a.window : 0) {}
  __device__ __forceinline__ bool has_scores(const AttnArgs &a) const { return rows <= FEW_ROWS && a.plan[AH_SCORES]; }
};

// Where the scores are there: a thread a token of request b's block
__device__ __forceinline__ void sum_scores(const AttnArgs &a, const int32_t *rq, const Weighed &w, int b, int block) {
  const int j = w.begin + (block - w.first_block) * WEIGHT_TOKENS + (int)threadIdx.x;
  if (j >= w.kv) return;
  const float *sc = a.scores + (int64_t)((uint64_t)(uint32_t)rq[5] | (uint64_t)(uint32_t)rq[6] << 32) + (j - w.begin);
  const int stride = rq[7], n_rows = w.rows * a.kv_heads;
  auto share = [&](int r, int &tok) {
    const int head = r / w.rows, row = r - head * w.rows;
    tok = row / a.group;
    const float lse = a.lse[(int64_t)(w.tok0 + tok) * a.q_heads + head * a.group + row - tok * a.group];
    const float e = exp2_(fmaf(sc[(int64_t)r * stride], a.c, -lse));
    return lse == -INFINITY ? 0.0f : e;
  };
  float x = 0.0f;
  int tok;
#pragma unroll 8
  for (int r = 0; r < n_rows; ++r) x += share(r, tok);
  if (x != x) {
    // A row whose own sum is no number makes that of all tokens, where one that does not see this token (its score is -infinity)
    // would have added 0: once more, over the rows of the tokens [j - pos0, behind), which see it.
    const int32_t page = a.table[(int64_t)b * a.table_stride + (j >> a.page_shift)];
    const int behind = (uint32_t)page >= (uint32_t)a.n_pages ? 0 : a.window > 0 ? j - w.pos0 + a.window : w.n;
    x = 0.0f;
#pragma unroll 1
    for (int r = 0; r < n_rows; ++r) {
      const float e = share(r, tok);
      x += tok >= j - w.pos0 && tok < behind ? e : 0.0f;
    }
  }
  a.weights[(int64_t)b * a.weights_stride + j] += x;
}

// Where they are not: 64 cached tokens from `base` on, whose keys of a head are in kf, and that head's rows [first, last_row) of those that see any
template <typename T, int D>
__device__ __forceinline__ void sum_rows(const AttnArgs &a, const Weighed &rq, const typename Traits<T>::vec8 (&kf)[4][D / 32], int head, int first,
                                         int last_row, int base, uint64_t bad, float (&w)[4][4]) {
  constexpr int CH = D / 32;
  using vec8 = typename Traits<T>::vec8;
  const int lane = threadIdx.x & 63, lrow = lane & 15, kg = lane >> 4;
  for (int r0 = first; r0 < last_row; r0 += 16) {
    const int row = r0 + lrow < rq.rows ? r0 + lrow : rq.rows - 1;
    const int tok = row / a.group, h = head * a.group + row - tok * a.group;
    const float lse = r0 + lrow < rq.rows ? a.lse[(int64_t)(rq.tok0 + tok) * a.q_heads + h] : -INFINITY;
    const uint16_t *qp = a.q + (int64_t)(rq.tok0 + tok) * a.q_stride + h * D + kg * 8;
    vec8 q[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) q[i] = as<vec8>(load16(qp + i * 32));
    const int last = rq.pos0 + tok, from = a.window > 0 ? last - a.window + 1 : 0;
    const uint64_t sees = lse == -INFINITY ? 0 : (run(from - base, last - base) & ~bad) >> kg * 4;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      f32x4 s{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < CH; ++i) s = Traits<T>::mfma(kf[tt][i], q[i], s);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[tt][i] += as<float>(as<uint32_t>(exp2_(fmaf(s[i], a.c, -lse))) & bit((uint32_t)(sees >> (tt >> 1) * 32), (tt & 1) * 16 + i));
    }
  }
}

// Rows that see any of 64 tokens from `base` on
struct Seeing {
  int lo, hi;
  __device__ __forceinline__ Seeing(const AttnArgs &a, const Weighed &rq, int base) {
    lo = base > rq.pos0 ? (base - rq.pos0) * a.group & ~15 : 0;
    const int64_t end = a.window > 0 ? ((int64_t)base + 63 - rq.pos0 + a.window) * a.group : rq.rows;
    hi = end < rq.rows ? (int)end : rq.rows;
  }
};

// What a lane's sixteen rows gave its tokens, for each of the tokens
template <typename F>
__device__ __forceinline__ void over_rows(const float (&w)[4][4], F take) {
  const int lane = threadIdx.x & 63, lrow = lane & 15, kg = lane >> 4;
#pragma unroll
  for (int tt = 0; tt < 4; ++tt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = w[tt][i];
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) x += __shfl_xor(x, d);
      if (lrow == 0) take(tt * 16 + kg * 4 + i, x);
    }
}

// ... which the two kinds of cache do by kernels of their own (csrc/attention.hip, csrc/attention8.hip); `most`: blocks of WEIGHT_TOKENS that there
// can be.  As many workgroups as the device holds at once: how many there are it knows.
template <typename T, int D>
int sum_weights(hipStream_t st, const AttnLayout &L, const AttnArgs &a, int64_t most);

template <typename T, int D, bool CODES>
int launch(hipStream_t st, const mlora_attention_plan &p, const AttnLayout &L, const AttnArgs &a) {
  if (int rc = a.lse ? launch_lists<T, D, true, CODES>(st, L, a) : launch_lists<T, D, false, CODES>(st, L, a)) return rc;
  if (L.tall_joins > 0) {
    hipLaunchKernelGGL((attend_join_kernel<T, D>), dim3((unsigned)(L.tall_joins * a.kv_heads), TALL_ROWS / JOIN_ROWS), dim3(THREADS), 0, st, a);
    if (int rc = check_launch("attend_join_kernel")) return rc;
  }
  if (a.weights && p.max_kv_len > 0) {
    const int64_t most = p.n_req * ((p.max_kv_len + WEIGHT_TOKENS - 1) / WEIGHT_TOKENS);
    if (int rc = sum_weights<T, D>(st, L, a, most)) return rc;
  }
  return MLORA_OK;
}

template <typename T, bool CODES>
int launch(hipStream_t st, const mlora_attention_plan &p, const AttnLayout &L, const AttnArgs &a) {
  switch (p.head_dim) {
    case 32: return launch<T, 32, CODES>(st, p, L, a);
    case 64: return launch<T, 64, CODES>(st, p, L, a);
    case 96: return launch<T, 96, CODES>(st, p, L, a);
    case 128: return launch<T, 128, CODES>(st, p, L, a);
    default: return launch<T, 256, CODES>(st, p, L, a);
  }
}

// What both entry points check and fill in.  `pool(a, n_pages)` checks the cache's operands and fills them in; it is asked for null
// pointers (`there`) only where there is work.
template <bool CODES, typename Pool>
int attention_call(const char *who, void *stream, const mlora_attention_plan *plan, void *workspace, size_t workspace_bytes, void *out,
                   int64_t out_stride, const void *q, int64_t q_stride, const int32_t *table, int64_t table_stride, int64_t table_width,
                   float scale, float *weights, int64_t weights_stride, mlora_dtype dtype, Pool pool) {
  if (int rc = check_attention_plan(plan, who)) return rc;
  if (!(scale > 0.0f) || scale > 1e30f) return fail(MLORA_ERR_INVALID, "%s: scale=%g must be positive", who, (double)scale);
  if (dtype != MLORA_F16 && dtype != MLORA_BF16) return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. %s: dtype=%d", who, (int)dtype);
  const AttnLayout L = attention_layout(*plan);
  if (!plan->dev || plan->bytes < (size_t)L.words * 4) return fail(MLORA_ERR_WORKSPACE, "%s: the plan's buffer is too small", who);
  const int64_t qw = (int64_t)plan->q_heads * plan->head_dim;
  AttnArgs a{};
  int64_t n_pages = 0;
  bool there = false;
  if (q_stride < qw || out_stride < qw) return fail(MLORA_ERR_INVALID, "%s: a row of q, out or the pool is shorter than its heads", who);
  if ((q_stride | out_stride) & 7 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15))
    return fail(MLORA_ERR_INVALID, "%s: rows of q, out and the pool must be multiples of 16 bytes and 16-byte aligned", who);
  if (int rc = pool(a, n_pages, there)) return rc;
  const int64_t pages = (plan->max_kv_len + plan->page_size - 1) / plan->page_size;
  if (table_width < pages || table_stride < table_width)
    return fail(MLORA_ERR_INVALID, "%s: a row of the table has %lld pages, max_kv_len=%lld needs %lld", who, (long long)table_width,
                (long long)plan->max_kv_len, (long long)pages);
  if (weights && weights_stride < plan->max_kv_len)
    return fail(MLORA_ERR_INVALID, "%s: a row of the weights is shorter than max_kv_len=%lld", who, (long long)plan->max_kv_len);
  if (plan->n_req == 0 || plan->n_tokens == 0 || plan->max_seq_len == 0) return MLORA_OK;
  // a pool without a whole page has no row to stand in for the ones that are not there
  if (!out || !q || (plan->max_kv_len > 0 && !table)) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  if (!there || n_pages == 0) return fail(MLORA_ERR_INVALID, "%s: the pool holds no page", who);
  const AttnWorkspace w = attention_workspace(*plan, L, weights != nullptr);
  if (w.bytes > 0 && (!workspace || (int64_t)workspace_bytes < w.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return fail(MLORA_ERR_WORKSPACE, "%s: workspace has %zu bytes (256-byte aligned), needs %lld", who, workspace ? workspace_bytes : 0,
                (long long)w.bytes);
  int shift = 0;
  while ((1 << shift) < plan->page_size) ++shift;
  a.plan = static_cast<const int32_t *>(plan->dev);
  a.out = static_cast<uint16_t *>(out);
  a.q = static_cast<const uint16_t *>(q);
  a.table = table;
  char *ws = static_cast<char *>(workspace);
  a.few_o = reinterpret_cast<float *>(ws + w.few_o);
  a.tall_o = reinterpret_cast<float *>(ws + w.tall_o);
  a.few_ml = reinterpret_cast<float4 *>(ws + w.few_ml);
  a.tall_ml = reinterpret_cast<float4 *>(ws + w.tall_ml);
  a.lse = weights ? reinterpret_cast<float *>(ws + w.lse) : nullptr;
  a.scores = reinterpret_cast<float *>(ws + w.scores);
  a.off_few = (int)L.off_few;
  a.off_tall = (int)L.off_tall;
  a.off_joins = (int)L.off_joins;
  a.off_tall_joins = (int)(L.off_joins + L.few_joins * AT_REC);
  a.off_arrive = (int)L.off_arrive;
  a.off_requests = (int)L.off_requests;
  a.off_shares = (int)L.off_shares;
  a.weights = weights;
  a.out_stride = out_stride;
  a.q_stride = q_stride;
  a.table_stride = table_stride;
  a.weights_stride = weights_stride;
  a.c = scale * 1.44269504088896340736f;
  a.q_heads = plan->q_heads;
  a.kv_heads = plan->kv_heads;
  a.group = (int)L.group;
  a.page_shift = shift;
  a.window = window_of(*plan);
  a.n_req = (int)plan->n_req;
  a.n_pages = (int)n_pages;
  hipStream_t st = (hipStream_t)stream;
  return dtype == MLORA_F16 ? launch<_Float16, CODES>(st, *plan, L, a) : launch<__bf16, CODES>(st, *plan, L, a);
}

}  // namespace

}  // namespace mlora
