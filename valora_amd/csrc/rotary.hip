// Rotary positions: every pair (a, b) of a head's first `rotary_dim` elements is turned by position * frequency,
//
//     a' = (a cos t - b sin t) * gain,   b' = (a sin t + b cos t) * gain,   t = 2 pi * position * freqs[pair]
//
// the others pass through; the result goes to where the part's `dst` says, which for k and v is the token's row of the paged
// pool, so the cache is written by the launch that rotates and k and v never go back to memory in between.
//
// `freqs` are in turns and in 64 bits: position * frequency is reduced to a fraction of a turn in 64 bits (a position of
// 10^6 in 32 bits would be off by 0.03 radians), the fraction is rounded to 32 bits (2^-25 turns) and sine and cosine are
// taken in 32 bits.  Each product is rounded to 16 bits once.
//
// Bound by bytes (8191 tokens, 32 query and 8 key heads of 128, bf16: 201 MB in 40 us, as a copy; one token: 3.1 us, a launch).  One
// workgroup per token (and, for few tokens, per piece of the token's heads): it works out the token's sines and cosines while
// the other operands are in flight, and every head uses them from LDS.
#include "kernel_common.h"

namespace mlora {

namespace {

struct RotaryArgs {
  mlora_rotary_part part[MLORA_ROTARY_PARTS];
  int units[MLORA_ROTARY_PARTS];      // units of all parts up to and with this one, per token
  const int64_t *positions, *loc;
  const double *freqs;
  int64_t n_rows;
  float gain;
  int head_dim, rotary_dim;
  int per_piece;                      // units of one workgroup
};

constexpr int RO_THREADS = 256;
constexpr int RO_MAX_PAIRS = 256;     // rotary_dim <= 512

// Row of the token in a destination: its own, or the one `loc` names (-1: none, nothing is written)
__device__ __forceinline__ int64_t dst_row(const mlora_rotary_part &p, int64_t token, int64_t row) {
  return (p.flags & MLORA_ROTARY_TO_ROWS) ? row : token;
}

__device__ __forceinline__ void sines(const RotaryArgs &a, int64_t pos, float2 *cs) {
  for (int i = threadIdx.x; i < a.rotary_dim / 2; i += RO_THREADS) {
    const double turns = (double)pos * a.freqs[i];
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = float2{c * a.gain, s * a.gain};
  }
}

// VEC: units of 16 bytes (a pair of them where the halves of a head are paired).  Otherwise a unit is one pair, or one
// element behind the rotated ones: any strides, any even rotary_dim.
template <typename T, bool INTERLEAVED, bool VEC>
__global__ __launch_bounds__(RO_THREADS) void rotary_kernel(RotaryArgs a) {
  __shared__ float2 cs[RO_MAX_PAIRS];
  const int64_t token = blockIdx.x;
  const int lo = blockIdx.y * a.per_piece, hi = min(lo + a.per_piece, a.units[MLORA_ROTARY_PARTS - 1]);
  const int64_t pos = a.positions[token];
  int64_t row = a.loc ? a.loc[token] : -1;
  if (row >= a.n_rows) row = -1;
  const int R = a.rotary_dim;
  const int turned = VEC ? (INTERLEAVED ? R / 8 : R / 16) : R / 2;         // units of a head that are rotated
  const int behind = VEC ? (a.head_dim - R) / 8 : a.head_dim - R;          // and that pass through

  bool ready = false;
  for (int u0 = lo; u0 < hi; u0 += RO_THREADS) {
    const int u = u0 + threadIdx.x;
    const uint16_t *src = nullptr;
    uint16_t *dst = nullptr;
    int at = 0, other = 0, pair = -1;      // element(s) of the head, first pair (-1: passes through)
    if (u < hi) {
      int k = 0;
#pragma unroll
      for (int i = 0; i + 1 < MLORA_ROTARY_PARTS; ++i) k += u >= a.units[i];
      const mlora_rotary_part &p = a.part[k];
      const int v = u - (k ? a.units[k - 1] : 0);
      const bool rotate = p.flags & MLORA_ROTARY_TURN;
      const int per_head = rotate ? turned + behind : (VEC ? a.head_dim / 8 : a.head_dim);
      const int head = v / per_head, w = v - head * per_head;
      if (rotate && w < turned) {
        if (VEC) {
          at = w * 8;
          other = INTERLEAVED ? at : at + R / 2;
          pair = INTERLEAVED ? w * 4 : w * 8;
        } else {
          at = INTERLEAVED ? 2 * w : w;
          other = INTERLEAVED ? at + 1 : at + R / 2;
          pair = w;
        }
      } else {
        at = (rotate ? R : 0) + (w - (rotate ? turned : 0)) * (VEC ? 8 : 1);
      }
      const int64_t to = dst_row(p, token, row);
      if (to >= 0) {
        src = static_cast<const uint16_t *>(p.src) + token * p.src_token_stride + head * p.src_head_stride;
        dst = static_cast<uint16_t *>(p.dst) + to * p.dst_token_stride + head * p.dst_head_stride;
      }
    }
    u32x4 x{0, 0, 0, 0}, y{0, 0, 0, 0};
    uint16_t xs = 0, ys = 0;
    if (src) {
      if constexpr (VEC) {
        x = load16(src + at);
        if (!INTERLEAVED && pair >= 0) y = load16(src + other);
      } else {
        xs = src[at];
        if (pair >= 0) ys = src[other];
      }
    }
    requested();
    if (!ready) {                          // (every thread of the workgroup comes here in its first round)
      sines(a, pos, cs);
      __syncthreads();
      ready = true;
    }
    if (!src) continue;
    if constexpr (VEC) {
      if (pair >= 0) {
        float f[8], g[8];
        unpack8<T>(x, f);
        if (INTERLEAVED) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 t = cs[pair + i];
            g[2 * i] = f[2 * i] * t.x - f[2 * i + 1] * t.y;
            g[2 * i + 1] = f[2 * i] * t.y + f[2 * i + 1] * t.x;
          }
          x = pack8<T>(g);
        } else {
          float h[8];
          unpack8<T>(y, h);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 t = cs[pair + i];
            g[i] = f[i] * t.x - h[i] * t.y;
            h[i] = f[i] * t.y + h[i] * t.x;
          }
          x = pack8<T>(g);
          store16(dst + other, pack8<T>(h));
        }
      }
      store16(dst + at, x);
    } else {
      if (pair >= 0) {
        const float f = Traits<T>::to_float(xs), h = Traits<T>::to_float(ys);
        const float2 t = cs[pair];
        xs = Traits<T>::from_float(f * t.x - h * t.y);
        dst[other] = Traits<T>::from_float(f * t.y + h * t.x);
      }
      dst[at] = xs;
    }
  }
}

template <typename T>
void launch(hipStream_t st, dim3 grid, const RotaryArgs &a, bool interleaved, bool vec) {
  auto *k = interleaved ? (vec ? rotary_kernel<T, true, true> : rotary_kernel<T, true, false>)
                        : (vec ? rotary_kernel<T, false, true> : rotary_kernel<T, false, false>);
  hipLaunchKernelGGL(k, grid, dim3(RO_THREADS), 0, st, a);
}

}  // namespace

// Whether heads of `dim` elements at row * row_stride + head * head_stride can share some.  Either the heads of a row lie within the room between
// two rows or the other way round; strides that interleave the two count as sharing.
bool share_elements(int64_t rows, int64_t row_stride, int64_t heads, int64_t head_stride, int64_t dim) {
  if ((rows > 1 && row_stride < dim) || (heads > 1 && head_stride < dim)) return true;
  if (rows <= 1 || heads <= 1) return false;
  const bool by_row = row_stride >= head_stride;
  const int64_t inner = by_row ? head_stride : row_stride, outer = by_row ? row_stride : head_stride, n = by_row ? heads : rows;
  return (outer - dim) / inner < n - 1;
}

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_rotary(void *stream, const mlora_rotary_part *parts, int32_t n_parts, const int64_t *positions,
                            const int64_t *loc, int64_t n_rows, int64_t T, int32_t head_dim, int32_t rotary_dim,
                            int32_t interleaved, const double *freqs, float gain, mlora_dtype dtype) {
  if (T < 0 || n_rows < 0 || n_parts < 1 || n_parts > MLORA_ROTARY_PARTS)
    return fail(MLORA_ERR_INVALID, "rotary: T=%lld n_rows=%lld n_parts=%d out of range", (long long)T, (long long)n_rows, n_parts);
  if (dtype != MLORA_F16 && dtype != MLORA_BF16)
    return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. rotary: dtype=%d", (int)dtype);
  if (head_dim < 2 || rotary_dim < 2 || (rotary_dim & 1) || rotary_dim > head_dim || rotary_dim > 2 * RO_MAX_PAIRS || head_dim > 4096)
    return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. rotary: head_dim=%d rotary_dim=%d (even, at most %d and head_dim)",
                head_dim, rotary_dim, 2 * RO_MAX_PAIRS);
  if (T > 0x7fffffff) return fail(MLORA_ERR_NO_KERNEL, "rotary: more than 2^31 - 1 tokens");
  if (!parts) return fail(MLORA_ERR_INVALID, "rotary: parts is null");
  RotaryArgs a{};
  bool vec = head_dim % 8 == 0 && rotary_dim % 16 == 0;
  for (int i = 0; i < n_parts; ++i) {
    const mlora_rotary_part &p = parts[i];
    if (p.heads < 0 || p.heads > 65536) return fail(MLORA_ERR_INVALID, "rotary: heads=%d out of range", p.heads);
    if (T > 0 && p.heads > 0 && (!p.src || !p.dst)) return fail(MLORA_ERR_INVALID, "rotary: null pointer");
    if ((p.flags & MLORA_ROTARY_TO_ROWS) && T > 0 && p.heads > 0 && !loc)
      return fail(MLORA_ERR_INVALID, "rotary: loc is null");
    const int64_t dst_rows = p.flags & MLORA_ROTARY_TO_ROWS ? n_rows : T;
    if (share_elements(dst_rows, p.dst_token_stride, p.heads, p.dst_head_stride, head_dim))
      return fail(MLORA_ERR_INVALID, "rotary: heads of a destination overlap");
    vec = vec && ((p.src_token_stride | p.src_head_stride | p.dst_token_stride | p.dst_head_stride) & 7) == 0 &&
          ((reinterpret_cast<uintptr_t>(p.src) | reinterpret_cast<uintptr_t>(p.dst)) & 15) == 0;
  }
  int64_t units = 0;
  for (int i = 0; i < MLORA_ROTARY_PARTS; ++i) {
    if (i < n_parts) {
      const bool rotate = parts[i].flags & MLORA_ROTARY_TURN;
      const int turned = !rotate ? 0 : vec ? (interleaved ? rotary_dim / 8 : rotary_dim / 16) : rotary_dim / 2;
      const int rest = head_dim - (rotate ? rotary_dim : 0);
      a.part[i] = parts[i];
      units += (int64_t)parts[i].heads * (turned + (vec ? rest / 8 : rest));
    }
    a.units[i] = (int)units;
  }
  if (T == 0 || units == 0) return MLORA_OK;
  if (!positions || !freqs) return fail(MLORA_ERR_INVALID, "rotary: null pointer");
  if (units > (1 << 30)) return fail(MLORA_ERR_NO_KERNEL, "rotary: too many heads");
  a.positions = positions;
  a.loc = loc;
  a.freqs = freqs;
  a.n_rows = n_rows;
  a.gain = gain;
  a.head_dim = head_dim;
  a.rotary_dim = rotary_dim;
  // Few tokens: a workgroup per round of units, so that a lone token's heads are not one workgroup's work after the other
  const int64_t rounds = (units + RO_THREADS - 1) / RO_THREADS;
  const int64_t pieces = T >= 512 ? 1 : rounds < 65535 ? rounds : 65535;
  a.per_piece = (int)((rounds + pieces - 1) / pieces * RO_THREADS);
  for (int64_t at = 0; at < T; at += most_blocks(RO_THREADS)) {
    RotaryArgs some = a;
    for (int i = 0; i < n_parts; ++i) {
      mlora_rotary_part &p = some.part[i];
      p.src = p.src ? static_cast<const uint16_t *>(p.src) + at * p.src_token_stride : nullptr;
      if (p.dst && !(p.flags & MLORA_ROTARY_TO_ROWS)) p.dst = static_cast<uint16_t *>(p.dst) + at * p.dst_token_stride;
    }
    some.positions += at;
    if (loc) some.loc += at;
    const dim3 grid((unsigned)(T - at < most_blocks(RO_THREADS) ? T - at : most_blocks(RO_THREADS)), (unsigned)((units + a.per_piece - 1) / a.per_piece));
    if (dtype == MLORA_F16) launch<_Float16>((hipStream_t)stream, grid, some, interleaved != 0, vec);
    else launch<__bf16>((hipStream_t)stream, grid, some, interleaved != 0, vec);
  }
  return check_launch("rotary_kernel");
}
