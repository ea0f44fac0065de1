// The norms around a layer's blocks (include/mlora.h): the block's output, normalised and gated where the model does that, joins the
// residual stream, and what the next block reads is normalised, in one pass.
//
// A row is held in the registers of one workgroup (or one wave) between its load and its stores; sums go over lanes, then waves, in a
// fixed order and 32 bits.  Variances are of differences from the mean, after it: no sum of squares loses them.
//
// Bound by bytes where rows are many: 8191 of 4096 with a gate, 268 MB in 46.9 us, 5.7 TB/s (part of it from the memory-side cache; a copy runs at
// 5.1).  Few rows are one row's chain: its loads, a sum for each norm, its stores: 256 of 5120 with two norms 4.7 us, one of 4096 2.9 of
// GPU time, which a launch takes too.
#include <type_traits>
#include <utility>

#include "kernel_common.h"

namespace mlora {

namespace {

// Runs of eight: a thread has one of up to NORM_ONE, which keeps its registers few and loads all it needs at once; rows of more would be workgroups
// of many waves that wait for each other, unless they are few and the chain counts (one / two runs a thread, rows of 5120 and of 7168 with two norms,
// us: 256 rows 4.8 / 5.2 and 5.4 / 5.5; 400 6.2 / 5.9 and 7.4 / 6.9; 512 6.6 / 6.2 and 7.9 / 7.5; 700 8.3 / 7.5 and 10.0 / 9.4; 2048 18.4 / 17.7
// and 26.2 / 22.1.  So the border lies near 300 rows, and 300 to 512 lose a twentieth.)
constexpr int NORM_ONE = 512, NORM_FEW_ROWS = 512;
constexpr int NORM_MAX = 32768;

// What lane l holds, and what the lane holds whose number differs in one way each: by quads, halves and rows of sixteen, rows, halves.  (No exchange
// goes through LDS, where a butterfly's six would wait one after the other.)
template <int CTRL>
__device__ __forceinline__ float plus_dpp(float x) {
  return x + as<float>((uint32_t)__builtin_amdgcn_mov_dpp((int)as<uint32_t>(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = plus_dpp<0xb1>(x);                 // quad_perm 1 0 3 2
  x = plus_dpp<0x4e>(x);                 // quad_perm 2 3 0 1
  x = plus_dpp<0x141>(x);                // row_half_mirror
  x = plus_dpp<0x140>(x);                // row_mirror
  typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
  const u32x2 rows = __builtin_amdgcn_permlane16_swap(as<uint32_t>(x), as<uint32_t>(x), false, false);
  x = as<float>(rows[0]) + as<float>(rows[1]);
  const u32x2 halves = __builtin_amdgcn_permlane32_swap(as<uint32_t>(x), as<uint32_t>(x), false, false);
  return as<float>(halves[0]) + as<float>(halves[1]);
}

// Over a row's lanes: a wave's, or with MANY those of all the workgroup's waves, 16 at most.  Every sum of a row has sixteen places of its own (0
// for waves that are not there), so one barrier each is enough.
constexpr int SUMS = 4, PLACES = 16;
template <bool MANY>
struct RowSum {
  float *part;
  __device__ __forceinline__ float operator()(float x) {
    x = wave_sum(x);
    if constexpr (MANY) {
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
      __syncthreads();
      f32x4 s = *reinterpret_cast<const f32x4 *>(part);
#pragma unroll
      for (int i = 4; i < PLACES; i += 4) s += *reinterpret_cast<const f32x4 *>(part + i);
      x = (s[0] + s[1]) + (s[2] + s[3]);
      part += PLACES;
    }
    return x;
  }
};

// Eight elements from `at` on; those behind the row are 0.  VEC: rows are whole runs of eight, at 16 bytes.  Otherwise a run is one access all the
// same, at whatever address, and the row's last one goes by elements (all by elements: 8000 rows of 4097 with a gate an element 208 us, now 81).
typedef u32x4 __attribute__((aligned(2))) u32x4_at2;
typedef f32x4 __attribute__((aligned(4))) f32x4_at4;
template <typename T, bool VEC>
__device__ __forceinline__ void load_row(const void *p, int64_t at, int left, float (&x)[8]) {
  const uint16_t *s = static_cast<const uint16_t *>(p) + at;
  u32x4 r{0, 0, 0, 0};
  if constexpr (VEC) {
    if (left > 0) r = load16(s);
  } else if (left >= 8) {
    r = *reinterpret_cast<const u32x4_at2 *>(s);
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < left) r[i / 2] |= (uint32_t)s[i] << i % 2 * 16;
  }
  unpack8<T>(r, x);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_row(void *p, int64_t at, int left, const float (&x)[8]) {
  uint16_t *d = static_cast<uint16_t *>(p) + at;
  const u32x4 r = pack8<T>(x);
  if constexpr (VEC) {
    if (left > 0) store16(d, r);
  } else if (left >= 8) {
    *reinterpret_cast<u32x4_at2 *>(d) = r;
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < left) d[i] = (uint16_t)(r[i / 2] >> i % 2 * 16);
  }
}

// A vector of the call, a thread's V runs of it.  EARLY: asked for with the row (behind a sum it would be a round trip more: 8191 rows of 4096
// with a gate 53.8 -> 47.1 us); where none is float and a thread has one run, as the registers of more would cost waves (two runs: 59.8 -> 76).
// Otherwise loaded where it is used.
template <typename T, bool VEC, int V, bool EARLY>
struct Vector {
  const void *p;
  bool f32;
  u32x4 x[EARLY ? V : 1];
  __device__ __forceinline__ Vector(const void *p_, bool f32_, int tid, int step, int H) : p(p_), f32(f32_) {
    if constexpr (EARLY)
      if (p)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int at = tid * 8 + v * step;
          x[v] = at < H ? load16(static_cast<const uint16_t *>(p) + at) : u32x4{0, 0, 0, 0};
        }
  }
  __device__ __forceinline__ void get(int v, int at, int left, float (&f)[8]) const {
    if constexpr (EARLY) {
      unpack8<T>(x[v], f);
    } else if (!f32) {
      load_row<T, VEC>(p, at, left, f);
    } else {
      const float *s = static_cast<const float *>(p) + at;
      f32x4 lo{0, 0, 0, 0}, hi = lo;
      if (left >= 8) {
        lo = *reinterpret_cast<const f32x4_at4 *>(s);
        hi = *reinterpret_cast<const f32x4_at4 *>(s + 4);
      } else {
#pragma unroll
        for (int i = 0; i < 7; ++i) {
          const float one = i < left ? s[i] : 0.0f;
          if (i < 4) lo[i] = one;
          else hi[i - 4] = one;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[i] = lo[i];
        f[4 + i] = hi[i];
      }
    }
  }
};

// x (of H elements, V runs of eight a thread) becomes its norm
template <bool MANY, int V, typename Vec>
__device__ __forceinline__ void normalise(float (&x)[V][8], const mlora_norm &n, const Vec &w, const Vec &b, int tid, int step, RowSum<MANY> &row_sum) {
  const int H = (int)n.H;
  const float inv = 1.0f / (float)H;
  float mean = 0.0f;
  if (n.layer) {
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += x[v][i];
    mean = row_sum(s) * inv;
  }
  float s = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[v][i] -= tid * 8 + v * step + i < H ? mean : 0.0f;
      s = fmaf(x[v][i], x[v][i], s);
    }
  const float r = 1.0f / sqrtf(row_sum(s) * inv + n.eps);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = tid * 8 + v * step;
    float f[8];
    w.get(v, at, H - at, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[v][i] *= r * (n.offset + f[i]);
    if (b.p) {
      b.get(v, at, H - at, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[v][i] += f[i];
    }
  }
}

// A workgroup a row, or a wave (four rows a workgroup)
template <typename T, bool VEC, bool MANY, int V, bool EARLY>
__global__ __launch_bounds__(MANY ? 1024 : 256) void block_norm_kernel(mlora_norm n) {
  __shared__ __align__(16) float part[SUMS * PLACES];
  RowSum<MANY> row_sum{part};
  constexpr int ROWS = MANY ? 1 : 4;
  const int step = MANY ? blockDim.x * 8 : 512;
  using Vec = Vector<T, VEC, V, EARLY>;
  const int64_t row = (int64_t)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x >> 6 : 0);
  if (row >= n.T) return;
  const int tid = ROWS > 1 ? threadIdx.x & 63 : threadIdx.x, H = (int)n.H;
  if (MANY && tid < SUMS * PLACES && (tid & (PLACES - 1)) >= (int)blockDim.x >> 6) part[tid] = 0.0f;
  float x[V][8], o[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = tid * 8 + v * step;
    if (n.block) load_row<T, VEC>(n.block, row * n.block_stride + at, H - at, o[v]);
    load_row<T, VEC>(n.x, row * n.x_stride + at, H - at, x[v]);
  }
  const Vec bw(n.block_weight, n.f32 & MLORA_NORM_F32_BLOCK_WEIGHT, tid, step, H), bb(n.block_bias, n.f32 & MLORA_NORM_F32_BLOCK_BIAS, tid, step, H);
  const Vec gate(n.gate && n.gate_column_stride ? static_cast<const char *>(n.gate) + row * n.gate_row_stride * (n.f32 & MLORA_NORM_F32_GATE ? 4 : 2) : nullptr,
                 n.f32 & MLORA_NORM_F32_GATE, tid, step, H);
  float row_gate = 1.0f;
  if (n.gate && !n.gate_column_stride) {
    const int64_t at = row * n.gate_row_stride;
    row_gate = n.f32 & MLORA_NORM_F32_GATE ? static_cast<const float *>(n.gate)[at] : Traits<T>::to_float(static_cast<const uint16_t *>(n.gate)[at]);
  }
  const Vec w(n.weight, n.f32 & MLORA_NORM_F32_WEIGHT, tid, step, H), b(n.bias, n.f32 & MLORA_NORM_F32_BIAS, tid, step, H);
  if (EARLY) requested();
  if (n.block) {
    if (n.block_weight) normalise<MANY, V>(o, n, bw, bb, tid, step, row_sum);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int at = tid * 8 + v * step;
      if (gate.p) {
        float g[8];
        gate.get(v, at, H - at, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[v][i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[v][i] = fmaf(n.block_scale, o[v][i] * row_gate, n.residual_scale * x[v][i]);
      if (n.residual_out) store_row<T, VEC>(n.residual_out, row * n.residual_stride + at, H - at, x[v]);
    }
  }
  if (!n.weight) return;
  normalise<MANY, V>(x, n, w, b, tid, step, row_sum);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = tid * 8 + v * step;
    store_row<T, VEC>(n.out, row * n.out_stride + at, H - at, x[v]);
  }
}

// `rows` rows from `at` on
mlora_norm rows_from(mlora_norm n, int64_t at, int64_t rows) {
  const auto read = [&](const void *&p, int64_t stride, int bytes) { p = p ? static_cast<const char *>(p) + at * stride * bytes : nullptr; };
  const auto written = [&](void *&p, int64_t stride) { p = p ? static_cast<char *>(p) + at * stride * 2 : nullptr; };
  read(n.x, n.x_stride, 2);
  read(n.block, n.block_stride, 2);
  read(n.gate, n.gate_row_stride, n.f32 & MLORA_NORM_F32_GATE ? 4 : 2);
  written(n.residual_out, n.residual_stride);
  written(n.out, n.out_stride);
  n.T = rows;
  return n;
}

template <typename T, bool VEC, bool EARLY>
int launch(hipStream_t st, const mlora_norm &n) {
  const int units = (int)((n.H + 7) / 8);
  const auto go = [&](auto many, auto v) {
    constexpr bool MANY = decltype(many)::value;
    constexpr int V = decltype(v)::value;
    const int threads = MANY ? ((units + V - 1) / V + 63) / 64 * 64 : 256;
    constexpr int ROWS = MANY ? 1 : 4;
    const int64_t most = most_blocks(threads) * ROWS;
    for (int64_t at = 0; at < n.T; at += most) {
      const mlora_norm part = rows_from(n, at, n.T - at < most ? n.T - at : most);
      hipLaunchKernelGGL((block_norm_kernel<T, VEC, MANY, V, EARLY && V == 1>), dim3((unsigned)((part.T + ROWS - 1) / ROWS)), dim3((unsigned)threads), 0,
                         st, part);
    }
    return check_launch("block_norm_kernel");
  };
  using std::integral_constant;
  using one = integral_constant<int, 1>;
  if (units <= 64) return go(std::false_type{}, one{});
  if (units <= NORM_ONE || (units <= 1024 && n.T <= NORM_FEW_ROWS)) return go(std::true_type{}, one{});
  if (units <= 2048) return go(std::true_type{}, integral_constant<int, 2>{});
  return go(std::true_type{}, integral_constant<int, 4>{});
}

}  // namespace

}  // namespace mlora

using namespace mlora;

// Rows of n's width in a tensor of the call
static Runs rows_of(const mlora_norm &n, const void *p, int64_t stride) { return {p, n.T, stride * 2, 1, 0, n.H * 2}; }

// Whether rows written at `d` can touch what other rows read at `s`: not where the two are the same rows
static bool overlap(const mlora_norm &n, const void *d, int64_t d_stride, const void *s, int64_t s_stride) {
  return !(d == s && (d_stride == s_stride || n.T == 1)) && share_memory(rows_of(n, d, d_stride), rows_of(n, s, s_stride));
}

extern "C" int mlora_block_norm(void *stream, const mlora_norm *norm, mlora_dtype dtype) {
  const char *who = "block_norm";
  if (!norm) return fail(MLORA_ERR_INVALID, "%s: norm is null", who);
  const mlora_norm &n = *norm;
  if (dtype != MLORA_F16 && dtype != MLORA_BF16) return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. %s: dtype=%d", who, (int)dtype);
  if (n.T < 0 || n.T > 0x7fffffff) return fail(MLORA_ERR_NO_KERNEL, "%s: T=%lld out of range", who, (long long)n.T);
  if (n.H < 1 || n.H > NORM_MAX) return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. %s: H=%lld (1 to %d)", who, (long long)n.H, NORM_MAX);
  if (!(n.eps >= 0.0f)) return fail(MLORA_ERR_INVALID, "%s: eps=%g must not be negative", who, (double)n.eps);
  if (!n.block && (n.block_weight || n.gate || n.residual_out)) return fail(MLORA_ERR_INVALID, "%s: block's operands without block", who);
  if (n.block_bias && !n.block_weight) return fail(MLORA_ERR_INVALID, "%s: block_bias without block_weight", who);
  if (n.bias && !n.weight) return fail(MLORA_ERR_INVALID, "%s: bias without weight", who);
  if (n.gate && (n.gate_row_stride < 0 || (n.gate_column_stride != 0 && n.gate_column_stride != 1)))
    return fail(MLORA_ERR_INVALID, "%s: elements of a row of the gate must be contiguous, or one, its rows in order", who);
  if (n.T > 1 && (n.x_stride < 0 || (n.block && n.block_stride < 0))) return fail(MLORA_ERR_INVALID, "%s: negative strides", who);
  if (n.T == 0) return MLORA_OK;
  void *out = n.weight ? n.out : nullptr;
  const int64_t gate_bytes = n.f32 & MLORA_NORM_F32_GATE ? 4 : 2;
  const Runs gate{n.gate, n.T, n.gate_row_stride * gate_bytes, 1, 0, (n.gate_column_stride ? n.H : 1) * gate_bytes};
  for (const auto &d : {std::make_pair((void *)n.residual_out, n.residual_stride), std::make_pair(out, n.out_stride)}) {
    if (d.first && n.T > 1 && d.second < n.H) return fail(MLORA_ERR_INVALID, "%s: rows of a result overlap", who);
    if (overlap(n, d.first, d.second, n.x, n.x_stride) || overlap(n, d.first, d.second, n.block, n.block_stride))
      return fail(MLORA_ERR_INVALID, "%s: a result overlaps other rows of an operand", who);
    const Runs to = rows_of(n, d.first, d.second);
    if (share_memory(to, gate)) return fail(MLORA_ERR_INVALID, "%s: a result overlaps the gate", who);
    const void *vectors[] = {n.weight, n.bias, n.block_weight, n.block_bias};
    for (int i = 0; i < 4; ++i)
      if (share_memory(to, {vectors[i], 1, 0, 1, 0, n.H * (n.f32 >> i & 1 ? 4 : 2)}))
        return fail(MLORA_ERR_INVALID, "%s: a result overlaps a vector", who);
  }
  if (out && n.residual_out && (out == n.residual_out || overlap(n, out, n.out_stride, n.residual_out, n.residual_stride)))
    return fail(MLORA_ERR_INVALID, "%s: the results overlap", who);
  if (!n.x || (n.weight && !n.out) || (!n.weight && !n.residual_out)) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  // rows that are whole runs of eight, at 16 bytes
  bool vec = n.H % 8 == 0;
  const auto row = [&](const void *p, int64_t stride) { vec = vec && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (!p || n.T == 1 || stride % 8 == 0); };
  row(n.x, n.x_stride);
  row(n.block, n.block_stride);
  row(n.residual_out, n.residual_stride);
  row(out, n.out_stride);
  row(n.gate_column_stride ? n.gate : nullptr, n.gate_row_stride);
  for (const void *p : {n.weight, n.bias, n.block_weight, n.block_bias}) row(p, 0);
  mlora_norm m = n;
  if (!m.block) m.residual_scale = 1.0f;
  hipStream_t st = (hipStream_t)stream;
  const bool early = vec && m.f32 == 0;
  if (dtype == MLORA_F16) return early ? launch<_Float16, true, true>(st, m) : vec ? launch<_Float16, true, false>(st, m) : launch<_Float16, false, false>(st, m);
  return early ? launch<__bf16, true, true>(st, m) : vec ? launch<__bf16, true, false>(st, m) : launch<__bf16, false, false>(st, m);
}
