// The norms around a layer's blocks (include/mlora.h): the block's output, normalised and gated where the model does that, joins the
// residual stream, and what the next block reads is normalised, in one pass.
//
// A row is held in the registers of one workgroup (or one wave) between its load and its stores; sums go over lanes, then waves, in a
// fixed order and 32 bits.  Variances are of differences from the mean, after it: no sum of squares loses them.
#include <type_traits>
#include <utility>

#include "kernel_common.h"

namespace mlora {

namespace {

constexpr int NORM_MAX = 32768, NORM_MAX_PLAIN = 16384;      // (wider rows element by element do not fit the registers)

template <int WAVES>
__device__ __forceinline__ float row_sum(float x, float *part) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  if constexpr (WAVES > 1) {
    __syncthreads();                     // (what was summed before has been read)
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) x += part[i];
  }
  return x;
}

// Eight elements from `at` on; those behind the row are 0
template <typename T, bool VEC>
__device__ __forceinline__ void load_row(const void *p, int64_t at, int left, float (&x)[8]) {
  const uint16_t *s = static_cast<const uint16_t *>(p) + at;
  if constexpr (VEC) {
    unpack8<T>(left > 0 ? load16(s) : u32x4{0, 0, 0, 0}, x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = Traits<T>::to_float(s[min(i, left - 1)]);           // (behind the row: its last)
      x[i] = i < left ? f : 0.0f;
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_row(void *p, int64_t at, int left, const float (&x)[8]) {
  uint16_t *d = static_cast<uint16_t *>(p) + at;
  if constexpr (VEC) {
    if (left > 0) store16(d, pack8<T>(x));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) d[i] = Traits<T>::from_float(x[i]);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void load_vector(const void *p, bool f32, int at, int left, float (&x)[8]) {
  if (!f32) return load_row<T, VEC>(p, at, left, x);
  const float *s = static_cast<const float *>(p) + at;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = s[min(i, left - 1)];
    x[i] = i < left ? f : 0.0f;
  }
}

// x (of H elements, V runs of eight a thread) becomes its norm
template <typename T, bool VEC, int WAVES, int V>
__device__ __forceinline__ void normalise(float (&x)[V][8], const mlora_norm &n, const void *w, bool w32, const void *b, bool b32, int tid, float *part) {
  constexpr int STEP = WAVES * 64 * 8;
  const int H = (int)n.H;
  const float inv = 1.0f / (float)H;
  float mean = 0.0f;
  if (n.layer) {
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += x[v][i];
    mean = row_sum<WAVES>(s, part) * inv;
  }
  float s = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[v][i] -= tid * 8 + v * STEP + i < H ? mean : 0.0f;
      s = fmaf(x[v][i], x[v][i], s);
    }
  const float r = 1.0f / sqrtf(row_sum<WAVES>(s, part) * inv + n.eps);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = tid * 8 + v * STEP;
    float wv[8], bv[8];
    load_vector<T, VEC>(w, w32, at, H - at, wv);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[v][i] *= r * (n.offset + wv[i]);
    if (b) {
      load_vector<T, VEC>(b, b32, at, H - at, bv);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[v][i] += bv[i];
    }
  }
}

// WAVES a row; where it is one, four rows a workgroup
template <typename T, bool VEC, int WAVES, int V>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void block_norm_kernel(mlora_norm n) {
  __shared__ float part[WAVES];
  constexpr int ROWS = WAVES == 1 ? 4 : 1, STEP = WAVES * 64 * 8;
  const int64_t row = (int64_t)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x >> 6 : 0);
  if (row >= n.T) return;
  const int tid = ROWS > 1 ? threadIdx.x & 63 : threadIdx.x, H = (int)n.H;
  float x[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = tid * 8 + v * STEP;
    load_row<T, VEC>(n.x, row * n.x_stride + at, H - at, x[v]);
  }
  if (n.block) {
    float o[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int at = tid * 8 + v * STEP;
      load_row<T, VEC>(n.block, row * n.block_stride + at, H - at, o[v]);
    }
    if (n.block_weight)
      normalise<T, VEC, WAVES, V>(o, n, n.block_weight, n.f32 & MLORA_NORM_F32_BLOCK_WEIGHT, n.block_bias, n.f32 & MLORA_NORM_F32_BLOCK_BIAS, tid, part);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int at = tid * 8 + v * STEP;
      if (n.gate) {
        float g[8];
        const bool f32 = n.f32 & MLORA_NORM_F32_GATE;
        if (n.gate_column_stride) {
          const char *p = static_cast<const char *>(n.gate) + row * n.gate_row_stride * (f32 ? 4 : 2);
          load_vector<T, VEC>(p, f32, at, H - at, g);
        } else {
          const int64_t to = row * n.gate_row_stride;
          const float one = f32 ? static_cast<const float *>(n.gate)[to] : Traits<T>::to_float(static_cast<const uint16_t *>(n.gate)[to]);
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] = one;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) o[v][i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[v][i] = fmaf(n.block_scale, o[v][i], n.residual_scale * x[v][i]);
      if (n.residual_out) store_row<T, VEC>(n.residual_out, row * n.residual_stride + at, H - at, x[v]);
    }
  }
  if (!n.weight) return;
  normalise<T, VEC, WAVES, V>(x, n, n.weight, n.f32 & MLORA_NORM_F32_WEIGHT, n.bias, n.f32 & MLORA_NORM_F32_BIAS, tid, part);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = tid * 8 + v * STEP;
    store_row<T, VEC>(n.out, row * n.out_stride + at, H - at, x[v]);
  }
}

template <typename T, bool VEC>
int launch(hipStream_t st, const mlora_norm &n) {
  const int units = (int)((n.H + 7) / 8);
  const auto go = [&](auto waves, auto v) {
    constexpr int W = decltype(waves)::value, V = decltype(v)::value;
    const int64_t blocks = W == 1 ? (n.T + 3) / 4 : n.T;
    hipLaunchKernelGGL((block_norm_kernel<T, VEC, W, V>), dim3((unsigned)blocks), dim3(W == 1 ? 256 : W * 64), 0, st, n);
    return check_launch("block_norm_kernel");
  };
  using std::integral_constant;
  if (units <= 64) return go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  if (units <= 128) return go(integral_constant<int, 2>{}, integral_constant<int, 1>{});
  if (units <= 256) return go(integral_constant<int, 4>{}, integral_constant<int, 1>{});
  if (units <= 512) return go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  if (units <= 1024) return go(integral_constant<int, 8>{}, integral_constant<int, 2>{});
  if (units <= 2048) return go(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  if constexpr (VEC) return go(integral_constant<int, 16>{}, integral_constant<int, 4>{});
  return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. block_norm: H=%lld above %d needs rows of 16-byte multiples, 16-byte aligned", (long long)n.H, NORM_MAX_PLAIN);
}

}  // namespace

}  // namespace mlora

using namespace mlora;

static bool meet(const char *a, int64_t a_bytes, const char *b, int64_t b_bytes) { return a && b && a < b + b_bytes && b < a + a_bytes; }

// Whether rows written at `d` can touch what other rows read at `s`: not where the two are the same rows
static bool overlap(const void *d, int64_t d_stride, const void *s, int64_t s_stride, int64_t T, int64_t H) {
  const char *a = static_cast<const char *>(d), *b = static_cast<const char *>(s);
  if (a == b && (d_stride == s_stride || T == 1)) return false;
  return meet(a, ((T - 1) * d_stride + H) * 2, b, ((T - 1) * s_stride + H) * 2);
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
  if (!n.x || (n.weight && !n.out) || (!n.weight && !n.residual_out)) return fail(MLORA_ERR_INVALID, "%s: null pointer", who);
  void *out = n.weight ? n.out : nullptr;
  for (const auto &d : {std::make_pair((void *)n.residual_out, n.residual_stride), std::make_pair(out, n.out_stride)}) {
    if (d.first && n.T > 1 && d.second < n.H) return fail(MLORA_ERR_INVALID, "%s: rows of a result overlap", who);
    if (overlap(d.first, d.second, n.x, n.x_stride, n.T, n.H) || overlap(d.first, d.second, n.block, n.block_stride, n.T, n.H))
      return fail(MLORA_ERR_INVALID, "%s: a result overlaps other rows of an operand", who);
    const char *to = static_cast<const char *>(d.first);
    const int64_t bytes = ((n.T - 1) * d.second + n.H) * 2;
    if (meet(to, bytes, static_cast<const char *>(n.gate),
             ((n.T - 1) * n.gate_row_stride + (n.gate_column_stride ? n.H : 1)) * (n.f32 & MLORA_NORM_F32_GATE ? 4 : 2)))
      return fail(MLORA_ERR_INVALID, "%s: a result overlaps the gate", who);
    const void *vectors[] = {n.weight, n.bias, n.block_weight, n.block_bias};
    for (int i = 0; i < 4; ++i)
      if (meet(to, bytes, static_cast<const char *>(vectors[i]), n.H * (n.f32 >> i & 1 ? 4 : 2)))
        return fail(MLORA_ERR_INVALID, "%s: a result overlaps a vector", who);
  }
  if (out && n.residual_out && (out == n.residual_out || overlap(out, n.out_stride, n.residual_out, n.residual_stride, n.T, n.H)))
    return fail(MLORA_ERR_INVALID, "%s: the results overlap", who);
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
  if (dtype == MLORA_F16) return vec ? launch<_Float16, true>(st, m) : launch<_Float16, false>(st, m);
  return vec ? launch<__bf16, true>(st, m) : launch<__bf16, false>(st, m);
}
