// The 8-bit cache's values: code * 2^e, an e4m3 code an element and one power of two (e8m0, a byte: e + 127) a token, key head and of k
// and v.  e is the least with which the head's largest element is at most 448, e4m3's largest value, within the bounds that make
// every code times its power a value of the model's type, so that reading back rounds nothing: in fp16 2^-9 * 2^-15 is the least value there is
// and 448 * 2^7 fits; in bf16 448 * 2^119 fits, and 2^-9 * 2^-117 is not subnormal.
#pragma once

#include "kernel_common.h"

namespace mlora {

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

template <typename T>
struct Powers;
template <>
struct Powers<_Float16> {
  static constexpr int LOWEST = -15, HIGHEST = 7;
};
template <>
struct Powers<__bf16> {
  static constexpr int LOWEST = -117, HIGHEST = 119;
};

// 2^e from the bytes {k's, v's} of a token and key head (the conversions below take a power's exponent alone)
__device__ __forceinline__ float k_power(uint32_t e) { return as<float>((e & 0xffu) << 23); }
__device__ __forceinline__ float v_power(uint32_t e) { return as<float>((e >> 8 & 0xffu) << 23); }

// Eight codes times a power: an instruction for two
template <typename T>
__device__ __forceinline__ typename Traits<T>::vec8 values_of(u32x2 codes, float power) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (__is_same(T, _Float16)) {
      r[2 * i] = as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[i], power, false));
      r[2 * i + 1] = as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[i], power, true));
    } else {
      r[2 * i] = as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[i], power, false));
      r[2 * i + 1] = as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[i], power, true));
    }
  }
  return as<typename Traits<T>::vec8>(r);
}

// The power of a head whose largest finite element is `largest`, as its byte.  448 is 1.75 * 2^8: above a fraction of .75 the sum carries.
template <typename T>
__device__ __forceinline__ uint32_t power_byte(float largest) {
  const int e = (int)((as<uint32_t>(largest) + 0x1fffffu) >> 23) - 8;
  return (uint32_t)min(max(e, Powers<T>::LOWEST + 127), Powers<T>::HIGHEST + 127);
}
// x in 32 bits for a conversion that is still to come: its first 20 bits behind the point, with the last of them set where more followed, so that
// what is next to the border of two codes, or above a power's largest value, stays on its side of it
__device__ __forceinline__ float sticky(double x) {
  const uint64_t b = as<uint64_t>(x);
  const uint32_t hi = (uint32_t)(b >> 32) | ((uint32_t)b ? 1u : 0u);
  return (float)as<double>((uint64_t)hi << 32);
}
// Eight elements as codes of the power 2^(byte - 127)
__device__ __forceinline__ u32x2 codes_of(const float (&x)[8], uint32_t byte) {
  const float down = as<float>((254u - byte) << 23);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float z = x[i] * down;
    y[i] = z != z ? z : __builtin_amdgcn_fmed3f(z, -448.0f, 448.0f);
  }
  u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
    r[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], w, true);
  }
  return r;
}

}  // namespace mlora
