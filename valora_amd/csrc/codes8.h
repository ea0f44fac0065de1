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
// The least float that is not below x >= 0
__device__ __forceinline__ float not_below(double x) {
  const float f = (float)x;
  return (double)f < x ? as<float>(as<uint32_t>(f) + 1) : f;
}
__device__ __forceinline__ float not_below(float x) { return x; }
// x in 32 bits for a conversion that is still to come: cut off, with the last bit set where something was, so that what is next to the border of
// two codes stays on its side of it
__device__ __forceinline__ float sticky(double x) {
  float f = (float)x;
  if ((double)f != x) {
    const uint32_t b = as<uint32_t>(f) - (fabs((double)f) > fabs(x) ? 1u : 0u);
    f = as<float>(b | 1u);
  }
  return f;
}
__device__ __forceinline__ float sticky(float x) { return x; }
// Eight elements as codes of the power 2^(byte - 127)
template <typename F>
__device__ __forceinline__ u32x2 codes_of(const F (&x)[8], uint32_t byte) {
  F down;                                          // 2^(127 - byte)
  if constexpr (sizeof(F) == 8) down = as<double>((uint64_t)(1023 + 127 - byte) << 52);
  else down = as<float>((254u - byte) << 23);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const F z = x[i] * down;
    const float f = sticky(z > (F)448 ? (F)448 : z < (F)-448 ? (F)-448 : z);
    y[i] = z != z ? NAN : f;
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
