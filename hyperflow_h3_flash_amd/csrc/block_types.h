// The two 16-bit element types of the attention block's operators: conversions and matrix products.
#pragma once

#include "common.h"

namespace hf {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct Bf16 {
  static constexpr uint32_t kExponent = 0x7f80u, kOne = 0x3f80u;
  static constexpr bool kNarrow = false;  // float32's exponents
  static __device__ __forceinline__ float lo(uint32_t pair) { return bf16_lo(pair); }
  static __device__ __forceinline__ float hi(uint32_t pair) { return bf16_hi(pair); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ v16f mfma(v4u a, v4u b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};

struct Fp16 {
  static constexpr uint32_t kExponent = 0x7c00u, kOne = 0x3c00u;
  static constexpr bool kNarrow = true;
  static __device__ __forceinline__ float lo(uint32_t pair) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(pair & 0xffffu));
  }
  static __device__ __forceinline__ float hi(uint32_t pair) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(pair >> 16));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {  // round to nearest even
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, h2));
  }
  static __device__ __forceinline__ v16f mfma(v4u a, v4u b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};

// Lane l exchanges with lane l ^ 32: max of both.
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Over lanes l, l ^ 16, l ^ 32 and l ^ 48.
__device__ __forceinline__ float quad_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quad_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

}  // namespace hf
