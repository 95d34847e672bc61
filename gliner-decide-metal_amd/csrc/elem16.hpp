// The two 16-bit element types of the packed-row operators: vector types,
// the MFMA forms, and a sum of two elements onto fp32 (subnormal elements count).
#pragma once

#include "gd_common.hpp"

namespace gd {

typedef __bf16 bf16_t;

template <class T>
struct Elem;

template <>
struct Elem<half_t> {
  typedef half2_t v2;
  typedef half4_t v4;
  typedef half8_t v8;
  static __device__ __forceinline__ float4_t mfma16(v8 a, v8 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float16_t mfma32(v8 a, v8 b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(v2 a, float c) {
    return __builtin_amdgcn_fdot2(a, (v2){(half_t)1.f, (half_t)1.f}, c, false);
  }
};

template <>
struct Elem<bf16_t> {
  typedef bf16_t v2 __attribute__((ext_vector_type(2)));
  typedef bf16_t v4 __attribute__((ext_vector_type(4)));
  typedef bf16_t v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float4_t mfma16(v8 a, v8 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float16_t mfma32(v8 a, v8 b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(v2 a, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(a, (v2){(bf16_t)1.f, (bf16_t)1.f}, c, false);
  }
};

}  // namespace gd
