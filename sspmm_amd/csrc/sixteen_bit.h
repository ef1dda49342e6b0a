// fp16 and bf16 under one set of names: conversions, and the matrix instructions that take them.
#ifndef SSPMM_AMD_SIXTEEN_BIT_H
#define SSPMM_AMD_SIXTEEN_BIT_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sspmm {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

struct Fp16 {
  typedef _Float16 vec8 __attribute__((ext_vector_type(8)));
  typedef _Float16 vec2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kExponent = 0x7c00;
  // two values rounded to nearest, ties to even, lo in the lower half
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const vec2 h = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, h);
  }
  static __device__ __forceinline__ float lower(uint32_t u) { return (float)__builtin_bit_cast(vec2, u)[0]; }
  static __device__ __forceinline__ float upper(uint32_t u) { return (float)__builtin_bit_cast(vec2, u)[1]; }
  static __device__ __forceinline__ floatx16 mfma_32x32x16(uintx4 a, uintx4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ floatx4 mfma_16x16x32(uintx4 a, uintx4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
  }
};

struct Bf16 {
  typedef __bf16 vec8 __attribute__((ext_vector_type(8)));
  typedef __bf16 vec2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kExponent = 0x7f80;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const vec2 h = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, h);
  }
  static __device__ __forceinline__ float lower(uint32_t u) { return __uint_as_float(u << 16); }
  static __device__ __forceinline__ float upper(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
  static __device__ __forceinline__ floatx16 mfma_32x32x16(uintx4 a, uintx4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ floatx4 mfma_16x16x32(uintx4 a, uintx4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
  }
};

// The eight values with zeros in place of infinities and NaN.
template <typename T>
__device__ __forceinline__ uintx4 finite_part(uintx4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((v[i] & T::kExponent) == T::kExponent) v[i] &= 0xffff0000u;
    if (((v[i] >> 16) & T::kExponent) == T::kExponent) v[i] &= 0xffffu;
  }
  return v;
}

}  // namespace sspmm
#endif
