// What kernels that read the paged cache in 8 bits share: its codes as operands of the matrix instructions.
#ifndef SSPMM_AMD_CACHE_CODES_H
#define SSPMM_AMD_CACHE_CODES_H

#include "lane_ops.h"
#include "sixteen_bit.h"

namespace sspmm {

__device__ __forceinline__ floatx4 mfma(uintx4 a, uintx4 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Fp16::vec8, a), __builtin_bit_cast(Fp16::vec8, b), c, 0, 0, 0);
}

// Eight codes as fp16, which holds either format's values exactly.
template <int FORMAT>
__device__ __forceinline__ uintx4 as_halfs(uint32_t lo, uint32_t hi) {
  uintx4 r;
  const uint32_t w[2] = {lo, hi};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (FORMAT == 0) {
      // 0x6400 + u is 1024 + u in fp16, u = code + 128
      const uint32_t u = w[i] ^ 0x80808080u;
      const Fp16::vec2 off = {(_Float16)1152, (_Float16)1152};
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(Fp16::vec2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off);
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(Fp16::vec2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off);
    } else {
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, false));
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, true));
    }
  }
  return r;
}

// Sums of values are kept in units of 2^16: probabilities are up to 2^15 and values of bf16 as large as 32 bits hold, and the sum must not overflow where the
// formula's does not.  (A scale may lose what is then below 32 bits' smallest number: 2^-127 of a value at most.)
constexpr float kValueUnit = 0x1p-16f;

}  // namespace sspmm
#endif
