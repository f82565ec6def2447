// What the kernels of the 16-bit operators share.
#pragma once

#include "mf_device.h"

namespace mf {

// D[16 rows, 16 columns] += A[16, 32] B[32, 16]: lane l holds eight k's from 8 (l / 16) on of A's row l % 16 and of B's column l % 16, and
// rows 4 (l / 16) .. + 3 of D's column l % 16
__device__ __forceinline__ f32x4_t mfma16(const uint4& a, const uint4& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// The activations on the hardware's exp2 and reciprocal (1 ulp each), from fp32 sums; the erf form on the library's erf.  The tanh form is
// x / (1 + e^(-2u)), which is 0.5 x (1 + tanh u) without its cancellation.
__device__ __forceinline__ float activate(float z, mf_activation act) {
  if (act == MF_ACT_SILU) return fast_silu(z);
  if (act == MF_ACT_GELU_TANH) return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.3022081986f * (z + 0.044715f * z * z * z)));
  if (act == MF_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  return z;
}

}  // namespace mf
