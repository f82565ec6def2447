// The projection of 16-bit weights with bias, activation and residual in its epilogue (mf_project).
#include "mf_dense16.h"
#include "mf_dense16_device.h"

namespace mf {

namespace {

// the result of a token's row j from its sum (and, gated, from the sum of the up row): one rounding, at the end
template <bool GATED>
__device__ __forceinline__ float epilogue(const mf_project_args& a, float z, float up, uint32_t j) {
  if (a.bias) {
    z += bf16_to_f(a.bias[j]);
    if (GATED) up += bf16_to_f(a.bias[a.m + j]);
  }
  z = activate(z, a.activation);
  return GATED ? z * up : z;
}

__device__ __forceinline__ void store_result(const mf_project_args& a, uint32_t i, uint32_t j, float v) {
  const size_t at = static_cast<size_t>(i) * a.y_stride + j, from = static_cast<size_t>(i) * a.residual_stride + j;
  if (a.y_f32) {
    if (a.residual) v += static_cast<const float*>(a.residual)[from];
    static_cast<float*>(a.y)[at] = v;
  } else {
    if (a.residual) v += bf16_to_f(static_cast<const uint16_t*>(a.residual)[from]);
    static_cast<uint16_t*>(a.y)[at] = narrow_bf16(v);
  }
}

// The simple form: a wave 16 rows of W and 64 tokens, operands straight from memory.
template <bool GATED>
__global__ __launch_bounds__(256) void project_kernel(const mf_project_args a) {
  const uint32_t lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const uint32_t j0 = blockIdx.x * 64 + (threadIdx.x >> 6) * 16, i0 = blockIdx.y * 64;
  if (j0 >= a.m) return;
  const uint16_t* w = a.w + static_cast<size_t>(min(j0 + r, a.m - 1)) * a.w_stride;
  const uint16_t* up = w + static_cast<size_t>(GATED ? a.m : 0) * a.w_stride;
  const uint16_t* x[4];
  for (uint32_t c = 0; c < 4; ++c) x[c] = a.x + static_cast<size_t>(min(i0 + c * 16 + r, a.t - 1)) * a.x_stride;
  f32x4_t sum[4] = {}, up_sum[4] = {};
  for (uint32_t k = g * 8; k - g * 8 < a.n; k += 32) {
    const uint32_t have = k < a.n ? a.n - k : 0;
    const uint4 wk = load_bf16x8_guarded(w + k, have);
    uint4 uk = wk;
    if (GATED) uk = load_bf16x8_guarded(up + k, have);
#pragma unroll
    for (uint32_t c = 0; c < 4; ++c) {
      const uint4 xk = load_bf16x8_guarded(x[c] + k, have);
      sum[c] = mfma16(wk, xk, sum[c]);
      if (GATED) up_sum[c] = mfma16(uk, xk, up_sum[c]);
    }
  }
#pragma unroll
  for (uint32_t c = 0; c < 4; ++c) {
    const uint32_t i = i0 + c * 16 + r;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      const uint32_t j = j0 + g * 4 + e;
      if (i < a.t && j < a.m) store_result(a, i, j, epilogue<GATED>(a, sum[c][e], up_sum[c][e], j));
    }
  }
}

}  // namespace

size_t project_workspace_bytes(uint32_t m, uint32_t n, uint32_t t, bool gated) { return 0; }

hipError_t launch_project(hipStream_t s, const mf_project_args& a, void* workspace) {
  const dim3 grid((a.m + 63) / 64, (a.t + 63) / 64);
  if (a.gated) project_kernel<true><<<grid, 256, 0, s>>>(a);
  else project_kernel<false><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace mf
