// The norms around a block with its gate and residual scale (mf_block_norm).
#include "mf_adapters.h"
#include "mf_device.h"

namespace mf {

namespace {

// sum over the workgroup, the same on every thread
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float sum = 0.0f;
  for (uint32_t w = 0; w < blockDim.x / 64; ++w) sum += part[w];
  return sum;
}

// one workgroup per row, an element at a time
template <bool F32>
__global__ __launch_bounds__(256) void block_norm_kernel(const mf_block_norm_args a) {
  __shared__ float part[4];
  const size_t row = blockIdx.x;
  uint16_t* h = a.hidden + row * a.hidden_stride;
  uint16_t* o = a.pre_weight ? a.out + row * a.out_stride : nullptr;
  auto block = [&](uint32_t i) {
    if constexpr (F32) return static_cast<const float*>(a.delta)[row * a.delta_stride + i];
    else return bf16_to_f(static_cast<const uint16_t*>(a.delta)[row * a.delta_stride + i]);
  };
  float post = 1.0f;
  if (a.post_weight) {
    float sum = 0.0f;
    for (uint32_t i = threadIdx.x; i < a.d; i += 256) sum = __builtin_fmaf(block(i), block(i), sum);
    post = 1.0f / __builtin_sqrtf(block_sum(sum, part) / static_cast<float>(a.d) + a.post_eps);
  }
  float row_gate = 1.0f;
  if (a.gate_kind == MF_GATE_ROW) row_gate = 1.0f / (1.0f + mf_exp(-bf16_to_f(a.gate[row * a.gate_stride])));
  float sum = 0.0f;
  for (uint32_t i = threadIdx.x; i < a.d; i += 256) {
    float v = bf16_to_f(h[i]);
    if (a.delta) {
      float b = block(i);
      if (a.post_weight) b = b * post * (bf16_to_f(a.post_weight[i]) + a.weight_bias);
      float g = row_gate;
      if (a.gate_kind == MF_GATE_ELEMENT) g = 1.0f / (1.0f + mf_exp(-bf16_to_f(a.gate[row * a.gate_stride + i])));
      if (a.gate_kind == MF_GATE_CHANNEL) g = bf16_to_f(a.gate[i]);
      const uint16_t hb = narrow_bf16(a.residual_scale * v + a.branch_scale * (b * g));
      h[i] = hb;
      v = bf16_to_f(hb);
    }
    sum = __builtin_fmaf(v, v, sum);
  }
  if (!a.pre_weight) return;
  const float pre = 1.0f / __builtin_sqrtf(block_sum(sum, part) / static_cast<float>(a.d) + a.pre_eps);
  for (uint32_t i = threadIdx.x; i < a.d; i += 256)
    o[i] = narrow_bf16(bf16_to_f(h[i]) * pre * (bf16_to_f(a.pre_weight[i]) + a.weight_bias));
}

}  // namespace

hipError_t launch_block_norm(hipStream_t s, const mf_block_norm_args& a) {
  if (a.delta_f32) block_norm_kernel<true><<<dim3(a.t), dim3(256), 0, s>>>(a);
  else block_norm_kernel<false><<<dim3(a.t), dim3(256), 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace mf
