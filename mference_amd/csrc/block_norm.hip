// The norms around a block with its gate and residual scale (mf_block_norm).
#include <type_traits>

#include "mf_adapters.h"
#include "mf_device.h"

namespace mf {

namespace {

// sum over the workgroup, the same on every thread (part: a word a wave; the calls of a kernel take turns on two of them)
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = wave_sum(v);
  if (blockDim.x == 64) return v;
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float sum = 0.0f;
  for (uint32_t w = 0; w < blockDim.x / 64; ++w) sum += part[w];
  return sum;
}

// 1 / (1 + e^-x) on the hardware's exp2 and reciprocal (1 ulp each): it scales a term of a sum that is narrowed to bf16 at once
__device__ __forceinline__ float gate_of(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f)); }

__device__ __forceinline__ float inverse_rms(float squares, uint32_t d, float eps) { return 1.0f / __builtin_sqrtf(squares / static_cast<float>(d) + eps); }

// eight elements of a row of which `have` exist (1..8; 0 behind them)
__device__ __forceinline__ void load8(const uint16_t* p, uint32_t have, float (&v)[8]) {
  if (have == 8) {
    const uint4 w = load_16_bytes(p);
    v[0] = bf16_lo(w.x), v[1] = bf16_hi(w.x), v[2] = bf16_lo(w.y), v[3] = bf16_hi(w.y);
    v[4] = bf16_lo(w.z), v[5] = bf16_hi(w.z), v[6] = bf16_lo(w.w), v[7] = bf16_hi(w.w);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) v[e] = e < have ? bf16_to_f(p[e]) : 0.0f;
  }
}
__device__ __forceinline__ void load8(const float* p, uint32_t have, float (&v)[8]) {
  if (have == 8) {
    __builtin_memcpy(&v[0], p, 16);
    __builtin_memcpy(&v[4], p + 4, 16);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) v[e] = e < have ? p[e] : 0.0f;
  }
}
__device__ __forceinline__ void store8(uint16_t* p, uint32_t have, const uint16_t (&v)[8]) {
  if (have == 8) {
    __builtin_memcpy(p, v, 16);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e)
      if (e < have) p[e] = v[e];
  }
}

// A workgroup a row, the row in registers: NV pieces of eight elements a thread, all that the row takes part in requested at once,
// in front of the first sum; two sums over the workgroup; every byte read and written once.
template <int NV, bool F32>
__global__ __launch_bounds__(1024) void block_norm_kernel(const mf_block_norm_args a) {
  __shared__ float part[2][16];
  using Delta = std::conditional_t<F32, float, uint16_t>;
  const size_t row = blockIdx.x;
  uint16_t* hidden = a.hidden + row * a.hidden_stride;
  const Delta* delta = static_cast<const Delta*>(a.delta) + row * a.delta_stride;
  uint32_t at[NV], have[NV];
  float h[NV][8], b[NV][8], g[NV][8], post_w[NV][8], pre_w[NV][8];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    at[k] = (k * blockDim.x + threadIdx.x) * 8;
    have[k] = at[k] < a.d ? min(a.d - at[k], 8u) : 0;
    if (!have[k]) continue;
    load8(hidden + at[k], have[k], h[k]);
    if (a.delta) load8(delta + at[k], have[k], b[k]);
    if (a.gate_kind == MF_GATE_ELEMENT) load8(a.gate + row * a.gate_stride + at[k], have[k], g[k]);
    if (a.gate_kind == MF_GATE_CHANNEL) load8(a.gate + at[k], have[k], g[k]);
    if (a.post_weight) load8(a.post_weight + at[k], have[k], post_w[k]);
    if (a.pre_weight) load8(a.pre_weight + at[k], have[k], pre_w[k]);
  }
  if (a.delta) {
    float branch = a.branch_scale;
    if (a.gate_kind == MF_GATE_ROW) branch *= gate_of(bf16_to_f(a.gate[row * a.gate_stride]));
    if (a.post_weight) {
      float squares = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (!have[k]) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) squares = __builtin_fmaf(b[k][e], b[k][e], squares);
      }
      const float inv = inverse_rms(block_sum(squares, part[0]), a.d, a.post_eps);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) b[k][e] = b[k][e] * inv * (post_w[k][e] + a.weight_bias);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!have[k]) continue;
      uint16_t out[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = b[k][e];
        if (a.gate_kind == MF_GATE_ELEMENT) v *= gate_of(g[k][e]);
        if (a.gate_kind == MF_GATE_CHANNEL) v *= g[k][e];
        out[e] = narrow_bf16(a.residual_scale * h[k][e] + branch * v);
        h[k][e] = bf16_to_f(out[e]);
      }
      store8(hidden + at[k], have[k], out);
    }
  }
  if (!a.pre_weight) return;
  float squares = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (static_cast<uint32_t>(e) < have[k]) squares = __builtin_fmaf(h[k][e], h[k][e], squares);
  }
  const float inv = inverse_rms(block_sum(squares, part[1]), a.d, a.pre_eps);
  uint16_t* o = a.out + row * a.out_stride;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (!have[k]) continue;
    uint16_t out[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = narrow_bf16(h[k][e] * inv * (pre_w[k][e] + a.weight_bias));
    store8(o + at[k], have[k], out);
  }
}

// rows that registers do not hold: three passes of the workgroup over its row
template <bool F32>
__global__ __launch_bounds__(1024) void block_norm_long_kernel(const mf_block_norm_args a) {
  __shared__ float part[2][16];
  using Delta = std::conditional_t<F32, float, uint16_t>;
  const size_t row = blockIdx.x;
  uint16_t* hidden = a.hidden + row * a.hidden_stride;
  const Delta* delta = static_cast<const Delta*>(a.delta) + row * a.delta_stride;
  float branch = a.branch_scale, inv = 1.0f;
  if (a.gate_kind == MF_GATE_ROW) branch *= gate_of(bf16_to_f(a.gate[row * a.gate_stride]));
  if (a.post_weight) {
    float squares = 0.0f;
    for (uint32_t at = threadIdx.x * 8; at < a.d; at += blockDim.x * 8) {
      float b[8];
      load8(delta + at, min(a.d - at, 8u), b);
#pragma unroll
      for (int e = 0; e < 8; ++e) squares = __builtin_fmaf(b[e], b[e], squares);
    }
    inv = inverse_rms(block_sum(squares, part[0]), a.d, a.post_eps);
  }
  float squares = 0.0f;
  for (uint32_t at = threadIdx.x * 8; at < a.d; at += blockDim.x * 8) {
    const uint32_t have = min(a.d - at, 8u);
    float h[8];
    load8(hidden + at, have, h);
    if (a.delta) {
      float b[8], w[8], g[8];
      load8(delta + at, have, b);
      if (a.post_weight) load8(a.post_weight + at, have, w);
      if (a.gate_kind == MF_GATE_ELEMENT) load8(a.gate + row * a.gate_stride + at, have, g);
      if (a.gate_kind == MF_GATE_CHANNEL) load8(a.gate + at, have, g);
      uint16_t out[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = b[e];
        if (a.post_weight) v = v * inv * (w[e] + a.weight_bias);
        if (a.gate_kind == MF_GATE_ELEMENT) v *= gate_of(g[e]);
        if (a.gate_kind == MF_GATE_CHANNEL) v *= g[e];
        out[e] = narrow_bf16(a.residual_scale * h[e] + branch * v);
        h[e] = bf16_to_f(out[e]);
      }
      store8(hidden + at, have, out);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (static_cast<uint32_t>(e) < have) squares = __builtin_fmaf(h[e], h[e], squares);
  }
  if (!a.pre_weight) return;
  inv = inverse_rms(block_sum(squares, part[1]), a.d, a.pre_eps);
  for (uint32_t at = threadIdx.x * 8; at < a.d; at += blockDim.x * 8) {
    const uint32_t have = min(a.d - at, 8u);
    float h[8], w[8];
    load8(hidden + at, have, h);  // (the thread's own stores)
    load8(a.pre_weight + at, have, w);
    uint16_t out[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = narrow_bf16(h[e] * inv * (w[e] + a.weight_bias));
    store8(a.out + row * a.out_stride + at, have, out);
  }
}

template <bool F32>
void launch(hipStream_t s, const mf_block_norm_args& a) {
  const uint32_t pieces = a.d / 8 + (a.d % 8 != 0);
  const dim3 grid(a.t);
  if (pieces > 2048) {
    block_norm_long_kernel<F32><<<grid, dim3(1024), 0, s>>>(a);
  } else if (pieces > 1024 || (pieces > 128 && a.t > 512)) {
    block_norm_kernel<2, F32><<<grid, dim3((pieces + 127) / 128 * 64), 0, s>>>(a);
  } else {
    block_norm_kernel<1, F32><<<grid, dim3((pieces + 63) / 64 * 64), 0, s>>>(a);
  }
}

}  // namespace

hipError_t launch_block_norm(hipStream_t s, const mf_block_norm_args& a) {
  if (a.delta_f32) launch<true>(s, a);
  else launch<false>(s, a);
  return hipGetLastError();
}

}  // namespace mf
