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

// eight elements of a row of which `have` exist (1..8; 0 behind them), as they lie in memory
struct Raw16 {
  uint4 w;
  __device__ __forceinline__ void load(const uint16_t* p, uint32_t have) {
    if (have == 8) {
      w = load_16_bytes(p);
    } else {
      uint32_t e[8];
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) e[k] = k < have ? p[k] : 0u;
      w = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
    }
  }
  __device__ __forceinline__ float operator[](int k) const {
    const uint32_t pair = k < 2 ? w.x : k < 4 ? w.y : k < 6 ? w.z : w.w;
    return k % 2 ? bf16_hi(pair) : bf16_lo(pair);
  }
};
struct Raw32 {
  float v[8];
  __device__ __forceinline__ void load(const float* p, uint32_t have) {
    if (have == 8) {
      __builtin_memcpy(&v[0], p, 16);
      __builtin_memcpy(&v[4], p + 4, 16);
    } else {
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) v[k] = k < have ? p[k] : 0.0f;
    }
  }
  __device__ __forceinline__ float operator[](int k) const { return v[k]; }
};
__device__ __forceinline__ uint32_t narrow_pair(float lo, float hi) { return static_cast<uint32_t>(narrow_bf16(lo)) | static_cast<uint32_t>(narrow_bf16(hi)) << 16; }
__device__ __forceinline__ void store8(uint16_t* p, uint32_t have, const uint4& v) {
  if (have == 8) {
    __builtin_memcpy(p, &v, 16);
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e)
      if (e < have) p[e] = static_cast<uint16_t>(w[e / 2] >> (e % 2 * 16));
  }
}

// A workgroup a row, the row in registers: NV pieces of eight elements a thread, all that the row takes part in requested at once,
// in front of the first sum, and kept as it lies in memory until it is used; two sums over the workgroup; every byte read and
// written once.  Long batches run at the rate of a copy: 8192 rows of 5120, all operands bf16, 71 us, 168 MB read and 168 written = 4.8 TB/s.  Short
// ones are the latency of a request, two sums and a launch: one row of 2048 2.7 us, eight of 2816 4.4, 777 of 4096 with an fp32 block output and a gate
// an element 11.4 us (25.7 + 12.7 MB).
// Calls of the simple form (three passes over the row) took 8.2, 8.8, 28 and 217 us, in the order of one, eight, 777 and 8192 rows.
template <int NV, bool F32>
__global__ __launch_bounds__(1024) void block_norm_kernel(const mf_block_norm_args a) {
  __shared__ float part[2][16];
  using Delta = std::conditional_t<F32, float, uint16_t>;
  using RawDelta = std::conditional_t<F32, Raw32, Raw16>;
  const size_t row = blockIdx.x;
  uint16_t* hidden = a.hidden + row * a.hidden_stride;
  const Delta* delta = static_cast<const Delta*>(a.delta) + row * a.delta_stride;
  uint32_t at[NV], have[NV];
  Raw16 h[NV], g[NV], post_w[NV], pre_w[NV];
  RawDelta b[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    at[k] = (k * blockDim.x + threadIdx.x) * 8;
    have[k] = at[k] < a.d ? min(a.d - at[k], 8u) : 0;
    if (!have[k]) continue;
    if (a.delta) b[k].load(delta + at[k], have[k]);
    h[k].load(hidden + at[k], have[k]);
    if (a.gate_kind == MF_GATE_ELEMENT) g[k].load(a.gate + row * a.gate_stride + at[k], have[k]);
    if (a.gate_kind == MF_GATE_CHANNEL) g[k].load(a.gate + at[k], have[k]);
    if (a.post_weight) post_w[k].load(a.post_weight + at[k], have[k]);
    if (a.pre_weight) pre_w[k].load(a.pre_weight + at[k], have[k]);
  }
  if (a.delta) {
    float branch = a.branch_scale, inv = 1.0f;
    if (a.gate_kind == MF_GATE_ROW) branch *= gate_of(bf16_to_f(a.gate[row * a.gate_stride]));
    if (a.post_weight) {
      float squares = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (!have[k]) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) squares = __builtin_fmaf(b[k][e], b[k][e], squares);
      }
      inv = inverse_rms(block_sum(squares, part[0]), a.d, a.post_eps);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!have[k]) continue;
      uint32_t out[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          v[i] = b[k][e + i];
          if (a.post_weight) v[i] = v[i] * inv * (post_w[k][e + i] + a.weight_bias);
          if (a.gate_kind == MF_GATE_ELEMENT) v[i] *= gate_of(g[k][e + i]);
          if (a.gate_kind == MF_GATE_CHANNEL) v[i] *= g[k][e + i];
          v[i] = a.residual_scale * h[k][e + i] + branch * v[i];
        }
        out[e / 2] = narrow_pair(v[0], v[1]);
      }
      h[k].w = make_uint4(out[0], out[1], out[2], out[3]);
      store8(hidden + at[k], have[k], h[k].w);
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
    uint32_t out[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      out[e / 2] = narrow_pair(h[k][e] * inv * (pre_w[k][e] + a.weight_bias), h[k][e + 1] * inv * (pre_w[k][e + 1] + a.weight_bias));
    store8(o + at[k], have[k], make_uint4(out[0], out[1], out[2], out[3]));
  }
}

// Rows that registers do not hold: three passes of the workgroup over its row, the later ones mostly from the caches.  Both norms, all operands bf16, us a
// pass: 512 rows of 32768 33.4, 2048 of 20000 78.8 (4.0 and 4.2 TB/s of the bytes that one pass would move; 2048 rows of 16384, in registers, 57.0 = 4.7),
// one row of 32768 11.0.
template <bool F32>
__global__ __launch_bounds__(1024) void block_norm_long_kernel(const mf_block_norm_args a) {
  __shared__ float part[2][16];
  using Delta = std::conditional_t<F32, float, uint16_t>;
  using RawDelta = std::conditional_t<F32, Raw32, Raw16>;
  const size_t row = blockIdx.x;
  uint16_t* hidden = a.hidden + row * a.hidden_stride;
  const Delta* delta = static_cast<const Delta*>(a.delta) + row * a.delta_stride;
  float branch = a.branch_scale, inv = 1.0f;
  if (a.gate_kind == MF_GATE_ROW) branch *= gate_of(bf16_to_f(a.gate[row * a.gate_stride]));
  if (a.post_weight) {
    float squares = 0.0f;
    for (uint32_t at = threadIdx.x * 8; at < a.d; at += blockDim.x * 8) {
      RawDelta b;
      b.load(delta + at, min(a.d - at, 8u));
#pragma unroll
      for (int e = 0; e < 8; ++e) squares = __builtin_fmaf(b[e], b[e], squares);
    }
    inv = inverse_rms(block_sum(squares, part[0]), a.d, a.post_eps);
  }
  float squares = 0.0f;
  for (uint32_t at = threadIdx.x * 8; at < a.d; at += blockDim.x * 8) {
    const uint32_t have = min(a.d - at, 8u);
    Raw16 h, w, g;
    h.load(hidden + at, have);
    if (a.delta) {
      RawDelta b;
      b.load(delta + at, have);
      if (a.post_weight) w.load(a.post_weight + at, have);
      if (a.gate_kind == MF_GATE_ELEMENT) g.load(a.gate + row * a.gate_stride + at, have);
      if (a.gate_kind == MF_GATE_CHANNEL) g.load(a.gate + at, have);
      uint32_t out[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          v[i] = b[e + i];
          if (a.post_weight) v[i] = v[i] * inv * (w[e + i] + a.weight_bias);
          if (a.gate_kind == MF_GATE_ELEMENT) v[i] *= gate_of(g[e + i]);
          if (a.gate_kind == MF_GATE_CHANNEL) v[i] *= g[e + i];
          v[i] = a.residual_scale * h[e + i] + branch * v[i];
        }
        out[e / 2] = narrow_pair(v[0], v[1]);
      }
      h.w = make_uint4(out[0], out[1], out[2], out[3]);
      store8(hidden + at, have, h.w);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (static_cast<uint32_t>(e) < have) squares = __builtin_fmaf(h[e], h[e], squares);
  }
  if (!a.pre_weight) return;
  inv = inverse_rms(block_sum(squares, part[1]), a.d, a.pre_eps);
  for (uint32_t at = threadIdx.x * 8; at < a.d; at += blockDim.x * 8) {
    const uint32_t have = min(a.d - at, 8u);
    Raw16 h, w;
    h.load(hidden + at, have);  // (the thread's own stores)
    w.load(a.pre_weight + at, have);
    uint32_t out[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) out[e / 2] = narrow_pair(h[e] * inv * (w[e] + a.weight_bias), h[e + 1] * inv * (w[e + 1] + a.weight_bias));
    store8(a.out + row * a.out_stride + at, have, make_uint4(out[0], out[1], out[2], out[3]));
  }
}

template <bool F32>
void launch(hipStream_t s, const mf_block_norm_args& a) {
  const uint32_t pieces = a.d / 8 + (a.d % 8 != 0);
  const dim3 grid(a.t);
  if (pieces > 2048) {
    block_norm_long_kernel<F32><<<grid, dim3(1024), 0, s>>>(a);
  } else if (pieces > 1024 || (pieces > 128 && a.t > 1024)) {
    // two pieces a thread where there are rows enough to fill the chip either way: the waves' common work is halved (us, one piece /
    // two: 8192 rows of 5120, all operands bf16, 93 / 70; 777 of 4096, fp32 block output and a gate an element, 11.6 / 12.2; 8 of 2816 4.4 / 5.1)
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
