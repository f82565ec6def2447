// The layer of 16-bit experts for a few tokens (mf_bf16_experts).
#include <algorithm>

#include "mf_dense16.h"
#include "mf_dense16_device.h"

namespace mf {

namespace {

constexpr uint32_t kWaves = 8;

// eight values from k on of a row of n (a multiple of 8); zeros behind it
__device__ __forceinline__ uint4 load8(const uint16_t* row, uint32_t k, uint32_t n) {
  return k < n ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0, 0, 0, 0);
}

// sum over the workgroup's first `waves` parts of word i
__device__ __forceinline__ float sum_parts(const float* part, uint32_t stride, uint32_t i) {
  float v = 0.0f;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) v += part[w * stride + i];
  return v;
}

// The first launch: activations of 16 gate and 16 up rows of one live expert (or of the shared one) for all of its routes.  The waves
// share the sum over d.  A workgroup finds its expert, the blockIdx.y-th that the batch names, and that expert's routes from the indices by itself; the
// first of an expert's workgroups writes them down for the second launch.
template <uint32_t NT>
__global__ __launch_bounds__(64 * kWaves) void experts_up_kernel(const Bf16ExpertsArgs a) {
  __shared__ uint32_t bits[MF_MAX_EXPERTS / 32], list[MF_BF16_EXPERTS_ROWS * MF_MAX_TOPK], mine_in[kWaves], front_in[kWaves];
  __shared__ float part[kWaves][2 * NT * 256];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
  const uint32_t most = a.most_live(), routes = a.route_count(), d = a.pool.d;
  if (blockIdx.y > most) {  // the shared expert's gate, a token a workgroup
    for (uint32_t i = blockIdx.x; i < a.t; i += gridDim.x) {
      const uint16_t* x = a.x + static_cast<size_t>(i) * a.x_stride;
      float v = 0.0f;
      for (uint32_t k = tid; k < d; k += 64 * kWaves) v = __builtin_fmaf(bf16_to_f(x[k]), bf16_to_f(a.pool.shared_gate[k]), v);
      v = wave_sum(v);
      if (lane == 0) part[wave][0] = v;
      __syncthreads();
      if (tid == 0) a.shared_gate[i] = sum_parts(&part[0][0], 2 * NT * 256, 0);
      __syncthreads();
    }
    return;
  }
  const bool shared = blockIdx.y == most;
  const uint32_t f = shared ? a.pool.shared_f : a.pool.f, j0 = blockIdx.x * 16;
  if (j0 >= f) return;
  uint32_t expert = 0, count = a.t;
  if (!shared) {
    const uint32_t e = tid < routes ? a.idx[tid] : ~0u;
    if (tid < MF_MAX_EXPERTS / 32) bits[tid] = 0;
    __syncthreads();
    const bool valid = e < a.pool.num_experts;
    if (valid) atomicOr(&bits[e / 32], 1u << (e & 31));
    __syncthreads();
    uint32_t rank = blockIdx.y, live = 0;
    expert = ~0u;
    for (uint32_t w = 0; w < MF_MAX_EXPERTS / 32; ++w) {
      uint32_t word = bits[w];
      const uint32_t here = __popc(word);
      if (rank >= live && rank < live + here) {
        for (uint32_t skip = rank - live; skip; --skip) word &= word - 1;
        expert = w * 32 + __ffs(static_cast<int>(word)) - 1;
      }
      live += here;
    }
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) a.plan[0] = live;
    if (expert == ~0u) return;
    const uint64_t mine = __ballot(valid && e == expert), front = __ballot(valid && e < expert);
    if (lane == 0) mine_in[wave] = __popcll(mine), front_in[wave] = __popcll(front);
    __syncthreads();
    uint32_t at = 0, first = 0;
    count = 0;
    for (uint32_t w = 0; w < kWaves; ++w) {
      if (w < wave) at += mine_in[w];
      count += mine_in[w];
      first += front_in[w];
    }
    if (valid && e == expert) {
      at += lanes_in_front(mine);
      list[at] = tid;
      if (blockIdx.x == 0) a.routes[first + at] = tid;
    }
    if (blockIdx.x == 0 && tid == 0) *reinterpret_cast<uint4*>(a.plan + 4 + 4 * blockIdx.y) = make_uint4(expert, first, count, 0);
    __syncthreads();
  }
  const uint16_t* w = shared ? a.pool.shared_gate_up : a.pool.gate_up + static_cast<size_t>(expert) * 2 * f * d;
  const uint16_t* gate = w + static_cast<size_t>(min(j0 + r, f - 1)) * d;
  const uint16_t* up = gate + static_cast<size_t>(f) * d;
  const uint16_t* bias = shared || !a.pool.gate_up_bias ? nullptr : a.pool.gate_up_bias + static_cast<size_t>(expert) * 2 * f;
  uint16_t* acts = shared ? a.shared_acts : a.acts;
  const size_t plane = static_cast<size_t>(shared ? a.t : routes) * f;
  const uint32_t steps = (d + 31) / 32, share = (steps + kWaves - 1) / kWaves;
  const uint32_t from = wave * share, to = min(from + share, steps);
  for (uint32_t base = 0; base < count; base += 16 * NT) {
    const uint16_t* x[NT];
#pragma unroll
    for (uint32_t c = 0; c < NT; ++c) {
      const uint32_t at = min(base + c * 16 + r, count - 1), token = shared ? at : list[at] / a.pool.top_k;
      x[c] = a.x + static_cast<size_t>(token) * a.x_stride;
    }
    f32x4_t zg[NT] = {}, zu[NT] = {};
    for (uint32_t step = from; step < to; ++step) {
      const uint32_t k = step * 32 + g * 8;
      const uint4 wg = load8(gate, k, d), wu = load8(up, k, d);
#pragma unroll
      for (uint32_t c = 0; c < NT; ++c) {
        uint4 xk = make_uint4(0, 0, 0, 0);
        if (k < d) xk = load_16_bytes(x[c] + k);
        zg[c] = mfma16(wg, xk, zg[c]);
        zu[c] = mfma16(wu, xk, zu[c]);
      }
    }
#pragma unroll
    for (uint32_t c = 0; c < NT; ++c)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        part[wave][(2 * c) * 256 + r * 16 + g * 4 + e] = zg[c][e];
        part[wave][(2 * c + 1) * 256 + r * 16 + g * 4 + e] = zu[c][e];
      }
    __syncthreads();
    for (uint32_t o = tid; o < NT * 256; o += 64 * kWaves) {
      const uint32_t c = o / 256, column = base + c * 16 + o % 256 / 16, j = j0 + o % 16;
      if (column < count && j < f) {
        float zg1 = sum_parts(&part[0][0], 2 * NT * 256, 2 * c * 256 + o % 256), zu1 = sum_parts(&part[0][0], 2 * NT * 256, (2 * c + 1) * 256 + o % 256);
        if (bias) zg1 += bf16_to_f(bias[j]), zu1 += bf16_to_f(bias[f + j]);
        const float act = activate(zg1, a.pool.activation) * zu1;
        const size_t at = static_cast<size_t>(shared ? column : list[column]) * f + j;
        const uint16_t high = narrow_bf16(act);
        acts[at] = high;
        acts[plane + at] = narrow_bf16(__builtin_isfinite(bf16_to_f(high)) ? act - bf16_to_f(high) : 0.0f);
      }
    }
    __syncthreads();
  }
}

// The second launch: 16 results of every token.  A wave takes a share of the live experts' (and the shared one's) down rows, every
// route's sum goes to LDS, and the weighted sums over a token's routes are made there in the order of their ranks.
__global__ __launch_bounds__(64 * kWaves) void experts_down_kernel(const Bf16ExpertsArgs a, uint32_t k_parts) {
  extern __shared__ float sums[];  // [k_parts][routes + shared rows][16]
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
  const uint32_t d = a.pool.d, routes = a.route_count(), rows = routes + (a.pool.shared_f ? a.t : 0), j0 = blockIdx.x * 16;
  const uint32_t live = a.plan[0], items = (live + (a.pool.shared_f ? 1 : 0)) * k_parts;
  for (uint32_t item = wave; item < items; item += kWaves) {
    const uint32_t entry = item / k_parts, k_part = item % k_parts;
    const bool shared = entry == live;
    const uint32_t f = shared ? a.pool.shared_f : a.pool.f;
    uint4 who = make_uint4(0, 0, a.t, 0);
    if (!shared) who = *reinterpret_cast<const uint4*>(a.plan + 4 + 4 * entry);
    const uint16_t* acts = shared ? a.shared_acts : a.acts;
    const size_t plane = static_cast<size_t>(shared ? a.t : routes) * f;
    const uint16_t* w = (shared ? a.pool.shared_down : a.pool.down + static_cast<size_t>(who.x) * d * f) + static_cast<size_t>(min(j0 + r, d - 1)) * f;
    const uint32_t steps = (f + 31) / 32, share = (steps + k_parts - 1) / k_parts, from = k_part * share, to = min(from + share, steps);
    for (uint32_t base = 0; base < who.z; base += 16) {
      const uint32_t at = min(base + r, who.z - 1), route = shared ? at : a.routes[who.y + at];
      const uint16_t* act = acts + static_cast<size_t>(route) * f;
      f32x4_t sum = {};
      for (uint32_t step = from; step < to; ++step) {
        const uint32_t k = step * 32 + g * 8;
        const uint4 wk = load8(w, k, f);
        sum = mfma16(wk, load8(act, k, f), sum);
        sum = mfma16(wk, load8(act + plane, k, f), sum);
      }
      if (base + r < who.z) *reinterpret_cast<f32x4_t*>(sums + (static_cast<size_t>(k_part) * rows + (shared ? routes : 0) + route) * 16 + g * 4) = sum;
    }
  }
  __syncthreads();
  for (uint32_t o = tid; o < a.t * 16; o += 64 * kWaves) {
    const uint32_t i = o / 16, row = o % 16, j = j0 + row;
    if (j >= d) continue;
    float v = a.residual ? bf16_to_f(a.residual[static_cast<size_t>(i) * a.residual_stride + j]) : 0.0f;
    for (uint32_t k = 0; k < a.pool.top_k; ++k) {
      const uint32_t route = i * a.pool.top_k + k, e = a.idx[route];
      if (e >= a.pool.num_experts) continue;
      float z = 0.0f;
      for (uint32_t p = 0; p < k_parts; ++p) z += sums[(static_cast<size_t>(p) * rows + route) * 16 + row];
      if (a.pool.down_bias) z += bf16_to_f(a.pool.down_bias[static_cast<size_t>(e) * d + j]);
      v += a.w[route] * z;
    }
    if (a.pool.shared_f) {
      float z = 0.0f;
      for (uint32_t p = 0; p < k_parts; ++p) z += sums[(static_cast<size_t>(p) * rows + routes + i) * 16 + row];
      if (a.pool.shared_gate) z *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a.shared_gate[i] * -1.4426950408889634f));
      v += z;
    }
    a.y[static_cast<size_t>(i) * a.y_stride + j] = narrow_bf16(v);
  }
}

size_t round16(size_t bytes) { return (bytes + 15) / 16 * 16; }

}  // namespace

void bf16_experts_layout(Bf16ExpertsArgs& a, void* workspace) {
  auto* p = static_cast<unsigned char*>(workspace);
  a.plan = reinterpret_cast<uint32_t*>(p);
  p += 16 + 16 * static_cast<size_t>(a.most_live());
  a.routes = reinterpret_cast<uint32_t*>(p);
  p += round16(4 * static_cast<size_t>(a.route_count()));
  a.shared_gate = reinterpret_cast<float*>(p);
  p += round16(4 * static_cast<size_t>(a.t));
  a.acts = reinterpret_cast<uint16_t*>(p);
  p += 4 * static_cast<size_t>(a.route_count()) * a.pool.f;  // (f is a multiple of 8)
  a.shared_acts = reinterpret_cast<uint16_t*>(p);
}

size_t bf16_experts_workspace_bytes(const mf_bf16_expert_pool& pool, uint32_t t) {
  Bf16ExpertsArgs a{};
  a.pool = pool;
  a.t = t;
  bf16_experts_layout(a, nullptr);
  return reinterpret_cast<uintptr_t>(a.shared_acts) + 4 * static_cast<size_t>(t) * pool.shared_f;
}

hipError_t launch_bf16_experts(hipStream_t s, const Bf16ExpertsArgs& a) {
  const mf_bf16_expert_pool& p = a.pool;
  const uint32_t widest = std::max(p.f, p.shared_f), rows = a.route_count() + (p.shared_f ? a.t : 0);
  const dim3 grid((widest + 15) / 16, a.most_live() + (p.shared_f ? p.shared_gate ? 2 : 1 : 0));
  if (a.t <= 16) experts_up_kernel<1><<<grid, 64 * kWaves, 0, s>>>(a);
  else experts_up_kernel<2><<<grid, 64 * kWaves, 0, s>>>(a);
  // parts of the sum over f, so that every wave has something to do when few experts are live
  uint32_t k_parts = 1;
  while (k_parts < 4 && a.most_live() * k_parts < 2 * kWaves && k_parts * rows <= 256) k_parts *= 2;
  const size_t lds = static_cast<size_t>(k_parts) * rows * 64;
  experts_down_kernel<<<dim3((p.d + 15) / 16), 64 * kWaves, lds, s>>>(a, k_parts);
  return hipGetLastError();
}

}  // namespace mf
