// Low-rank adapters of many requests beside a shared projection (mf_adapter_apply) and the grouping of a batch's rows by
// adapter (mf_adapter_group).
#include <algorithm>

#include "mf_adapters.h"
#include "mf_device.h"

namespace mf {

namespace {

// ------------------------------------------------------------------ rows by adapter

__device__ __forceinline__ uint32_t adapter_key(int32_t id, uint32_t n) { return static_cast<uint32_t>(id) < n ? static_cast<uint32_t>(id) : n; }

// A stable counting sort by one workgroup: thread k owns key k of the counts, and the rows are walked in order.
__global__ __launch_bounds__(1024) void adapter_group_kernel(const int32_t* __restrict__ ids, uint32_t t, uint32_t n, AdapterPlan plan) {
  __shared__ uint32_t start[MF_MAX_ADAPTERS + 2];
  for (uint32_t k = threadIdx.x; k <= n; k += blockDim.x) {
    uint32_t count = 0;
    for (uint32_t i = 0; i < t; ++i) count += adapter_key(ids[i], n) == k;
    start[k + 1] = count;
  }
  if (threadIdx.x == 0) start[0] = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t tiles = 0;
    for (uint32_t k = 0; k < n; ++k) {
      const uint32_t count = start[k + 1];
      for (uint32_t at = 0; at < count; at += plan.tile_rows)
        plan.tiles[tiles++] = make_uint2(k | min(count - at, plan.tile_rows) << 16, start[k] + at);
      start[k + 1] += start[k];
    }
    plan.header[0] = t;
    plan.header[1] = n;
    plan.header[2] = tiles;
    plan.header[3] = plan.tile_rows;
  }
  __syncthreads();
  for (uint32_t k = threadIdx.x; k <= n; k += blockDim.x) {
    plan.offsets[k] = start[k];
    uint32_t at = start[k];
    for (uint32_t i = 0; i < t; ++i)
      if (adapter_key(ids[i], n) == k) plan.rows[at++] = i;
  }
}

// ------------------------------------------------------------------ A x

__device__ __forceinline__ uint32_t live_rank(const AdapterArgs& a, uint32_t adapter) { return a.ranks ? min(a.ranks[adapter], a.rank) : a.rank; }

// one wave per (row, target, row of A)
__global__ __launch_bounds__(64) void adapter_shrink_kernel(const AdapterArgs a) {
  const uint32_t row = blockIdx.x, col = blockIdx.y;
  const uint32_t adapter = adapter_key(a.ids[row], a.num_adapters);
  if (adapter >= a.num_adapters) return;
  const uint32_t target = col / a.rank, r = col % a.rank;
  if (r >= live_rank(a, adapter)) return;
  const uint16_t* x = a.x + static_cast<size_t>(row) * a.x_stride;
  const uint16_t* w = a.target[target].a + (static_cast<size_t>(adapter) * a.rank + r) * a.n;
  float sum = 0.0f;
  for (uint32_t i = threadIdx.x; i < a.n; i += 64) sum = __builtin_fmaf(bf16_to_f(x[i]), bf16_to_f(w[i]), sum);
  sum = wave_sum(sum);
  if (threadIdx.x == 0) a.v[static_cast<size_t>(row) * a.cols + col] = sum * (a.scales ? a.scales[adapter] : 1.0f);
}

// ------------------------------------------------------------------ y += B v

// one thread per result
template <bool F32>
__global__ __launch_bounds__(256) void adapter_expand_kernel(const AdapterArgs a) {
  const uint32_t row = blockIdx.x;
  const AdapterArgs::Target tg = a.target[blockIdx.z];
  const uint32_t adapter = adapter_key(a.ids[row], a.num_adapters);
  const uint32_t j = blockIdx.y * 256 + threadIdx.x;
  if (adapter >= a.num_adapters || j >= tg.m) return;
  const uint32_t rank = live_rank(a, adapter);
  const float* v = a.v + static_cast<size_t>(row) * a.cols + blockIdx.z * a.rank;
  const uint16_t* b = tg.b + (static_cast<size_t>(adapter) * tg.m + j) * a.rank;
  float sum = 0.0f;
  for (uint32_t r = 0; r < rank; ++r) sum = __builtin_fmaf(v[r], bf16_to_f(b[r]), sum);
  const size_t at = static_cast<size_t>(row) * tg.y_stride + j;
  if constexpr (F32) static_cast<float*>(tg.y)[at] += sum;
  else {
    uint16_t* y = static_cast<uint16_t*>(tg.y) + at;
    *y = narrow_bf16(bf16_to_f(*y) + sum);
  }
}

}  // namespace

hipError_t launch_adapter_group(hipStream_t s, const int32_t* ids, uint32_t t, uint32_t n, uint32_t* plan) {
  adapter_group_kernel<<<dim3(1), dim3(1024), 0, s>>>(ids, t, n, AdapterPlan::at(plan, t, n));
  return hipGetLastError();
}

size_t adapter_workspace_bytes(uint32_t num_targets, uint32_t rank, uint32_t n, uint32_t t) {
  return static_cast<size_t>(t) * num_targets * rank * sizeof(float);
}

hipError_t launch_adapter_apply(hipStream_t s, const AdapterArgs& a, bool y_f32) {
  uint32_t m = 0;
  for (uint32_t k = 0; k < a.num_targets; ++k) m = std::max(m, a.target[k].m);
  adapter_shrink_kernel<<<dim3(a.t, a.num_targets * a.rank), dim3(64), 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid(a.t, (m + 255) / 256, a.num_targets);
  if (y_f32) adapter_expand_kernel<true><<<grid, dim3(256), 0, s>>>(a);
  else adapter_expand_kernel<false><<<grid, dim3(256), 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace mf
