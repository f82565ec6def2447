// The operators of layers kept in 16 bits (projections, head norms, experts) as api.hip and their kernels see them.
#pragma once

#include "mf_internal.h"

namespace mf {

// projection.hip
size_t project_workspace_bytes(uint32_t m, uint32_t n, uint32_t t, bool gated);
hipError_t launch_project(hipStream_t s, const mf_project_args& a, void* workspace);

// head_norms.hip
hipError_t launch_head_norms(hipStream_t s, const mf_head_norms_args& a);

// bf16_experts.hip
struct Bf16ExpertsArgs {
  mf_bf16_expert_pool pool;
  const uint16_t* x;
  const uint32_t* idx;
  const float* w;
  const uint16_t* residual;
  uint16_t* y;
  uint32_t t, x_stride, residual_stride, y_stride;
  // the workspace
  float* shared_gate;  // [t]: logits of the shared expert's gate
  uint16_t* acts;      // [2][routes, f]: what is left of the activations' 32 bits in two bf16 terms, one plane each
  uint16_t* shared_acts;  // [2][t, shared_f]
  float* route_sums;   // [parts][routes + t, d], beyond eight tokens (t: of the shared expert)

  __host__ __device__ uint32_t route_count() const { return t * pool.top_k; }
  __host__ __device__ uint32_t most_live() const { return pool.num_experts < route_count() ? pool.num_experts : route_count(); }
  // runs of at most `rows` routes of one expert
  __host__ __device__ uint32_t most_tiles(uint32_t rows) const { return most_live() + (route_count() - most_live()) / rows; }
};
size_t bf16_experts_workspace_bytes(const mf_bf16_expert_pool& p, uint32_t t);
// the workspace's parts
void bf16_experts_layout(Bf16ExpertsArgs& a, void* workspace);
hipError_t launch_bf16_experts(hipStream_t s, const Bf16ExpertsArgs& a);

}  // namespace mf
