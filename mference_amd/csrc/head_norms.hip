// The norms of query and key heads with the rotation by their positions (mf_head_norms).
#include "mf_dense16.h"
#include "mf_dense16_device.h"

namespace mf {

namespace {

// The simple form: a wave a head of a row, the head in LDS.
__global__ __launch_bounds__(256) void head_norms_kernel(const mf_head_norms_args a) {
  __shared__ float rows[4][1024];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, heads = a.q.heads + a.k.heads;
  const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 4 + wave;
  float* z = rows[wave];
  const bool live = at < static_cast<uint64_t>(heads) * a.t;
  const uint32_t row = live ? static_cast<uint32_t>(at / heads) : 0;
  uint32_t head = live ? static_cast<uint32_t>(at % heads) : 0;
  const bool is_q = head < a.q.heads;
  const mf_head_rows& h = is_q ? a.q : a.k;
  if (!is_q) head -= a.q.heads;
  const uint16_t* x = h.x + static_cast<size_t>(row) * h.row_stride + static_cast<size_t>(head) * h.head_stride;
  uint16_t* out = h.out + static_cast<size_t>(row) * h.out_row_stride + static_cast<size_t>(head) * h.out_head_stride;
  float squares = 0.0f;
  if (live)
    for (uint32_t e = lane; e < a.head_dim; e += 64) {
      z[e] = bf16_to_f(x[e]);
      squares = __builtin_fmaf(z[e], z[e], squares);
    }
  squares = wave_sum(squares);
  if (live && h.weight) {
    const float inv = 1.0f / __builtin_sqrtf(squares / static_cast<float>(a.head_dim) + a.eps);
    for (uint32_t e = lane; e < a.head_dim; e += 64) z[e] = z[e] * inv * (bf16_to_f(h.weight[e]) + a.weight_bias);
  }
  __syncthreads();
  if (!live) return;
  const uint32_t rot = a.positions ? a.rotary_dim : 0, pairs = rot / 2;
  for (uint32_t p = lane; p < pairs; p += 64) {
    const uint32_t axis = a.axis_of_pair ? a.axis_of_pair[p] : 0;
    float c = 1.0f, s = 0.0f;
    if (axis < a.axes) {
      const double turns = a.positions[static_cast<size_t>(axis) * a.position_stride + row] * (static_cast<double>(a.inv_freq[p]) * 0.15915494309189533577);
      sincospif(2.0f * static_cast<float>(turns - __builtin_rint(turns)), &s, &c);
      c *= a.rotation_scale;
      s *= a.rotation_scale;
    }
    const uint32_t i = a.interleaved ? 2 * p : p, j = a.interleaved ? 2 * p + 1 : p + pairs;
    out[i] = narrow_bf16(z[i] * c - z[j] * s);
    out[j] = narrow_bf16(z[j] * c + z[i] * s);
  }
  for (uint32_t e = rot + lane; e < a.head_dim; e += 64) out[e] = narrow_bf16(z[e]);
}

}  // namespace

hipError_t launch_head_norms(hipStream_t s, const mf_head_norms_args& a) {
  const uint64_t heads = static_cast<uint64_t>(a.q.heads + a.k.heads) * a.t;
  head_norms_kernel<<<dim3(static_cast<uint32_t>((heads + 3) / 4)), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace mf
