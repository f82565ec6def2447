// The norms of query and key heads with the rotation by their positions (mf_head_norms).
#include <algorithm>

#include "mf_dense16.h"
#include "mf_dense16_device.h"

namespace mf {

namespace {

// Cosine and sine of a pair's angle at a row.  The number of turns is made and reduced to half a turn in fp64: 2^31 steps of a pair that turns once a step
// leave 2^-22 of a turn.  A pair without an axis is copied, since by cosine 1 and sine 0 an infinity in it would not stay alone: its sine is a NaN that no arithmetic makes.
constexpr uint32_t kNoTurn = 0x7FEDCBA9u;
__device__ __forceinline__ bool turns(const float2& cs) { return __float_as_uint(cs.y) != kNoTurn; }
__device__ __forceinline__ float2 turn_of(const mf_head_norms_args& a, uint32_t pair, uint32_t row) {
  const uint32_t axis = a.axis_of_pair ? a.axis_of_pair[pair] : 0;
  if (axis >= a.axes) return make_float2(1.0f, __uint_as_float(kNoTurn));
  const double turns = a.positions[static_cast<size_t>(axis) * a.position_stride + row] * (static_cast<double>(a.inv_freq[pair]) * 0.15915494309189533577);
  float s, c;
  sincospif(2.0f * static_cast<float>(turns - __builtin_rint(turns)), &s, &c);
  return make_float2(c * a.rotation_scale, s * a.rotation_scale);
}

__device__ __forceinline__ float inverse_rms(float squares, const mf_head_norms_args& a) { return 1.0f / __builtin_sqrtf(squares / static_cast<float>(a.head_dim) + a.eps); }

// V values of 16 bits, as they lie in memory
template <int V> struct Piece {
  static constexpr int kWords = (V + 1) / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const uint16_t* p) {
    if constexpr (V == 1) w[0] = *p;
    else __builtin_memcpy(w, p, 2 * V);
  }
  __device__ __forceinline__ float operator[](int i) const { return i % 2 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]); }
};

// V results from p on
template <int V>
__device__ __forceinline__ void store_piece(uint16_t* p, const float (&y)[V]) {
  if constexpr (V == 1) {
    *p = narrow_bf16(y[0]);
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int e = 0; e < V / 2; ++e) w[e] = narrow_bf16(y[2 * e]) | static_cast<uint32_t>(narrow_bf16(y[2 * e + 1])) << 16;
    __builtin_memcpy(p, w, 2 * V);
  }
}

// A wave a row (or some of its heads, where there are few rows).  2^log_lanes lanes a head, each with V pairs: both elements of every pair in one lane, in two pieces of V that lie
// together; what is not rotated is dealt out the same way.  The wave's lanes share the row's cosines and sines: each makes some, LDS hands them on while the first heads
// are on their way.  The next heads are requested before this turn's are worked on.  What bounds it is memory: 8192 rows, 40 + 8 heads of 128, 201 MB in 38.1 us, 5.3 TB/s; at 777 rows
// of 32 + 8, 6.5 us, the loads and then the stores of one round.  The same bytes in heads of 72 (V = 4) 75 us, of 50 (V = 1) 111.
// Six waves a SIMD, 80 registers of a lane: with five, batches of 5120 to 6144 waves take a second round (6100 rows, 16 + 16 heads of 64: 13.6 us, 12.5 so).
template <int V>
__global__ __launch_bounds__(256, 6) void head_norms_kernel(const mf_head_norms_args a, uint32_t log_lanes, uint32_t chunk, uint32_t chunks) {
  __shared__ float2 tables[4][64 * V];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint64_t task = static_cast<uint64_t>(blockIdx.x) * 4 + wave;
  if (task >= static_cast<uint64_t>(a.t) * chunks) return;  // (no barrier below)
  const uint32_t row = static_cast<uint32_t>(task / chunks), heads = a.q.heads + a.k.heads, begin = static_cast<uint32_t>(task % chunks) * chunk, end = min(begin + chunk, heads);
  const uint32_t lanes = 1u << log_lanes, slot = lane & (lanes - 1), step = 64 >> log_lanes, slots = a.head_dim / (2 * V), rot = a.rotary_dim, pairs = rot / 2, turned = pairs / V;
  const bool live = slot < slots, rotates = slot < turned;
  // where the lane's two pieces lie in a head
  const uint32_t first = !rotates ? rot + (slot - turned) * 2 * V : a.interleaved ? slot * 2 * V : slot * V, second = rotates && !a.interleaved ? first + pairs : first + V;
  Piece<V> now[2], next[2], wq[2], wk[2];
  const auto place = [&](uint32_t head, bool out) {
    const bool k = head >= a.q.heads;
    const mf_head_rows &q = a.q, &o = a.k;
    const uint32_t in = k ? head - q.heads : head;
    const uint32_t rs = out ? (k ? o.out_row_stride : q.out_row_stride) : (k ? o.row_stride : q.row_stride), hs = out ? (k ? o.out_head_stride : q.out_head_stride) : (k ? o.head_stride : q.head_stride);
    return static_cast<size_t>(row) * rs + static_cast<size_t>(in) * hs;
  };
  const auto request = [&](Piece<V>(&p)[2], uint32_t head) {
    if (!live || head >= end) return;
    const uint16_t* x = (head >= a.q.heads ? a.k.x : a.q.x) + place(head, false);
    p[0].load(x + first);
    p[1].load(x + second);
  };
  uint32_t head = begin + (lane >> log_lanes);
  request(now, head);
  if (live && a.q.weight && a.q.heads) wq[0].load(a.q.weight + first), wq[1].load(a.q.weight + second);
  if (live && a.k.weight && a.k.heads) wk[0].load(a.k.weight + first), wk[1].load(a.k.weight + second);
  float2* table = tables[wave];
  for (uint32_t p = lane; p < pairs; p += 64) table[p] = turn_of(a, p, row);
  issue_fence();  // (a wave's own LDS accesses keep their order)
  float c[V], s[V];
  uint32_t turn = 0;  // bit e: pair e of the lane has an axis
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float2 cs = rotates ? table[slot * V + e] : make_float2(1.0f, 0.0f);
    turn |= rotates && turns(cs) ? 1u << e : 0u;
    c[e] = cs.x;
    s[e] = cs.y;
  }
  for (uint32_t base = begin; base < end; base += step, head += step) {
    request(next, head + step);
    const bool is_k = head >= a.q.heads;
    float z[2][V];
    float squares = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        z[h][e] = live && head < end ? now[h][e] : 0.0f;
        squares = __builtin_fmaf(z[h][e], z[h][e], squares);
      }
    squares = group_sum(squares, lanes);
    if (is_k ? a.k.weight != nullptr : a.q.weight != nullptr) {
      const float inv = inverse_rms(squares, a);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < V; ++e) z[h][e] = z[h][e] * inv * ((is_k ? wk[h][e] : wq[h][e]) + a.weight_bias);
    }
    if (live && head < end) {
      uint16_t* out = (is_k ? a.k.out : a.q.out) + place(head, true);
      float y[2][V];
      if (V > 1 && a.interleaved) {  // neighbours are a pair: of element i = h V + e pair i / 2 of the lane
#pragma unroll
        for (int p = 0; p < V; ++p) {
          const float l = z[2 * p / V][2 * p % V], r = z[(2 * p + 1) / V][(2 * p + 1) % V];
          y[2 * p / V][2 * p % V] = (turn >> p & 1) ? l * c[p] - r * s[p] : l;
          y[(2 * p + 1) / V][(2 * p + 1) % V] = (turn >> p & 1) ? r * c[p] + l * s[p] : r;
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          y[0][e] = (turn >> e & 1) ? z[0][e] * c[e] - z[1][e] * s[e] : z[0][e];
          y[1][e] = (turn >> e & 1) ? z[1][e] * c[e] + z[0][e] * s[e] : z[1][e];
        }
      }
      store_piece<V>(out + first, y[0]);
      store_piece<V>(out + second, y[1]);
    }
    now[0] = next[0];
    now[1] = next[1];
  }
}

// Heads that lanes cannot share out in equal pieces (an odd size, pairs of an odd number in a long head): a wave a head, the head in LDS.  The same bytes in heads
// of 130: 222 us.
__global__ __launch_bounds__(256) void head_norms_any_kernel(const mf_head_norms_args a) {
  __shared__ float rows[4][1024];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, heads = a.q.heads + a.k.heads;
  float* z = rows[wave];
  for (uint64_t at = static_cast<uint64_t>(blockIdx.x) * 4 + wave; at < static_cast<uint64_t>(heads) * a.t; at += static_cast<uint64_t>(gridDim.x) * 4) {
    const uint32_t row = static_cast<uint32_t>(at / heads);
    uint32_t head = static_cast<uint32_t>(at % heads);
    const bool is_q = head < a.q.heads;
    const mf_head_rows& h = is_q ? a.q : a.k;
    if (!is_q) head -= a.q.heads;
    const uint16_t* x = h.x + static_cast<size_t>(row) * h.row_stride + static_cast<size_t>(head) * h.head_stride;
    uint16_t* out = h.out + static_cast<size_t>(row) * h.out_row_stride + static_cast<size_t>(head) * h.out_head_stride;
    float squares = 0.0f;
    issue_fence();  // (a wave's own LDS accesses keep their order)
    for (uint32_t e = lane; e < a.head_dim; e += 64) {
      z[e] = bf16_to_f(x[e]);
      squares = __builtin_fmaf(z[e], z[e], squares);
    }
    squares = wave_sum(squares);
    if (h.weight) {
      const float inv = inverse_rms(squares, a);
      for (uint32_t e = lane; e < a.head_dim; e += 64) z[e] = z[e] * inv * (bf16_to_f(h.weight[e]) + a.weight_bias);
    }
    issue_fence();
    const uint32_t rot = a.rotary_dim, pairs = rot / 2;
    for (uint32_t p = lane; p < pairs; p += 64) {
      const float2 cs = turn_of(a, p, row);
      const uint32_t i = a.interleaved ? 2 * p : p, j = a.interleaved ? 2 * p + 1 : p + pairs;
      out[i] = narrow_bf16(z[i] * cs.x - z[j] * cs.y);
      out[j] = narrow_bf16(z[j] * cs.x + z[i] * cs.y);
      if (!turns(cs)) {  // (seldom: stored over the turned)
        out[i] = narrow_bf16(z[i]);
        out[j] = narrow_bf16(z[j]);
      }
    }
    for (uint32_t e = rot + lane; e < a.head_dim; e += 64) out[e] = narrow_bf16(z[e]);
  }
}

template <int V>
hipError_t launch_pieces(hipStream_t s, const mf_head_norms_args& a) {
  const uint32_t heads = a.q.heads + a.k.heads, slots = a.head_dim / (2 * V);
  uint32_t log_lanes = 0;
  while (1u << log_lanes < slots) ++log_lanes;
  // a row's heads to several waves while there are waves enough for them
  const uint32_t step = 64 >> log_lanes, turns = (heads + step - 1) / step;
  uint32_t each = 1;
  while (each < turns && static_cast<uint64_t>(a.t) * ((turns + each - 1) / each) > device_cu_count() * 16) ++each;
  const uint32_t chunk = each * step, chunks = (heads + chunk - 1) / chunk;
  head_norms_kernel<V><<<dim3(static_cast<uint32_t>((static_cast<uint64_t>(a.t) * chunks + 3) / 4)), 256, 0, s>>>(a, log_lanes, chunk, chunks);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_head_norms(hipStream_t s, const mf_head_norms_args& a) {
  const auto fits = [&](uint32_t v) { return a.head_dim % (2 * v) == 0 && a.rotary_dim % (2 * v) == 0 && a.head_dim / (2 * v) <= 64; };
  if (fits(8)) return launch_pieces<8>(s, a);
  if (fits(4)) return launch_pieces<4>(s, a);
  if (fits(1)) return launch_pieces<1>(s, a);
  const uint64_t waves = static_cast<uint64_t>(a.q.heads + a.k.heads) * a.t;
  head_norms_any_kernel<<<dim3(static_cast<uint32_t>(std::min<uint64_t>((waves + 3) / 4, 1u << 20))), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace mf
