// The layer of 16-bit experts for a few tokens (mf_bf16_experts).
#include <algorithm>

#include "mf_dense16.h"
#include "mf_dense16_device.h"

namespace mf {

namespace {

constexpr uint32_t kRoutes = MF_BF16_EXPERTS_ROWS * MF_MAX_TOPK;

// A batch names few experts (its live ones).  Where a wave's lanes hold all of its routes they are found by ballots, in the order in which the batch
// names them; beyond 64 routes in the order of their numbers, by a workgroup.  Both launches find them for themselves, which costs less than handing them over.
constexpr uint32_t kFew = 64;

// calls found(number, expert, lanes of its routes) for every live expert until it returns true (e: the lane's expert, or one that is none)
template <class Found>
__device__ __forceinline__ void each_live(uint32_t e, uint32_t num_experts, Found found) {
  uint64_t left = __ballot(e < num_experts);
  for (uint32_t number = 0; left; ++number) {
    const uint32_t expert = __builtin_amdgcn_readlane(e, __ffsll(static_cast<unsigned long long>(left)) - 1);
    const uint64_t mine = __ballot(e == expert);
    if (found(number, expert, mine)) return;
    left &= ~mine;
  }
}

// ------------------------------------------------------------------ activations

constexpr uint32_t kUpWaves = 4, kUpStages = 3;

// The first launch: activations of 16 gate and 16 up rows of one live expert (blockIdx.y: which), or of the shared one, for all of its routes, eight (XI = 2: 16) at
// a time.  The call is the rows' stream; the waves share the sum over d.
template <int XI, bool ALIGNED>
__global__ __launch_bounds__(64 * kUpWaves) void experts_up_kernel(const Bf16ExpertsArgs a) {
  constexpr int kLoads = 4 + XI, kRing = kUpStages * kLoads * 64;
  __shared__ uint4 rings[kUpWaves * kRing];
  __shared__ uint32_t bits[MF_MAX_EXPERTS / 32], list[kRoutes], counts[2];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
  const uint32_t most = a.most_live(), routes = a.route_count(), d = a.pool.d;
  float* part = reinterpret_cast<float*>(rings);
  if (blockIdx.y > most) {  // the shared expert's gate, a token a workgroup
    for (uint32_t i = blockIdx.x; i < a.t; i += gridDim.x) {
      const uint16_t* x = a.x + static_cast<size_t>(i) * a.x_stride;
      float v = 0.0f;
      for (uint32_t k = tid; k < d; k += 64 * kUpWaves) v = __builtin_fmaf(bf16_to_f(x[k]), bf16_to_f(a.pool.shared_gate[k]), v);
      v = wave_sum(v);
      if (lane == 0) part[wave] = v;
      __syncthreads();
      if (tid == 0) a.shared_gate[i] = part[0] + part[1] + part[2] + part[3];
      __syncthreads();
    }
    return;
  }
  const bool shared = blockIdx.y == most;
  const uint32_t f = shared ? a.pool.shared_f : a.pool.f, j0 = blockIdx.x * 16;
  if (j0 >= f) return;
  uint32_t expert = ~0u, count = a.t;
  if (shared) {
    if (tid < a.t) list[tid] = tid;
    expert = 0;
  } else if (routes <= kFew) {
    const uint32_t e = lane < routes ? a.idx[lane] : ~0u;
    each_live(e, a.pool.num_experts, [&](uint32_t number, uint32_t live, uint64_t mine) {
      if (number < blockIdx.y) return false;
      expert = live;
      count = __popcll(mine);
      if (wave == 0 && e == live) list[lanes_in_front(mine)] = lane;
      return true;
    });
    if (expert == ~0u) return;
  } else {
    if (tid < MF_MAX_EXPERTS / 32) bits[tid] = 0;
    if (tid == 0) counts[0] = 0;
    __syncthreads();
    uint32_t e[kRoutes / (64 * kUpWaves)];
#pragma unroll
    for (uint32_t k = 0; k < kRoutes / (64 * kUpWaves); ++k) {
      const uint32_t route = k * 64 * kUpWaves + tid;
      e[k] = route < routes ? a.idx[route] : ~0u;
      if (e[k] < a.pool.num_experts) atomicOr(&bits[e[k] / 32], 1u << (e[k] & 31));
    }
    __syncthreads();
    uint32_t live = 0;
    for (uint32_t w = 0; w < MF_MAX_EXPERTS / 32; ++w) {
      uint32_t word = bits[w];
      const uint32_t here = __popc(word);
      if (blockIdx.y >= live && blockIdx.y < live + here) {
        for (uint32_t skip = blockIdx.y - live; skip; --skip) word &= word - 1;
        expert = w * 32 + __ffs(static_cast<int>(word)) - 1;
      }
      live += here;
    }
    if (expert == ~0u) return;
    // (the order of an expert's routes changes no result: each is a column of its own)
#pragma unroll
    for (uint32_t k = 0; k < kRoutes / (64 * kUpWaves); ++k)
      if (e[k] == expert) list[atomicAdd(&counts[0], 1u)] = k * 64 * kUpWaves + tid;
    __syncthreads();
    count = counts[0];
  }
  __syncthreads();
  expert = __builtin_amdgcn_readfirstlane(expert);
  count = __builtin_amdgcn_readfirstlane(count);
  const uint32_t share = ((d + 63) / 64 + kUpWaves - 1) / kUpWaves, from = min(wave * share * 64, d), to = min(from + share * 64, d), begin = to > from ? from : 0;
  const uint16_t* w = (shared ? a.pool.shared_gate_up : a.pool.gate_up + static_cast<size_t>(expert) * 2 * f * d) + static_cast<size_t>(j0) * d + begin;
  const uint16_t* bias = shared || !a.pool.gate_up_bias ? nullptr : a.pool.gate_up_bias + static_cast<size_t>(expert) * 2 * f;
  uint16_t* acts = shared ? a.shared_acts : a.acts;
  const size_t plane = static_cast<size_t>(shared ? a.t : routes) * f;
  for (uint32_t base = 0; base < count; base += 8 * XI) {
    RowAt<ALIGNED> at[kLoads];
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const uint32_t row = q % 2 * 8 + lane / 8;
      if (q < 4) {
        at[q] = (static_cast<RowAt<ALIGNED>>(min(row, f - 1 - j0)) * d + lane_piece(lane)) * 2;
      } else {
        const uint32_t route = list[min(base + row, count - 1)], token = shared ? route : route / a.pool.top_k;
        at[q] = (static_cast<RowAt<ALIGNED>>(token) * a.x_stride + lane_piece(lane)) * 2;
      }
    }
    f32x4_t zg = {}, zu = {};
    stream_rows<true, ALIGNED, kUpStages, XI>(w, w + static_cast<size_t>(f) * d, a.x + begin, at, to - from, rings + wave * kRing, zg, zu);
    __syncthreads();
    *reinterpret_cast<f32x4_t*>(part + wave * 512 + r * 16 + g * 4) = zg;
    *reinterpret_cast<f32x4_t*>(part + wave * 512 + 256 + r * 16 + g * 4) = zu;
    __syncthreads();
    const uint32_t column = tid / 16, j = j0 + tid % 16;
    if (column < 8 * XI && base + column < count && j < f) {
      float gate = 0.0f, up = 0.0f;
#pragma unroll
      for (uint32_t v = 0; v < kUpWaves; ++v) gate += part[v * 512 + tid], up += part[v * 512 + 256 + tid];
      if (bias) gate += bf16_to_f(bias[j]), up += bf16_to_f(bias[f + j]);
      const float act = activate(gate, a.pool.activation) * up;
      const size_t to_at = static_cast<size_t>(list[base + column]) * f + j;
      const uint16_t high = narrow_bf16(act);
      acts[to_at] = high;
      acts[plane + to_at] = narrow_bf16(__builtin_isfinite(bf16_to_f(high)) ? act - bf16_to_f(high) : 0.0f);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ results

constexpr uint32_t kDownWaves = 8;

// The second launch: ROWS results of every token.  The work is cut into items, the rows of one expert's down matrix times up to 8 XI of its routes over a part of f, dealt to the
// waves; a wave's items are one stream through its ring.  Every route's sum goes to LDS, and the weighted sums over a token's routes are made there in the
// order of their ranks, the parts of a sum in theirs.
template <int ROWS, int XI, int STAGES>
__global__ __launch_bounds__(64 * kDownWaves) void experts_down_kernel(const Bf16ExpertsArgs a, uint32_t part_blocks, uint32_t parts) {
  constexpr uint32_t kW = ROWS / 8, kLoads = kW + 2 * XI, kStage = kLoads * 64, kTile = 8 * XI;
  extern __shared__ uint4 whole_lds[];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
  const uint32_t d = a.pool.d, routes = a.route_count(), shared_rows = a.pool.shared_f ? a.t : 0, rows = routes + shared_rows, j0 = blockIdx.x * ROWS;
  float* sums = reinterpret_cast<float*>(whole_lds + kDownWaves * STAGES * kStage);          // [parts][rows][ROWS]
  uint32_t* list = reinterpret_cast<uint32_t*>(sums + static_cast<size_t>(parts) * rows * ROWS);  // [routes]: by tile
  uint2* tiles = reinterpret_cast<uint2*>(list + (routes + 1) / 2 * 2);                      // expert | routes << 16, first; at most `routes` of them
  __shared__ uint32_t tile_count, hist[MF_MAX_EXPERTS], wave_sums[2][kDownWaves];
  if (routes <= kFew) {
    if (wave == 0) {
      const uint32_t e = lane < routes ? a.idx[lane] : ~0u;
      uint32_t first = 0, n = 0;
      each_live(e, a.pool.num_experts, [&](uint32_t, uint32_t live, uint64_t mine) {
        const uint32_t count = __popcll(mine);
        if (e == live) list[first + lanes_in_front(mine)] = lane;
        for (uint32_t k = 0; k < count; k += kTile, ++n)
          if (lane == 0) tiles[n] = make_uint2(live | min(count - k, kTile) << 16, first + k);
        first += count;
        return false;
      });
      if (lane == 0) tile_count = n;
    }
  } else {
    // a thread an expert and a route
    static_assert(64 * kDownWaves >= MF_MAX_EXPERTS && 64 * kDownWaves >= kRoutes, "a thread each");
    const uint32_t e = tid < routes ? a.idx[tid] : ~0u;
    hist[tid] = 0;
    __syncthreads();
    if (e < a.pool.num_experts) atomicAdd(&hist[e], 1u);
    __syncthreads();
    const uint32_t count = hist[tid], mine = (count + kTile - 1) / kTile;
    uint32_t first = count, tile = mine;
#pragma unroll
    for (uint32_t s = 1; s < 64; s *= 2) {
      const uint32_t c = __shfl_up(first, s), t = __shfl_up(tile, s);
      if (lane >= s) first += c, tile += t;
    }
    if (lane == 63) wave_sums[0][wave] = first, wave_sums[1][wave] = tile;
    __syncthreads();
    first -= count;
    tile -= mine;
    for (uint32_t w = 0; w < wave; ++w) first += wave_sums[0][w], tile += wave_sums[1][w];
    for (uint32_t k = 0; k < mine; ++k) tiles[tile + k] = make_uint2(tid | min(count - k * kTile, kTile) << 16, first + k * kTile);
    if (tid == 64 * kDownWaves - 1) tile_count = tile + mine;
    hist[tid] = first;  // (from here on: where the next route of the expert goes; their order changes no result)
    __syncthreads();
    if (e < a.pool.num_experts) list[atomicAdd(&hist[e], 1u)] = tid;
  }
  __syncthreads();
  // items: the shared expert's first (its f may be the longest), then the tiles of routes
  const uint32_t shared_tiles = (shared_rows + kTile - 1) / kTile, shared_blocks = (a.pool.shared_f + 63) / 64, routed_blocks = (a.pool.f + 63) / 64;
  const uint32_t shared_parts = (shared_blocks + part_blocks - 1) / part_blocks, routed_parts = (routed_blocks + part_blocks - 1) / part_blocks;
  const uint32_t shared_items = shared_tiles * shared_parts, items = shared_items + __builtin_amdgcn_readfirstlane(tile_count) * routed_parts;
  struct Item {
    const uint16_t *w, *act, *low;  // down rows; the activations' two terms
    uint32_t f, first, blocks, count, from, part;
    bool shared;
  };
  const auto item_of = [&](uint32_t n) {
    Item it;
    it.shared = n < shared_items;
    const uint32_t in = it.shared ? n : n - shared_items, per = it.shared ? shared_parts : routed_parts, tile = in / per;
    it.part = in % per;
    it.f = it.shared ? a.pool.shared_f : a.pool.f;
    it.from = it.part * part_blocks * 64;
    it.blocks = (min(it.f - it.from, part_blocks * 64) + 63) / 64;
    if (it.shared) {
      it.first = tile * kTile;
      it.count = min(a.t - it.first, kTile);
      it.w = a.pool.shared_down;
      it.act = a.shared_acts;
      it.low = it.act + static_cast<size_t>(a.t) * it.f;
    } else {
      const uint2 t = tiles[tile];
      const uint32_t who = __builtin_amdgcn_readfirstlane(t.x);
      it.first = __builtin_amdgcn_readfirstlane(t.y);
      it.count = who >> 16;
      it.w = a.pool.down + static_cast<size_t>(who & 0xFFFF) * d * it.f;
      it.act = a.acts;
      it.low = it.act + static_cast<size_t>(routes) * it.f;
    }
    it.w = uniform(it.w + static_cast<size_t>(j0) * it.f + it.from);
    it.act = uniform(it.act + it.from);
    it.low = uniform(it.low + it.from);
    return it;
  };
  const auto route_of = [&](const Item& it, uint32_t column) {
    const uint32_t at = it.first + min(column, it.count - 1);
    return it.shared ? at : list[at];
  };
  // the requests' place in the stream runs ahead of the products'
  const uint32_t ring = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(whole_lds))) + wave * STAGES * kStage * 16, piece = lane_piece(lane);
  uint32_t ask_item = wave, ask_block = 0, at[kW + XI];
  Item ask{};
  const auto ask_next = [&] {
    ask = item_of(ask_item);
#pragma unroll
    for (uint32_t q = 0; q < kW; ++q) at[q] = (min(q * 8 + lane / 8, d - 1 - j0) * ask.f + piece) * 2;
#pragma unroll
    for (uint32_t q = 0; q < XI; ++q) at[kW + q] = (route_of(ask, q * 8 + lane / 8) * ask.f + piece) * 2;
  };
  const auto request = [&](uint32_t stage) {
    const uint32_t k = ask_block * 64, left = ask.f - ask.from - k;  // (of the row: 64 and more but in its last block)
    const uint32_t back = piece >= left ? piece * 2 : 0, to = ring + stage * kStage * 16;
#pragma unroll
    for (uint32_t q = 0; q < kW; ++q) load_to_lds_from(ask.w + k, at[q] - back, to + q * 1024);
#pragma unroll
    for (uint32_t q = 0; q < XI; ++q) {
      load_to_lds_from(ask.act + k, at[kW + q] - back, to + (kW + q) * 1024);
      load_to_lds_from(ask.low + k, at[kW + q] - back, to + (kW + XI + q) * 1024);
    }
    if (++ask_block < ask.blocks) return;
    if (ask_item + kDownWaves < items) {
      ask_item += kDownWaves;
      ask_block = 0;
      ask_next();
    } else {
      ask_block = ask.blocks - 1;  // behind the end: the last block again
    }
  };
  if (wave < items) {
    const uint32_t mine = ROWS == 16 ? place_of(r, g) : place_of(r & 7, g), mine_x = XI == 2 ? place_of(r, g) : place_of(r & 7, g);
    ask_next();
#pragma unroll
    for (uint32_t s = 0; s < STAGES; ++s) request(s);
    uint32_t item = wave, block = 0;
    Item now = item_of(item);
    f32x4_t sum = {};
    for (bool more = true; more;) {
#pragma unroll
      for (uint32_t s = 0; s < STAGES; ++s) {
        if (!more) break;
        const uint4* stage = whole_lds + wave * STAGES * kStage + s * kStage;
        wait_loads<(STAGES - 1) * kLoads>();
        uint4 fw[2], fh[2], fl[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          fw[h] = stage[mine ^ h * 4];
          fh[h] = stage[kW * 64 + (mine_x ^ h * 4)];
          fl[h] = stage[(kW + XI) * 64 + (mine_x ^ h * 4)];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read
        request(s);
        const uint32_t left = now.f - now.from - block * 64;
        if (left < 64) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t keep = (h * 4 + g) * 8 < left ? ~0u : 0u;
            fw[h] = masked(fw[h], keep);
            fh[h] = masked(fh[h], keep);
            fl[h] = masked(fl[h], keep);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sum = mfma16(fw[h], fh[h], sum);
          sum = mfma16(fw[h], fl[h], sum);
        }
        if (++block < now.blocks) continue;
        if (r < now.count && g * 4 < ROWS)
          *reinterpret_cast<f32x4_t*>(sums + (static_cast<size_t>(now.part) * rows + (now.shared ? routes : 0) + route_of(now, r)) * ROWS + g * 4) = sum;
        sum = f32x4_t{};
        block = 0;
        item += kDownWaves;
        more = item < items;
        if (more) now = item_of(item);
      }
    }
    wait_loads<0>();
  }
  __syncthreads();
  for (uint32_t o = tid; o < a.t * ROWS; o += 64 * kDownWaves) {
    const uint32_t i = o / ROWS, row = o % ROWS, j = j0 + row;
    if (j >= d) continue;
    float v = a.residual ? bf16_to_f(a.residual[static_cast<size_t>(i) * a.residual_stride + j]) : 0.0f;
    for (uint32_t k = 0; k < a.pool.top_k; ++k) {
      const uint32_t route = i * a.pool.top_k + k, e = a.idx[route];
      if (e >= a.pool.num_experts) continue;
      float z = 0.0f;
      for (uint32_t p = 0; p < routed_parts; ++p) z += sums[(static_cast<size_t>(p) * rows + route) * ROWS + row];
      if (a.pool.down_bias) z += bf16_to_f(a.pool.down_bias[static_cast<size_t>(e) * d + j]);
      v += a.w[route] * z;
    }
    if (shared_rows) {
      float z = 0.0f;
      for (uint32_t p = 0; p < shared_parts; ++p) z += sums[(static_cast<size_t>(p) * rows + routes + i) * ROWS + row];
      if (a.pool.shared_gate) z *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a.shared_gate[i] * -1.4426950408889634f));
      v += z;
    }
    a.y[static_cast<size_t>(i) * a.y_stride + j] = narrow_bf16(v);
  }
}

template <int ROWS, int XI, int STAGES>
hipError_t launch_down(hipStream_t s, const Bf16ExpertsArgs& a) {
  const mf_bf16_expert_pool& p = a.pool;
  const uint32_t routes = a.route_count(), rows = routes + (p.shared_f ? a.t : 0), longest = (std::max(p.f, p.shared_f) + 63) / 64;
  // parts of the sum over f, so that every wave has something to do when few experts are live
  uint32_t parts = 1;
  while (parts < 4 && a.most_live() * parts < 3 * kDownWaves && parts * 2 * rows * ROWS <= 4096 && longest > parts) parts *= 2;
  const uint32_t part_blocks = (longest + parts - 1) / parts;
  const size_t lds = kDownWaves * STAGES * (ROWS / 8 + 2 * XI) * 1024 + static_cast<size_t>(parts) * rows * ROWS * 4 + (routes + 1) / 2 * 8 + routes * 8;
  const hipError_t e = allow_lds<experts_down_kernel<ROWS, XI, STAGES>>(lds, 156 * 1024);
  if (e != hipSuccess) return e;
  experts_down_kernel<ROWS, XI, STAGES><<<dim3((p.d + ROWS - 1) / ROWS), 64 * kDownWaves, lds, s>>>(a, part_blocks, parts);
  return hipGetLastError();
}

size_t round16(size_t bytes) { return (bytes + 15) / 16 * 16; }

}  // namespace

void bf16_experts_layout(Bf16ExpertsArgs& a, void* workspace) {
  auto* p = static_cast<unsigned char*>(workspace);
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
  const uint32_t widest = std::max(p.f, p.shared_f);
  const dim3 grid((widest + 15) / 16, a.most_live() + (p.shared_f ? p.shared_gate ? 2 : 1 : 0));
  const bool aligned = aligned16(a.x) && a.x_stride % 8 == 0 && a.x_stride < 1u << 24;  // (offsets of 32 bits)
  if (a.t <= 8) {
    if (aligned) experts_up_kernel<1, true><<<grid, 64 * kUpWaves, 0, s>>>(a);
    else experts_up_kernel<1, false><<<grid, 64 * kUpWaves, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return p.d / 16 < device_cu_count() ? launch_down<8, 1, 4>(s, a) : launch_down<16, 1, 4>(s, a);
  }
  if (aligned) experts_up_kernel<2, true><<<grid, 64 * kUpWaves, 0, s>>>(a);
  else experts_up_kernel<2, false><<<grid, 64 * kUpWaves, 0, s>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? launch_down<16, 2, 2>(s, a) : e;
}

}  // namespace mf
