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

// calls found(expert, lanes of its routes) for every live expert until it returns true (e: the lane's expert, or one that is none)
template <class Found>
__device__ __forceinline__ void each_live(uint32_t e, uint32_t num_experts, Found found) {
  uint64_t left = __ballot(e < num_experts);
  while (left) {
    const uint32_t expert = __builtin_amdgcn_readlane(e, __ffsll(static_cast<unsigned long long>(left)) - 1);
    const uint64_t mine = __ballot(e == expert);
    if (found(expert, mine)) return;
    left &= ~mine;
  }
}

// ------------------------------------------------------------------ activations

constexpr uint32_t kUpWaves = 2, kUpStages = 2;

// The first launch: activations of 16 gate and 16 up rows of one live expert, or of the shared one, for eight (XI = 2: 16) of its routes: a tile (blockIdx.y).  Its work is
// the reading of W, rows of d in lines of 128 bytes: a workgroup's two waves share d and each streams its part of the 32 rows through a ring of two stages in LDS; the matrix
// cores' sums meet in LDS.  What bounds it is the memory: 206 MB in 42 us (8 tokens, 23 live experts of 704 x 2816 beside a shared one of 2112: 4.9 TB/s, the rate of a large copy);
// 218 MB in 55 us where popular experts have several tiles, which read their rows again (61 tokens, 26 live of 1024 x 2048); 37.7 MB in 9 us (one token, 8 of 512 x 2048 beside a
// shared one), of which the way to the expert's number and the first lines is the larger part.  Measured beside it, at the first two: four waves 46 and 58 us; three stages
// 46 and 63, fewer workgroups fitting on a unit; waves with 16 + 16 rows of their own and all of d, 59 and 77; an expert's tiles one after the other in a workgroup, 68 at 61 tokens.
template <int XI, bool ALIGNED>
__global__ __launch_bounds__(64 * kUpWaves) void experts_up_kernel(const Bf16ExpertsArgs a) {
  constexpr int kLoads = 4 + XI, kRing = kUpStages * kLoads * 64;
  constexpr uint32_t kTile = 8 * XI;
  __shared__ uint4 rings[kUpWaves * kRing];
  __shared__ uint32_t hist[MF_MAX_EXPERTS], list[kRoutes], sums[kRoutes / 64], found[3];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
  const uint32_t most = a.most_tiles(kTile), routes = a.route_count(), d = a.pool.d, shared_tiles = a.pool.shared_f ? (a.t + kTile - 1) / kTile : 0;
  float* part = reinterpret_cast<float*>(rings);
  if (blockIdx.y >= most + shared_tiles) {  // the shared expert's gate, a token a workgroup
    for (uint32_t i = blockIdx.x; i < a.t; i += gridDim.x) {
      const uint16_t* x = a.x + static_cast<size_t>(i) * a.x_stride;
      float v = 0.0f;
      for (uint32_t k = tid; k < d; k += 64 * kUpWaves) v = __builtin_fmaf(bf16_to_f(x[k]), bf16_to_f(a.pool.shared_gate[k]), v);
      v = wave_sum(v);
      if (lane == 0) part[wave] = v;
      __syncthreads();
      if (tid == 0) a.shared_gate[i] = part[0] + part[1];
      __syncthreads();
    }
    return;
  }
  const bool shared = blockIdx.y >= most;
  const uint32_t f = shared ? a.pool.shared_f : a.pool.f;
  const uint32_t j0 = blockIdx.x * 16;
  if (j0 >= f) return;
  uint32_t expert = ~0u, count = a.t, base = (blockIdx.y - most) * kTile;
  if (shared) {
    if (tid < a.t) list[tid] = tid;
    expert = 0;
  } else if (routes <= kFew) {
    const uint32_t e = lane < routes ? a.idx[lane] : ~0u;
    uint32_t tile = 0;
    each_live(e, a.pool.num_experts, [&](uint32_t live, uint64_t mine) {
      count = __popcll(mine);
      base = (blockIdx.y - tile) * kTile;
      tile += (count + kTile - 1) / kTile;
      if (tile <= blockIdx.y) return false;
      expert = live;
      if (wave == 0 && e == live) list[lanes_in_front(mine)] = lane;
      return true;
    });
    if (expert == ~0u) return;
  } else {
    constexpr uint32_t kThreads = 64 * kUpWaves, kEach = MF_MAX_EXPERTS / kThreads, kTurns = kRoutes / kThreads;
    static_assert(kEach * kThreads == MF_MAX_EXPERTS && kTurns * kThreads == kRoutes, "the threads share out experts and routes");
    for (uint32_t k = tid; k < MF_MAX_EXPERTS; k += kThreads) hist[k] = 0;
    if (tid == 0) found[0] = ~0u;
    __syncthreads();
    uint32_t e[kTurns];
#pragma unroll
    for (uint32_t k = 0; k < kTurns; ++k) {
      const uint32_t route = k * kThreads + tid;
      e[k] = route < routes ? a.idx[route] : ~0u;
      if (e[k] < a.pool.num_experts) atomicAdd(&hist[e[k]], 1u);
    }
    __syncthreads();
    uint32_t tiles = 0;
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) tiles += (hist[tid * kEach + k] + kTile - 1) / kTile;
    uint32_t tile = tiles;
#pragma unroll
    for (uint32_t s = 1; s < 64; s *= 2) {
      const uint32_t v = __shfl_up(tile, s);
      if (lane >= s) tile += v;
    }
    if (lane == 63) sums[wave] = tile;
    __syncthreads();
    tile -= tiles;
    for (uint32_t w = 0; w < wave; ++w) tile += sums[w];
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
      const uint32_t here = hist[tid * kEach + k], own = (here + kTile - 1) / kTile;
      if (blockIdx.y >= tile && blockIdx.y < tile + own) found[0] = tid * kEach + k, found[1] = here, found[2] = (blockIdx.y - tile) * kTile;
      tile += own;
    }
    __syncthreads();
    expert = found[0];
    if (expert == ~0u) return;
    count = found[1];
    base = found[2];
    // an expert's routes in the order of their numbers: its tiles are other workgroups' too
#pragma unroll
    for (uint32_t k = 0; k < kTurns; ++k) {
      const uint64_t mine = __ballot(e[k] == expert);
      if (lane == 0) sums[k * kUpWaves + wave] = __popcll(mine);
    }
    __syncthreads();
    uint32_t at = 0;
#pragma unroll
    for (uint32_t k = 0; k < kTurns; ++k) {
      const uint64_t mine = __ballot(e[k] == expert);
      uint32_t first = at;
      for (uint32_t w = 0; w < kUpWaves; ++w) {
        if (w < wave) first += sums[k * kUpWaves + w];
        at += sums[k * kUpWaves + w];
      }
      if (e[k] == expert) list[first + lanes_in_front(mine)] = k * kThreads + tid;
    }
  }
  __syncthreads();
  expert = __builtin_amdgcn_readfirstlane(expert);
  count = __builtin_amdgcn_readfirstlane(count);
  base = __builtin_amdgcn_readfirstlane(base);
  const uint32_t share = ((d + 63) / 64 + kUpWaves - 1) / kUpWaves, from = min(wave * share * 64, d), to = min(from + share * 64, d), begin = to > from ? from : 0;
  const uint16_t* matrix = (shared ? a.pool.shared_gate_up : a.pool.gate_up + static_cast<size_t>(expert) * 2 * f * d) + begin;
  const uint16_t* bias = shared || !a.pool.gate_up_bias ? nullptr : a.pool.gate_up_bias + static_cast<size_t>(expert) * 2 * f;
  uint16_t* acts = shared ? a.shared_acts : a.acts;
  const size_t plane = static_cast<size_t>(shared ? a.t : routes) * f;
  // eight or 16 routes through 16 + 16 rows
  const auto rows_of = [&](auto columns) {
    constexpr int kX = decltype(columns)::value, kN = 4 + kX;
    RowAt<ALIGNED> at[kN];
#pragma unroll
    for (int q = 0; q < kN; ++q) {
      const uint32_t row = q % 2 * 8 + lane / 8;
      if (q < 4) {
        at[q] = (static_cast<RowAt<ALIGNED>>(min(row, f - 1 - j0)) * d + lane_piece(lane)) * 2;
      } else {
        const uint32_t route = list[min(base + row, count - 1)], token = shared ? route : route / a.pool.top_k;
        at[q] = (static_cast<RowAt<ALIGNED>>(token) * a.x_stride + lane_piece(lane)) * 2;
      }
    }
    const uint16_t* w = matrix + static_cast<size_t>(j0) * d;
    f32x4_t zg = {}, zu = {};
    stream_rows<true, ALIGNED, kUpStages, kX>(w, w + static_cast<size_t>(f) * d, a.x + begin, at, to - from, rings + wave * kRing, zg, zu);
    __syncthreads();
    *reinterpret_cast<f32x4_t*>(part + wave * 512 + r * 16 + g * 4) = zg;
    *reinterpret_cast<f32x4_t*>(part + wave * 512 + 256 + r * 16 + g * 4) = zu;
    __syncthreads();
    for (uint32_t o = tid; o < 128 * kX; o += 64 * kUpWaves) {
      const uint32_t column = o / 16, j = j0 + o % 16;
      if (base + column >= count || j >= f) continue;
      float gate = 0.0f, up = 0.0f;
#pragma unroll
      for (uint32_t v = 0; v < kUpWaves; ++v) gate += part[v * 512 + o], up += part[v * 512 + 256 + o];
      if (bias) gate += bf16_to_f(bias[j]), up += bf16_to_f(bias[f + j]);
      const float act = activate(gate, a.pool.activation) * up;
      const size_t to_at = static_cast<size_t>(list[base + column]) * f + j;
      // (nearer to 2^128 than to the last bf16: cut off, since the first term would be an infinity and the second cannot take that back)
      const uint16_t near = narrow_bf16(act), high = __builtin_isfinite(act) && !__builtin_isfinite(bf16_to_f(near)) ? static_cast<uint16_t>(__float_as_uint(act) >> 16) : near;
      acts[to_at] = high;
      acts[plane + to_at] = narrow_bf16(__builtin_isfinite(act) ? act - bf16_to_f(high) : 0.0f);
    }
  };
  if (XI == 2 && count - base > 8) rows_of(std::integral_constant<int, 2>{});
  else rows_of(std::integral_constant<int, 1>{});
}

// ------------------------------------------------------------------ results

// How the second launch is cut: rows of a workgroup, and parts of the sums over f, which a workgroup's waves share up to eight tokens and workgroups of their own take beyond.
struct DownCut {
  uint32_t rows, routed_blocks, shared_blocks, parts;  // (blocks: of 64 of f, in a part)
};

// The second launch: up to ROWS results of every token.  The work is cut into items, the rows of one expert's down matrix times up to 8 XI of its routes over a part of f,
// dealt to a workgroup's waves; a wave's items are one stream through its ring in LDS, whose requests run over an item's end into the next.  Up to eight tokens every route's sum
// goes to LDS and the weighted sums over a token's routes are made there, in the order of their ranks, the parts of a sum in theirs; beyond, the sums go to memory and a third launch adds
// them up in that order: no atomics either way, so calls repeat to the bit.  The activations come as two bf16 terms (32 bits narrowed to 16 would cost the layer half a step more than
// the result's own rounding).  What bounds it: 103 MB in 28 us (8 tokens, d 2816: 256 workgroups of 11 rows; 176 of 16 took 47); 109 MB in 34 us (61 tokens; with all routes' sums in
// LDS there was room for rings of two stages, not four, and it took 46), 4 TB/s with the rows that several tiles read; 18.9 MB in 10 us (one token), the way from idx to the
// rows to the sums; 16 waves 11 us.
template <int ROWS, int XI, int STAGES, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void experts_down_kernel(const Bf16ExpertsArgs a, const DownCut cut) {
  constexpr bool kJoin = XI > 1;  // beyond eight tokens the third launch adds up
  constexpr uint32_t kW = ROWS / 8, kLoads = kW + 2 * XI, kStage = kLoads * 64, kTile = 8 * XI, kM = (ROWS + 15) / 16, kThreads = 64 * WAVES;
  extern __shared__ uint4 whole_lds[];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4, group = blockIdx.y;
  const uint32_t d = a.pool.d, routes = a.route_count(), shared_rows = a.pool.shared_f ? a.t : 0, rows = routes + shared_rows, j0 = blockIdx.x * cut.rows, own_rows = min(cut.rows, d - j0);
  float* sums = reinterpret_cast<float*>(whole_lds + WAVES * STAGES * kStage);                      // [parts][rows][ROWS]
  uint32_t* list = reinterpret_cast<uint32_t*>(sums + (kJoin ? 0 : static_cast<size_t>(cut.parts) * rows * ROWS));  // [routes]: by tile
  uint2* tiles = reinterpret_cast<uint2*>(list + (routes + 1) / 2 * 2);                             // expert | routes << 16, first; at most `routes` of them
  uint2* named = tiles + routes;                                                                    // [routes]: expert, weight
  uint2* table = named + (kJoin ? 0 : routes);                                                                    // a group's items: expert | routes << 16 | part << 24, first
  __shared__ uint32_t tile_count, hist[MF_MAX_EXPERTS], wave_sums[2][WAVES];
  for (uint32_t k = tid; !kJoin && k < routes; k += kThreads) named[k] = make_uint2(a.idx[k], __float_as_uint(a.w[k]));
  if (XI == 1 || routes <= kFew) {  // (eight tokens have no more)
    if (wave == 0) {
      const uint32_t e = lane < routes ? a.idx[lane] : ~0u;
      uint32_t first = 0, n = 0;
      each_live(e, a.pool.num_experts, [&](uint32_t live, uint64_t mine) {
        const uint32_t count = __popcll(mine);
        if (e == live) list[first + lanes_in_front(mine)] = lane;
        for (uint32_t k = 0; k < count; k += kTile, ++n)
          if (lane == 0) tiles[n] = make_uint2(live | min(count - k, kTile) << 16, first + k);
        first += count;
        return false;
      });
      if (lane == 0) tile_count = n;
    }
  } else if constexpr (XI > 1) {
    // a thread two neighbouring experts (or one)
    constexpr uint32_t kEach = MF_MAX_EXPERTS / kThreads;
    static_assert(kEach * kThreads == MF_MAX_EXPERTS, "the threads share out the experts");
    for (uint32_t k = tid; k < MF_MAX_EXPERTS; k += kThreads) hist[k] = 0;
    __syncthreads();
    for (uint32_t k = tid; k < routes; k += kThreads) {
      const uint32_t e = a.idx[k];
      if (e < a.pool.num_experts) atomicAdd(&hist[e], 1u);
    }
    __syncthreads();
    uint32_t count[kEach], all = 0, all_tiles = 0;
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
      count[k] = hist[tid * kEach + k];
      all += count[k];
      all_tiles += (count[k] + kTile - 1) / kTile;
    }
    uint32_t first = all, tile = all_tiles;
#pragma unroll
    for (uint32_t s = 1; s < 64; s *= 2) {
      const uint32_t c = __shfl_up(first, s), t = __shfl_up(tile, s);
      if (lane >= s) first += c, tile += t;
    }
    if (lane == 63) wave_sums[0][wave] = first, wave_sums[1][wave] = tile;
    __syncthreads();
    first -= all;
    tile -= all_tiles;
    for (uint32_t w = 0; w < wave; ++w) first += wave_sums[0][w], tile += wave_sums[1][w];
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
      const uint32_t e = tid * kEach + k;
      for (uint32_t c = 0; c < count[k]; c += kTile) tiles[tile++] = make_uint2(e | min(count[k] - c, kTile) << 16, first + c);
      hist[e] = first;  // (from here on: where the next route of the expert goes; their order changes no result)
      first += count[k];
    }
    if (tid == kThreads - 1) tile_count = tile;
    __syncthreads();
    for (uint32_t k = tid; k < routes; k += kThreads) {
      const uint32_t e = a.idx[k];
      if (e < a.pool.num_experts) list[atomicAdd(&hist[e], 1u)] = k;
    }
  }
  __syncthreads();
  // items: the shared expert's first (its f may be the longest), then the tiles of routes; a tile's parts side by side
  const auto parts_of = [&](uint32_t f, uint32_t blocks) { return kJoin ? group * blocks * 64 < f ? 1u : 0u : (f + blocks * 64 - 1) / (blocks * 64); };
  const uint32_t shared_parts = parts_of(a.pool.shared_f, cut.shared_blocks), routed_parts = parts_of(a.pool.f, cut.routed_blocks);
  const uint32_t shared_items = (shared_rows + kTile - 1) / kTile * shared_parts, items = shared_items + __builtin_amdgcn_readfirstlane(tile_count) * routed_parts;
  struct Item {
    const uint16_t *w, *act, *low;  // down rows; the activations' two terms
    uint32_t f, first, blocks, count, left, part;
    bool shared;
  };
  for (uint32_t n = tid; n < items; n += kThreads) {
    const bool shared = n < shared_items;
    const uint32_t in = shared ? n : n - shared_items, per = shared ? shared_parts : routed_parts, part = in % per, first = in / per * kTile;
    const uint2 it = shared ? make_uint2(min(shared_rows - first, kTile) << 16, first) : tiles[in / per];
    table[n] = make_uint2(it.x | part << 24, it.y);
  }
  __syncthreads();
  const auto item_of = [&](uint32_t n) {
    const uint2 e = table[n];
    const uint32_t who = __builtin_amdgcn_readfirstlane(e.x), expert = who & 0xFFFF;
    Item it;
    it.first = __builtin_amdgcn_readfirstlane(e.y);
    it.count = who >> 16 & 0xFF;
    it.part = who >> 24;
    it.shared = n < shared_items;
    it.f = it.shared ? a.pool.shared_f : a.pool.f;
    const uint32_t blocks = it.shared ? cut.shared_blocks : cut.routed_blocks, from = (kJoin ? group : it.part) * blocks * 64;
    it.left = it.f - from;
    it.blocks = (min(it.left, blocks * 64) + 63) / 64;
    it.w = (it.shared ? a.pool.shared_down : a.pool.down) + (static_cast<size_t>(expert) * d + j0) * it.f + from;
    it.act = (it.shared ? a.shared_acts : a.acts) + from;
    it.low = it.act + static_cast<size_t>(it.shared ? a.t : routes) * it.f;
    return it;
  };
  const auto route_of = [&](const Item& it, uint32_t column) {
    const uint32_t at = it.first + min(column, it.count - 1);
    return it.shared ? at : list[at];
  };
  // the requests' place in the stream runs ahead of the products'
  const uint32_t ring = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(whole_lds))) + wave * STAGES * kStage * 16, piece = lane_piece(lane);
  uint32_t ask_item = wave, ask_block = 0, w_at[kW], act_at[XI];
  Item ask{};
  const auto ask_next = [&] {
    ask = item_of(ask_item);
#pragma unroll
    for (uint32_t q = 0; q < kW; ++q) w_at[q] = (min(q * 8 + lane / 8, own_rows - 1) * ask.f + piece) * 2;
#pragma unroll
    for (uint32_t q = 0; q < XI; ++q) act_at[q] = (route_of(ask, q * 8 + lane / 8) * ask.f + piece) * 2;
  };
  const auto request = [&](uint32_t stage) {
    const uint32_t k = __builtin_amdgcn_readfirstlane(ask_block * 64), left = ask.left - k;  // (of the row: 64 and more but in its last block)
    const uint32_t back = piece >= left ? piece * 2 : 0, to = ring + stage * kStage * 16;
#pragma unroll
    for (uint32_t q = 0; q < kW; ++q) load_to_lds_from(uniform(ask.w + k), w_at[q] - back, to + q * 1024);
#pragma unroll
    for (uint32_t q = 0; q < XI; ++q) {
      load_to_lds_from(uniform(ask.act + k), act_at[q] - back, to + (kW + q) * 1024);
      load_to_lds_from(uniform(ask.low + k), act_at[q] - back, to + (kW + XI + q) * 1024);
    }
    if (++ask_block < ask.blocks) return;
    if (ask_item + WAVES < items) {
      ask_item += WAVES;
      ask_block = 0;
      ask_next();
    } else {
      ask_block = ask.blocks - 1;  // behind the end: the last block again
    }
  };
  if (wave < items) {
    const uint32_t mine = ROWS >= 16 ? place_of(r, g) : place_of(r & 7, g), mine_x = XI == 2 ? place_of(r, g) : place_of(r & 7, g);
    ask_next();
#pragma unroll
    for (uint32_t s = 0; s < STAGES; ++s) request(s);
    uint32_t item = wave, block = 0;
    Item now = item_of(item);
    f32x4_t sum[kM] = {};
    for (bool more = true; more;) {
#pragma unroll
      for (uint32_t s = 0; s < STAGES; ++s) {
        if (!more) break;
        const uint4* stage = whole_lds + wave * STAGES * kStage + s * kStage;
        wait_loads<(STAGES - 1) * kLoads>();
        uint4 fw[kM][2], fh[2], fl[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (uint32_t m = 0; m < kM; ++m) fw[m][h] = stage[m * 128 + (mine ^ h * 4)];
          fh[h] = stage[kW * 64 + (mine_x ^ h * 4)];
          fl[h] = stage[(kW + XI) * 64 + (mine_x ^ h * 4)];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read
        request(s);
        const uint32_t left = now.left - block * 64;
        if (left < 64) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t keep = (h * 4 + g) * 8 < left ? ~0u : 0u;
#pragma unroll
            for (uint32_t m = 0; m < kM; ++m) fw[m][h] = masked(fw[m][h], keep);
            fh[h] = masked(fh[h], keep);
            fl[h] = masked(fl[h], keep);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (uint32_t m = 0; m < kM; ++m) {
            sum[m] = mfma16(fw[m][h], fh[h], sum[m]);
            sum[m] = mfma16(fw[m][h], fl[h], sum[m]);
          }
        if (++block < now.blocks) continue;
        const size_t row = static_cast<size_t>(kJoin ? group : now.part) * rows + (now.shared ? routes : 0) + route_of(now, r);
        float* out = (kJoin ? a.route_sums + row * d + j0 : sums + row * ROWS) + g * 4;
#pragma unroll
        for (uint32_t m = 0; m < kM; ++m) {
          if (r < now.count && m * 16 + g * 4 < (kJoin ? own_rows : ROWS)) *reinterpret_cast<f32x4_t*>(out + m * 16) = sum[m];
          sum[m] = f32x4_t{};
        }
        block = 0;
        item += WAVES;
        more = item < items;
        if (more) now = item_of(item);
      }
    }
    wait_loads<0>();
  }
  if constexpr (kJoin) return;
  __syncthreads();
  for (uint32_t o = tid; o < a.t * ROWS; o += kThreads) {
    const uint32_t i = o / ROWS, row = o % ROWS, j = j0 + row;
    if (row >= own_rows) continue;
    float v = 0.0f;
    for (uint32_t k0 = 0; k0 < a.pool.top_k; k0 += 4) {
      uint2 who[4];
      float bias[4];
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {  // (loads of four at a time)
        who[k] = named[i * a.pool.top_k + min(k0 + k, a.pool.top_k - 1)];
        if (k0 + k >= a.pool.top_k || who[k].x >= a.pool.num_experts) who[k].x = ~0u;
        bias[k] = a.pool.down_bias && who[k].x != ~0u ? bf16_to_f(a.pool.down_bias[static_cast<size_t>(who[k].x) * d + j]) : 0.0f;
      }
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        if (who[k].x == ~0u) continue;
        float z = 0.0f;
        for (uint32_t p = 0; p < routed_parts; ++p) z += sums[(static_cast<size_t>(p) * rows + i * a.pool.top_k + k0 + k) * ROWS + row];
        v += __uint_as_float(who[k].y) * (z + bias[k]);
      }
    }
    if (shared_rows) {
      float z = 0.0f;
      for (uint32_t p = 0; p < shared_parts; ++p) z += sums[(static_cast<size_t>(p) * rows + routes + i) * ROWS + row];
      if (a.pool.shared_gate) z *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a.shared_gate[i] * -1.4426950408889634f));
      v += z;
    }
    if (a.residual) v += bf16_to_f(a.residual[static_cast<size_t>(i) * a.residual_stride + j]);
    a.y[static_cast<size_t>(i) * a.y_stride + j] = narrow_bf16(v);
  }
}

// The third launch, beyond eight tokens: four neighbouring results of a token a thread, the weighted sums of its routes in the order of their ranks, the parts of a sum in theirs.
template <uint32_t GROUPS>
__global__ __launch_bounds__(64) void experts_join_kernel(const Bf16ExpertsArgs a, const DownCut cut) {
  const uint32_t d = a.pool.d, at = blockIdx.x * 64 + threadIdx.x, i = at / (d / 4), j = at % (d / 4) * 4, routes = a.route_count(), rows = routes + (a.pool.shared_f ? a.t : 0);
  if (i >= a.t) return;
  const auto load = [&](f32x4_t* z, uint32_t row, uint32_t f, uint32_t blocks, bool is) {  // (a short f has fewer parts)
#pragma unroll
    for (uint32_t p = 0; p < GROUPS; ++p) z[p] = is && p * blocks * 64 < f ? *reinterpret_cast<const f32x4_t*>(a.route_sums + (static_cast<size_t>(p) * rows + row) * d + j) : f32x4_t{};
  };
  const auto whole = [](const f32x4_t* z) {
    f32x4_t sum = z[0];
#pragma unroll
    for (uint32_t p = 1; p < GROUPS; ++p) sum += z[p];
    return sum;
  };
  // (the loads of all ranks at once: one after the other they took 10.9 us, so 8.0: 61 tokens of 8 routes, 2048 results, four parts, 16 MB)
  f32x4_t v = {}, z[MF_MAX_TOPK][GROUPS];
  uint32_t e[MF_MAX_TOPK];
  float w[MF_MAX_TOPK];
#pragma unroll
  for (uint32_t k = 0; k < MF_MAX_TOPK; ++k) {
    const uint32_t route = i * a.pool.top_k + min(k, a.pool.top_k - 1);
    e[k] = k < a.pool.top_k ? a.idx[route] : ~0u;
    w[k] = a.w[route];
  }
#pragma unroll
  for (uint32_t k = 0; k < MF_MAX_TOPK; ++k) load(z[k], i * a.pool.top_k + k, a.pool.f, cut.routed_blocks, e[k] < a.pool.num_experts);
#pragma unroll
  for (uint32_t k = 0; k < MF_MAX_TOPK; ++k) {
    if (e[k] >= a.pool.num_experts) continue;
    f32x4_t sum = whole(z[k]);
    if (a.pool.down_bias)
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[c] += bf16_to_f(a.pool.down_bias[static_cast<size_t>(e[k]) * d + j + c]);
    v += w[k] * sum;
  }
  if (a.pool.shared_f) {
    load(z[0], routes + i, a.pool.shared_f, cut.shared_blocks, true);
    f32x4_t sum = whole(z[0]);
    if (a.pool.shared_gate) sum *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a.shared_gate[i] * -1.4426950408889634f));
    v += sum;
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (a.residual) v[c] += bf16_to_f(a.residual[static_cast<size_t>(i) * a.residual_stride + j + c]);
    a.y[static_cast<size_t>(i) * a.y_stride + j + c] = narrow_bf16(v[c]);
  }
}

// Beyond eight tokens: parts of the sums over f in workgroups of their own, until every unit has one of 20 rows or more.  16 tokens, 12 live
// experts of 1024 x 2048: 32 us in one, 16.6 + 4.8 in four; 32 tokens, 27 live of 704 x 2816: 37 in two of 24 rows.
uint32_t groups_of(const mf_bf16_expert_pool& p) {
  uint32_t groups = 1;
  while (groups < 4 && p.d * groups < device_cu_count() * 20) groups *= 2;
  return groups;
}

// Rows of a workgroup, at most `most`, that give every unit the same number of workgroups.  (Fewer than four would read little but activations.)
uint32_t rows_of_workgroup(uint32_t d, uint32_t groups, uint32_t most, uint32_t cus) {
  const uint32_t rounds = (d * groups + cus * most - 1) / (cus * most);
  return std::min(std::max((d * groups + cus * rounds - 1) / (cus * rounds), 4u), most);
}

template <int ROWS, int XI, int STAGES, int WAVES>
hipError_t launch_down(hipStream_t s, const Bf16ExpertsArgs& a, uint32_t own_rows, uint32_t groups) {
  const mf_bf16_expert_pool& p = a.pool;
  const uint32_t routes = a.route_count(), rows = routes + (p.shared_f ? a.t : 0), longest = (std::max(p.f, p.shared_f) + 63) / 64;
  DownCut cut = {own_rows, ((p.f + 63) / 64 + groups - 1) / groups, ((p.shared_f + 63) / 64 + groups - 1) / groups, 1};
  if (XI == 1) {  // parts, so that every wave has something to do when few experts are live
    while (cut.parts < 4 && a.most_live() * cut.parts < 2 * WAVES && cut.parts * 2 * rows * ROWS <= 4096 && longest > cut.parts) cut.parts *= 2;
    cut.routed_blocks = cut.shared_blocks = (longest + cut.parts - 1) / cut.parts;
  }
  const size_t items = static_cast<size_t>(routes + (p.shared_f ? (a.t + 8 * XI - 1) / (8 * XI) : 0)) * cut.parts;
  const size_t own = XI == 1 ? static_cast<size_t>(cut.parts) * rows * ROWS * 4 + routes * 8 : 0;
  const size_t lds = WAVES * STAGES * (ROWS / 8 + 2 * XI) * 1024 + own + (routes + 1) / 2 * 8 + routes * 8 + items * 8;
  hipError_t e = allow_lds<experts_down_kernel<ROWS, XI, STAGES, WAVES>>(lds, 154 * 1024);
  if (e != hipSuccess) return e;
  experts_down_kernel<ROWS, XI, STAGES, WAVES><<<dim3((p.d + own_rows - 1) / own_rows, groups), 64 * WAVES, lds, s>>>(a, cut);
  e = hipGetLastError();
  if (XI == 1 || e != hipSuccess) return e;
  const dim3 grid((a.t * (p.d / 4) + 63) / 64);
  if (groups == 1) experts_join_kernel<1><<<grid, 64, 0, s>>>(a, cut);
  else if (groups == 2) experts_join_kernel<2><<<grid, 64, 0, s>>>(a, cut);
  else experts_join_kernel<4><<<grid, 64, 0, s>>>(a, cut);
  return hipGetLastError();
}

template <int XI>
hipError_t launch_up(hipStream_t s, const Bf16ExpertsArgs& a) {
  const mf_bf16_expert_pool& p = a.pool;
  const uint32_t shared = p.shared_f ? (a.t + 8 * XI - 1) / (8 * XI) + (p.shared_gate ? 1 : 0) : 0;
  const dim3 grid((std::max(p.f, p.shared_f) + 15) / 16, a.most_tiles(8 * XI) + shared);
  if (aligned16(a.x) && a.x_stride % 8 == 0 && a.x_stride < 1u << 24) experts_up_kernel<XI, true><<<grid, 64 * kUpWaves, 0, s>>>(a);  // (offsets of 32 bits)
  else experts_up_kernel<XI, false><<<grid, 64 * kUpWaves, 0, s>>>(a);
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
  p += 4 * static_cast<size_t>(a.t) * a.pool.shared_f;
  a.route_sums = reinterpret_cast<float*>(p);
}

size_t bf16_experts_workspace_bytes(const mf_bf16_expert_pool& pool, uint32_t t) {
  Bf16ExpertsArgs a{};
  a.pool = pool;
  a.t = t;
  bf16_experts_layout(a, nullptr);
  return reinterpret_cast<uintptr_t>(a.route_sums) + (t > 8 ? 4 * static_cast<size_t>(groups_of(pool)) * (a.route_count() + (pool.shared_f ? t : 0)) * pool.d : 0);
}

hipError_t launch_bf16_experts(hipStream_t s, const Bf16ExpertsArgs& a) {
  const mf_bf16_expert_pool& p = a.pool;
  const hipError_t e = a.t <= 8 ? launch_up<1>(s, a) : launch_up<2>(s, a);
  if (e != hipSuccess) return e;
  const uint32_t cus = device_cu_count();
  if (a.t <= 8) {
    const uint32_t rows = rows_of_workgroup(p.d, 1, 16, cus);
    return rows <= 8 ? launch_down<8, 1, 4, 8>(s, a, rows, 1) : launch_down<16, 1, 4, 8>(s, a, rows, 1);
  }
  const uint32_t groups = groups_of(p);
  return launch_down<32, 2, 4, 4>(s, a, (rows_of_workgroup(p.d, groups, 32, cus) + 3) / 4 * 4, groups);  // (four results a store)
}

}  // namespace mf
