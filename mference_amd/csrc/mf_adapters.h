// The low-rank adapters as api.hip and adapters.hip see them.
#pragma once

#include "mf_internal.h"

namespace mf {

// mf_adapter_group's words.  Behind the two public lists: four words that say what the plan is of (t, adapters, tiles, rows a
// tile), and the tiles: runs of at most tile_rows rows of one adapter, x = adapter | rows << 16, y = where its rows start in
// the list.
struct AdapterPlan {
  uint32_t* rows;     // [t]
  uint32_t* offsets;  // [n + 1]
  uint32_t* header;   // [4]
  uint2* tiles;       // [most_tiles]
  uint32_t* runs;     // [runs][n + 1]: rows of every key in each run, where there are several
  uint32_t tile_rows, most_tiles;

  // tile i of an adapter whose rows start at `at` in the list
  __device__ uint2 tile(uint32_t adapter, uint32_t at, uint32_t count, uint32_t i) const {
    return make_uint2(adapter | min(count - i * tile_rows, tile_rows) << 16, at + i * tile_rows);
  }
  // rows a tile: what a wave of the products holds at once.  Where a batch has few rows an adapter the wide tiles would be
  // mostly empty.
  static uint32_t rows_of_tile(uint32_t t, uint32_t n) { return t / 32 >= n ? 64 : 16; }
  static uint32_t tiles_of(uint32_t t, uint32_t n) { return t / rows_of_tile(t, n) + (n < t ? n : t); }
  static size_t header_word(uint32_t t, uint32_t n) { return (static_cast<size_t>(t) + n + 1 + 3) / 4 * 4; }
  // the sort: rows a lane takes one after the other, and workgroups of 1024 lanes
  static uint32_t turns_of(uint32_t t) { return t <= 1024 ? 1 : t <= 4096 ? 4 : t <= 32768 ? 1 : t <= 262144 ? 4 : 16; }
  static uint32_t runs_of(uint32_t t) { return t <= 4096 ? 1 : (t + 1024 * turns_of(t) - 1) / (1024 * turns_of(t)); }
  static size_t words(uint32_t t, uint32_t n) {
    return header_word(t, n) + 4 + 2 * static_cast<size_t>(tiles_of(t, n)) + (runs_of(t) > 1 ? static_cast<size_t>(runs_of(t)) * (n + 1) : 0);
  }
  static AdapterPlan at(uint32_t* p, uint32_t t, uint32_t n) {
    uint32_t* h = p + header_word(t, n);
    return {p, p + t, h, reinterpret_cast<uint2*>(h + 4), h + 4 + 2 * static_cast<size_t>(tiles_of(t, n)), rows_of_tile(t, n), tiles_of(t, n)};
  }
};

struct AdapterArgs {
  struct Target {
    const uint16_t* a;
    const uint16_t* b;
    void* y;
    uint32_t m, y_stride;
  };
  Target target[MF_MAX_ADAPTER_TARGETS];
  const uint32_t* ranks;
  const float* scales;
  const uint16_t* x;
  const int32_t* ids;
  float* v;  // [splits, t, cols]: c_a A x in parts, targets side by side
  uint32_t num_targets, num_adapters, rank, n, t, x_stride, cols, splits, by_xcd;
  uint32_t run_blocks, first_run[MF_MAX_ADAPTER_TARGETS + 1];  // a workgroup's share of the results: blocks of 64, and where each target's begin
  AdapterPlan plan;  // tiles null: the rows as they lie
};

hipError_t launch_adapter_group(hipStream_t s, const int32_t* ids, uint32_t t, uint32_t n, uint32_t* plan);
size_t adapter_workspace_bytes(uint32_t num_targets, uint32_t rank, uint32_t n, uint32_t t);
hipError_t launch_adapter_apply(hipStream_t s, AdapterArgs a, bool y_f32);

// block_norm.hip
hipError_t launch_block_norm(hipStream_t s, const mf_block_norm_args& a);

}  // namespace mf
