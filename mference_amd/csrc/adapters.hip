// Low-rank adapters of many requests beside a shared projection (mf_adapter_apply) and the grouping of a batch's rows by
// adapter (mf_adapter_group).
#include <algorithm>
#include <type_traits>

#include "mf_adapters.h"
#include "mf_device.h"

namespace mf {

namespace {

// ------------------------------------------------------------------ rows by adapter

__device__ __forceinline__ uint32_t adapter_key(int32_t id, uint32_t n) { return static_cast<uint32_t>(id) < n ? static_cast<uint32_t>(id) : n; }

// A stable counting sort.  A wave owns IT * 64 consecutive rows and takes 64 of them at a time: the lanes that hold the same key find
// each other by a ballot for every bit of it, a row's place among its wave's rows of that key is the count so far plus the lanes in
// front of it, and the lane in front raises the count.  No atomics: the order is the rows'.  Counts of a wave fit 16 bits (IT <= 16).
template <int IT>
struct RowRanks {
  uint32_t key[IT], rank[IT];  // rank within the wave's rows of the key
  uint64_t valid[IT];

  __device__ __forceinline__ void find(const int32_t* __restrict__ ids, uint32_t first, uint32_t t, uint32_t n, uint16_t* counts) {
    const uint32_t lane = threadIdx.x & 63, bits = 32 - __builtin_clz(n);
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const uint32_t i = first + k * 64 + lane;
      key[k] = i < t ? adapter_key(ids[i], n) : n;
    }
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      valid[k] = __ballot(first + k * 64 + lane < t);
      uint64_t same = valid[k];
      for (uint32_t b = 0; b < bits; ++b) {
        const bool set = (key[k] >> b) & 1;
        const uint64_t with = __ballot(set);
        same &= set ? with : ~with;
      }
      const uint32_t in_front = __builtin_popcountll(same & ((1ull << lane) - 1));
      if ((valid[k] >> lane) & 1) {
        const uint32_t before = counts[key[k]];
        rank[k] = before + in_front;
        if (in_front == 0) counts[key[k]] = static_cast<uint16_t>(before + __builtin_popcountll(same));
      }
      asm volatile("" ::: "memory");  // the next 64 read what these have left
      __builtin_amdgcn_wave_barrier();
    }
  }
};

// exclusive sums over the workgroup of two numbers a thread
__device__ __forceinline__ uint2 block_exclusive(uint2 v, uint2* part) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint2 sum = v;
#pragma unroll
  for (uint32_t by = 1; by < 64; by *= 2) {
    const uint32_t x = __shfl_up(sum.x, by), y = __shfl_up(sum.y, by);
    if (lane >= by) sum.x += x, sum.y += y;
  }
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  uint2 before = make_uint2(sum.x - v.x, sum.y - v.y);
  for (uint32_t w = 0; w < wave; ++w) before.x += part[w].x, before.y += part[w].y;
  return before;
}

// One workgroup for a run of rows.  COUNT: it leaves how many rows of every key the run has, and that is all.  Otherwise it adds up
// those counts of all runs (a thread a key), knows from them where every key's rows start and where its own go, and writes its rows;
// the lists of adapters and tiles are dealt out over the workgroups.  A batch of one run needs no counting launch in front.
template <int IT, bool COUNT>
__global__ __launch_bounds__(1024) void adapter_group_kernel(const int32_t* __restrict__ ids, uint32_t t, uint32_t n, AdapterPlan plan) {
  __shared__ uint16_t counts[16 * (MF_MAX_ADAPTERS + 1)];  // [wave][key]; then where a wave's rows of a key start among the run's
  __shared__ uint32_t starts[MF_MAX_ADAPTERS + 1];         // where the run's rows of a key go
  __shared__ uint2 part[16];
  const uint32_t waves = blockDim.x / 64, keys = n + 1, wave = threadIdx.x >> 6;
  for (uint32_t k = threadIdx.x; k < waves * keys; k += blockDim.x) counts[k] = 0;
  __syncthreads();
  RowRanks<IT> mine;
  const uint32_t first = (blockIdx.x * waves + wave) * (IT * 64);
  mine.find(ids, first, t, n, counts + wave * keys);
  __syncthreads();
  uint2 total = make_uint2(0, 0);  // rows and tiles of thread k's key
  uint32_t before = 0;             // its rows in the runs in front
  for (uint32_t k = threadIdx.x; k < keys; k += blockDim.x) {  // (a second turn for the last key of the largest pool only)
    uint32_t own = 0;
    for (uint32_t w = 0; w < waves; ++w) {
      const uint32_t c = counts[w * keys + k];
      counts[w * keys + k] = static_cast<uint16_t>(own);  // at most 16 * 16 * 64 rows in front
      own += c;
    }
    if constexpr (COUNT) {
      plan.runs[static_cast<size_t>(blockIdx.x) * keys + k] = own;
    } else if (k < n) {
      total.x = own;
      if (gridDim.x > 1) {
        total.x = 0;
        for (uint32_t r = 0; r < gridDim.x; ++r) {
          const uint32_t c = plan.runs[static_cast<size_t>(r) * keys + k];
          before += r < blockIdx.x ? c : 0;
          total.x += c;
        }
      }
      total.y = (total.x + plan.tile_rows - 1) / plan.tile_rows;
    }
  }
  if constexpr (!COUNT) {
    const uint2 at = block_exclusive(total, part);
    const uint32_t k = threadIdx.x;
    if (k < n) {
      starts[k] = at.x + before;
      if (k % gridDim.x == blockIdx.x) {
        plan.offsets[k] = at.x;
        for (uint32_t i = 0; i < total.y; ++i)
          plan.tiles[at.y + i] = make_uint2(k | min(total.x - i * plan.tile_rows, plan.tile_rows) << 16, at.x + i * plan.tile_rows);
      }
    }
    if (k == n - 1) {  // behind all adapters: the rows without one.  What of them lies in the runs in front is what the adapters leave.
      const uint32_t with = at.x + total.x;
      starts[n] = with;
      if (blockIdx.x == 0) {
        plan.offsets[n] = with;
        plan.header[0] = t;
        plan.header[1] = n;
        plan.header[2] = at.y + total.y;
        plan.header[3] = plan.tile_rows;
      }
    }
    __syncthreads();
    if (gridDim.x > 1) {
      for (uint32_t r = threadIdx.x; r < blockIdx.x; r += blockDim.x) atomicAdd(&starts[n], plan.runs[static_cast<size_t>(r) * keys + n]);  // whole numbers: any order
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (!((mine.valid[i] >> (threadIdx.x & 63)) & 1)) continue;
      plan.rows[starts[mine.key[i]] + counts[wave * keys + mine.key[i]] + mine.rank[i]] = first + i * 64 + (threadIdx.x & 63);
    }
  }
}

// ------------------------------------------------------------------ which rows meet which adapter

__device__ __forceinline__ uint32_t live_rank(const AdapterArgs& a, uint32_t adapter) { return a.ranks ? min(a.ranks[adapter], a.rank) : a.rank; }

// ROWS rows of the batch, a lane each (ROWS <= 64; the lanes behind hold none), and the adapters that they meet.  With a plan they are
// (a part of) one of its tiles, of one adapter; without one they are consecutive rows, whose adapters are taken one after the other in
// the order of their first rows.  Every wave finds them for itself.
template <int ROWS>
struct Meeting {
  uint32_t row;    // this lane's
  uint32_t key;    // its adapter, num_adapters where it has no row or no adapter
  uint64_t left;   // lanes whose adapter is still to come

  // PLAN_ROWS: rows of a tile of the plan
  __device__ __forceinline__ Meeting(const AdapterArgs& a, uint32_t tile, uint32_t lane) : row(0), key(a.num_adapters) {
    if (a.plan.tiles && a.plan.header[0] == a.t && a.plan.header[1] == a.num_adapters) {
      const uint32_t parts = a.plan.tile_rows / ROWS, of = tile / parts, from = tile % parts * ROWS;
      if (of < a.plan.header[2] && of < a.plan.most_tiles) {
        const uint2 rec = a.plan.tiles[of];
        const uint32_t count = rec.x >> 16;
        if (lane < ROWS && from + lane < count && rec.y + from + lane < a.t) {
          row = a.plan.rows[rec.y + from + lane];
          if (row < a.t) key = min(rec.x & 0xFFFFu, a.num_adapters);
          else row = 0;
        }
      }
    } else {
      const uint32_t r = tile * ROWS + lane;
      if (lane < ROWS && r < a.t) {
        row = r;
        key = adapter_key(a.ids[r], a.num_adapters);
      }
    }
    left = __ballot(key < a.num_adapters);
  }
  // the next adapter, and the lanes that have it; false when there is none left
  __device__ __forceinline__ bool next(uint32_t& adapter, uint64_t& lanes, uint32_t& lead) {
    if (!left) return false;
    lead = static_cast<uint32_t>(__builtin_ctzll(left));
    adapter = __builtin_amdgcn_readlane(key, lead);
    lanes = __ballot(key == adapter);
    left &= ~lanes;
    return true;
  }
};

__device__ __forceinline__ f32x4_t mfma16(const uint4& a, const uint4& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// ------------------------------------------------------------------ v = c A x
//
// Operands of v_mfma_f32_16x16x32_bf16 are eight consecutive elements of a row a lane, of x (16 rows of the batch) and of A (16 ranks):
// 16-byte loads straight into the registers that the instruction reads.  A workgroup takes RT * 16 rows, CF blocks of 16 ranks and a
// window of the row length; its eight waves take 64 elements (a line of 128 bytes) in turn and add their sums through LDS.  A rank
// beyond the adapter's, and a row of another one, is a column or a row of the product that nobody reads.
constexpr uint32_t kShrinkWaves = 8;

template <int RT, int CF>
__global__ __launch_bounds__(kShrinkWaves * 64) void adapter_shrink_kernel(const AdapterArgs a) {
  __shared__ f32x4_t part[kShrinkWaves][RT * CF][64];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t split = blockIdx.y % a.splits, group = blockIdx.y / a.splits;
  const uint32_t blocks = (a.rank + 15) / 16;  // of 16 ranks, a target
  const uint32_t units = a.n / 64, u0 = units * split / a.splits, u1 = units * (split + 1) / a.splits;
  const uint32_t in_row = (lane >> 4) * 8;
  Meeting<RT * 16> meeting(a, blockIdx.x, lane);
  uint32_t adapter, lead;
  uint64_t lanes;
  for (uint32_t turn = 0; meeting.next(adapter, lanes, lead); ++turn) {
    if (turn % gridDim.z != blockIdx.z) continue;
    const uint32_t rank = live_rank(a, adapter);
    const float scale = a.scales ? a.scales[adapter] : 1.0f;
    const uint16_t* xp[RT];
    const uint16_t* wp[CF];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const uint32_t at = r * 16 + (lane & 15);
      const uint32_t row = __shfl(meeting.row, (lanes >> at) & 1 ? at : lead);
      xp[r] = a.x + static_cast<size_t>(row) * a.x_stride + in_row;
    }
    bool any = false;
#pragma unroll
    for (int c = 0; c < CF; ++c) {
      const uint32_t cb = group * CF + c, target = cb / blocks, first = cb % blocks * 16;
      const bool live = target < a.num_targets && first < rank;
      any |= live;
      const uint32_t r = first + (lane & 15);
      wp[c] = a.target[live ? target : 0].a + (static_cast<size_t>(adapter) * a.rank + (live && r < rank ? r : 0)) * a.n + in_row;
    }
    if (!any) continue;
    f32x4_t acc[RT][CF];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < CF; ++c) acc[r][c] = f32x4_t{0, 0, 0, 0};
    const auto step = [&](auto n_units, uint32_t u) {  // that many of the wave's units, all requested before the first is used
      constexpr int kUnits = decltype(n_units)::value;
      uint4 xv[RT][2 * kUnits], wv[CF][2 * kUnits];
#pragma unroll
      for (int k = 0; k < 2 * kUnits; ++k) {
        const uint32_t at = (u + k / 2 * kShrinkWaves) * 64 + k % 2 * 32;
#pragma unroll
        for (int r = 0; r < RT; ++r) xv[r][k] = load_16_bytes(xp[r] + at);
#pragma unroll
        for (int c = 0; c < CF; ++c) wv[c][k] = *reinterpret_cast<const uint4*>(wp[c] + at);
      }
#pragma unroll
      for (int k = 0; k < 2 * kUnits; ++k)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int c = 0; c < CF; ++c) acc[r][c] = mfma16(xv[r][k], wv[c][k], acc[r][c]);
    };
    uint32_t u = u0 + wave;
    for (; u + kShrinkWaves < u1; u += 2 * kShrinkWaves) step(std::integral_constant<int, 2>{}, u);
    if (u < u1) step(std::integral_constant<int, 1>{}, u);
    __syncthreads();  // (the parts of the adapter before have been read)
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < CF; ++c) part[wave][r * CF + c][lane] = acc[r][c];
    __syncthreads();
    for (uint32_t f = wave; f < RT * CF; f += kShrinkWaves) {
      f32x4_t sum[kShrinkWaves];
#pragma unroll
      for (uint32_t w = 0; w < kShrinkWaves; ++w) sum[w] = part[w][f][lane];
#pragma unroll
      for (uint32_t by = 1; by < kShrinkWaves; by *= 2)
#pragma unroll
        for (uint32_t w = 0; w < kShrinkWaves; w += 2 * by) sum[w] += sum[w + by];
      const uint32_t cb = group * CF + f % CF, target = cb / blocks, r = cb % blocks * 16 + (lane & 15);
      const uint32_t row0 = f / CF * 16 + (lane >> 4) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t row = __shfl(meeting.row, row0 + i);
        if (target < a.num_targets && r < rank && ((lanes >> (row0 + i)) & 1))
          a.v[(static_cast<size_t>(split) * a.t + row) * a.cols + target * a.rank + r] = sum[0][i] * scale;
      }
    }
  }
}

// ------------------------------------------------------------------ y += B v
//
// The second product with B as the instruction's first operand (16 results) and v as its second (16 rows), so that a lane ends with
// four consecutive results of one row for every 16: results are dealt to the operand's rows such that those come together to 16 bytes
// of y.  v goes in as TERMS bf16 numbers whose sum it is (to 16 bits, or all 24): the upper half of its bits, the same of what is left,
// and the rest; an infinity stays in the first.
template <int TERMS>
__device__ __forceinline__ void split_terms(const float (&v)[8], uint4 (&out)[TERMS]) {
  float rest[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) rest[e] = v[e];
#pragma unroll
  for (int k = 0; k < TERMS; ++k) {
    if (k == TERMS - 1) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = static_cast<uint32_t>(narrow_bf16(rest[2 * e])) | static_cast<uint32_t>(narrow_bf16(rest[2 * e + 1])) << 16;
      out[k] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      out[k] = make_uint4(upper_halves(rest[0], rest[1]), upper_halves(rest[2], rest[3]), upper_halves(rest[4], rest[5]), upper_halves(rest[6], rest[7]));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float top = __uint_as_float(__float_as_uint(rest[e]) & 0xFFFF0000u);
        rest[e] = __builtin_isfinite(rest[e]) ? rest[e] - top : 0.0f;
      }
    }
  }
}

// the first `n` of eight bf16 numbers (n < 8), zeros behind
__device__ __forceinline__ uint4 keep_bf16(uint4 v, uint32_t n) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) w[e] = 2 * e + 1 < n ? w[e] : 2 * e < n ? w[e] & 0xFFFFu : 0u;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A workgroup takes RT * 16 rows and a run of a target's results.  It adds up the parts of v and leaves its terms in LDS as the
// operands that the instruction reads; its waves then take 64 results in turn, the y and B of the next ones requested before the
// present ones are worked on.
template <int RT, bool F32>
__global__ __launch_bounds__(256) void adapter_expand_kernel(const AdapterArgs a) {
  constexpr int kTerms = F32 ? 3 : 2, kPer = F32 ? 4 : 8, kChunks = 16 / kPer;  // results to 16 bytes; such pieces a lane holds of a row
  using Elem = std::conditional_t<F32, float, uint16_t>;
  extern __shared__ uint4 operand[];  // [32 ranks][RT][kTerms][lane]
  const uint32_t lane = threadIdx.x & 63, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t run = blockIdx.x, target = 0;
  while (run >= a.first_run[target + 1]) ++target;
  run -= a.first_run[target];
  const AdapterArgs::Target tg = a.target[target];
  const uint32_t m_blocks = (tg.m + 63) / 64, end = min(m_blocks, (run + 1) * a.run_blocks);
  Meeting<RT * 16> meeting(a, blockIdx.y, lane);
  uint32_t adapter, lead;
  uint64_t lanes;
  for (uint32_t turn = 0; meeting.next(adapter, lanes, lead); ++turn) {
    if (turn % gridDim.z != blockIdx.z) continue;
    const uint16_t* bp = tg.b + static_cast<size_t>(adapter) * tg.m * a.rank;
    Elem* yp[RT];
    bool mine[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const uint32_t at = r * 16 + (lane & 15);
      mine[r] = (lanes >> at) & 1;
      yp[r] = static_cast<Elem*>(tg.y) + static_cast<size_t>(__shfl(meeting.row, mine[r] ? at : lead)) * tg.y_stride;
    }
    const auto load_y = [&](uint32_t block, uint4 (&yv)[RT][kChunks]) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint32_t m = block * 64 + c * 4 * kPer + q * kPer;
          if (mine[r] && m + kPer <= tg.m) yv[r][c] = load_16_bytes(yp[r] + m);
        }
    };
    const auto load_b = [&](uint32_t block, uint32_t k, uint4 (&bv)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t p = lane & 15;
        const uint32_t m = block * 64 + (F32 ? 16 * j + p : 32 * (j >> 1) + 8 * (p >> 2) + 4 * (j & 1) + (p & 3));
        if (k < a.rank) bv[j] = *reinterpret_cast<const uint4*>(bp + static_cast<size_t>(min(m, tg.m - 1)) * a.rank + k);
      }
    };
    uint32_t block = run * a.run_blocks + wave;
    uint4 yv[RT][kChunks], bv[4];
    if (block < end) {
      load_y(block, yv);
      load_b(block, q * 8, bv);
    }
    const uint32_t rank = live_rank(a, adapter), kb = (rank + 31) / 32;
    __syncthreads();  // (the operands of the adapter before have been read)
    for (uint32_t slot = threadIdx.x; slot < kb * RT * 64; slot += 256) {
      const uint32_t at = slot / 64 % RT * 16 + (slot & 15), k = slot / (64 * RT) * 32 + (slot >> 4) % 4 * 8, have = k < rank ? min(rank - k, 8u) : 0;
      float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      const uint32_t row = __shfl(meeting.row, at);
      if (have && ((lanes >> at) & 1)) {
        const float* p = a.v + static_cast<size_t>(row) * a.cols + target * a.rank + k;
        const size_t part = static_cast<size_t>(a.t) * a.cols;
        for (uint32_t s = 0; s < a.splits; s += 4) {  // four parts requested at once
          float4 lo[4], hi[4];
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const float4* w = reinterpret_cast<const float4*>(p + min(s + i, a.splits - 1) * part);
            lo[i] = w[0], hi[i] = w[1];
          }
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            if (s + i >= a.splits) continue;
            v[0] += lo[i].x, v[1] += lo[i].y, v[2] += lo[i].z, v[3] += lo[i].w;
            v[4] += hi[i].x, v[5] += hi[i].y, v[6] += hi[i].z, v[7] += hi[i].w;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = static_cast<uint32_t>(e) < have ? v[e] : 0.0f;
      uint4 terms[kTerms];
      split_terms<kTerms>(v, terms);
#pragma unroll
      for (int i = 0; i < kTerms; ++i) operand[(slot / 64 * kTerms + i) * 64 + (slot & 63)] = terms[i];
    }
    __syncthreads();
    for (; block < end; block += 4) {
      uint4 next_y[RT][kChunks], next_b[4];
      if (block + 4 < end) {
        load_y(block + 4, next_y);
        load_b(block + 4, q * 8, next_b);
      }
      f32x4_t acc[RT][4];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[r][j] = f32x4_t{0, 0, 0, 0};
      for (uint32_t b = 0; b < kb; ++b) {
        const uint32_t k = b * 32 + q * 8, have = k < rank ? min(rank - k, 8u) : 0;
        if (b) load_b(block, k, bv);
        if (rank % 32) {
#pragma unroll
          for (int j = 0; j < 4; ++j) bv[j] = have < 8 ? keep_bf16(bv[j], have) : bv[j];
        }
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int i = kTerms - 1; i >= 0; --i) {  // the small terms first
            const uint4 term = operand[((b * RT + r) * kTerms + i) * 64 + lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[r][j] = mfma16(bv[j], term, acc[r][j]);
          }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (!mine[r]) continue;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint32_t m = block * 64 + c * 4 * kPer + q * kPer;
          float add[kPer];
#pragma unroll
          for (int e = 0; e < kPer; ++e) add[e] = acc[r][F32 ? c : 2 * c + e / 4][e % 4];
          if (m + kPer <= tg.m) {
            uint32_t w[4] = {yv[r][c].x, yv[r][c].y, yv[r][c].z, yv[r][c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (F32) w[e] = __float_as_uint(__uint_as_float(w[e]) + add[e]);
              else w[e] = static_cast<uint32_t>(narrow_bf16(bf16_lo(w[e]) + add[2 * e])) | static_cast<uint32_t>(narrow_bf16(bf16_hi(w[e]) + add[2 * e + 1])) << 16;
            }
            __builtin_memcpy(yp[r] + m, w, 16);
          } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
              if (m + e >= tg.m) continue;
              if constexpr (F32) yp[r][m + e] += add[e];
              else yp[r][m + e] = narrow_bf16(bf16_to_f(yp[r][m + e]) + add[e]);
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) yv[r][c] = next_y[r][c];
#pragma unroll
      for (int j = 0; j < 4; ++j) bv[j] = next_b[j];
    }
  }
}

// Parts of the sum over n: workgroups for one and a half times the CUs, of eight units of 64 elements (one a wave) or more, and few
// parts where there are many rows (every part of v is written and read again).
constexpr uint32_t kMostSplits = 16, kShrinkGroups = 384;
uint32_t shrink_splits(uint32_t t, uint32_t n) {
  return std::max(1u, std::min({kShrinkGroups / ((t + 15) / 16), n / 64 / kShrinkWaves, kMostSplits}));
}

template <int RT>
void launch_shrink(hipStream_t s, const AdapterArgs& a, uint32_t tiles, uint32_t turns) {
  const uint32_t blocks = (a.rank + 15) / 16 * a.num_targets;
  const auto go = [&](auto cf) {
    constexpr int kCols = decltype(cf)::value;
    adapter_shrink_kernel<RT, kCols><<<dim3(tiles, (blocks + kCols - 1) / kCols * a.splits, turns), dim3(kShrinkWaves * 64), 0, s>>>(a);
  };
  if (blocks == 1) go(std::integral_constant<int, 1>{});
  else if (blocks == 2) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, 4>{});
}

template <int RT, bool F32>
hipError_t launch_expand(hipStream_t s, AdapterArgs& a, uint32_t tiles, uint32_t turns) {
  uint32_t blocks = 0;
  for (uint32_t k = 0; k < a.num_targets; ++k) blocks += (a.target[k].m + 63) / 64;
  // runs of results: workgroups for eight times the CUs where there is so much to do
  a.run_blocks = std::max<uint32_t>(1, static_cast<uint32_t>(static_cast<uint64_t>(blocks) * tiles / (4 * 2048))) * 4;
  a.first_run[0] = 0;
  for (uint32_t k = 0; k < MF_MAX_ADAPTER_TARGETS; ++k)
    a.first_run[k + 1] = k < a.num_targets ? a.first_run[k] + ((a.target[k].m + 63) / 64 + a.run_blocks - 1) / a.run_blocks : 0xFFFFFFFFu;
  const size_t lds = static_cast<size_t>((a.rank + 31) / 32) * RT * (F32 ? 3 : 2) * 1024;
  hipError_t e = allow_lds<adapter_expand_kernel<RT, F32>>(lds, 64 * 1024);
  if (e != hipSuccess) return e;
  adapter_expand_kernel<RT, F32><<<dim3(a.first_run[a.num_targets], tiles, turns), dim3(256), lds, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_adapter_group(hipStream_t s, const int32_t* ids, uint32_t t, uint32_t n, uint32_t* plan) {
  const AdapterPlan p = AdapterPlan::at(plan, t, n);
  const uint32_t runs = AdapterPlan::runs_of(t), it = AdapterPlan::turns_of(t);
  const auto go = [&](auto turns) {
    constexpr int kTurns = decltype(turns)::value;
    if (runs == 1) {  // threads for the rows, and one for every adapter
      const uint32_t threads = std::max((t + kTurns * 64 - 1) / (kTurns * 64) * 64, (n + 63) / 64 * 64);
      adapter_group_kernel<kTurns, false><<<dim3(1), dim3(threads), 0, s>>>(ids, t, n, p);
      return;
    }
    adapter_group_kernel<kTurns, true><<<dim3(runs), dim3(1024), 0, s>>>(ids, t, n, p);
    adapter_group_kernel<kTurns, false><<<dim3(runs), dim3(1024), 0, s>>>(ids, t, n, p);
  };
  if (it == 1) go(std::integral_constant<int, 1>{});
  else if (it == 4) go(std::integral_constant<int, 4>{});
  else go(std::integral_constant<int, 16>{});
  return hipGetLastError();
}

size_t adapter_workspace_bytes(uint32_t num_targets, uint32_t rank, uint32_t n, uint32_t t) {
  // rows times parts, and no less than for any smaller t: the parts fall as one over the tiles of 16 rows
  const uint64_t most = std::max<uint64_t>(t, std::min<uint64_t>(kShrinkGroups * 16, static_cast<uint64_t>(t) * shrink_splits(1, n)));
  return most * num_targets * rank * sizeof(float);
}

hipError_t launch_adapter_apply(hipStream_t s, AdapterArgs a, bool y_f32) {
  a.splits = shrink_splits(a.t, a.n);
  const bool planned = a.plan.tiles != nullptr;
  const bool wide = planned ? a.plan.tile_rows == 64 : a.t > 256;  // 32 rows a workgroup instead of 16
  const uint32_t rows = wide ? 32 : 16;
  const uint32_t tiles = std::max((a.t + rows - 1) / rows, planned ? a.plan.most_tiles * (a.plan.tile_rows / rows) : 0);
  // consecutive rows of a short batch: the adapters of a tile side by side
  const uint32_t turns = planned || tiles > 4 ? 1 : std::min({a.t, a.num_adapters, 16u});
  if (wide) launch_shrink<2>(s, a, tiles, turns);
  else launch_shrink<1>(s, a, tiles, turns);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (wide) return y_f32 ? launch_expand<2, true>(s, a, tiles, turns) : launch_expand<2, false>(s, a, tiles, turns);
  return y_f32 ? launch_expand<1, true>(s, a, tiles, turns) : launch_expand<1, false>(s, a, tiles, turns);
}

}  // namespace mf
