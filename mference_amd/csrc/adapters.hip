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
// window of the row length; its four waves take 64 elements (a line of 128 bytes) in turn and add their sums through LDS.  A rank
// beyond the adapter's, and a row of another one, is a column or a row of the product that nobody reads.
template <int RT, int CF>
__global__ __launch_bounds__(256) void adapter_shrink_kernel(const AdapterArgs a) {
  __shared__ f32x4_t part[4][RT * CF][64];
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
        const uint32_t at = (u + k / 2 * 4) * 64 + k % 2 * 32;
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
    for (; u + 4 < u1; u += 8) step(std::integral_constant<int, 2>{}, u);
    if (u < u1) step(std::integral_constant<int, 1>{}, u);
    __syncthreads();  // (the parts of the adapter before have been read)
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < CF; ++c) part[wave][r * CF + c][lane] = acc[r][c];
    __syncthreads();
    const float scale = a.scales ? a.scales[adapter] : 1.0f;
    for (uint32_t f = wave; f < RT * CF; f += 4) {
      const f32x4_t sum = (part[0][f][lane] + part[1][f][lane]) + (part[2][f][lane] + part[3][f][lane]);
      const uint32_t cb = group * CF + f % CF, target = cb / blocks, r = cb % blocks * 16 + (lane & 15);
      const uint32_t row0 = f / CF * 16 + (lane >> 4) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t row = __shfl(meeting.row, row0 + i);
        if (target < a.num_targets && r < rank && ((lanes >> (row0 + i)) & 1))
          a.v[(static_cast<size_t>(split) * a.t + row) * a.cols + target * a.rank + r] = sum[i] * scale;
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

template <int RT, bool F32>
__global__ __launch_bounds__(256) void adapter_expand_kernel(const AdapterArgs a) {
  constexpr int kTerms = F32 ? 3 : 2, kPer = F32 ? 4 : 8, kChunks = 16 / kPer;  // results to 16 bytes; such pieces a lane holds of a row
  using Elem = std::conditional_t<F32, float, uint16_t>;
  const uint32_t lane = threadIdx.x & 63, q = lane >> 4;
  uint32_t block = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), target = 0;
  while (target < a.num_targets && block >= (a.target[target].m + 63) / 64) block -= (a.target[target++].m + 63) / 64;
  if (target >= a.num_targets) return;
  const AdapterArgs::Target tg = a.target[target];
  const uint32_t m0 = block * 64;
  Meeting<RT * 16> meeting(a, blockIdx.y, lane);
  uint32_t adapter, lead;
  uint64_t lanes;
  for (uint32_t turn = 0; meeting.next(adapter, lanes, lead); ++turn) {
    if (turn % gridDim.z != blockIdx.z) continue;
    const uint32_t rank = live_rank(a, adapter);
    Elem* yp[RT];
    const float* vp[RT];
    uint4 yv[RT][kChunks];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const uint32_t at = r * 16 + (lane & 15);
      const bool mine = (lanes >> at) & 1;
      const uint32_t row = __shfl(meeting.row, mine ? at : lead);
      vp[r] = a.v + static_cast<size_t>(row) * a.cols + target * a.rank;
      yp[r] = static_cast<Elem*>(tg.y) + static_cast<size_t>(row) * tg.y_stride;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const uint32_t m = m0 + c * 4 * kPer + q * kPer;
        if (mine && m + kPer <= tg.m) yv[r][c] = load_16_bytes(yp[r] + m);
      }
    }
    f32x4_t acc[RT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[r][j] = f32x4_t{0, 0, 0, 0};
    for (uint32_t k0 = 0; k0 < rank; k0 += 32) {
      const uint32_t k = k0 + q * 8, have = k < rank ? min(rank - k, 8u) : 0;
      uint4 bv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t p = lane & 15;
        const uint32_t m = m0 + (F32 ? 16 * j + p : 32 * (j >> 1) + 8 * (p >> 2) + 4 * (j & 1) + (p & 3));
        bv[j] = make_uint4(0, 0, 0, 0);
        if (have) bv[j] = *reinterpret_cast<const uint4*>(tg.b + (static_cast<size_t>(adapter) * tg.m + min(m, tg.m - 1)) * a.rank + k);
        if (have < 8) bv[j] = keep_bf16(bv[j], have);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (have) {
          for (uint32_t s = 0; s < a.splits; ++s) {
            const float4* p = reinterpret_cast<const float4*>(vp[r] + static_cast<size_t>(s) * a.t * a.cols + k);
            const float4 lo = p[0], hi = p[1];
            v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
            v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = static_cast<uint32_t>(e) < have ? v[e] : 0.0f;
        uint4 terms[kTerms];
        split_terms<kTerms>(v, terms);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int s = kTerms - 1; s >= 0; --s) acc[r][j] = mfma16(bv[j], terms[s], acc[r][j]);  // the small ones first
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if (!((lanes >> (r * 16 + (lane & 15))) & 1)) continue;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const uint32_t m = m0 + c * 4 * kPer + q * kPer;
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
  }
}

// Parts of the sum over n: as many as give the chip a workgroup a CU or two, but at least four units of 64 elements a part, and few
// where there are many rows (every part of v is written and read again).
uint32_t shrink_splits(uint32_t t, uint32_t n) {
  const uint32_t tiles = (t + 15) / 16, units = n / 64;
  return std::max(1u, std::min({512u / tiles, units / 4, 32u}));
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
  // rows times parts, and no less than for any smaller t: parts fall as 512 / (t / 16)
  const uint64_t most = std::max<uint64_t>(t, std::min<uint64_t>(512 * 16, static_cast<uint64_t>(t) * shrink_splits(1, n)));
  return most * num_targets * rank * sizeof(float);
}

hipError_t launch_adapter_apply(hipStream_t s, AdapterArgs a, bool y_f32) {
  constexpr int kCols = 4;
  a.splits = shrink_splits(a.t, a.n);
  const uint32_t col_blocks = (a.rank + 15) / 16 * a.num_targets, groups = (col_blocks + kCols - 1) / kCols;
  const bool planned = a.plan.tiles != nullptr;
  // consecutive rows: several adapters of a tile at once where a batch has few tiles
  const uint32_t tiles16 = std::max((a.t + 15) / 16, planned ? a.plan.most_tiles * (a.plan.tile_rows / 16) : 0);
  const uint32_t turns = planned ? 1 : std::min({a.t, a.num_adapters, tiles16 > 16 ? 2u : 16u});
  adapter_shrink_kernel<1, kCols><<<dim3(tiles16, groups * a.splits, turns), dim3(256), 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  uint32_t blocks = 0;
  for (uint32_t k = 0; k < a.num_targets; ++k) blocks += (a.target[k].m + 63) / 64;
  const uint32_t wide = planned ? a.plan.tile_rows == 64 : a.t > 256;
  if (wide) {
    const dim3 grid((blocks + 3) / 4, std::max((a.t + 63) / 64, planned ? a.plan.most_tiles : 0), turns);
    if (y_f32) adapter_expand_kernel<4, true><<<grid, dim3(256), 0, s>>>(a);
    else adapter_expand_kernel<4, false><<<grid, dim3(256), 0, s>>>(a);
  } else {
    const dim3 grid((blocks + 3) / 4, tiles16, turns);
    if (y_f32) adapter_expand_kernel<1, true><<<grid, dim3(256), 0, s>>>(a);
    else adapter_expand_kernel<1, false><<<grid, dim3(256), 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace mf
