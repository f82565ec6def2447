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

  __device__ __forceinline__ void find(const int32_t* __restrict__ ids, uint32_t first, uint32_t t, uint32_t n, uint16_t* counts) {
    const uint32_t lane = threadIdx.x & 63, bits = 32 - __builtin_clz(n);
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const uint32_t i = first + k * 64 + lane;
      key[k] = i < t ? adapter_key(ids[i], n) : n;
    }
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const bool valid = first + k * 64 + lane < t;
      uint64_t same = __ballot(valid);
      for (uint32_t b = 0; b < bits; ++b) {
        const bool set = (key[k] >> b) & 1;
        const uint64_t with = __ballot(set);
        same &= set ? with : ~with;
      }
      const uint32_t in_front = lanes_in_front(same);
      if (valid) {
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
// the lists of adapters and tiles are dealt out over the workgroups.  A batch of one run needs no counting launch in front: up to 4096
// rows, where one workgroup's turns still cost less than a second launch.  Four bytes a row are read and written: what it takes is latency (ids,
// ballots, two scans, scattered stores): 200 rows 2.8 us, 16384 rows 3.7 + 6.8 us.  Calls of the simple form (a thread an adapter that
// reads all rows) took 27 and 1829 us.
constexpr uint32_t kOwnTiles = 4;

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
        for (uint32_t r = 0; r < gridDim.x; r += 16) {  // sixteen requested at once
          uint32_t c[16];
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) c[i] = plan.runs[static_cast<size_t>(min(r + i, gridDim.x - 1)) * keys + k];
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) {
            before += r + i < blockIdx.x ? c[i] : 0;
            total.x += r + i < gridDim.x ? c[i] : 0;
          }
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
        for (uint32_t i = 0; i < min(total.y, kOwnTiles); ++i) plan.tiles[at.y + i] = plan.tile(k, at.x, total.x, i);
      }
    }
    // an adapter with many rows: its wave deals out its tiles (16384 rows of one adapter 13.9 -> 6.2 us)
    for (uint64_t many = __ballot(k < n && k % gridDim.x == blockIdx.x && total.y > kOwnTiles); many; many &= many - 1) {
      const int of = __builtin_ctzll(many);
      const uint32_t key = __shfl(k, of), x = __shfl(at.x, of), y = __shfl(at.y, of), rows = __shfl(total.x, of), tiles = __shfl(total.y, of);
      for (uint32_t i = kOwnTiles + (threadIdx.x & 63); i < tiles; i += 64) plan.tiles[y + i] = plan.tile(key, x, rows, i);
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
      const uint32_t row = first + i * 64 + (threadIdx.x & 63);
      if (row < t) plan.rows[starts[mine.key[i]] + counts[wave * keys + mine.key[i]] + mine.rank[i]] = row;
    }
  }
}

// ------------------------------------------------------------------ which rows meet which adapter

// (a number below zero, for callers whose tables are signed, is no rank)
__device__ __forceinline__ uint32_t live_rank(const AdapterArgs& a, uint32_t adapter) {
  return a.ranks ? static_cast<uint32_t>(max(0, min(static_cast<int>(a.ranks[adapter]), static_cast<int>(a.rank)))) : a.rank;
}

// ROWS rows of the batch, a lane each (ROWS <= 32; the lanes behind hold none), and the adapters that they meet.  With a plan they are
// (a part of) one of its tiles, of one adapter; without one they are consecutive rows, whose adapters are taken one after the other in
// the order of their first rows.  Every wave finds them for itself.
template <int ROWS>
struct Meeting {
  static_assert(ROWS <= 32, "the lanes' bits are a word");
  uint32_t row;    // this lane's
  uint32_t key;    // its adapter, num_adapters where it has no row or no adapter
  // Lanes whose adapter is still to come.  A word: a 64-bit shift by a register reads a second one behind it, and where the amount lay in
  // the last register of a wave some lanes got a wrong mask and took another row's x.
  uint32_t left;

  __device__ __forceinline__ Meeting(const AdapterArgs& a, uint32_t tile, uint32_t lane) : row(0), key(a.num_adapters) {
    bool planned = false;
    uint4 head = make_uint4(0, 0, 0, 0);
    uint2 rec = make_uint2(0, 0);
    uint32_t of = 0, from = 0;
    if (a.plan.tiles) {
      const uint32_t parts = a.plan.tile_rows / ROWS;
      of = tile / parts, from = tile % parts * ROWS;
      head = *reinterpret_cast<const uint4*>(a.plan.header);
      rec = a.plan.tiles[min(of, a.plan.most_tiles - 1)];
      planned = head.x == a.t && head.y == a.num_adapters;  // (what another batch left is not used)
    }
    if (planned) {
      const uint32_t count = rec.x >> 16, at = rec.y + from + lane;
      if (of < min(head.z, a.plan.most_tiles) && lane < ROWS && from + lane < count && at < a.t) {
        row = a.plan.rows[at];
        if (row < a.t) key = min(rec.x & 0xFFFFu, a.num_adapters);
        else row = 0;
      }
    } else {
      const uint32_t r = tile * ROWS + lane;
      if (lane < ROWS && r < a.t) {
        row = r;
        key = adapter_key(a.ids[r], a.num_adapters);
      }
    }
    left = static_cast<uint32_t>(__ballot(key < a.num_adapters));
  }
  // the next adapter, and the lanes that have it; false when there is none left
  __device__ __forceinline__ bool next(uint32_t& adapter, uint32_t& lanes, uint32_t& lead) {
    if (!left) return false;
    lead = static_cast<uint32_t>(__builtin_ctz(left));
    adapter = __builtin_amdgcn_readlane(key, lead);
    lanes = static_cast<uint32_t>(__ballot(key == adapter));
    left &= ~lanes;
    return true;
  }
};

__device__ __forceinline__ f32x4_t mfma16(const uint4& a, const uint4& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// ------------------------------------------------------------------ v = c A x
//
// v_mfma_f32_16x16x32_bf16 wants eight consecutive elements of a row a lane, and neighbouring lanes on different rows.  Loaded that
// way a request touches 64 lines of memory for its 1024 bytes; so eight lanes take a line of 128 bytes, and the operands come from
// LDS, where every wave has a place of its own: no barrier.  The 16-byte pieces of a row lie there exclusive-ored with the row's
// number, so that neither side meets a bank twice.  A rank beyond the adapter's, and a row of another one, is a column or a row of
// the product that nobody reads.
constexpr int kWaves = 8;

// What a wave stages at once: 64 elements of RT * 16 rows of x and of CF * 16 rows of A
template <int RT, int CF>
struct Stage {
  static constexpr int kLoads = 2 * (RT + CF), kBytes = kLoads * 1024;
  const uint16_t* x[2 * RT];  // the lane's row of each request, its piece of the line included
  const uint16_t* w[CF];      // the adapter's rows of each block of 16 ranks
  uint32_t in_w[CF][2];       // the lane's place there
  uint32_t used;              // bit i: one of the rows of x of request i is the adapter's (the others need not be there)

  __device__ __forceinline__ void rows_of_x(const AdapterArgs& a, uint32_t my_row, uint32_t lanes, uint32_t lead) {
    const uint32_t lane = threadIdx.x & 63, piece = (lane & 7) ^ (lane >> 3);
    used = 0;
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) {
      used |= (lanes >> (i * 8)) & 0xFFu ? 1u << i : 0u;
      const uint32_t at = i * 8 + (lane >> 3);
      const uint32_t row = __shfl(my_row, (lanes >> at) & 1 ? at : lead);
      x[i] = a.x + static_cast<size_t>(row) * a.x_stride + piece * 8;
    }
  }
  // block c of 16 ranks: from rank `first` on of the adapter's A, of which `have` exist
  __device__ __forceinline__ void rows_of_a(int c, const uint16_t* adapter, uint32_t n, uint32_t first, uint32_t have) {
    const uint32_t lane = threadIdx.x & 63, piece = (lane & 7) ^ (lane >> 3);
    w[c] = first < have ? adapter + static_cast<size_t>(first) * n : adapter;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t r = i * 8 + (lane >> 3);
      in_w[c][i] = (first + r < have ? r * n : 0) + piece * 8;
    }
  }

  // The wave's part of the products over the units of 64 elements from u0 to u1, WAVES apart, left in `part` [block][lane].  It
  // requests UNITS of them before it uses the first.  place: kBytes of LDS.
  template <int WAVES, int UNITS>
  __device__ __forceinline__ void multiply(uint32_t u0, uint32_t u1, uint4* place, f32x4_t* part) const {
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f32x4_t acc[RT][CF];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < CF; ++c) acc[r][c] = f32x4_t{0, 0, 0, 0};
    for (uint32_t u = u0 + wave; u < u1; u += UNITS * WAVES) {
      uint4 v[UNITS][kLoads];
#pragma unroll
      for (int k = 0; k < UNITS; ++k) {
        if (u + k * WAVES >= u1) break;
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i)
          if (used >> i & 1) v[k][i] = load_16_bytes(x[i] + (u + k * WAVES) * 64);
#pragma unroll
        for (int i = 0; i < 2 * CF; ++i) v[k][2 * RT + i] = *reinterpret_cast<const uint4*>(w[i / 2] + (u + k * WAVES) * 64 + in_w[i / 2][i % 2]);
      }
      issue_fence();
#pragma unroll
      for (int k = 0; k < UNITS; ++k) {
        if (u + k * WAVES >= u1) break;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          if (i >= 2 * RT || (used >> i & 1)) place[i * 64 + lane] = v[k][i];
        lane_order();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t at = (lane & 15) * 8 + ((h * 4 + (lane >> 4)) ^ (lane & 7));
          uint4 xo[RT], wo[CF];
#pragma unroll
          for (int r = 0; r < RT; ++r) xo[r] = place[r * 128 + at];
#pragma unroll
          for (int c = 0; c < CF; ++c) wo[c] = place[(RT + c) * 128 + at];
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int c = 0; c < CF; ++c) acc[r][c] = mfma16(wo[c], xo[r], acc[r][c]);
        }
        lane_order();
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < CF; ++c) part[(r * CF + c) * 64 + lane] = acc[r][c];
  }
  // other lanes' LDS stores in front of this come before this lane's loads behind it (a wave's LDS instructions run in order)
  static __device__ __forceinline__ void lane_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
};

// the waves' parts of four sums, `apart` from each other
template <int WAVES>
__device__ __forceinline__ f32x4_t add_parts(const f32x4_t* part, uint32_t apart) {
  f32x4_t sum[WAVES];
#pragma unroll
  for (int w = 0; w < WAVES; ++w) sum[w] = part[w * apart];
#pragma unroll
  for (int by = 1; by < WAVES; by *= 2)
#pragma unroll
    for (int w = 0; w < WAVES; w += 2 * by) sum[w] += sum[w + by];
  return sum[0];
}

// units requested at once: what 128 registers a lane hold
template <int RT, int CF> constexpr int kUnitsAhead = 6 - RT - CF;

// The first of two launches: v to memory, in parts over n.  It reads x once for every RT * 16 rows and two blocks of ranks, and those
// rows of A; matrix instructions are a few percent of its time.  Bound by the loads' latency: a wave has two to four
// units in flight and often no more than three turns.  777 rows of 4096, rank 64, two targets: 12.4 us, 14.5 MB from memory; 4096 rows of
// 5120, rank 16, two targets: 18.9 us, 45.6 MB = 2.4 TB/s; eight rows of 17408, rank 16: 5.6 us.
// The simple form of both launches (a dot product a wave, a result a thread) took 932 and 4263 us for the two prompts.
template <int RT, int CF>
__global__ __launch_bounds__(kWaves * 64, 4) void adapter_shrink_kernel(const AdapterArgs a) {
  using S = Stage<RT, CF>;
  __shared__ uint4 places[kWaves * S::kBytes / 16];  // a wave's place holds its part of the sums when it is done
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint4* place = places + wave * (S::kBytes / 16);
  // Parts side by side: with eight of them (or their multiples) every XCD has a window of x and A of its own.  The groups of ranks that
  // read the same part of x are on one XCD too, and run together.
  // (3875 rows of 11392, rank 64, two targets: 54 -> 46 us)
  const uint32_t blocks = (a.rank + 15) / 16;  // of 16 ranks, a target
  const uint32_t groups = (blocks * a.num_targets + CF - 1) / CF;
  const uint32_t pair = blockIdx.x / 8 / groups * 8 + blockIdx.x % 8, group = blockIdx.x / 8 % groups, split = pair % a.splits;
  const uint32_t units = a.n / 64, u0 = units * split / a.splits, u1 = units * (split + 1) / a.splits;
  Meeting<RT * 16> meeting(a, pair / a.splits, lane);  // (none behind the last pair)
  uint32_t adapter, lanes, lead;
  for (uint32_t turn = 0; meeting.next(adapter, lanes, lead); ++turn) {
    if (turn % gridDim.z != blockIdx.z) continue;
    const uint32_t rank = live_rank(a, adapter);
    const float scale = a.scales ? a.scales[adapter] : 1.0f;
    S stage;
    stage.rows_of_x(a, meeting.row, lanes, lead);
    bool any = false;
#pragma unroll
    for (int c = 0; c < CF; ++c) {
      const uint32_t cb = group * CF + c, target = cb / blocks, first = cb % blocks * 16;
      const bool live = target < a.num_targets && first < rank;
      any |= live;
      stage.rows_of_a(c, a.target[live ? target : 0].a + static_cast<size_t>(adapter) * a.rank * a.n, a.n, first, live ? rank : 0);
    }
    if (!any) continue;
    __syncthreads();  // (the parts of the adapter before have been read)
    stage.template multiply<kWaves, kUnitsAhead<RT, CF>>(u0, u1, place, reinterpret_cast<f32x4_t*>(place));
    __syncthreads();
    for (uint32_t f = wave; f < RT * CF; f += kWaves) {
      const f32x4_t sum = add_parts<kWaves>(reinterpret_cast<f32x4_t*>(places) + f * 64 + lane, S::kBytes / 16) * scale;
      const uint32_t cb = group * CF + f % CF, target = cb / blocks, r = cb % blocks * 16 + (lane >> 4) * 4;
      const uint32_t at = f / CF * 16 + (lane & 15), row = __shfl(meeting.row, at);
      if (target < a.num_targets && r < rank && ((lanes >> at) & 1))  // (four ranks: rank of the pool is a multiple of eight)
        *reinterpret_cast<f32x4_t*>(a.v + (static_cast<size_t>(split) * a.t + row) * a.cols + target * a.rank + r) = sum;
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

// A workgroup's share of the results of one adapter's rows: its waves take 64 results in turn, the y and B of the next ones requested
// before the present ones are worked on.  DEEP: B of the next 32 ranks in their place, and y no earlier than its results' first B; that is for
// fp32 results of 32 rows, whose y takes most registers, and ranks past 32 (2000 rows, two times 4096, rank 48 43 -> 36 us, 64 45 -> 41, 128 62 -> 57;
// bf16 results 55 -> 57, fp32 ones of 16 rows 11.2 -> 12.3, of rank 16 251 -> 290).
template <int RT, bool F32, int WAVES, bool DEEP>
struct Expand {
  static constexpr int kTerms = F32 ? 3 : 2, kPer = F32 ? 4 : 8, kChunks = 16 / kPer;  // results to 16 bytes; such pieces a lane holds of a row
  using Elem = std::conditional_t<F32, float, uint16_t>;

  const uint16_t* bp;
  uint32_t m, rank_of_pool, q, in_b[4];  // in_b: the lane's elements of a block of 64 rows of B
  Elem* yp[RT];
  bool mine[RT];
  uint4 yv[RT][kChunks], bv[4];

  __device__ __forceinline__ void load_y(uint32_t block, uint4 (&v)[RT][kChunks]) const {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const uint32_t at = block * 64 + c * 4 * kPer + q * kPer;
        if (mine[r] && at + kPer <= m) v[r][c] = load_16_bytes(yp[r] + at);
      }
  }
  static __device__ __forceinline__ uint32_t row_of_b(int j, uint32_t p) { return F32 ? 16 * j + p : 32 * (j >> 1) + 8 * (p >> 2) + 4 * (j & 1) + (p & 3); }
  __device__ __forceinline__ void load_b(uint32_t block, uint32_t k0, uint4 (&v)[4]) const {
    const uint16_t* base = bp + static_cast<size_t>(block) * 64 * rank_of_pool + k0;
    const uint32_t rows = m - block * 64;
    if (k0 + q * 8 >= rank_of_pool) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t in = in_b[j];
      if (rows < 64) in = min(row_of_b(j, threadIdx.x & 15), rows - 1) * rank_of_pool + q * 8;
      v[j] = *reinterpret_cast<const uint4*>(base + in);
    }
  }
  // requests the wave's first results
  __device__ __forceinline__ Expand(const AdapterArgs& a, const AdapterArgs::Target& tg, uint32_t adapter, uint32_t my_row, uint32_t lanes,
                                    uint32_t lead, uint32_t block, uint32_t end) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t p = lane & 15;
    q = lane >> 4;
    m = tg.m, rank_of_pool = a.rank;
#pragma unroll
    for (int j = 0; j < 4; ++j) in_b[j] = row_of_b(j, p) * a.rank + q * 8;
    bp = tg.b + static_cast<size_t>(adapter) * m * a.rank;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const uint32_t at = r * 16 + p;
      mine[r] = (lanes >> at) & 1;
      yp[r] = static_cast<Elem*>(tg.y) + static_cast<size_t>(__shfl(my_row, mine[r] ? at : lead)) * tg.y_stride;
    }
    if (block < end) {
      if constexpr (!DEEP) load_y(block, yv);
      load_b(block, 0, bv);
    }
  }
  // operand: [32 ranks][RT][kTerms][lane], the terms of v
  __device__ __forceinline__ void run(uint32_t block, uint32_t end, uint32_t rank, const uint4* operand) {
    const uint32_t lane = threadIdx.x & 63, kb = (rank + 31) / 32;
    for (; block < end; block += WAVES) {
      [[maybe_unused]] uint4 next_y[RT][kChunks];
      uint4 next_b[4];
      if constexpr (DEEP) {
        load_y(block, yv);
      } else if (block + WAVES < end) {
        load_y(block + WAVES, next_y);
        load_b(block + WAVES, 0, next_b);
      }
      f32x4_t acc[RT][4];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[r][j] = f32x4_t{0, 0, 0, 0};
      for (uint32_t b = 0; b < kb; ++b) {
        const uint32_t k = b * 32 + q * 8, have = k < rank ? min(rank - k, 8u) : 0;
        if constexpr (DEEP) {
          const bool more = b + 1 < kb;
          if (more || block + WAVES < end) load_b(more ? block : block + WAVES, more ? b * 32 + 32 : 0, next_b);
        } else {
          if (b) load_b(block, b * 32, bv);
        }
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
        if constexpr (DEEP) {
#pragma unroll
          for (int j = 0; j < 4; ++j) bv[j] = next_b[j];
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (!mine[r]) continue;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint32_t at = block * 64 + c * 4 * kPer + q * kPer;
          float add[kPer];
#pragma unroll
          for (int e = 0; e < kPer; ++e) add[e] = acc[r][F32 ? c : 2 * c + e / 4][e % 4];
          if (at + kPer <= m) {
            uint32_t w[4] = {yv[r][c].x, yv[r][c].y, yv[r][c].z, yv[r][c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (F32) w[e] = __float_as_uint(__uint_as_float(w[e]) + add[e]);
              else w[e] = static_cast<uint32_t>(narrow_bf16(bf16_lo(w[e]) + add[2 * e])) | static_cast<uint32_t>(narrow_bf16(bf16_hi(w[e]) + add[2 * e + 1])) << 16;
            }
            __builtin_memcpy(yp[r] + at, w, 16);
          } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
              if (at + e >= m) continue;
              if constexpr (F32) yp[r][at + e] += add[e];
              else yp[r][at + e] = narrow_bf16(bf16_to_f(yp[r][at + e]) + add[e]);
            }
          }
        }
      }
      if constexpr (!DEEP) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int c = 0; c < kChunks; ++c) yv[r][c] = next_y[r][c];
#pragma unroll
        for (int j = 0; j < 4; ++j) bv[j] = next_b[j];
      }
    }
  }
};

// Slot `slot` of the operand: eight ranks (k on) of the tile's row `at`
template <int RT>
__device__ __forceinline__ void place_of_slot(uint32_t slot, uint32_t& at, uint32_t& k) {
  at = slot / 64 % RT * 16 + (slot & 15);
  k = slot / (64 * RT) * 32 + (slot >> 4) % 4 * 8;
}
template <int RT, int TERMS>
__device__ __forceinline__ void store_terms(uint4* operand, uint32_t slot, const float (&v)[8]) {
  uint4 terms[TERMS];
  split_terms<TERMS>(v, terms);
#pragma unroll
  for (int i = 0; i < TERMS; ++i) operand[(slot / 64 * TERMS + i) * 64 + (slot & 63)] = terms[i];
}

// which target, and which of its blocks of 64 results, a workgroup has
struct Share {
  uint32_t target, first, end;
  __device__ __forceinline__ Share(const AdapterArgs& a, uint32_t run) : target(0) {
    while (run >= a.first_run[target + 1]) ++target;
    first = (run - a.first_run[target]) * a.run_blocks;
    end = min((a.target[target].m + 63) / 64, first + a.run_blocks);
  }
};

// The second of two launches.  A workgroup takes RT * 16 rows and a run of a target's results, and adds up the parts of v itself: a
// third launch that did would cost more.  Long batches are bound by y, which is read and written once: 4096 rows, rank 16, two times 17408,
// 138 us, 345 MB read and 285 written = 4.6 TB/s, where a copy reaches 4.8.  Short ones are bound by a chain of requests (rows and
// adapters 1.1 us, parts of v 2.9, products and y 1.8): 777 rows, rank 64, two times 2048, 11.3 us; eight rows, 5120 in fp32, 6.6 us.  Tried: eight
// waves (no gain), y past the caches (no gain), whole lines of y in 8-byte pieces (199 us where it took 146), a wave's results one behind the
// other (rows that start inside a line 108 -> 126 us).  Such rows cost: two times 13992 (16-byte places) 108 us where whole lines would take 85,
// 13999 (2-byte places) 152.
constexpr uint32_t kExpandWaves = 4;

template <int RT, bool F32, bool DEEP>
__global__ __launch_bounds__(kExpandWaves * 64) void adapter_expand_kernel(const AdapterArgs a) {
  extern __shared__ uint4 operand[];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Share share(a, blockIdx.x);
  const AdapterArgs::Target tg = a.target[share.target];
  Meeting<RT * 16> meeting(a, blockIdx.y, lane);
  uint32_t adapter, lanes, lead;
  for (uint32_t turn = 0; meeting.next(adapter, lanes, lead); ++turn) {
    if (turn % gridDim.z != blockIdx.z) continue;
    Expand<RT, F32, kExpandWaves, DEEP> expand(a, tg, adapter, meeting.row, lanes, lead, share.first + wave, share.end);
    const uint32_t rank = live_rank(a, adapter);
    __syncthreads();  // (the operands of the adapter before have been read)
    for (uint32_t slot = threadIdx.x; slot < (rank + 31) / 32 * RT * 64; slot += kExpandWaves * 64) {
      uint32_t at, k;
      place_of_slot<RT>(slot, at, k);
      const uint32_t have = k < rank ? min(rank - k, 8u) : 0, row = __shfl(meeting.row, at);
      float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (have && ((lanes >> at) & 1)) {
        const float* p = a.v + static_cast<size_t>(row) * a.cols + share.target * a.rank + k;
        const size_t part = static_cast<size_t>(a.t) * a.cols;
        constexpr uint32_t kAhead = RT == 1 ? 8 : 4;  // parts requested at once
        for (uint32_t s = 0; s < a.splits; s += kAhead) {
          float4 lo[kAhead], hi[kAhead];
#pragma unroll
          for (uint32_t i = 0; i < kAhead; ++i) {
            const float4* w = reinterpret_cast<const float4*>(p + min(s + i, a.splits - 1) * part);
            lo[i] = w[0], hi[i] = w[1];
          }
#pragma unroll
          for (uint32_t i = 0; i < kAhead; ++i) {
            if (s + i >= a.splits) continue;
            v[0] += lo[i].x, v[1] += lo[i].y, v[2] += lo[i].z, v[3] += lo[i].w;
            v[4] += hi[i].x, v[5] += hi[i].y, v[6] += hi[i].z, v[7] += hi[i].w;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = static_cast<uint32_t>(e) < have ? v[e] : 0.0f;
      store_terms<RT, Expand<RT, F32, kExpandWaves, DEEP>::kTerms>(operand, slot, v);
    }
    __syncthreads();
    if (rank) expand.run(share.first + wave, share.end, rank, operand);
  }
}

// ------------------------------------------------------------------ both in one launch
//
// Every workgroup makes the v of its rows and its target for itself, over the whole of n, and goes on to its results: nothing goes
// through memory in between, and there is no second launch.  Workgroups that share rows make the same v, on compute units that
// would have nothing else to do.  One row of 2048, rank 16, two times 512: 5.5 us (ids 0.8, addresses 0.7, the loop over n 1.3, the
// waves' sums 1.0, results 0.8; the rest starts and ends the launch).  Four rows of 5120, rank 32, two times 17408: 10.4 us, of which 4.2 are
// the loop, which draws 410 KB of x and A through a CU's L1, 40 bytes a clock of 64.  200 mixed rows of 2816, rank 24, two
// times 2112: 11.5 us, 25 MB from memory.  Sixteen waves, and more units in flight, were no gain.
//
// Two workgroups a CU need 128 registers a lane: bf16 results and ranks up to 16 fit them with two units in flight instead of four (2169 rows,
// rank 8, two times 809, 21.2 -> 17.5 us; 3000 rows, rank 16, 27.4 -> 22.8; one row 5.6 -> 5.5).  The others would spill: fp32 8.9 -> 10.8 us
// on 700 rows, two blocks of ranks 11.9 -> 16.0 on 200.
template <int CF, bool F32> constexpr bool kTwoACu = CF == 1 && !F32;
template <int CF, bool F32>
__global__ __launch_bounds__(kWaves * 64, (kTwoACu<CF, F32> ? 4 : 2)) void adapter_fused_kernel(const AdapterArgs a) {
  constexpr int kTerms = F32 ? 3 : 2;
  using S = Stage<1, CF>;
  __shared__ uint4 lds[kWaves * S::kBytes / 16 + kTerms * 64];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint4* place = lds + wave * (S::kBytes / 16);  // the wave's; its part of the sums later on
  uint4* operand = lds + kWaves * (S::kBytes / 16);
  const uint32_t runs = a.first_run[a.num_targets];
  // workgroups of one tile share x and A: on one XCD where there are tiles for all of them (200 mixed rows of 2816, rank 24, two times
  // 2112: 14.3 -> 12.9 us, 1500 rows of 2048, rank 32, two times 2048: 21.2 -> 20.4)
  const uint32_t tile = a.by_xcd ? blockIdx.x / 8 / runs * 8 + blockIdx.x % 8 : blockIdx.x / runs;
  const Share share(a, (a.by_xcd ? blockIdx.x / 8 : blockIdx.x) % runs);
  const AdapterArgs::Target tg = a.target[share.target];
  Meeting<16> meeting(a, tile, lane);
  uint32_t adapter, lanes, lead;
  for (uint32_t turn = 0; meeting.next(adapter, lanes, lead); ++turn) {
    if (turn % gridDim.z != blockIdx.z) continue;
    S stage;
    stage.rows_of_x(a, meeting.row, lanes, lead);
    Expand<1, F32, kWaves, false> expand(a, tg, adapter, meeting.row, lanes, lead, share.first + wave, share.end);
#pragma unroll
    for (int c = 0; c < CF; ++c) stage.rows_of_a(c, tg.a + static_cast<size_t>(adapter) * a.rank * a.n, a.n, c * 16, a.rank);  // not waiting for its own rank
    if (turn) __syncthreads();  // (the parts of the adapter before have been read)
    stage.template multiply<kWaves, (kTwoACu<CF, F32> ? 2 : kUnitsAhead<1, CF>)>(0, a.n / 64, place, reinterpret_cast<f32x4_t*>(place));
    const uint32_t rank = live_rank(a, adapter);
    const float scale = a.scales ? a.scales[adapter] : 1.0f;
    __syncthreads();
    if (wave < CF) {  // a block of ranks a wave; a lane of the operand has eight of a row: its own four and those of the lane 16 behind
      const f32x4_t lo = add_parts<kWaves>(reinterpret_cast<f32x4_t*>(lds) + wave * 64 + lane, S::kBytes / 16) * scale;
      f32x4_t hi;
#pragma unroll
      for (int e = 0; e < 4; ++e) hi[e] = __shfl_down(lo[e], 16);
      const uint32_t k = wave * 16 + (lane >> 4) * 4;
      float v[8];
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) v[e] = k + e < rank ? (e < 4 ? lo[e] : hi[e - 4]) : 0.0f;
      if ((lane & 16) == 0) store_terms<1, kTerms>(operand, wave * 32 + (lane >> 5) * 16 + (lane & 15), v);
    }
    if (CF == 1 && wave == 1) {  // the ranks from 16 on: none
      const float none[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (lane >= 32) store_terms<1, kTerms>(operand, lane, none);
    }
    __syncthreads();
    if (rank) expand.run(share.first + wave, share.end, rank, operand);
  }
}

// Parts of the sum over n: for two workgroups a CU, of eight units of 64 elements (one a wave) or more; few of them where there are
// many rows, since every part of v is written and read again (777 rows of 4096, rank 64, two targets: four parts 11.6 + 13.4 us, five 12.7 +
// 14.5, eight 13.0 + 15.0), unless a workgroup has all ranks (2000 rows of 16384, rank 16, two times 1024: four 26.4 + 11.4 us, eight 18.7 + 13.0).
constexpr uint32_t kMostSplits = 16, kShrinkGroups = 512;
uint32_t shrink_splits(uint32_t t, uint32_t n, uint32_t blocks) {
  const bool all = t > 256 && blocks <= 2;
  // two units a wave where there is a workgroup a CU without any parts (2578 rows of 1600, rank 128, two targets: three parts 26.5 us, one 18.8)
  const uint32_t least = t > 256 && (t + 31) / 32 * ((blocks + 1) / 2) >= 256 ? 2 : 1;
  return std::max(1u, std::min({kShrinkGroups * (all ? 2 : 1) / ((t + 15) / 16), n / 64 / (kWaves * least), t <= 256 ? kMostSplits : all ? 8u : 4u}));
}

// deals the results of all targets to workgroups, `least` blocks of 64 or more each, and so many that there are no more than `most`
// workgroups; but fewer where less than `fill` would be left
void deal_results(AdapterArgs& a, uint32_t tiles, uint32_t least, uint32_t fill, uint32_t most, uint32_t waves) {
  uint64_t blocks = 0;
  for (uint32_t k = 0; k < a.num_targets; ++k) blocks += (a.target[k].m + 63) / 64;
  blocks *= tiles;
  a.run_blocks = static_cast<uint32_t>(std::max<uint64_t>((blocks + most - 1) / most, std::min<uint64_t>(least, (blocks + fill - 1) / fill)));
  a.run_blocks = (a.run_blocks + waves - 1) / waves * waves;
  a.first_run[0] = 0;
  for (uint32_t k = 0; k < MF_MAX_ADAPTER_TARGETS; ++k)
    a.first_run[k + 1] = k < a.num_targets ? a.first_run[k] + ((a.target[k].m + 63) / 64 + a.run_blocks - 1) / a.run_blocks : 0xFFFFFFFFu;
}

template <int RT>
hipError_t launch_shrink(hipStream_t s, const AdapterArgs& a, uint32_t tiles, uint32_t turns) {
  const uint32_t blocks = (a.rank + 15) / 16 * a.num_targets;
  const auto go = [&](auto cf) {
    constexpr int kCols = decltype(cf)::value;
    adapter_shrink_kernel<RT, kCols><<<dim3((tiles * a.splits + 7) / 8 * 8 * ((blocks + kCols - 1) / kCols), 1, turns), dim3(kWaves * 64), 0, s>>>(a);
  };
  if (blocks == 1) go(std::integral_constant<int, 1>{});
  else go(std::integral_constant<int, 2>{});
  return hipGetLastError();
}

template <int RT, bool F32>
hipError_t launch_expand(hipStream_t s, AdapterArgs& a, uint32_t tiles, uint32_t turns) {
  // Four blocks a wave pay for its start, if a few workgroups a CU remain (us a pass with one block a wave / so): 3875 rows, rank 64, two
  // times 4608, 63 / 52; 1402 rows, rank 32, two times 6251 in fp32, 47 / 38; 4096 rows, rank 16, two times 17408, 139 / 135 (six blocks: 144);
  // 62 rows, rank 16, two times 8256, 12 / 9; there 2048 workgroups were no gain.
  deal_results(a, tiles > 16 ? tiles : tiles * turns, 16, RT == 1 ? 1024 : 2048, 8192, kExpandWaves);
  constexpr uint32_t kBlock = RT * (F32 ? 3 : 2) * 1024;  // of 32 ranks
  static_assert(MF_MAX_ADAPTER_RANK / 32 * kBlock <= 48 * 1024, "what a launch may ask for without further ado");
  const uint32_t lds = (a.rank + 31) / 32 * kBlock;
  const dim3 grid(a.first_run[a.num_targets], tiles, turns), block(kExpandWaves * 64);
  if constexpr (RT == 2 && F32) {
    if (a.rank > 32) {
      adapter_expand_kernel<RT, F32, true><<<grid, block, lds, s>>>(a);
      return hipGetLastError();
    }
  }
  adapter_expand_kernel<RT, F32, false><<<grid, block, lds, s>>>(a);
  return hipGetLastError();
}

struct Tiling {
  uint32_t tiles, turns, shrink_turns, expand_turns;
  Tiling(const AdapterArgs& a, uint32_t rows) {
    const bool planned = a.plan.tiles != nullptr;
    tiles = std::max((a.t + rows - 1) / rows, planned ? a.plan.most_tiles * (a.plan.tile_rows / rows) : 0);
    // Consecutive rows of a short batch: the adapters of a tile side by side.  Us a pass, all of one tile's after one another / side by
    // side: 80 rows of several requests, one launch of rank 16, 2048 to two times 2048, 13.4 / 7.0, of one request 6.8 / 6.9, but 1000 rows
    // of one request 9.6 / 11.4; the second of two launches of rank 64, two times 4096, 80 rows 15.4 / 9.4 (one request 7.9 / 8.1), 777 rows, two
    // times 2048, 13.5 / 11.0 (9.5 / 9.8), 2000 rows 32.4 / 34.1.  The first of two launches has workgroups for its parts of n and groups of ranks
    // too: 1000 rows of 8192 (32 tiles of 32 rows) 12.7 / 11.1, 1402 rows 12.0 / 13.6, 200 rows of 5120 (13 tiles of 16) 10.2 / 13.4; 257 to 512 rows (9
    // to 16 tiles of 32) go either way and take one: 300 rows of 4096, rank 64, 9.6 / 8.4, 512 rows of 17408, rank 16, 14.1 / 9.4, of 4096, rank 64, 10.2 / 9.2,
    // rank 128 13.2 / 15.5.
    const auto at_once = [&](uint32_t most) { return planned ? 1 : std::min({a.t, a.num_adapters, most}); };
    turns = at_once(tiles <= 4 ? 16 : tiles <= 16 ? 4 : 1);
    shrink_turns = at_once(tiles <= 4 ? 16 : tiles > 16 && tiles <= 32 ? 2 : 1);
    expand_turns = at_once(tiles <= 4 ? 16 : tiles <= 16 ? 4 : tiles <= 48 ? 2 : 1);
  }
};

template <bool F32>
hipError_t launch_fused(hipStream_t s, AdapterArgs& a) {
  const Tiling g(a, 16);
  const uint32_t rows = g.tiles * g.turns, groups = std::max(1u, 256 / rows) * rows;  // one workgroup a CU, or one for all results of a tile
  deal_results(a, rows, 1, groups, groups, kWaves);
  a.by_xcd = g.tiles >= 32;
  const dim3 grid(a.first_run[a.num_targets] * (a.by_xcd ? (g.tiles + 7) / 8 * 8 : g.tiles), 1, g.turns), block(kWaves * 64);
  if (a.rank <= 16) adapter_fused_kernel<1, F32><<<grid, block, 0, s>>>(a);
  else adapter_fused_kernel<2, F32><<<grid, block, 0, s>>>(a);
  return hipGetLastError();
}

template <int RT, bool F32>
hipError_t launch_two(hipStream_t s, AdapterArgs& a) {
  const Tiling g(a, RT * 16);
  a.splits = shrink_splits(a.t, a.n, (a.rank + 15) / 16 * a.num_targets);
  const hipError_t e = launch_shrink<RT>(s, a, g.tiles, g.shrink_turns);
  return e != hipSuccess ? e : launch_expand<RT, F32>(s, a, g.tiles, g.expand_turns);
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
  const uint64_t most = std::max<uint64_t>(t, std::min<uint64_t>(kShrinkGroups * 2 * 16, static_cast<uint64_t>(t) * shrink_splits(1, n, 1)));
  return most * num_targets * rank * sizeof(float);
}

hipError_t launch_adapter_apply(hipStream_t s, AdapterArgs a, bool y_f32) {
  uint64_t results = 0;
  for (uint32_t k = 0; k < a.num_targets; ++k) results += a.target[k].m;
  results *= a.t;
  // One launch where v costs a workgroup little (two blocks of ranks, half a megabyte of x and A) and the results are not so many that
  // their streaming decides.  Us of one launch / of the two (which cost one more to start), two projections: one row of 2048, rank 16, 5.4 /
  // 8.8; of 5120, rank 32, 9.8 / 9.7; of 17408, rank 8, 14.5 / 10.4; eight rows of eight adapters, 5120, rank 16, 9.6 / 11.2; 1000 rows of
  // 17408, rank 16, 31.5 / 19.9; 2048 to 2048, rank 32, 2000 rows 21.7 / 26.6, 4000 rows 33.0 / 37.9; to 4096 (33 million results) 52.3 / 50.6;
  // 512 rows, 5120 to 17408 (18 million), 33.0 / 30.4.
  if (a.rank <= 32 && static_cast<uint64_t>(a.rank + 16) * a.n * sizeof(uint16_t) <= (512u << 10) && results <= (16u << 20))
    return y_f32 ? launch_fused<true>(s, a) : launch_fused<false>(s, a);
  const bool wide = a.plan.tiles ? a.plan.tile_rows == 64 : a.t > 256;  // 32 rows a workgroup instead of 16
  if (wide) return y_f32 ? launch_two<2, true>(s, a) : launch_two<2, false>(s, a);
  return y_f32 ? launch_two<1, true>(s, a) : launch_two<1, false>(s, a);
}

}  // namespace mf
