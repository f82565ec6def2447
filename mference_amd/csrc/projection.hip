// The projection of 16-bit weights with bias, activation and residual in its epilogue (mf_project).
#include <algorithm>
#include <type_traits>

#include "mf_dense16.h"
#include "mf_dense16_device.h"

namespace mf {

namespace {

// ------------------------------------------------------------------ epilogue

// four neighbouring values from p on, of which `have` exist (0 behind them); at any address (memory takes unaligned accesses)
__device__ __forceinline__ f32x4_t load4(const float* p, uint32_t have) {
  f32x4_t v = {};
  if (have >= 4) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 3; ++e)
      if (e < have) v[e] = p[e];
  }
  return v;
}
__device__ __forceinline__ f32x4_t load4(const uint16_t* p, uint32_t have) {
  uint32_t lo = 0, hi = 0;
  if (have >= 4) {
    __builtin_memcpy(&lo, p, 4);
    __builtin_memcpy(&hi, p + 2, 4);
  } else {
    lo = p[0] | (have > 1 ? static_cast<uint32_t>(p[1]) << 16 : 0u);
    hi = have > 2 ? p[2] : 0u;
  }
  return f32x4_t{bf16_lo(lo), bf16_hi(lo), bf16_lo(hi), bf16_hi(hi)};
}
__device__ __forceinline__ void store4(float* p, const f32x4_t& v, uint32_t have) {
  if (have >= 4) {
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 3; ++e)
      if (e < have) p[e] = v[e];
  }
}
__device__ __forceinline__ void store4(uint16_t* p, const f32x4_t& v, uint32_t have) {
  const uint2 w = make_uint2(narrow_bf16(v[0]) | static_cast<uint32_t>(narrow_bf16(v[1])) << 16, narrow_bf16(v[2]) | static_cast<uint32_t>(narrow_bf16(v[3])) << 16);
  if (have >= 4) {
    __builtin_memcpy(p, &w, 8);
  } else {
    p[0] = static_cast<uint16_t>(w.x);
    if (have > 1) p[1] = static_cast<uint16_t>(w.x >> 16);
    if (have > 2) p[2] = static_cast<uint16_t>(w.y);
  }
}

// Results j .. j + 3 of row i, those of them in front of `end`, from their sums (and, gated, from those of their up rows): one rounding, at the end.
template <bool GATED>
__device__ __forceinline__ void finish4(const mf_project_args& a, uint32_t i, uint32_t j, uint32_t end, f32x4_t z, f32x4_t up) {
  const uint32_t have = end - j;
  if (a.bias) {
    z += load4(a.bias + j, have);
    if (GATED) up += load4(a.bias + a.m + j, have);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    z[e] = activate(z[e], a.activation);
    if (GATED) z[e] *= up[e];
  }
  const size_t at = static_cast<size_t>(i) * a.y_stride + j, from = static_cast<size_t>(i) * a.residual_stride + j;
  if (a.y_f32) {
    if (a.residual) z += load4(static_cast<const float*>(a.residual) + from, have);
    store4(static_cast<float*>(a.y) + at, z, have);
  } else {
    if (a.residual) z += load4(static_cast<const uint16_t*>(a.residual) + from, have);
    store4(static_cast<uint16_t*>(a.y) + at, z, have);
  }
}

// ------------------------------------------------------------------ tiles

struct TileArgs {
  mf_project_args p;
  float* parts;          // several parts of the sum over n: [parts][t][rows], else null
  uint32_t part_blocks;  // blocks of 64 a part
  uint32_t part_count;
  uint32_t row_tiles, token_tiles;
};

// Workgroups are dealt to the eight XCDs in turn: each takes a range of the tiles of its own, and in it groups of eight token tiles side by side,
// so that what its CUs read at a time is in its L2 for the others (a part of the sum is a range of its own).
__device__ __forceinline__ void tile_of(const TileArgs& a, uint32_t id, uint32_t* row_tile, uint32_t* token_tile) {
  const uint32_t total = a.row_tiles * a.token_tiles, xcd = id % 8, each = total / 8, rest = total % 8;
  const uint32_t at = xcd * each + min(xcd, rest) + id / 8;
  const uint32_t group = at / (8 * a.row_tiles), first = group * 8, wide = min(a.token_tiles - first, 8u), in = at - group * 8 * a.row_tiles;
  *row_tile = in / wide;
  *token_tile = first + in % wide;
}

// the largest divisor of n that is no larger than `most`
constexpr int largest_part(int n, int most) {
  int part = most < n ? most : n;
  while (n % part) --part;
  return part;
}

// A workgroup TM tokens x TN rows of W (gated: TN / 2 gate rows and their up rows), WM x WN waves, sums in registers.  The operands go straight to LDS in blocks
// of 64 values of n, a whole line of 128 bytes a row at a time, STAGES - 1 blocks ahead.  A block is two steps of the matrix cores; a wave reads a step's operands into
// registers while the matrix cores work on the step before, so that a block costs one barrier and no wait for LDS.  The eight pieces of a row are turned by
// the row's number, so that 16 lanes that read the same piece of 16 rows meet all banks.  A workgroup starts at a block of its own (`skew`), so that neighbours do not wait
// for the same lines at once (3 %).  What bounds it is LDS, at 128 bytes a clock (119 measured): for a block of 128 x 192 the waves read 131 KB and the requests write 41, together
// 0.56 us at 2.4 GHz; a block takes 0.53, the matrix cores need 0.32 of them (777 rows 1280 -> 5120, bias and gelu: 24.0 us, of which 10 stand in front of the first block and
// behind the last and 3 are the bias and the gelu).  Of 256 x 256 LDS and the matrix cores need 0.85 us each of 1.5 (4096 rows 5120 -> 17408, gated: 1205 to 1225 us, 1.2 PFLOP/s; the library's
// product without the gate 1194 to 1275).  200 rows 2816 -> 2113, tiles of 32 x 64: 9.6 us, 22 blocks one behind the other in either half of n, 0.27 each, and 4 around them.  Waves of four or fewer (kSpread) deal their reads and
// requests out among the matrix instructions by hand; eight leave it to the scheduler's groups, as the order by hand would take registers that spill.
template <int TM, int TN, int WM, int WN, int KG, int STAGES, bool GATED, bool ALIGNED>
__global__ __launch_bounds__(64 * WM * WN * KG) void project_tile_kernel(const TileArgs t) {
  constexpr bool kSpread = WM * WN <= 4;
  constexpr int kWaves = WM * WN, kLoads = (TM + TN) / 8 / kWaves, MT = TM / WM / 16, NT = TN / WN / 16;
  constexpr int kStage = (TM + TN) * 128;  // bytes
  using At = std::conditional_t<ALIGNED, uint32_t, uint64_t>;
  static_assert(kLoads * kWaves * 8 == TM + TN && (!GATED || NT % 2 == 0), "tiles deal out evenly");
  extern __shared__ uint4 whole_lds[];
  const mf_project_args& a = t.p;
  const uint32_t tid = threadIdx.x, lane = tid & 63, group = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6) / kWaves, wave = __builtin_amdgcn_readfirstlane(tid >> 6) % kWaves;
  const uint32_t wm = wave / WN, wn = wave % WN;
  uint32_t row_tile, token_tile;
  tile_of(t, blockIdx.x, &row_tile, &token_tile);
  constexpr uint32_t kRows = GATED ? TN / 2 : TN, kHalf = TN / WN / 2;
  const uint32_t i0 = token_tile * TM, j0 = row_tile * kRows;
  // this workgroup's part of the sum, and in it its groups' shares
  const uint32_t part_from = blockIdx.y * t.part_blocks * 64, part_to = min(part_from + t.part_blocks * 64, a.n), blocks = ((part_to - part_from + 63) / 64 + KG - 1) / KG;
  const uint32_t from = min(part_from + group * blocks * 64, part_to), to = min(from + blocks * 64, part_to);

  const uint32_t full = __builtin_amdgcn_readfirstlane((to - from) / 64), rest = __builtin_amdgcn_readfirstlane((to - from) % 64);
  const uint32_t last = __builtin_amdgcn_readfirstlane(rest || !full ? full : full - 1);
  const uint32_t skew = __builtin_amdgcn_readfirstlane(min(blockIdx.x / 8 % 8, last));
  uint4* lds = whole_lds + group * (STAGES * kStage / 16);
  // A lane's pieces of a block: eight rows an instruction, eight lanes a row, from a uniform base and a lane's offset.  What lies behind the sum's end
  // is left out when it is multiplied: a lane that would read there reads the start of the last block again.
  const uint16_t* src[kLoads];
  const uint32_t piece = lane_piece(lane), back = piece >= rest ? piece * 2 : 0;  // (elements; bytes)
  // Eight rows from a uniform base with one offset a lane for all of them, but where rows end among the eight: rows behind the last are that row again (their results are
  // not stored).  Kept to so few registers because a spilled one, read back, waits for every block that is on its way: 256 x 256 has 9 to 11 in scratch all the same, of which every
  // second block reads six back right behind the next block's requests.
  const uint32_t x_edge = (min(a.t - i0, static_cast<uint32_t>(TM)) - 1) / 8 * 8, w_edge = (min(a.m - j0, kRows) - 1) / 8 * 8;
  constexpr bool kMixed = TM % (kLoads * 8) != 0;  // a wave may have rows of both
  const auto offset_of = [&](uint32_t most, uint32_t stride) { return (static_cast<At>(min(lane / 8, most)) * stride + piece) * 2; };  // (bytes)
  const bool of_x = wave * kLoads * 8 < TM;  // (where all are of one kind, they share these)
  const At whole = offset_of(7, of_x ? a.x_stride : a.w_stride);
  const At edge = offset_of(of_x ? a.t - 1 - i0 - x_edge : a.m - 1 - j0 - w_edge, of_x ? a.x_stride : a.w_stride);
  const At w_whole = kMixed ? offset_of(7, a.w_stride) : whole, w_last = kMixed ? offset_of(a.m - 1 - j0 - w_edge, a.w_stride) : edge;
  uint32_t at_edge = 0;  // bit q: instruction q's rows end among its eight, or in front of them
#pragma unroll
  for (int q = 0; q < kLoads; ++q) {
    const uint32_t first = (wave * kLoads + q) * 8, begin = to > from ? from : 0;
    if (first < TM) {
      src[q] = a.x + static_cast<size_t>(i0 + min(first, x_edge)) * a.x_stride + begin;
      at_edge |= (first >= x_edge ? 1u : 0u) << q;
    } else {
      uint32_t j = first - TM, up = 0;
      if (GATED) {
        const uint32_t in = j % (TN / WN);
        j = j / (TN / WN) * kHalf + in % kHalf;
        up = in >= kHalf ? a.m : 0;
      }
      src[q] = a.w + (static_cast<size_t>(j0) + min(j, w_edge) + up) * a.w_stride + begin;
      at_edge |= (j >= w_edge ? 1u : 0u) << q;
    }
    src[q] = uniform(src[q]);
  }
  at_edge = __builtin_amdgcn_readfirstlane(at_edge);
  const auto lane_at = [&](int q) -> At {
    const uint32_t ends = at_edge >> q & 1, of_w = kMixed && (wave * kLoads + q) * 8 >= TM;
    const At plain = of_w ? w_whole + 0 : whole + 0, cut = of_w ? w_last + 0 : edge + 0;  // (values: a choice between variables would put them into memory)
    return ends ? cut + 0 : plain + 0;
  };
  const uint32_t lds_at = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds))) + wave * kLoads * 1024;
  uint4 held[ALIGNED ? 1 : kLoads];
  const auto request_one = [&](int q, uint32_t block, uint32_t stage) {
    block = min(block, last);
    const bool broken = block == full;
    if (block < full) block = block + skew < full ? block + skew : block + skew - full;
    block = __builtin_amdgcn_readfirstlane(block);
    if constexpr (ALIGNED) {
      load_to_lds_from(src[q] + block * 64, lane_at(q) - (back & (broken ? ~0u : 0u)), lds_at + stage * kStage + q * 1024);
    } else {
      const uint16_t* p = src[q] + block * 64 + lane_at(q) / 2;
      if (!broken) held[q] = load_16_bytes(p);
      else held[q] = piece < rest ? load_bf16x8_guarded(p, rest - piece) : make_uint4(0, 0, 0, 0);
    }
  };
  const auto request = [&](uint32_t block, uint32_t stage) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q) request_one(q, block, stage);
  };
  const auto place = [&](uint32_t stage) {
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int q = 0; q < kLoads; ++q) lds[stage * (kStage / 16) + (wave * kLoads + q) * 64 + lane] = held[q];
    }
  };
  const uint32_t r = lane & 15, g = lane >> 4, mine = r * 8 + (g ^ (r & 7));
  f32x4_t sum[NT][MT] = {};
  uint4 fx[2][MT], fw[2][NT];
  const auto read_one = [&](int k, int half, uint32_t stage) {
    const uint4* p = lds + stage * (kStage / 16) + (mine ^ half * 4);
    if (k < NT) fw[half][k] = p[(TM / 16 + wn * NT + k) * 128];
    else fx[half][k - NT] = p[(wm * MT + k - NT) * 128];
  };
  const auto read = [&](int half, uint32_t stage) {
#pragma unroll
    for (int k = 0; k < MT + NT; ++k) read_one(k, half, stage);
  };
  // A step of the matrix cores.  Between its instructions, in their shadow: the other half's operands are read (from `stage`), and where `ask` the next block's
  // pieces are requested.
  const auto multiply = [&](int half, uint32_t stage, bool ask, uint32_t block, uint32_t into) {
    constexpr int kAll = MT * NT, kReads = MT + NT;
    if constexpr (kSpread) {
#pragma unroll
      for (int i = 0; i < kAll; ++i) {
#pragma unroll
        for (int k = i * kReads * 2 / kAll; k < (i + 1) * kReads * 2 / kAll; ++k)
          if (k < kReads) read_one(k, half ^ 1, stage);
        if (ask)
#pragma unroll
          for (int q = i * kLoads / kAll; q < (i + 1) * kLoads / kAll; ++q) request_one(q, block, into);
        sum[i / MT][i % MT] = mfma16(fw[half][i / MT], fx[half][i % MT], sum[i / MT][i % MT]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      if (ask) {
        request(block, into);
      }
      read(half ^ 1, stage);
#pragma unroll
      for (int i = 0; i < kAll; ++i) sum[i / MT][i % MT] = mfma16(fw[half][i / MT], fx[half][i % MT], sum[i / MT][i % MT]);
      // the reads in front, between the first matrix instructions
#pragma unroll
      for (int k = 0; k < kReads; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, kAll / kReads, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, kAll - kAll / kReads * kReads, 0);
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES; ++s) {
    if (!ALIGNED && s == STAGES - 1) break;
    request(s, s);
    place(s);
  }
  if (ALIGNED) wait_loads<(STAGES - 1) * kLoads>();
  __syncthreads();
  read(0, 0);
  for (uint32_t base = 0; base < full; base += STAGES) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      if (base + s >= full) break;
      if (!ALIGNED) request(base + s + STAGES - 1, (s + STAGES - 1) % STAGES);
      multiply(0, s, false, 0, 0);
      // every wave has the block's last operands, and the next block is there
      if constexpr (ALIGNED) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * kLoads) : "memory");
        __builtin_amdgcn_s_barrier();
        issue_fence();
      } else {
        place((s + STAGES - 1) % STAGES);
        __syncthreads();
      }
      multiply(1, (s + 1) % STAGES, ALIGNED, base + s + STAGES, s);
    }
  }
  if (KG > 1)  // (a group whose share ends earlier waits with the others)
    for (uint32_t b = full; b < blocks; ++b) __syncthreads();
  if (rest) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h) read(1, full % STAGES);
      const uint32_t keep = (h * 4 + g) * 8 < rest ? ~0u : 0u;
#pragma unroll
      for (int c = 0; c < MT; ++c) fx[h][c] = masked(fx[h][c], keep);
#pragma unroll
      for (int c = 0; c < NT; ++c) fw[h][c] = masked(fw[h][c], keep);
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m) sum[c][m] = mfma16(fw[h][c], fx[h][m], sum[c][m]);
    }
  }
  if (ALIGNED) wait_loads<0>();

  // The sums go through LDS, a part of the wave's tokens at a time, so that a lane gets four neighbours of a token and neighbouring lanes the next ones; the
  // pieces of a token are turned by its number, so that the lanes' tokens meet all banks.  The groups' sums are added here, each group finishing its share.
  constexpr uint32_t kPieces = NT * 4, kGroupLds = STAGES * kStage / 16, kWaveLds = kGroupLds / kWaves;
  constexpr int kSlab = largest_part(MT, kWaveLds / (64 * NT));
  static_assert(kSlab * 16 * kPieces % 64 == 0, "the lanes take turns evenly");
  const auto turned = [](uint32_t token, uint32_t p) { return (p + token * (kPieces < 16 ? kPieces : 16) / 16) % kPieces; };  // (token: of 16)
  const f32x4_t* all = reinterpret_cast<const f32x4_t*>(whole_lds) + wave * kWaveLds;
  f32x4_t* out = reinterpret_cast<f32x4_t*>(lds) + wave * kWaveLds;
  __syncthreads();
#pragma unroll
  for (int m0 = 0; m0 < MT; m0 += kSlab) {
#pragma unroll
    for (int m = 0; m < kSlab; ++m)
#pragma unroll
      for (int c = 0; c < NT; ++c) out[(m * 16 + r) * kPieces + turned(r, c * 4 + g)] = sum[c][m0 + m];
    if (KG > 1) __syncthreads();
    else issue_fence();  // (a wave's own LDS accesses keep their order)
    constexpr uint32_t kAcross = GATED ? kPieces / 2 : kPieces;  // pieces of results a token
    for (uint32_t at = group * 64 + lane; at < kSlab * 16 * kAcross; at += 64 * KG) {
      const uint32_t token = at / kAcross, p = at % kAcross, i = i0 + (wm * MT + m0) * 16 + token, j = j0 + wn * (kAcross * 4) + p * 4;
      if (i >= a.t || j >= a.m) continue;
      const uint32_t z_at = token * kPieces + turned(token % 16, p), up_at = token * kPieces + turned(token % 16, GATED ? p + kAcross : p);
      f32x4_t z = all[z_at], up = all[up_at];
#pragma unroll
      for (int k = 1; k < KG; ++k) {
        z += all[k * kGroupLds + z_at];
        if (GATED) up += all[k * kGroupLds + up_at];
      }
      if (t.parts) {
        float* part = t.parts + (static_cast<size_t>(blockIdx.y) * a.t + i) * (GATED ? 2 : 1) * a.m + j;
        store4(part, z, a.m - j);
        if (GATED) store4(part + a.m, up, a.m - j);
      } else {
        finish4<GATED>(a, i, j, a.m, z, up);
      }
    }
    if (KG > 1) __syncthreads();
    else issue_fence();
  }
}

// Results whose sums over n were made in parts: four neighbours a thread, the parts in their order.  (20 rows 8200 -> 1100: 16.7 us in one
// part, 10.5 in four with this launch; 100 rows 8200 -> 4100: 34.7 and 26.7.)
template <bool GATED>
__global__ __launch_bounds__(256) void project_parts_kernel(const TileArgs t) {
  const mf_project_args& a = t.p;
  const uint32_t across = (a.m + 3) / 4;
  const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= static_cast<uint64_t>(a.t) * across) return;
  const uint32_t i = static_cast<uint32_t>(at / across), j = static_cast<uint32_t>(at % across) * 4;
  const size_t width = (GATED ? 2 : 1) * static_cast<size_t>(a.m), plane = width * a.t;
  const float* part = t.parts + i * width + j;
  f32x4_t z = {}, up = {};
  for (uint32_t k = 0; k < t.part_count; ++k) {
    z += load4(part + k * plane, a.m - j);
    if (GATED) up += load4(part + k * plane + a.m, a.m - j);
  }
  finish4<GATED>(a, i, j, a.m, z, up);
}

// ------------------------------------------------------------------ few rows

// Up to 16 tokens: the call is W's stream.  A workgroup up to 16 rows of W (and, gated, their up rows), its waves share the sum over n, each with a ring in LDS that it fills itself with whole
// lines of 128 bytes.  Four rows 5120 -> 17408, gated: 63.5 us, 5.6 TB/s; eight 17408 -> 5120: 32.9 us, 5.4 TB/s (operands straight from memory in the matrix cores' order touch 64 bytes of a row at a time: 2.2 TB/s; eight rows
// an instruction without LDS: 4.7).
template <bool GATED, bool ALIGNED, int WAVES, int STAGES, int XI>
__global__ __launch_bounds__(64 * WAVES) void project_rows_kernel(const mf_project_args a, uint32_t rows) {
  constexpr int kW = GATED ? 4 : 2, kLoads = kW + XI;
  extern __shared__ uint4 whole_lds[];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4, j0 = blockIdx.x * rows, own = min(rows, a.m - j0);
  // a wave's share of n, in whole blocks
  const uint32_t share = ((a.n + 63) / 64 + WAVES - 1) / WAVES, from = min(wave * share * 64, a.n), to = min(from + share * 64, a.n), begin = to > from ? from : 0;
  RowAt<ALIGNED> at[kLoads];
#pragma unroll
  for (int q = 0; q < kLoads; ++q) {
    const uint32_t row = q % 2 * 8 + lane / 8;
    at[q] = ((q < kW ? static_cast<RowAt<ALIGNED>>(min(row, own - 1)) * a.w_stride : static_cast<RowAt<ALIGNED>>(min(row, a.t - 1)) * a.x_stride) + lane_piece(lane)) * 2;
  }
  const uint16_t* w = a.w + static_cast<size_t>(j0) * a.w_stride + begin;
  f32x4_t sum = {}, up_sum = {};
  stream_rows<GATED, ALIGNED, STAGES, XI>(w, w + static_cast<size_t>(a.m) * a.w_stride, a.x + begin, at, to - from, whole_lds + wave * STAGES * kLoads * 64, sum, up_sum);
  __syncthreads();
  f32x4_t* part = reinterpret_cast<f32x4_t*>(whole_lds);
  part[wave * 128 + lane] = sum;
  if (GATED) part[wave * 128 + 64 + lane] = up_sum;
  __syncthreads();
  if (wave) return;
  const uint32_t j = j0 + g * 4;
  if (r >= a.t || g * 4 >= own) return;
#pragma unroll
  for (int v = 1; v < WAVES; ++v) {
    sum += part[v * 128 + lane];
    if (GATED) up_sum += part[v * 128 + 64 + lane];
  }
  finish4<GATED>(a, r, j, j0 + own, sum, up_sum);
}

template <bool GATED, bool ALIGNED, int WAVES, int STAGES, int XI>
hipError_t launch_rows(hipStream_t s, const mf_project_args& a, uint32_t rows) {
  constexpr int kLds = WAVES * STAGES * ((GATED ? 4 : 2) + XI) * 1024;
  const hipError_t e = allow_lds<project_rows_kernel<GATED, ALIGNED, WAVES, STAGES, XI>>(kLds, kLds);
  if (e != hipSuccess) return e;
  project_rows_kernel<GATED, ALIGNED, WAVES, STAGES, XI><<<dim3((a.m + rows - 1) / rows), 64 * WAVES, kLds, s>>>(a, rows);
  return hipGetLastError();
}

template <int TM, int TN, int WM, int WN, int KG, int STAGES, bool GATED, bool ALIGNED>
hipError_t launch_tiles(hipStream_t s, TileArgs& a) {
  constexpr uint32_t kRows = GATED ? TN / 2 : TN;
  constexpr int kLds = KG * STAGES * (TM + TN) * 128;
  a.row_tiles = (a.p.m + kRows - 1) / kRows;
  a.token_tiles = (a.p.t + TM - 1) / TM;
  const hipError_t e = allow_lds<project_tile_kernel<TM, TN, WM, WN, KG, STAGES, GATED, ALIGNED>>(kLds, kLds);
  if (e != hipSuccess) return e;
  project_tile_kernel<TM, TN, WM, WN, KG, STAGES, GATED, ALIGNED><<<dim3(a.row_tiles * a.token_tiles, a.part_count), 64 * WM * WN * KG, kLds, s>>>(a);
  return hipGetLastError();
}

}  // namespace

// Sums over n in parts, where the tiles leave CUs idle: what they may take, by the most parts and bytes that are considered.
constexpr uint32_t kMostParts = 16;
constexpr uint64_t kMostPartBytes = 16u << 20;

size_t project_workspace_bytes(uint32_t m, uint32_t n, uint32_t t, bool gated) {
  const uint64_t rows = gated ? 2ull * m : m;
  if (t <= 16 || n < 512 || rows >= 32ull * device_cu_count()) return 0;  // (the smallest tiles have 32 rows)
  return static_cast<size_t>(std::min(kMostPartBytes, kMostParts * 4 * rows * t));
}

namespace {

// The shapes of tiles, and what they cost: us for a block of 64 values of n where every CU has the tiles that fit it at once (one, or two of 128 x 128 in two stages), where the chip has
// more than two tiles a CU (the caches then hold less of what they share), and in front of and behind the blocks.  Measured over 1 .. 4096 tokens and seven pairs of
// sizes; the choice is within 10 % of the best shape in most of them.  A third stage is worth more than the second workgroup that it costs while there are no tiles for one:
// 128 x 128 at 512 tokens, 5120 -> 5120: 40.0 us in three stages, 56.5 in two; at 1024 tokens 80 and 63.
struct Shape {
  uint32_t tokens, rows;
  float block, block_many, fixed;
  uint32_t a_cu;
  bool unaligned;  // has a form for rows that are no whole 16 bytes
};
constexpr Shape kShapes[] = {{32, 32, 0.09f, 0.1f, 3.7f, 1, true},      {32, 64, 0.133f, 0.15f, 4.0f, 1, false},     {64, 64, 0.178f, 0.2f, 4.3f, 1, true},
                             {64, 128, 0.267f, 0.33f, 5.0f, 1, false},  {128, 128, 0.65f, 0.97f, 9.5f, 2, true},     {128, 128, 0.385f, 0.5f, 7.7f, 1, false},
                             {128, 192, 0.53f, 0.79f, 10.0f, 1, false}, {256, 128, 0.8f, 0.92f, 9.0f, 1, false},     {256, 192, 1.35f, 1.42f, 10.0f, 1, false},
                             {256, 256, 1.5f, 1.62f, 13.0f, 1, false}};

template <bool GATED, bool ALIGNED>
hipError_t launch_shape(hipStream_t s, TileArgs& t, float* workspace) {
  const mf_project_args& a = t.p;
  const uint32_t cus = device_cu_count(), rows = GATED ? 2 * a.m : a.m;
  // Few rows: sixteen of W a workgroup while every CU has one at most, else as many as give every CU the same number of workgroups (8 rows 17408 -> 5120: 32.6 us with 10, 39.4 with 16;
  // four 5120 -> 17408, gated: 65.9 with 14, 70.2 with 16).  Two waves where there are workgroups for every CU and one stream of W each (32.6 us, four waves 35.1), four where there are
  // fewer (8192 -> 1024: 6.7, two 8.5) or two streams (12 rows 5120 -> 17408, gated: 69.6, two 74.9).
  if (a.t <= 16) {
    const uint32_t blocks = (a.m + 15) / 16, rounds = (blocks + cus - 1) / cus, few = rounds == 1 ? 16 : (a.m + cus * rounds - 1) / (cus * rounds);
    if (GATED || blocks < cus) return a.t <= 8 ? launch_rows<GATED, ALIGNED, 4, 3, 1>(s, a, few) : launch_rows<GATED, ALIGNED, 4, 3, 2>(s, a, few);
    return a.t <= 8 ? launch_rows<false, ALIGNED, 2, 4, 1>(s, a, few) : launch_rows<false, ALIGNED, 2, 4, 2>(s, a, few);
  }
  int best = 0;
  uint32_t blocks = (a.n + 63) / 64, parts = 1;
  float least = 3.4e38f;
  for (int k = 0; k < 10; ++k) {
    const Shape& h = kShapes[k];
    if (!ALIGNED && !h.unaligned) continue;
    const uint64_t tiles = static_cast<uint64_t>((a.t + h.tokens - 1) / h.tokens) * ((rows + h.rows - 1) / h.rows);
    for (uint32_t p = 1; p <= (workspace ? kMostParts : 1); p *= 2) {
      const uint64_t bytes = 4ull * p * a.t * rows, rounds = (tiles * p + cus * h.a_cu - 1) / (cus * h.a_cu);
      if (p > 1 && (tiles * p > cus || blocks / p < 4 || bytes > kMostPartBytes)) break;
      float us = h.fixed + static_cast<float>(rounds * ((blocks + p - 1) / p)) * (tiles * p > 2 * cus ? h.block_many : h.block);
      if (p > 1) us += 3.5f + static_cast<float>(bytes) / 2e6f;  // the launch that adds the parts, and their way to memory and back
      if (us < least) least = us, best = k, parts = p;
    }
  }
  t.part_blocks = (blocks + parts - 1) / parts;
  t.part_count = (blocks + t.part_blocks - 1) / t.part_blocks;
  t.parts = t.part_count > 1 ? workspace : nullptr;
  switch (best) {
    case 0: return launch_tiles<32, 32, 2, 1, 2, 4, GATED, ALIGNED>(s, t);
    case 2: return launch_tiles<64, 64, 2, 2, 1, 4, GATED, ALIGNED>(s, t);
    case 4: return launch_tiles<128, 128, 2, 4, 1, 2, GATED, ALIGNED>(s, t);
  }
  if constexpr (ALIGNED) {
    switch (best) {
      case 1: return launch_tiles<32, 64, 2, 2, 2, 4, GATED, true>(s, t);
      case 3: return launch_tiles<64, 128, 2, 4, 1, 3, GATED, true>(s, t);
      case 5: return launch_tiles<128, 128, 2, 4, 1, 3, GATED, true>(s, t);
      case 6: return launch_tiles<128, 192, 4, 2, 1, 3, GATED, true>(s, t);
      case 7: return launch_tiles<256, 128, 4, 2, 1, 3, GATED, true>(s, t);
      case 8: return launch_tiles<256, 192, 4, 2, 1, 2, GATED, true>(s, t);
      case 9: return launch_tiles<256, 256, 2, 4, 1, 2, GATED, true>(s, t);
    }
  }
  return hipErrorUnknown;
}

}  // namespace

hipError_t launch_project(hipStream_t s, const mf_project_args& a, void* workspace) {
  TileArgs t{};
  t.p = a;
  // whole pieces of 16 bytes, and rows near enough for a tile's offsets of 32 bits
  constexpr uint32_t kFar = 1u << 27;
  const bool aligned = aligned16(a.x) && aligned16(a.w) && a.x_stride % 8 == 0 && a.w_stride % 8 == 0 && a.n % 8 == 0 && a.x_stride < kFar && a.w_stride < kFar;
  float* parts = project_workspace_bytes(a.m, a.n, a.t, a.gated != 0) ? static_cast<float*>(workspace) : nullptr;
  const hipError_t e = a.gated ? (aligned ? launch_shape<true, true>(s, t, parts) : launch_shape<true, false>(s, t, parts))
                               : (aligned ? launch_shape<false, true>(s, t, parts) : launch_shape<false, false>(s, t, parts));
  if (e != hipSuccess || !t.parts) return e;
  const dim3 grid(static_cast<uint32_t>((static_cast<uint64_t>(a.t) * ((a.m + 3) / 4) + 255) / 256));
  if (a.gated) project_parts_kernel<true><<<grid, 256, 0, s>>>(t);
  else project_parts_kernel<false><<<grid, 256, 0, s>>>(t);
  return hipGetLastError();
}

}  // namespace mf
