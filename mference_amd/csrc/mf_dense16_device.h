// What the kernels of the 16-bit operators share.
#pragma once

#include <type_traits>

#include "mf_device.h"

namespace mf {

// D[16 rows, 16 columns] += A[16, 32] B[32, 16]: lane l holds eight k's from 8 (l / 16) on of A's row l % 16 and of B's column l % 16, and
// rows 4 (l / 16) .. + 3 of D's column l % 16
__device__ __forceinline__ f32x4_t mfma16(const uint4& a, const uint4& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// z Phi(z) = z (1 + erf(z / sqrt 2)) / 2.  The tail H = erfc(|z| / sqrt 2) / 2 is e^(-z^2 / 2) t p(t), t = 1 / (1 + 0.35 |z|), p a least-maximum fit of degree 8 over
// |z| <= 14 (2^-24.9 relative); Phi is H for negative arguments and 1 - H for the others, so that nothing cancels: 1 + erf in fp32 loses a twentieth of the result at -5
// and all of it from -5.5 on.  2^-20.8 relative near 0, (z^2 + 19) 2^-23 far out.  777 rows 1280 -> 5120: 27.4 us, with 1 + the
// library's erf 30.0, with its erfc 31.3.
__device__ __forceinline__ float gelu(float z) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35f, __builtin_fabsf(z), 1.0f));
  float p = -0.0291459281f;
  p = __builtin_fmaf(p, t, 0.143971682f);
  p = __builtin_fmaf(p, t, -0.255714238f);
  p = __builtin_fmaf(p, t, 0.159174129f);
  p = __builtin_fmaf(p, t, -0.0231098142f);
  p = __builtin_fmaf(p, t, 0.105507992f);
  p = __builtin_fmaf(p, t, 0.119832873f);
  p = __builtin_fmaf(p, t, 0.139861867f);
  p = __builtin_fmaf(p, t, 0.139621407f);
  const float h = t * __builtin_amdgcn_exp2f(z * z * -0.72134752044f) * p;
  return z * (z < 0.0f ? h : 1.0f - h);
}

// The activations on the hardware's exp2 and reciprocal (1 ulp each), from fp32 sums.  The tanh form is x / (1 + e^(-2u)), which is 0.5 x (1 + tanh u) without its cancellation.
__device__ __forceinline__ float activate(float z, mf_activation act) {
  if (act == MF_ACT_SILU) return fast_silu(z);
  if (act == MF_ACT_GELU_TANH) return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.3022081986f * (z + 0.044715f * z * z * z)));
  if (act == MF_ACT_GELU) return gelu(z);
  return z;
}

// v where `keep` is ~0, zeros where it is 0
__device__ __forceinline__ uint4 masked(const uint4& v, uint32_t keep) { return make_uint4(v.x & keep, v.y & keep, v.z & keep, v.w & keep); }

// a pointer that is the same in all lanes, as one for the compiler too (the builtin gives an int)
template <class T>
__device__ __forceinline__ T* uniform(T* pointer) {
  const auto p = reinterpret_cast<uint64_t>(pointer);
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(p >> 32)), lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(p));
  return reinterpret_cast<T*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// load_to_lds (mf_device.h) from a uniform base and a lane's byte offset: no 64-bit address a lane
__device__ __forceinline__ void load_to_lds_from(const void* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(lds), "v"(offset), "s"(base) : "memory");
}

// ------------------------------------------------------------------ rows as a stream

// A lane's byte offset of a row, 32 bits where the rows come straight to LDS.
template <bool ALIGNED> using RowAt = std::conditional_t<ALIGNED, uint32_t, uint64_t>;

// Which 16 bytes of a block of 64 values a lane brings of its row (eight lanes a row, a line of 128 bytes), turned by the row's number so that 16 lanes that
// read the same piece of 16 rows meet all banks; and where row r's piece g (0 .. 3) of a block lies (the second half's: ^ 4).
__device__ __forceinline__ uint32_t lane_piece(uint32_t lane) { return ((lane & 7) ^ lane / 8) * 8; }
__device__ __forceinline__ uint32_t place_of(uint32_t r, uint32_t g) { return r * 8 + (g ^ (r & 7)); }

// sum (and up_sum) += 16 rows of w (and of up) times up to 8 XI rows of x, over `length` values, by one wave: the call is the rows' stream.  Whole lines go through a ring of
// STAGES blocks of 64 values in LDS that is this wave's own, so that it waits for no other; `at` are the lanes' byte offsets of 2 (4) instructions of eight rows of w (and
// up) and XI of x, the lane's piece included.  What lies behind the end is left out when it is multiplied: a lane that would read there reads the
// start of its last block again.  Rows that are no whole 16 bytes (ALIGNED false) pass through registers.
template <bool GATED, bool ALIGNED, int STAGES, int XI>
__device__ __forceinline__ void stream_rows(const uint16_t* w, const uint16_t* up, const uint16_t* x, const RowAt<ALIGNED> (&at)[(GATED ? 4 : 2) + XI], uint32_t length, uint4* lds,
                                            f32x4_t& sum, f32x4_t& up_sum) {
  constexpr int kW = GATED ? 4 : 2, kLoads = kW + XI, kStage = kLoads * 64;  // instructions a block, 16-byte pieces a stage
  const uint32_t lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, piece = lane_piece(lane);
  const uint32_t full = __builtin_amdgcn_readfirstlane(length / 64), rest = __builtin_amdgcn_readfirstlane(length % 64), last = rest || !full ? full : full - 1;
  const uint32_t lds_at = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds))), back = piece >= rest ? piece * 2 : 0;
  w = uniform(w);
  x = uniform(x);
  if (GATED) up = uniform(up);
  uint4 held[ALIGNED ? 1 : kLoads];
  const auto request = [&](uint32_t block, uint32_t stage) {
    block = min(block, last);
    const bool broken = block == full;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const uint16_t* p = (q >= kW ? x : q >= 2 ? up : w) + block * 64;
      if constexpr (ALIGNED) {
        load_to_lds_from(p, at[q] - (back & (broken ? ~0u : 0u)), lds_at + (stage * kStage + q * 64) * 16);
      } else {
        p += at[q] / 2;
        if (!broken) held[q] = load_16_bytes(p);
        else held[q] = piece < rest ? load_bf16x8_guarded(p, rest - piece) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  const auto place = [&](uint4* stage) {
    if constexpr (!ALIGNED) {
      issue_fence();  // (a wave's own LDS accesses keep their order)
#pragma unroll
      for (int q = 0; q < kLoads; ++q) stage[q * 64 + lane] = held[q];
      issue_fence();
    }
  };
  const uint32_t mine = place_of(r, g), mine_x = XI == 2 ? mine : place_of(r & 7, g);
  uint4 fw[2], fu[2], fx[2];
  const auto read = [&](const uint4* stage) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      fw[h] = stage[mine ^ h * 4];
      if (GATED) fu[h] = stage[128 + (mine ^ h * 4)];
      fx[h] = stage[kW * 64 + (mine_x ^ h * 4)];
    }
  };
  const auto multiply = [&] {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum = mfma16(fw[h], fx[h], sum);
      if (GATED) up_sum = mfma16(fu[h], fx[h], up_sum);
    }
  };
#pragma unroll
  for (int s = 0; s < (ALIGNED ? STAGES : 1); ++s) request(s, s);
  for (uint32_t base = 0; base < full; base += STAGES) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      if (base + s >= full) break;
      uint4* stage = lds + s * kStage;
      if constexpr (ALIGNED) {
        wait_loads<(STAGES - 1) * kLoads>();
        read(stage);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read
        request(base + s + STAGES, s);
      } else {
        place(stage);
        request(base + s + 1, 0);
        read(stage);
      }
      multiply();
    }
  }
  if (rest) {
    if (ALIGNED) wait_loads<0>();
    uint4* stage = lds + full % STAGES * kStage;
    place(stage);
    read(stage);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t keep = (h * 4 + g) * 8 < rest ? ~0u : 0u;
      fw[h] = masked(fw[h], keep);
      if (GATED) fu[h] = masked(fu[h], keep);
      fx[h] = masked(fx[h], keep);
    }
    multiply();
  }
  if (ALIGNED) wait_loads<0>();
}

}  // namespace mf
