// Drives the low-rank adapters and the norm between two blocks through include/mfmoe.hpp and checks them against loops in 64 bits.
//
//   adapters_test cpu   sizes and refusals (no GPU needed)
//   adapters_test gpu   rows by adapter, their corrections in bf16 and fp32, the norms around a block
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>

#include "mfmoe.hpp"

static int g_fail = 0;
#define EXPECT(cond, ...)                              \
  do {                                                 \
    if (!(cond)) {                                     \
      ++g_fail;                                        \
      std::printf("FAIL %s:%d: ", __FILE__, __LINE__); \
      std::printf(__VA_ARGS__);                        \
      std::printf("\n");                               \
    }                                                  \
  } while (0)

#define HIP_OK(call)                                                                     \
  do {                                                                                   \
    hipError_t e_ = (call);                                                              \
    if (e_ != hipSuccess) {                                                              \
      std::printf("HIP error %s at %s:%d\n", hipGetErrorString(e_), __FILE__, __LINE__); \
      std::exit(2);                                                                      \
    }                                                                                    \
  } while (0)

template <typename T> static T* to_device(const std::vector<T>& v) {
  T* p = nullptr;
  HIP_OK(hipMalloc(&p, v.size() * sizeof(T) + 16));
  HIP_OK(hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice));
  return p;
}
template <typename T> static std::vector<T> to_host(const T* p, size_t n) {
  std::vector<T> v(n);
  HIP_OK(hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
  return v;
}

static float widen(uint16_t b) {
  const uint32_t w = static_cast<uint32_t>(b) << 16;
  float f;
  std::memcpy(&f, &w, 4);
  return f;
}
static uint16_t narrow(float f) {
  uint32_t w;
  std::memcpy(&w, &f, 4);
  return static_cast<uint16_t>((w + 0x7FFFu + ((w >> 16) & 1u)) >> 16);
}
// numbers of [-1, 1) in steps of 1/64: exact in bf16
static uint32_t g_state = 12345;
static float next_number() {
  g_state = g_state * 1664525u + 1013904223u;
  return static_cast<float>(static_cast<int>(g_state >> 25) - 64) / 64.0f;
}
static std::vector<uint16_t> numbers(size_t n) {
  std::vector<uint16_t> v(n);
  for (auto& x : v) x = narrow(next_number());
  return v;
}

template <typename F> static mf_status status_of(F f) {
  try {
    f();
  } catch (const mf::Error& e) {
    return e.status;
  }
  return MF_OK;
}

static void test_sizes() {
  mf_adapter_pool pool{4, 16, 128, nullptr, nullptr};
  EXPECT(mf_adapter_workspace_bytes(&pool, 2, 8) > 0, "workspace");
  pool.rank = 12;
  EXPECT(mf_adapter_workspace_bytes(&pool, 2, 8) == 0, "a rank that is no multiple of eight");
  EXPECT(mf_adapter_plan_bytes(10, 4) >= 4 * (10 + 5) && mf_adapter_plan_bytes(10, 0) == 0, "plan");
  EXPECT(mf_adapter_group(nullptr, nullptr, nullptr, 1, 1, nullptr, 0) == MF_ERR_INVALID_ARGUMENT, "no context");
  EXPECT(mf_block_norm(nullptr, nullptr, nullptr) == MF_ERR_INVALID_ARGUMENT, "no arguments");
}

// What a result may be off by: its own rounding, half a step (eps / 2 of its magnitude), and what the fp32 sums and the terms of A x
// leave, which for these sizes (|v| < n, |correction| < rank n) stays below 2^-16 of the sum of magnitudes.
static void test_adapters(const mf::MetalContext& ctx, bool float32, bool planned) {
  const uint32_t t = 37, n = 192, m[2] = {70, 33}, adapters = 5, rank = 24;
  const uint32_t ranks[adapters] = {24, 0, 7, 16, 9};
  const float scales[adapters] = {0.5f, 2.0f, -1.0f, 0.25f, 1.5f};
  std::vector<int32_t> ids(t);
  for (uint32_t i = 0; i < t; ++i) ids[i] = static_cast<int32_t>(i * 7 % (adapters + 1)) - (i % 11 == 0 ? 8 : 0);
  const auto x = numbers(size_t(t) * n);
  auto* d_x = to_device(x);
  auto* d_ids = to_device(ids);
  auto* d_ranks = to_device(std::vector<uint32_t>(ranks, ranks + adapters));
  auto* d_scales = to_device(std::vector<float>(scales, scales + adapters));
  const mf_adapter_pool pool{adapters, rank, n, d_ranks, d_scales};
  const mf::AdapterGrouping grouping(ctx, adapters);
  const mf::LowRankAdapters low(ctx, pool);
  uint32_t* plan = nullptr;
  if (planned) {
    plan = to_device(std::vector<uint32_t>(grouping.planBytes(t) / 4));
    grouping.encode(nullptr, d_ids, t, plan, grouping.planBytes(t));
    const auto rows = to_host(plan, t + adapters + 1);
    uint32_t at = 0;
    for (uint32_t a = 0; a <= adapters; ++a) {
      EXPECT(rows[t + a] == at, "adapter %u starts at %u, not %u", a, rows[t + a], at);
      for (uint32_t i = 0; i < t; ++i) {
        const bool has = ids[i] >= 0 && ids[i] < static_cast<int32_t>(adapters);
        if (a == adapters ? has : !has || ids[i] != static_cast<int32_t>(a)) continue;
        EXPECT(at < t && rows[at] == i, "row %u is not at %u", i, at);
        ++at;
      }
    }
    EXPECT(status_of([&] { grouping.encode(nullptr, d_ids, t, plan, 16); }) == MF_ERR_SCRATCH_TOO_SMALL, "a plan without room");
  }
  std::vector<uint16_t> a[2], b[2], y[2];
  mf_adapter_target targets[2];
  for (int s = 0; s < 2; ++s) {
    a[s] = numbers(size_t(adapters) * rank * n), b[s] = numbers(size_t(adapters) * m[s] * rank), y[s] = numbers(size_t(t) * m[s]);
    std::vector<float> wide(y[s].size());
    for (size_t i = 0; i < wide.size(); ++i) wide[i] = widen(y[s][i]);
    targets[s] = {to_device(a[s]), to_device(b[s]), float32 ? static_cast<void*>(to_device(wide)) : to_device(y[s]), m[s], m[s]};
  }
  const size_t need = low.workspaceBytes(2, t);
  auto* workspace = to_device(std::vector<uint8_t>(need));
  EXPECT(status_of([&] { low.encode(nullptr, targets, 2, d_x, n, d_ids, t, float32, plan, workspace, need - 1); }) == MF_ERR_SCRATCH_TOO_SMALL, "a workspace without room");
  low.encode(nullptr, targets, 2, d_x, n, d_ids, t, float32, plan, workspace, need);
  HIP_OK(hipDeviceSynchronize());
  for (int s = 0; s < 2; ++s) {
    std::vector<float> got(size_t(t) * m[s]);
    if (float32) got = to_host(static_cast<float*>(targets[s].y), got.size());
    else {
      const auto bits = to_host(static_cast<uint16_t*>(targets[s].y), got.size());
      for (size_t i = 0; i < got.size(); ++i) got[i] = widen(bits[i]);
    }
    for (uint32_t i = 0; i < t; ++i) {
      const bool has = ids[i] >= 0 && ids[i] < static_cast<int32_t>(adapters);
      const uint32_t k = has ? ids[i] : 0, live = has ? ranks[k] : 0;
      std::vector<double> v(live);
      for (uint32_t r = 0; r < live; ++r)
        for (uint32_t e = 0; e < n; ++e) v[r] += double(widen(a[s][(size_t(k) * rank + r) * n + e])) * widen(x[size_t(i) * n + e]);
      for (uint32_t j = 0; j < m[s]; ++j) {
        const double old = widen(y[s][size_t(i) * m[s] + j]);
        double want = old, most = std::fabs(old);
        for (uint32_t r = 0; r < live; ++r) {
          const double term = scales[k] * v[r] * widen(b[s][(size_t(k) * m[s] + j) * rank + r]);
          want += term, most += std::fabs(term);
        }
        const double off = std::fabs(got[size_t(i) * m[s] + j] - want), may = std::fabs(want) * (float32 ? std::ldexp(1.0, -24) : std::ldexp(1.0, -8)) + most * std::ldexp(1.0, -16);
        EXPECT(live ? off <= may : got[size_t(i) * m[s] + j] == old, "target %d row %u result %u: %g, not %g", s, i, j, got[size_t(i) * m[s] + j], want);
      }
    }
    HIP_OK(hipFree(const_cast<uint16_t*>(targets[s].a)));
    HIP_OK(hipFree(const_cast<uint16_t*>(targets[s].b)));
    HIP_OK(hipFree(targets[s].y));
  }
  for (void* p : {static_cast<void*>(d_x), static_cast<void*>(d_ids), static_cast<void*>(d_ranks), static_cast<void*>(d_scales), static_cast<void*>(plan), static_cast<void*>(workspace)})
    if (p) HIP_OK(hipFree(p));
  std::printf("adapters, %s results, %s: ok\n", float32 ? "fp32" : "bf16", planned ? "grouped" : "as they lie");
}

// hidden is narrowed once (2^-8 of it); out is the norm of that, narrowed once more, so it is compared with the norm of what the call
// left in hidden; fp32 in between (2^-16 covers sums of 100 terms and the gate)
static void test_block_norm(const mf::MetalContext& ctx) {
  const uint32_t t = 5, d = 100;
  const float eps = 1e-6f;
  const auto hidden = numbers(size_t(t) * d), delta = numbers(size_t(t) * d), post = numbers(d), pre = numbers(d), gate = numbers(t);
  auto* d_hidden = to_device(hidden);
  auto* d_out = to_device(std::vector<uint16_t>(size_t(t) * d));
  auto* d_delta = to_device(delta);
  auto* d_post = to_device(post);
  auto* d_pre = to_device(pre);
  auto* d_gate = to_device(gate);
  auto args = mf::BlockNorm::arguments(d_hidden, d_delta, t, d, eps);
  args.post_weight = d_post, args.pre_weight = d_pre, args.out = d_out, args.gate = d_gate, args.gate_kind = MF_GATE_ROW;
  args.branch_scale = 0.5f;
  const mf::BlockNorm norm(ctx);
  norm.encode(nullptr, args);
  HIP_OK(hipDeviceSynchronize());
  const auto h = to_host(d_hidden, size_t(t) * d), out = to_host(d_out, size_t(t) * d);
  for (uint32_t i = 0; i < t; ++i) {
    double sd = 0, sh = 0;
    for (uint32_t e = 0; e < d; ++e) sd += std::pow(widen(delta[i * d + e]), 2.0), sh += std::pow(widen(h[i * d + e]), 2.0);
    const double inv_d = 1 / std::sqrt(sd / d + eps), inv_h = 1 / std::sqrt(sh / d + eps), g = 0.5 / (1 + std::exp(-double(widen(gate[i]))));
    for (uint32_t e = 0; e < d; ++e) {
      const double old = widen(hidden[i * d + e]), b = g * widen(delta[i * d + e]) * inv_d * widen(post[e]), want = old + b;
      EXPECT(std::fabs(widen(h[i * d + e]) - want) <= std::fabs(want) * std::ldexp(1.0, -8) + (std::fabs(old) + std::fabs(b)) * std::ldexp(1.0, -16), "hidden %u %u", i, e);
      const double o = widen(h[i * d + e]) * inv_h * widen(pre[e]);
      EXPECT(std::fabs(widen(out[i * d + e]) - o) <= std::fabs(o) * (std::ldexp(1.0, -8) + std::ldexp(1.0, -16)), "out %u %u", i, e);
    }
  }
  args.out = nullptr;
  EXPECT(status_of([&] { norm.encode(nullptr, args); }) == MF_ERR_INVALID_ARGUMENT, "a norm without a place for its result");
  for (uint16_t* p : {d_hidden, d_out, d_delta, d_post, d_pre, d_gate}) HIP_OK(hipFree(p));
  std::printf("block norm: ok\n");
}

int main(int argc, char** argv) {
  const std::string mode = argc > 1 ? argv[1] : "cpu";
  test_sizes();
  if (mode == "gpu") {
    const mf::MetalContext ctx;
    for (bool float32 : {false, true})
      for (bool planned : {false, true}) test_adapters(ctx, float32, planned);
    test_block_norm(ctx);
  }
  if (g_fail) return 1;
  std::printf("adapters_test: ok\n");
  return 0;
}
