// Drives the operators of layers kept in 16 bits through include/mfmoe.hpp and checks them against loops in 64 bits.
//
//   dense16_test cpu   sizes and refusals (no GPU needed)
//   dense16_test gpu   a projection, head norms, a layer of experts
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
// a number of [-1, 1) in steps of 1/64: exact in bf16
static uint32_t g_state = 4711;
static uint16_t next_number() {
  g_state = g_state * 1664525u + 1013904223u;
  const float f = static_cast<float>(static_cast<int>(g_state >> 25) - 64) / 64.0f;
  uint32_t w;
  std::memcpy(&w, &f, 4);
  return static_cast<uint16_t>(w >> 16);
}
static std::vector<uint16_t> numbers(size_t n) {
  std::vector<uint16_t> v(n);
  for (auto& x : v) x = next_number();
  return v;
}
// one rounding to bf16 (2^-8) and fp32 sums of numbers of that size (1e-4 of the largest partial sums here)
static bool near(float got, double want) { return std::fabs(got - want) <= std::fabs(want) / 256.0 + 2e-3; }

template <typename F> static mf_status status_of(F f) {
  try {
    f();
  } catch (const mf::Error& e) {
    return e.status;
  }
  return MF_OK;
}

static void test_sizes() {
  EXPECT(mf_project_workspace_bytes(0, 64, 1, 0) == 0, "no rows of W");
  mf_bf16_expert_pool p{};
  p.num_experts = 4, p.top_k = 2, p.d = 64, p.f = 32;
  EXPECT(mf_bf16_experts_workspace_bytes(&p, 5) > 0, "five tokens");
  EXPECT(mf_bf16_experts_workspace_bytes(&p, MF_BF16_EXPERTS_ROWS + 1) == 0, "too many tokens");
  p.f = 30;
  EXPECT(mf_bf16_experts_workspace_bytes(&p, 5) == 0, "a width that is no multiple of 8");
  EXPECT(mf_project(nullptr, nullptr, nullptr, nullptr, 0) == MF_ERR_INVALID_ARGUMENT, "null");
  EXPECT(mf_head_norms(nullptr, nullptr, nullptr) == MF_ERR_INVALID_ARGUMENT, "null");
  EXPECT(mf_bf16_experts(nullptr, nullptr, nullptr, nullptr, 0, nullptr, nullptr, nullptr, 0, 0, nullptr, 0, nullptr, 0) == MF_ERR_INVALID_ARGUMENT, "null");
  std::printf("sizes and refusals: ok\n");
}

static void test_projection(const mf::MetalContext& ctx) {
  const uint32_t t = 5, m = 37, n = 72;
  const auto x = numbers(t * n), w = numbers(2 * m * n), b = numbers(2 * m), r = numbers(t * m);
  uint16_t *dx = to_device(x), *dw = to_device(w), *db = to_device(b), *dr = to_device(r);
  const mf::Projection op(ctx, dw, m, n, db, MF_ACT_SILU, true);
  EXPECT(status_of([&] { op.encode(nullptr, dx, t, dx); }) == MF_ERR_INVALID_ARGUMENT, "x as the result");
  op.encode(nullptr, dx, t, dr, false, dr);  // in place
  HIP_OK(hipDeviceSynchronize());
  const auto y = to_host(dr, t * m);
  for (uint32_t i = 0; i < t; ++i)
    for (uint32_t j = 0; j < m; ++j) {
      double z = widen(b[j]), u = widen(b[m + j]);
      for (uint32_t k = 0; k < n; ++k) z += static_cast<double>(widen(x[i * n + k])) * widen(w[j * n + k]), u += static_cast<double>(widen(x[i * n + k])) * widen(w[(m + j) * n + k]);
      const double want = widen(r[i * m + j]) + z / (1.0 + std::exp(-z)) * u;
      EXPECT(near(widen(y[i * m + j]), want), "row %u column %u: %g, not %g", i, j, widen(y[i * m + j]), want);
    }
  for (void* p : {dx, dw, db, dr}) HIP_OK(hipFree(p));
  std::printf("projection: ok\n");
}

static void test_head_norms(const mf::MetalContext& ctx) {
  const uint32_t t = 3, heads = 4, dim = 32, pairs = 8;
  const auto q = numbers(t * heads * dim), w = numbers(dim);
  const std::vector<int32_t> positions = {100000, 7, 0, 3, 1, 2};  // two axes
  std::vector<float> freq(pairs);
  std::vector<uint8_t> axis(pairs);
  for (uint32_t p = 0; p < pairs; ++p) freq[p] = std::pow(10000.0f, -static_cast<float>(p) / pairs), axis[p] = p % 2;
  uint16_t *dq = to_device(q), *dw = to_device(w);
  int32_t* dp = to_device(positions);
  float* df = to_device(freq);
  uint8_t* da = to_device(axis);
  auto a = mf::HeadNorms::arguments(dq, heads, t, dim, dw, 1e-6f);
  a.positions = dp, a.inv_freq = df, a.axis_of_pair = da, a.rotary_dim = 2 * pairs, a.axes = 2;
  const mf::HeadNorms op(ctx);
  auto bad = a;
  bad.rotary_dim = 34;
  EXPECT(status_of([&] { op.encode(nullptr, bad); }) == MF_ERR_DIMENSION_MISMATCH, "more rotated than there is");
  op.encode(nullptr, a);
  HIP_OK(hipDeviceSynchronize());
  const auto y = to_host(dq, t * heads * dim);
  for (uint32_t i = 0; i < t; ++i)
    for (uint32_t h = 0; h < heads; ++h) {
      const uint16_t* from = &q[(i * heads + h) * dim];
      double squares = 0, z[32], want[32];
      for (uint32_t e = 0; e < dim; ++e) squares += static_cast<double>(widen(from[e])) * widen(from[e]);
      for (uint32_t e = 0; e < dim; ++e) want[e] = z[e] = widen(from[e]) / std::sqrt(squares / dim + 1e-6) * widen(w[e]);
      for (uint32_t p = 0; p < pairs; ++p) {
        const double angle = static_cast<double>(positions[axis[p] * t + i]) * freq[p], c = std::cos(angle), s = std::sin(angle);
        want[p] = z[p] * c - z[p + pairs] * s;
        want[p + pairs] = z[p + pairs] * c + z[p] * s;
      }
      for (uint32_t e = 0; e < dim; ++e) {
        const float got = widen(y[(i * heads + h) * dim + e]);
        EXPECT(near(got, want[e]), "row %u head %u element %u: %g, not %g", i, h, e, got, want[e]);
      }
    }
  for (void* p : {static_cast<void*>(dq), static_cast<void*>(dw), static_cast<void*>(dp), static_cast<void*>(df), static_cast<void*>(da)}) HIP_OK(hipFree(p));
  std::printf("head norms: ok\n");
}

static void test_experts(const mf::MetalContext& ctx) {
  const uint32_t t = 3, d = 40, f = 24, e = 5, k = 2;
  const auto x = numbers(t * d), up = numbers(e * 2 * f * d), down = numbers(e * d * f);
  const std::vector<uint32_t> idx = {4, 0, 1, 4, 9, 2};  // 9: no expert
  const std::vector<float> w = {0.5f, 0.25f, 1.0f, -0.5f, 3.0f, 0.125f};
  mf_bf16_expert_pool pool{};
  uint16_t *dup = to_device(up), *ddown = to_device(down), *dx = to_device(x), *dy = to_device(std::vector<uint16_t>(t * d, 0x7FC0));
  uint32_t* di = to_device(idx);
  float* dw = to_device(w);
  pool.gate_up = dup, pool.down = ddown, pool.num_experts = e, pool.top_k = k, pool.d = d, pool.f = f, pool.activation = MF_ACT_GELU_TANH;
  const mf::Bf16Experts op(ctx, pool);
  void* ws = nullptr;
  HIP_OK(hipMalloc(&ws, op.workspaceBytes(t)));
  EXPECT(status_of([&] { op.encode(nullptr, dx, di, dw, t, dy, nullptr, ws, op.workspaceBytes(t) - 1); }) == MF_ERR_SCRATCH_TOO_SMALL, "a short workspace");
  op.encode(nullptr, dx, di, dw, t, dy, nullptr, ws, op.workspaceBytes(t));
  HIP_OK(hipDeviceSynchronize());
  const auto y = to_host(dy, t * d);
  for (uint32_t i = 0; i < t; ++i) {
    std::vector<double> want(d, 0.0);
    for (uint32_t r = 0; r < k; ++r) {
      const uint32_t ex = idx[i * k + r];
      if (ex >= e) continue;
      for (uint32_t j = 0; j < f; ++j) {
        double g = 0, u = 0;
        for (uint32_t c = 0; c < d; ++c) g += static_cast<double>(widen(x[i * d + c])) * widen(up[(ex * 2 * f + j) * d + c]), u += static_cast<double>(widen(x[i * d + c])) * widen(up[(ex * 2 * f + f + j) * d + c]);
        const double a = 0.5 * g * (1.0 + std::tanh(std::sqrt(2.0 / M_PI) * (g + 0.044715 * g * g * g))) * u;
        for (uint32_t o = 0; o < d; ++o) want[o] += w[i * k + r] * a * widen(down[(ex * d + o) * f + j]);
      }
    }
    for (uint32_t o = 0; o < d; ++o) EXPECT(near(widen(y[i * d + o]), want[o]), "row %u column %u: %g, not %g", i, o, widen(y[i * d + o]), want[o]);
  }
  for (void* p : {static_cast<void*>(dup), static_cast<void*>(ddown), static_cast<void*>(dx), static_cast<void*>(dy), static_cast<void*>(di), static_cast<void*>(dw), ws}) HIP_OK(hipFree(p));
  std::printf("experts: ok\n");
}

int main(int argc, char** argv) {
  const std::string mode = argc > 1 ? argv[1] : "";
  if (mode == "cpu") {
    test_sizes();
  } else if (mode == "gpu") {
    const mf::MetalContext ctx(0);
    test_projection(ctx);
    test_head_norms(ctx);
    test_experts(ctx);
  } else {
    std::printf("usage: dense16_test cpu|gpu\n");
    return 2;
  }
  if (!g_fail) std::printf("dense16_test: ok\n");
  return g_fail ? 1 : 0;
}
