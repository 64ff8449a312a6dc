// gradients_test.cc -- gloo_amd.hpp's Gradients and mx on one GPU: values small
// enough to be exact, the header's refusals.  Exit status 0 = all passed.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <stdexcept>
#include <vector>

#include "gloo_amd/gloo_amd.hpp"

namespace {

int g_failures = 0;

#define EXPECT(cond)                                                  \
  do {                                                                \
    if (!(cond)) {                                                    \
      std::fprintf(stderr, "FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      g_failures++;                                                   \
    }                                                                 \
  } while (0)

template <typename T>
struct Device {
  T* p = nullptr;
  explicit Device(const std::vector<T>& v) {
    if (hipMalloc((void**)&p, v.size() * sizeof(T)) != hipSuccess ||
        hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) {
      throw std::runtime_error("device memory");
    }
  }
  ~Device() { (void)hipFree(p); }
  std::vector<T> get(size_t n) const {
    std::vector<T> v(n);
    if (hipDeviceSynchronize() != hipSuccess ||
        hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost) != hipSuccess) {
      throw std::runtime_error("copy back");
    }
    return v;
  }
};

void gradients() {
  using gloo_amd::Gradients;
  Device<float> a(std::vector<float>(1000, 3.0f));
  Device<gloo_amd::bfloat16> b(std::vector<gloo_amd::bfloat16>(
      4000, gloo_amd::bfloat16{0x3f80}));  // 1.0
  Device<float> out(std::vector<float>(1000, 0.0f));
  Gradients g(Gradients::List().add(a.p, 1000, out.p).add(b.p, 4000));
  EXPECT(g.device() == 0);
  Device<char> ws(std::vector<char>(g.workspaceBytes()));
  Device<float> norm({0.0f});
  Device<double> sum({0.0});
  g.powerSum(2, sum.p, ws.p, nullptr);
  EXPECT(sum.get(1)[0] == 13000.0);
  g.norm(1, norm.p, ws.p, nullptr);
  EXPECT(norm.get(1)[0] == 7000.0f);
  g.clipNorm(1e9, norm.p, ws.p, nullptr);  // nothing to clip: a copy, and in place
  EXPECT(out.get(1000)[999] == 3.0f && b.get(1)[0].x == 0x3f80);
  Device<double> four({4.0});
  g.clipNormOf(four.p, 1.0, norm.p, nullptr);  // norm 2 -> about a half
  EXPECT(norm.get(1)[0] == 2.0f);
  const float v = out.get(1000)[999];
  EXPECT(v > 1.49999f && v <= 1.5f && b.get(4000)[3999].x == 0x3f00);
  bool refused = false;
  try {
    g.norm(3, norm.p, ws.p, nullptr);
  } catch (const gloo_amd::EnforceNotMet&) {
    refused = true;
  }
  EXPECT(refused);
}

void messages() {
  const size_t n = 100;
  std::vector<float> x(n);
  for (size_t i = 0; i < n; i++) x[i] = (float)((int)(i % 13) - 6);  // -6..6
  Device<float> d(x), back(std::vector<float>(n, 0.0f));
  Device<char> p(std::vector<char>(gloo_amd::mx::payloadBytes(n), 1));
  Device<char> q(std::vector<char>(gloo_amd::mx::payloadBytes(n), 1));
  gloo_amd::mx::quantize(p.p, d.p, n, nullptr);
  gloo_amd::mx::reduceN(back.p, {p.p, p.p}, n, nullptr, 0.5f);
  std::vector<float> y = back.get(n);
  for (size_t i = 0; i < n; i++) {
    const float want = x[i] == 5 ? 4 : x[i] == -5 ? -4 : x[i];
    EXPECT(y[i] == want);
  }
  gloo_amd::mx::requantizeN(q.p, {p.p}, n, nullptr);
  EXPECT(q.get(gloo_amd::mx::payloadBytes(n)) == p.get(gloo_amd::mx::payloadBytes(n)));
}

}  // namespace

int main() {
  try {
    gradients();
    messages();
  } catch (const std::exception& e) {
    std::fprintf(stderr, "FAIL: %s\n", e.what());
    return 1;
  }
  if (g_failures == 0) std::printf("all passed\n");
  return g_failures == 0 ? 0 : 1;
}
