// gradients_host_test.cc -- what glx_mx_* and glx_gradients_* decide on the
// host, on two imagined GPUs: the HIP functions that these calls use are defined
// here, and an executable's definitions come before the runtime's, so every
// launch is written down and none happens.  Needs no GPU.
//   gradients_host_test CASE     exit status 0 = passed
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstring>
#include <map>
#include <string>
#include <utility>
#include <vector>

#include "gloo_amd/glx.h"

namespace {

int g_failures = 0;

#define EXPECT(cond)                                                       \
  do {                                                                     \
    if (!(cond)) {                                                         \
      std::fprintf(stderr, "FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      g_failures++;                                                        \
    }                                                                      \
  } while (0)

// ---- the imagined machine ---------------------------------------------------

// Addresses: a stretch of memory per GPU, one of pinned host memory; all others
// are pageable host memory.
constexpr uintptr_t kStretch = uintptr_t(1) << 44;
constexpr int kDevices = 2;
char* device(int d, size_t at) { return (char*)(kStretch * (d + 1) + at); }
char* pinned(size_t at) { return (char*)(kStretch * (kDevices + 1) + at); }
char* pageable(size_t at) { return (char*)(kStretch * (kDevices + 2) + at); }

struct Launch {
  std::string kernel;
  int device;
  hipStream_t stream;
  void** args;  // valid during the launch only
};
struct Machine {
  int current = 0, lookups = 0, frees = 0;
  size_t next = kStretch / 2;  // of hipMalloc
  hipError_t error = hipSuccess;
  hipStreamCaptureMode mode = hipStreamCaptureModeGlobal;
  std::vector<Launch> launches;
  void (*onLaunch)(const Launch&) = nullptr;
};
Machine m;

std::map<const void*, std::string>& kernels() {  // filled before main()
  static std::map<const void*, std::string> k;
  return k;
}

hipError_t left(hipError_t e) {
  if (e != hipSuccess) m.error = e;
  return e;
}

}  // namespace

extern "C" {

hipError_t hipGetLastError() {
  const hipError_t e = m.error;
  m.error = hipSuccess;
  return e;
}
hipError_t hipGetDevice(int* d) {
  *d = m.current;
  return hipSuccess;
}
hipError_t hipSetDevice(int d) {
  if (d < 0 || d >= kDevices) return left(hipErrorInvalidDevice);
  m.current = d;
  return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) {
  *v = 256;
  return hipSuccess;
}
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* a, const void* p) {
  m.lookups++;
  std::memset(a, 0, sizeof(*a));
  const uintptr_t s = (uintptr_t)p / kStretch;
  if (s < 1 || s > kDevices + 1) return left(hipErrorInvalidValue);
  a->type = s <= kDevices ? hipMemoryTypeDevice : hipMemoryTypeHost;
  a->device = s <= kDevices ? (int)s - 1 : 0;
  a->devicePointer = (void*)p;
  return hipSuccess;
}
hipError_t hipMalloc(void** p, size_t n) {
  *p = device(m.current, m.next);
  m.next += (n + 4095) / 4096 * 4096;
  return hipSuccess;
}
hipError_t hipMemcpy(void*, const void*, size_t, hipMemcpyKind) { return hipSuccess; }
hipError_t hipFree(void* p) {
  m.frees++;
  // a capture under way in any thread makes what is not relaxed fail
  EXPECT(m.mode == hipStreamCaptureModeRelaxed);
  EXPECT((uintptr_t)p / kStretch == (uintptr_t)m.current + 1);  // it waits for this device
  return hipSuccess;
}
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode* mode) {
  std::swap(m.mode, *mode);
  return hipSuccess;
}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*,
                           void*, void*, void*, int*) {
  kernels()[host] = name;
}
namespace {
dim3 g_grid, g_block;
size_t g_shared;
hipStream_t g_stream;
}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t s) {
  g_grid = grid, g_block = block, g_shared = shared, g_stream = s;
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* s) {
  *grid = g_grid, *block = g_block, *shared = g_shared, *s = g_stream;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3, dim3, void** args, size_t, hipStream_t s) {
  m.launches.push_back({kernels()[f], m.current, s, args});
  if (m.onLaunch != nullptr) m.onLaunch(m.launches.back());
  return hipSuccess;
}

}  // extern "C"

namespace {

const glx_stream_t kStream = (glx_stream_t)0x1234;

// A refusal: its message, nothing launched, the device as it was, and no error
// that the next HIP call would be taken to have made.
void refused(int line, int status, const char* message) {
  const bool ok = status == GLX_ERR_ENFORCE && std::strstr(glx_last_error(), message) != nullptr &&
                  m.launches.empty() && m.current == 0 && m.error == hipSuccess;
  if (!ok) {
    std::fprintf(stderr, "FAIL line %d: status %d, \"%s\" for \"%s\", %zu launches\n", line, status,
                 glx_last_error(), message, m.launches.size());
    g_failures++;
  }
  m.launches.clear();
  m.error = hipSuccess;
}
#define REFUSED(call, message) refused(__LINE__, call, message)

// One launch of a kernel on a device, and the current device back.
void launched(int line, int status, const char* kernel, int dev) {
  const bool ok = status == GLX_OK && m.launches.size() == 1 &&
                  m.launches[0].kernel.find(kernel) != std::string::npos &&
                  m.launches[0].device == dev && m.launches[0].stream == kStream && m.current == 0;
  if (!ok) {
    std::fprintf(stderr, "FAIL line %d: status %d \"%s\", %zu launches, the first %s on %d\n", line,
                 status, glx_last_error(), m.launches.size(),
                 m.launches.empty() ? "-" : m.launches[0].kernel.c_str(),
                 m.launches.empty() ? -1 : m.launches[0].device);
    g_failures++;
  }
  m.launches.clear();
}
#define LAUNCHED(call, kernel, dev) launched(__LINE__, call, kernel, dev)

// ---- cases ------------------------------------------------------------------

constexpr size_t kN = 4099, kMiB = 1 << 20;

void mxPointers() {
  const int f32 = GLX_FLOAT32;
  char *pay = device(0, 0), *x = device(0, kMiB), *r = device(0, 2 * kMiB), *host = pageable(0);
  float *ro = (float*)device(0, 3 * kMiB), *rf = (float*)r;
  auto quantize = [&](void* payload, void* src, void* res, float* out) {
    return glx_mx_quantize(f32, payload, src, (float*)res, out, kN, kStream);
  };
  REFUSED(quantize(host, x, r, ro), "not a device pointer");
  REFUSED(quantize(pay, host, r, ro), "x is");
  REFUSED(quantize(pay, x, host, ro), "residual is");
  REFUSED(quantize(pay, x, r, (float*)host), "residual_out is");
  REFUSED(quantize(pay, host, nullptr, nullptr), "x is");
  LAUNCHED(quantize(pay, x, r, ro), "quantize", 0);
  LAUNCHED(quantize(pay, x, r, rf), "quantize", 0);
  LAUNCHED(quantize(pay, x, nullptr, nullptr), "quantize", 0);
  // what a kernel reaches may be pinned host memory
  LAUNCHED(quantize(pay, pinned(0), r, (float*)pinned(kMiB)), "quantize", 0);
  LAUNCHED(quantize(device(1, 0), device(1, kMiB), nullptr, nullptr), "quantize", 1);

  for (int k = 1; k <= 16; k++) {
    std::vector<const void*> src;
    for (int j = 0; j < k; j++) src.push_back(device(0, (4 + j) * kMiB));
    auto reduce = [&](void* dst) {
      return glx_mx_reduce_n(f32, dst, src.data(), k, kN, 0.5f, kStream);
    };
    auto requantize = [&](void* to) {
      return glx_mx_requantize_n(to, src.data(), k, kN, 0.5f, kStream);
    };
    LAUNCHED(reduce(x), "reduce_n", 0);
    LAUNCHED(requantize(pay), "requantize_n", 0);
    LAUNCHED(requantize((void*)src[0]), "requantize_n", 0);
    REFUSED(reduce(host), "not a device pointer");
    REFUSED(requantize(host), "not a device pointer");
    for (int j = 0; j < k; j++) {
      const void* was = src[j];
      src[j] = host;
      const std::string name = "payload " + std::to_string(j) + " is";
      REFUSED(reduce(x), name.c_str());
      REFUSED(requantize(pay), name.c_str());
      src[j] = pinned(0);
      LAUNCHED(reduce(x), "reduce_n", 0);
      src[j] = was;
    }
  }
}

// The calls on a stated device look nothing up.
void mxOn() {
  const void* src[2] = {device(1, kMiB), device(1, 2 * kMiB)};
  m.lookups = 0;
  LAUNCHED(glx_mx_quantize_on(1, GLX_FLOAT32, device(1, 0), device(1, kMiB), nullptr, nullptr, kN,
                              kStream),
           "quantize", 1);
  LAUNCHED(glx_mx_reduce_n_on(1, GLX_BFLOAT16, device(1, 0), src, 2, kN, 1, kStream), "reduce_n",
           1);
  LAUNCHED(glx_mx_requantize_n_on(1, device(1, 0), src, 2, kN, 1, kStream), "requantize_n", 1);
  EXPECT(m.lookups == 0);
  REFUSED(glx_mx_reduce_n_on(-1, GLX_FLOAT32, device(1, 0), src, 2, kN, 1, kStream), "negative");
  REFUSED(glx_mx_requantize_n_on(1, device(1, kMiB + 16), src, 2, kN, 1, kStream), "overlaps");
  EXPECT(glx_mx_reduce_n_on(kDevices, GLX_FLOAT32, device(1, 0), src, 2, kN, 1, kStream) ==
         GLX_ERR_HIP);
  EXPECT(m.launches.empty() && m.current == 0);
}

// A list in device 0's memory: `n` tensors of `count` floats, `stride` bytes
// apart from `at` on; with `outs` clipped to as many others.
struct List {
  glx_gradients* g = nullptr;
  std::vector<void*> grads, outs;
  List(int n, size_t count, size_t stride, size_t at, long outsAt = -1) {
    for (int i = 0; i < n; i++) {
      grads.push_back(device(0, at + i * stride));
      if (outsAt >= 0) outs.push_back(device(0, outsAt + i * stride));
    }
    const std::vector<size_t> counts(n, count);
    const std::vector<int> types(n, GLX_FLOAT32);
    g = glx_gradients_create(grads.data(), outsAt < 0 ? nullptr : outs.data(), counts.data(),
                             types.data(), n);
    EXPECT(g != nullptr);
  }
  ~List() { glx_gradients_destroy(g); }
};

// Device memory, apart from the tensors and the scalar.
void workspace() {
  // three tensors of 4 MiB, 8 MiB apart from 64 MiB on; outputs from 128 MiB on
  const size_t at = 64 * kMiB, oat = 128 * kMiB, count = kMiB, step = 8 * kMiB;
  List list(3, count, step, at, oat);
  const size_t bytes = glx_gradients_workspace_bytes(list.g);
  EXPECT(bytes > 0 && bytes % 8 == 0);
  char *out = device(0, 0), *good = device(0, kMiB);
  void* sum = device(0, 64);
  using Call = int (*)(const List&, void* out, void* sum, void* ws);
  const Call calls[] = {
      [](const List& l, void* o, void*, void* w) {
        return glx_gradients_norm(l.g, 2, o, GLX_FLOAT32, w, kStream);
      },
      [](const List& l, void*, void* s, void* w) {
        return glx_gradients_power_sum(l.g, 1, s, w, kStream);
      },
      [](const List& l, void* o, void*, void* w) {
        return glx_gradients_clip(l.g, 1, 2, nullptr, o, GLX_FLOAT32, w, kStream);
      },
      [](const List& l, void*, void*, void* w) {
        return glx_gradients_clip(l.g, 1, 2, nullptr, nullptr, 0, w, kStream);
      },
  };
  for (const Call call : calls) {
    for (const size_t base : {at, oat}) {
      for (const size_t i : {0, 1, 2}) {
        char* t = device(0, base + i * step);
        char* end = t + count * 4;
        for (char* w : {t - bytes + 8, t, t + 4096, end - bytes, end - 8}) {
          REFUSED(call(list, out, sum, w), "workspace lies in a tensor");
        }
        for (char* w : {t - bytes, end}) {
          EXPECT(call(list, out, sum, w) == GLX_OK && m.launches.size() == 2);
          m.launches.clear();
        }
      }
    }
    REFUSED(call(list, out, sum, pageable(0)), "not a device pointer");
    REFUSED(call(list, out, sum, pinned(0)), "not a device pointer");
    REFUSED(call(list, out, sum, nullptr), "workspace is null");
    REFUSED(call(list, out, sum, good + 4), "misaligned");
    EXPECT(call(list, out, sum, good) == GLX_OK && m.launches.size() == 2);
    m.launches.clear();
  }
  REFUSED(calls[0](list, good + bytes - 8, sum, good), "in the workspace");
  // a workspace around a whole tensor
  List tiny(400, 16, 128, at);
  EXPECT(glx_gradients_workspace_bytes(tiny.g) > 400 * 4);
  REFUSED(calls[0](tiny, out, sum, device(0, at + 200 * 128 - 8)), "workspace lies in a tensor");
  // a power sum given: no partials
  LAUNCHED(glx_gradients_clip(list.g, 1, 2, sum, out, GLX_FLOAT32, nullptr, kStream), "clip", 0);
}

// Calls run where the tensors are, and scalars and workspaces are there too; a
// list without elements runs where its result goes.
void devices() {
  for (const bool tensors : {false, true}) {  // no tensors at all, and empty ones
    std::vector<void*> none(3, nullptr);
    const std::vector<size_t> counts(3, 0);
    const std::vector<int> types(3, GLX_BFLOAT16);
    glx_gradients* g =
        glx_gradients_create(none.data(), nullptr, counts.data(), types.data(), tensors ? 3 : 0);
    EXPECT(g != nullptr && glx_gradients_workspace_bytes(g) == 0);
    EXPECT(glx_gradients_device(g) == 0);  // the current one
    for (int d = 0; d < kDevices; d++) {
      void *out = device(d, 0), *sum = device(d, 64);
      LAUNCHED(glx_gradients_norm(g, 2, out, GLX_FLOAT32, nullptr, kStream), "short", d);
      LAUNCHED(glx_gradients_power_sum(g, 2, sum, nullptr, kStream), "short", d);
      LAUNCHED(glx_gradients_clip(g, 1, 2, nullptr, out, GLX_FLOAT32, nullptr, kStream), "short",
               d);
      LAUNCHED(glx_gradients_clip(g, 1, 2, sum, out, GLX_FLOAT32, nullptr, kStream), "clip", d);
      REFUSED(glx_gradients_clip(g, 1, 2, sum, device(1 - d, 0), GLX_FLOAT32, nullptr, kStream),
              "another device");
    }
    // neither tensors nor a result: nothing to do
    EXPECT(glx_gradients_clip(g, 1, 2, nullptr, nullptr, 0, nullptr, kStream) == GLX_OK);
    EXPECT(glx_gradients_clip(g, 1, 2, device(1, 0), nullptr, 0, nullptr, kStream) == GLX_OK);
    EXPECT(m.launches.empty());
    REFUSED(glx_gradients_clip(g, -1, 2, nullptr, nullptr, 0, nullptr, kStream), "max_norm");
    glx_gradients_destroy(g);
  }
  for (const size_t count : {10, 1 << 20}) {  // one workgroup, and many
    List list(3, count, 8 * kMiB, 64 * kMiB);
    EXPECT(glx_gradients_device(list.g) == 0);
    void *out = device(0, 0), *sum = device(0, 64), *ws = device(0, kMiB);
    void *far = device(1, 0), *farWs = device(1, kMiB);
    REFUSED(glx_gradients_norm(list.g, 2, far, GLX_FLOAT32, ws, kStream), "out is on another");
    REFUSED(glx_gradients_power_sum(list.g, 2, far, ws, kStream), "out is on another");
    REFUSED(glx_gradients_clip(list.g, 1, 2, nullptr, far, GLX_FLOAT32, ws, kStream),
            "norm is on another");
    REFUSED(glx_gradients_clip(list.g, 1, 2, far, out, GLX_FLOAT32, ws, kStream),
            "power_sum is on another");
    if (glx_gradients_workspace_bytes(list.g) > 0) {
      REFUSED(glx_gradients_norm(list.g, 2, out, GLX_FLOAT32, farWs, kStream),
              "workspace is on another");
      REFUSED(glx_gradients_clip(list.g, 1, 2, nullptr, nullptr, 0, farWs, kStream),
              "workspace is on another");
    }
    m.current = 1;  // another device is current
    EXPECT(glx_gradients_norm(list.g, 2, out, GLX_FLOAT32, ws, kStream) == GLX_OK);
    EXPECT(glx_gradients_clip(list.g, 1, 2, sum, nullptr, 0, nullptr, kStream) == GLX_OK);
    for (const Launch& l : m.launches) EXPECT(l.device == 0);
    EXPECT(m.launches.size() >= 2 && m.current == 1);
    m.launches.clear();
    m.current = 0;
  }
  void* two[2] = {device(0, 0), device(1, 0)};
  const size_t counts[2] = {4, 4};
  const int types[2] = {GLX_FLOAT32, GLX_FLOAT32};
  EXPECT(glx_gradients_create(two, nullptr, counts, types, 2) == nullptr &&
         std::strstr(glx_last_error(), "tensor 1 is on another device") != nullptr);
}

void destroy() {
  glx_gradients_destroy(nullptr);
  for (int d = 0; d < kDevices; d++) {
    void* p = device(d, 0);
    const size_t count = 1000;
    const int type = GLX_FLOAT32;
    glx_gradients* g = glx_gradients_create(&p, nullptr, &count, &type, 1);
    EXPECT(g != nullptr && m.frees == d && m.current == 0);
    glx_gradients_destroy(g);
    EXPECT(m.frees == d + 1 && m.current == 0 && m.mode == hipStreamCaptureModeGlobal);
  }
}

int g_chunks, g_streamed;  // of the last sum

void seeSum(const Launch& l) {
  if (l.kernel.find("power_partials") == std::string::npos) return;
  g_chunks = *(int*)l.args[1];
  g_streamed = *(int*)l.args[2];
}

// What a clip will read again is loaded to stay in the cache: the last 256 MiB,
// whatever the tensors' sizes.  A norm alone keeps nothing.
void cached() {
  m.onLaunch = seeSum;
  const size_t cache = 256 * kMiB;
  struct { int n; size_t count; } lists[] = {
      {50000, 1024}, {100000, 1024}, {300000, 250}, {64, kMiB}, {65, kMiB}, {300, kMiB + 1},
      {3, 100 * kMiB}, {1, 1 << 20}, {70000, 1025}};
  for (const auto& c : lists) {
    const size_t bytes = c.count * 4;
    List list(c.n, c.count, (bytes + 15) / 16 * 16, 4096 * kMiB);
    void *out = device(0, 0), *sum = device(0, 64), *ws = device(0, kMiB);
    EXPECT(glx_gradients_clip(list.g, 1, 2, nullptr, out, GLX_FLOAT32, ws, kStream) == GLX_OK);
    // whole chunks of 16 KiB, cut by the tensors' ends
    const size_t per = (bytes + 16383) / 16384, kept = g_chunks - g_streamed;
    EXPECT(bytes * c.n < 256 * kMiB || (size_t)g_chunks == per * c.n);
    size_t tail = 0;  // bytes of the kept chunks
    for (size_t i = 0; i < kept; i++) {
      tail += i % per == 0 && bytes % 16384 != 0 ? bytes % 16384 : 16384;
    }
    if (bytes * c.n <= cache) {
      EXPECT(g_streamed == 0);
    } else {
      EXPECT(tail <= cache && tail > cache - 16384);
    }
    const int clipped = g_streamed;
    EXPECT(glx_gradients_power_sum(list.g, 2, sum, ws, kStream) == GLX_OK);
    EXPECT(g_streamed == clipped);
    EXPECT(glx_gradients_norm(list.g, 2, out, GLX_FLOAT32, ws, kStream) == GLX_OK);
    EXPECT(g_streamed == g_chunks);
    m.launches.clear();
  }
}

const std::map<std::string, void (*)()> kCases = {
    {"mx_pointers", mxPointers},
    {"mx_on", mxOn},
    {"workspace", workspace},
    {"devices", devices},
    {"destroy", destroy},
    {"cached", cached},
};

}  // namespace

int main(int argc, char** argv) {
  const auto c = argc == 2 ? kCases.find(argv[1]) : kCases.end();
  if (c == kCases.end()) return 2;
  c->second();
  if (g_failures == 0) std::printf("passed\n");
  return g_failures == 0 ? 0 : 1;
}
