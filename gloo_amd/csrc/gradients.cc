// gradients.cc -- GradientList: checks, the chunk table, the calls.
#include "gradients.h"

#include <algorithm>
#include <cmath>

#include "common.h"

namespace gloo {

namespace {

size_t elementSize(int dtype) {
  switch (dtype) {
    case GLX_FLOAT64: return 8;
    case GLX_FLOAT32: return 4;
    case GLX_FLOAT16:
    case GLX_BFLOAT16: return 2;
  }
  return 0;
}

int kindOf(double p) {
  if (p == 2.0) return glx::kGradNorm2;
  if (p == 1.0) return glx::kGradNorm1;
  GLX_ENFORCE(std::isinf(p) && p > 0, "gradients: the norm is 1, 2 or infinity, not ", p);
  return glx::kGradNormInf;
}

void checkOut(const void* out, int dtype) {
  GLX_ENFORCE(dtype == GLX_FLOAT32 || dtype == GLX_FLOAT64,
              "gradients: the norm is written as float32 or float64");
  GLX_ENFORCE((uintptr_t)out % (dtype == GLX_FLOAT32 ? 4 : 8) == 0,
              "gradients: misaligned scalar");
}

struct Span {
  uintptr_t at, end;
  size_t tensor;
  bool out;
};

// Every byte is written by at most one tensor, and none that another reads.
void checkOverlap(std::vector<Span> spans) {
  std::sort(spans.begin(), spans.end(),
            [](const Span& a, const Span& b) { return a.at < b.at; });
  for (size_t i = 1; i < spans.size(); i++) {
    GLX_ENFORCE(spans[i - 1].end <= spans[i].at, "gradients: tensors ", spans[i - 1].tensor,
                " and ", spans[i].tensor, " share memory",
                spans[i - 1].out != spans[i].out ? " (a gradient and an output)" : "");
  }
}

}  // namespace

int deviceOf(const void* p) {
  hipPointerAttribute_t a;
  GLX_HIP_CHECK(hipPointerGetAttributes(&a, p));
  GLX_ENFORCE(a.type == hipMemoryTypeDevice, "not a device pointer");
  return a.device;
}

DeviceScope::DeviceScope(int device) {
  int cur = -1;
  if (device < 0 || hipGetDevice(&cur) != hipSuccess || cur == device) return;
  GLX_HIP_CHECK(hipSetDevice(device));
  was_ = cur;
}

DeviceScope::~DeviceScope() {
  if (was_ >= 0) (void)hipSetDevice(was_);
}

GradientList::GradientList(const std::vector<void*>& grads, const std::vector<void*>& outs,
                           const std::vector<size_t>& counts, const std::vector<int>& dtypes) {
  std::vector<Span> spans;
  size_t bytes = 0;
  for (size_t i = 0; i < grads.size(); i++) {
    const size_t es = elementSize(dtypes[i]);
    GLX_ENFORCE(es != 0, "gradients: tensor ", i, " is not of a floating type");
    if (counts[i] == 0) continue;
    GLX_ENFORCE(counts[i] <= (size_t(1) << 60) / es, "gradients: tensor ", i, " is too long");
    const size_t len = counts[i] * es;
    const uintptr_t g = (uintptr_t)grads[i], o = outs.empty() ? g : (uintptr_t)outs[i];
    GLX_ENFORCE(g != 0 && o != 0, "gradients: tensor ", i, " has no memory");
    GLX_ENFORCE(g % es == 0 && o % es == 0, "gradients: tensor ", i,
                " is not aligned to its elements");
    spans.push_back({g, g + len, i, false});
    if (o != g) spans.push_back({o, o + len, i, true});
    bytes += len;
  }
  checkOverlap(spans);

  if (spans.empty()) {
    GLX_HIP_CHECK(hipGetDevice(&device_));
  } else {
    device_ = deviceOf((void*)spans[0].at);
    for (const Span& p : spans) {
      GLX_ENFORCE(deviceOf((void*)p.at) == device_, "gradients: tensor ", p.tensor,
                  " is on another device");
    }
  }
  DeviceScope scope(device_);
  int cus = 0;
  GLX_HIP_CHECK(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device_));

  // Chunks of 64 KiB, shorter for lists too small to give every workgroup one.
  const size_t groups = (size_t)std::max(cus, 1) * 8;
  const size_t chunk =
      std::min<size_t>(64 << 10, std::max<size_t>(4 << 10, bytes / groups / 4096 * 4096));
  std::vector<glx::GradChunk> table;
  for (size_t i = 0; i < grads.size(); i++) {
    const size_t es = elementSize(dtypes[i]), per = chunk / es;
    char* g = (char*)grads[i];
    char* o = outs.empty() ? g : (char*)outs[i];
    for (size_t at = 0; at < counts[i]; at += per) {
      table.push_back({g + at * es, o + at * es, (uint32_t)std::min(per, counts[i] - at),
                       (uint32_t)dtypes[i]});
    }
  }
  GLX_ENFORCE(table.size() < (size_t(1) << 31), "gradients: the list is too long");
  nchunks_ = (int)table.size();
  grid_ = (int)std::max<size_t>(1, std::min(table.size(), groups));
  if (nchunks_ > 0) {
    const size_t n = table.size() * sizeof(glx::GradChunk);
    GLX_HIP_CHECK(hipMalloc((void**)&chunks_, n));
    const hipError_t e = hipMemcpy(chunks_, table.data(), n, hipMemcpyHostToDevice);
    if (e != hipSuccess) (void)hipFree(chunks_);
    GLX_HIP_CHECK(e);
  }
}

GradientList::~GradientList() {
  if (chunks_ != nullptr) (void)hipFree(chunks_);
}

void GradientList::powerSum(double p, void* sum, void* workspace, hipStream_t s) const {
  const int kind = kindOf(p);
  GLX_ENFORCE(sum != nullptr && workspace != nullptr, "gradients: null pointer");
  checkOut(sum, GLX_FLOAT64);
  checkOut(workspace, GLX_FLOAT64);
  DeviceScope scope(device_);
  double* part = (double*)workspace;
  GLX_HIP_CHECK(glx::launch_power_partials(kind, chunks_, nchunks_, grid_, part, s));
  GLX_HIP_CHECK(glx::launch_power_finish(kind, part, grid_, false, sum, GLX_FLOAT64, s));
}

void GradientList::norm(double p, void* out, int outDtype, void* workspace,
                        hipStream_t s) const {
  const int kind = kindOf(p);
  GLX_ENFORCE(out != nullptr && workspace != nullptr, "gradients: null pointer");
  checkOut(out, outDtype);
  checkOut(workspace, GLX_FLOAT64);
  DeviceScope scope(device_);
  double* part = (double*)workspace;
  GLX_HIP_CHECK(glx::launch_power_partials(kind, chunks_, nchunks_, grid_, part, s));
  GLX_HIP_CHECK(glx::launch_power_finish(kind, part, grid_, true, out, outDtype, s));
}

void GradientList::clip(double maxNorm, double p, const void* powerSum, void* out, int outDtype,
                        void* workspace, hipStream_t s) const {
  const int kind = kindOf(p);
  GLX_ENFORCE(maxNorm >= 0, "gradients: max_norm is a number >= 0, not ", maxNorm);
  GLX_ENFORCE(powerSum != nullptr || workspace != nullptr, "gradients: null workspace");
  checkOut(out, outDtype);
  checkOut(powerSum != nullptr ? powerSum : workspace, GLX_FLOAT64);
  DeviceScope scope(device_);
  const double* part = (const double*)powerSum;
  int nparts = 1;
  if (part == nullptr) {
    GLX_HIP_CHECK(glx::launch_power_partials(kind, chunks_, nchunks_, grid_, (double*)workspace,
                                             s));
    part = (const double*)workspace;
    nparts = grid_;
  }
  GLX_HIP_CHECK(glx::launch_clip(kind, chunks_, nchunks_, grid_, part, nparts, maxNorm, out,
                                 outDtype, s));
}

}  // namespace gloo
