// gradients.cc -- GradientList: checks, the chunk table, the calls.
#include "gradients.h"

#include <algorithm>
#include <cmath>

#include "common.h"

namespace gloo {

namespace {

// Lists of up to 64 chunks of 4 KiB are summed by one workgroup (64 chunks of f32:
// 4.2 us, two launches 6.1), but only half as many are also clipped by it: the
// CU that does it alone needs 6.1 us for 32 chunks and 7.7 for 64, of 16-bit
// values 9.1, two launches 6.4 for any of them.
constexpr int kShortClipChunks = 32;
constexpr size_t kCachedBytes = size_t(256) << 20;  // the Infinity Cache

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

bool aligned(const void* p, int dtype) { return (uintptr_t)p % elementSize(dtype) == 0; }

using Span = GradientList::Span;

// Every byte is written by at most one tensor, and none that another reads.
void checkOverlap(std::vector<Span>& spans) {
  std::sort(spans.begin(), spans.end(),
            [](const Span& a, const Span& b) { return a.at < b.at; });
  for (size_t i = 1; i < spans.size(); i++) {
    GLX_ENFORCE(spans[i - 1].end <= spans[i].at, "gradients: tensors ", spans[i - 1].tensor,
                " and ", spans[i].tensor, " share memory",
                spans[i - 1].out != spans[i].out ? " (a gradient and an output)" : "");
  }
}

}  // namespace

namespace {

hipPointerAttribute_t attributesOf(const void* p) {
  hipPointerAttribute_t a;
  if (hipPointerGetAttributes(&a, p) != hipSuccess) {
    (void)hipGetLastError();  // not the next launch's error
    a.type = hipMemoryTypeUnregistered;
  }
  return a;
}

}  // namespace

int deviceOf(const void* p) {
  const hipPointerAttribute_t a = attributesOf(p);
  GLX_ENFORCE(a.type == hipMemoryTypeDevice, "not a device pointer");
  return a.device;
}

bool reachable(const void* p) { return attributesOf(p).type != hipMemoryTypeUnregistered; }

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
  std::vector<Span>& spans = spans_;
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

  // Chunks of 16 KiB, one pass of a workgroup's loads, cut at 16-byte boundaries
  // of the gradient; shorter where that would leave workgroups without one.
  const size_t groups = (size_t)std::max(cus, 1) * 4;
  const size_t chunk = std::min<size_t>(
      16 << 10, std::max(glx::kGradShortBytes, bytes / groups / 4096 * 4096));
  std::vector<glx::GradChunk> table;
  for (size_t i = 0; i < grads.size(); i++) {
    const size_t es = elementSize(dtypes[i]), per = chunk / es;
    char* g = (char*)grads[i];
    char* o = outs.empty() ? g : (char*)outs[i];
    const size_t lead = (uintptr_t)g % 16 / es;
    for (size_t at = 0, n; at < counts[i]; at += n) {
      n = std::min(at == 0 ? per - lead : per, counts[i] - at);
      table.push_back({g + at * es, o + at * es, (uint32_t)n, (uint32_t)dtypes[i]});
    }
  }
  // one workgroup of 256 threads per chunk, below 2^32 threads
  GLX_ENFORCE(table.size() < (size_t(1) << 24) - 8, "gradients: the list is too long");
  nchunks_ = (int)table.size();
  short_ = nchunks_ <= glx::kGradShortChunks && chunk <= glx::kGradShortBytes;
  shortClip_ = short_ && nchunks_ <= kShortClipChunks;
  // The last chunks that fit the cache together stay.  Counted in bytes, since a
  // tensor's last chunk may be short: clip of 50000 tensors of 4 KiB 141 us, 151 if
  // each were taken for 16 KiB.
  streamed_ = nchunks_;
  for (size_t kept = 0; streamed_ > 0; streamed_--) {
    const glx::GradChunk& c = table[streamed_ - 1];
    kept += c.n * elementSize(c.dtype);
    if (kept > kCachedBytes) break;
  }
  grid_ = (int)std::max<size_t>(1, std::min(table.size(), groups));
  if (nchunks_ > 0) {
    const size_t n = table.size() * sizeof(glx::GradChunk);
    hipError_t e = hipMalloc((void**)&chunks_, n);
    if (e == hipSuccess) {
      e = hipMemcpy(chunks_, table.data(), n, hipMemcpyHostToDevice);
      if (e != hipSuccess) (void)hipFree(chunks_);
    }
    if (e != hipSuccess) (void)hipGetLastError();  // not the next launch's error
    GLX_HIP_CHECK(e);
  }
}

// hipFree waits for the device's work first.  It runs in the relaxed mode: a
// capture that this thread or another one has under way, of a graph that need not
// know the list, would be lost to it otherwise.
GradientList::~GradientList() {
  if (chunks_ == nullptr) return;
  int cur = device_;
  (void)hipGetDevice(&cur);
  if (cur != device_) (void)hipSetDevice(device_);
  hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
  const bool relaxed = hipThreadExchangeStreamCaptureMode(&mode) == hipSuccess;
  const hipError_t e = hipFree(chunks_);
  if (relaxed) (void)hipThreadExchangeStreamCaptureMode(&mode);
  if (cur != device_) (void)hipSetDevice(cur);
  if (e != hipSuccess) (void)hipGetLastError();  // not the next launch's error
}

// Memory of a call outside the tensors, which other workgroups read and write.
void GradientList::checkApart(const void* p, size_t bytes, const char* what) const {
  const uintptr_t at = (uintptr_t)p, end = at + bytes;
  // spans_ is sorted and without overlap: only the last one that begins before
  // the end can reach it
  auto i = std::lower_bound(spans_.begin(), spans_.end(), end,
                            [](const Span& s, uintptr_t e) { return s.at < e; });
  GLX_ENFORCE(i == spans_.begin() || (i - 1)->end <= at, "gradients: ", what,
              " lies in a tensor's memory");
}

// The device of p, which is that of the tensors, if there are any.
int GradientList::checkPlace(const void* p, const char* what) const {
  const int device = deviceOf(p);
  GLX_ENFORCE(nchunks_ == 0 || device == device_, "gradients: ", what,
              " is on another device than the tensors");
  return device;
}

// A scalar outside the tensors, on their device; returns the device.
int GradientList::checkScalar(const void* p, int dtype, const char* what) const {
  GLX_ENFORCE(dtype == GLX_FLOAT32 || dtype == GLX_FLOAT64, "gradients: ", what,
              " is a float32 or float64");
  GLX_ENFORCE(p != nullptr && aligned(p, dtype), "gradients: ", what, " is null or misaligned");
  checkApart(p, elementSize(dtype), what);
  return checkPlace(p, what);
}

// The partials' memory: on the tensors' device, apart from them and the result.
void GradientList::checkWorkspace(const void* p, const void* scalar) const {
  GLX_ENFORCE(p != nullptr && aligned(p, GLX_FLOAT64),
              "gradients: workspace is null or misaligned");
  const size_t bytes = (size_t)grid_ * sizeof(double);
  const uintptr_t w = (uintptr_t)p, end = w + bytes;
  const uintptr_t q = (uintptr_t)scalar;
  GLX_ENFORCE(scalar == nullptr || q < w || q >= end,
              "gradients: a scalar lies in the workspace");
  checkApart(p, bytes, "workspace");
  checkPlace(p, "workspace");
}

void GradientList::sum(int kind, bool root, int streamed, void* out, int outDtype,
                       void* workspace, hipStream_t s) const {
  const int device = checkScalar(out, outDtype, "out");
  if (!short_) checkWorkspace(workspace, out);
  DeviceScope scope(device);
  if (short_) {
    GLX_HIP_CHECK(
        glx::launch_short(kind, chunks_, nchunks_, false, 0, root, out, outDtype, s));
    return;
  }
  double* part = (double*)workspace;
  GLX_HIP_CHECK(
      glx::launch_power_partials(kind, chunks_, nchunks_, streamed, grid_, part, s));
  GLX_HIP_CHECK(glx::launch_power_finish(kind, part, grid_, root, out, outDtype, s));
}

void GradientList::powerSum(double p, void* out, void* workspace, hipStream_t s) const {
  sum(kindOf(p), false, streamed_, out, GLX_FLOAT64, workspace, s);  // a clip will follow
}

void GradientList::norm(double p, void* out, int outDtype, void* workspace,
                        hipStream_t s) const {
  sum(kindOf(p), true, nchunks_, out, outDtype, workspace, s);
}

void GradientList::clip(double maxNorm, double p, const void* powerSum, void* out, int outDtype,
                        void* workspace, hipStream_t s) const {
  const int kind = kindOf(p);
  GLX_ENFORCE(maxNorm >= 0, "gradients: max_norm is a number >= 0, not ", maxNorm);
  int device = device_;
  if (out != nullptr) device = checkScalar(out, outDtype, "norm");
  if (powerSum != nullptr) {
    const int place = checkScalar(powerSum, GLX_FLOAT64, "power_sum");
    GLX_ENFORCE(out == nullptr || place == device,
                "gradients: norm is on another device than power_sum");
    const uintptr_t q = (uintptr_t)powerSum, o = (uintptr_t)out;
    GLX_ENFORCE(out == nullptr || o + elementSize(outDtype) <= q || o >= q + sizeof(double),
                "gradients: norm and power_sum share memory");
  } else if (!shortClip_) {
    checkWorkspace(workspace, out);
  }
  if (nchunks_ == 0 && out == nullptr) return;
  DeviceScope scope(device);
  const double* part = (const double*)powerSum;
  int nparts = 1;
  if (part == nullptr) {
    if (shortClip_) {
      GLX_HIP_CHECK(
          glx::launch_short(kind, chunks_, nchunks_, true, maxNorm, true, out, outDtype, s));
      return;
    }
    GLX_HIP_CHECK(glx::launch_power_partials(kind, chunks_, nchunks_, streamed_, grid_,
                                             (double*)workspace, s));
    part = (const double*)workspace;
    nparts = grid_;
  }
  GLX_HIP_CHECK(glx::launch_clip(kind, chunks_, nchunks_, part, nparts, maxNorm, out, outDtype,
                                 s));
}

}  // namespace gloo
