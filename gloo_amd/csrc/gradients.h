// gradients.h -- the global norm of a list of gradient tensors, and clipping
// by it: the host side (gradients.cc) and the kernels' launchers
// (gradient_kernels.hip).
#pragma once

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include <vector>

namespace glx {

// What one workgroup takes at a time: n elements of one tensor, and where
// their clipped values go (dst == src: in place).
struct GradChunk {
  const void* src;
  void* dst;
  uint32_t n;
  uint32_t dtype;
};

// The most chunks, of kGradShortBytes at most, that one workgroup does alone.
constexpr int kGradShortChunks = 64;
constexpr size_t kGradShortBytes = 4 << 10;

constexpr int kGradNorm1 = 0, kGradNorm2 = 1, kGradNormInf = 2;

// part[b] = sum of |x|^p (maximum for inf) over workgroup b's chunks, in
// double.  grid workgroups; part has grid words.  The first `streamed` chunks are
// read past the caches, the others to stay there for a clip.
hipError_t launch_power_partials(int kind, const GradChunk* chunks, int nchunks, int streamed,
                                 int grid, double* part, hipStream_t s);
// The fold of nparts partials: the power sum itself (root = false, out double)
// or the norm (root = true, out float or double by outDtype).
hipError_t launch_power_finish(int kind, const double* part, int nparts, bool root, void* out,
                               int outDtype, hipStream_t s);
// dst = x * min(1, maxNorm / (norm + 1e-6)) over all chunks, the norm folded
// from the partials; the norm to `out` if not null.
hipError_t launch_clip(int kind, const GradChunk* chunks, int nchunks, const double* part,
                       int nparts, double maxNorm, void* out, int outDtype, hipStream_t s);
// Power sum or norm (root) to `out` if not null, and with `clip` the clipping
// too (root is true then), in one launch of one workgroup.  At most
// kGradShortChunks chunks of at most kGradShortBytes.
hipError_t launch_short(int kind, const GradChunk* chunks, int nchunks, bool clip,
                        double maxNorm, bool root, void* out, int outDtype, hipStream_t s);

}  // namespace glx

namespace gloo {

// The current device, set to `device` (if >= 0) for a scope.
class DeviceScope {
 public:
  explicit DeviceScope(int device);
  ~DeviceScope();
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int was_ = -1;
};

// The device whose memory p is in (EnforceNotMet: not device memory).
int deviceOf(const void* p);

// Whether kernels can reach p: memory of a device, or host memory pinned for it.
bool reachable(const void* p);

// A list of gradient tensors on one device, laid out once into a table of
// chunks in device memory.  Read-only afterwards: any number of calls may run
// at once, each with a workspace of its own.
class GradientList {
 public:
  struct Span {  // memory of a tensor
    uintptr_t at, end;
    size_t tensor;
    bool out;
  };

  GradientList(const std::vector<void*>& grads, const std::vector<void*>& outs,
               const std::vector<size_t>& counts, const std::vector<int>& dtypes);
  ~GradientList();
  GradientList(const GradientList&) = delete;
  GradientList& operator=(const GradientList&) = delete;

  int device() const { return device_; }
  size_t workspaceBytes() const { return shortClip_ ? 0 : (size_t)grid_ * sizeof(double); }
  void powerSum(double p, void* sum, void* workspace, hipStream_t s) const;
  void norm(double p, void* out, int outDtype, void* workspace, hipStream_t s) const;
  void clip(double maxNorm, double p, const void* powerSum, void* out, int outDtype,
            void* workspace, hipStream_t s) const;

 private:
  void sum(int kind, bool root, int streamed, void* out, int outDtype, void* workspace,
           hipStream_t s) const;

  void checkApart(const void* p, size_t bytes, const char* what) const;
  int checkPlace(const void* p, const char* what) const;
  int checkScalar(const void* p, int dtype, const char* what) const;
  void checkWorkspace(const void* p, const void* scalar) const;

  std::vector<Span> spans_;  // sorted
  int device_ = 0;  // of the tensors; without any, the one current at creation
  int grid_ = 1;            // workgroups of the sum, and partials
  bool short_ = false;      // one workgroup sums it all
  bool shortClip_ = false;  // and clips it
  int nchunks_ = 0;
  int streamed_ = 0;        // chunks that a clip will not find in the cache anyway
  glx::GradChunk* chunks_ = nullptr;  // device memory
};

}  // namespace gloo
