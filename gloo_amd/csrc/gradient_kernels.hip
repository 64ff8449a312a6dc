// gradient_kernels.hip -- the global norm of many gradient tensors and
// clipping by it, for CDNA4 (gfx950).
//
//   S = sum over all tensors of |x|^p (p = 1, 2), or max |x| (p = inf)
//   N = S^(1/p);  out = x * min(1, maxNorm / (N + 1e-6))
//
// Both are bound by HBM: the sum reads every element once, the clip reads it
// again and writes it.  The tensors come as a table of chunks (gradients.h),
// dealt to workgroups in turn, so that hundreds of tensors of any sizes cost
// one launch.  S is accumulated in double: the square of an fp32 value is exact
// there and cannot overflow or vanish.  No atomics: workgroup b writes partial
// b, and whoever needs the sum folds the partials in one fixed order, so the
// same list gives the same bits every time.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "elem_ops.h"
#include "gradients.h"

namespace glx {
namespace {

// Global memory: pointers read from a table would otherwise be taken for
// generic ones and loaded with flat instructions.
#define GLX_GLOBAL __attribute__((address_space(1)))
// 16 bytes at an address that is only aligned to its elements: views into a
// bucket start anywhere.
typedef v4u __attribute__((aligned(2))) v4u_any;

struct F64 { using S = double; };
struct F32 { using S = float; };
struct F16 { using S = _Float16; };
struct BF16 { using S = __bf16; };

// ---- power sum ------------------------------------------------------------

// NaN wins over every number, as in the sums.
__device__ __forceinline__ double max_nan(double a, double b) {
  return (a > b || a != a) ? a : b;
}

template <int KIND>
__device__ __forceinline__ double join(double a, double b) {
  return KIND == kGradNormInf ? max_nan(a, b) : a + b;
}

template <int KIND>
__device__ __forceinline__ double power_add(double acc, double x) {
  if (KIND == kGradNorm2) return __builtin_fma(x, x, acc);
  if (KIND == kGradNorm1) return acc + __builtin_fabs(x);
  return max_nan(acc, __builtin_fabs(x));
}

template <typename T, int KIND>
__device__ __forceinline__ double chunk_power(const GradChunk& g, double acc) {
  using S = typename T::S;
  constexpr int V = 16 / sizeof(S), U = 4;
  const GLX_GLOBAL S* x = (const GLX_GLOBAL S*)g.src;
  const uint32_t nvec = g.n / V;
  const GLX_GLOBAL v4u_any* v = (const GLX_GLOBAL v4u_any*)x;
  for (uint32_t base = threadIdx.x; base < nvec; base += kBlock * U) {
    union { v4u v; S s[V]; } r[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t i = base + u * kBlock;
      r[u].v = i < nvec ? (v4u)v[i] : (v4u)(0u);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
      for (int e = 0; e < V; e++) acc = power_add<KIND>(acc, (double)r[u].s[e]);
    }
  }
  const uint32_t i = nvec * V + threadIdx.x;
  if (i < g.n) acc = power_add<KIND>(acc, (double)x[i]);
  return acc;
}

// The workgroup's values joined in a fixed order; the result in every thread.
template <int KIND>
__device__ __forceinline__ double block_join(double v) {
  __shared__ double wave[kBlock / 64];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = join<KIND>(v, __shfl_xor(v, d, 64));
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = wave[0];
#pragma unroll
  for (int w = 1; w < kBlock / 64; w++) r = join<KIND>(r, wave[w]);
  return r;
}

template <int KIND>
__global__ __launch_bounds__(kBlock) void power_partials_kernel(const GradChunk* chunks,
                                                                int nchunks, double* part) {
  double acc = 0;
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
    const GradChunk g = chunks[c];
    switch (g.dtype) {
      case GLX_FLOAT64: acc = chunk_power<F64, KIND>(g, acc); break;
      case GLX_FLOAT32: acc = chunk_power<F32, KIND>(g, acc); break;
      case GLX_FLOAT16: acc = chunk_power<F16, KIND>(g, acc); break;
      default: acc = chunk_power<BF16, KIND>(g, acc);
    }
  }
  acc = block_join<KIND>(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

template <int KIND>
__device__ __forceinline__ double fold_partials(const double* part, int nparts) {
  double acc = 0;
  for (int i = threadIdx.x; i < nparts; i += kBlock) acc = join<KIND>(acc, part[i]);
  return block_join<KIND>(acc);
}

template <int KIND>
__device__ __forceinline__ double root_of(double s) {
  return KIND == kGradNorm2 ? __builtin_sqrt(s) : s;
}

__device__ __forceinline__ void put_scalar(void* out, int dtype, double v) {
  if (dtype == GLX_FLOAT32) {
    *static_cast<float*>(out) = (float)v;
  } else {
    *static_cast<double*>(out) = v;
  }
}

template <int KIND>
__global__ __launch_bounds__(kBlock) void power_finish_kernel(const double* part, int nparts,
                                                              bool root, void* out,
                                                              int outDtype) {
  const double s = fold_partials<KIND>(part, nparts);
  if (threadIdx.x == 0) put_scalar(out, outDtype, root ? root_of<KIND>(s) : s);
}

// ---- clip -----------------------------------------------------------------

// x * c in fp32 (fp64 for fp64), rounded once to the element's type.
__device__ __forceinline__ double scaled(double x, double c) { return x * c; }
__device__ __forceinline__ float scaled(float x, double c) { return x * (float)c; }
__device__ __forceinline__ _Float16 scaled(_Float16 x, double c) {
  return (_Float16)((float)x * (float)c);
}
__device__ __forceinline__ __bf16 scaled(__bf16 x, double c) {
  return (__bf16)((float)x * (float)c);
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const GradChunk& g, double c) {
  using S = typename T::S;
  constexpr int V = 16 / sizeof(S), U = 4;
  const GLX_GLOBAL S* x = (const GLX_GLOBAL S*)g.src;
  GLX_GLOBAL S* y = (GLX_GLOBAL S*)g.dst;
  const uint32_t nvec = g.n / V;
  const GLX_GLOBAL v4u_any* vx = (const GLX_GLOBAL v4u_any*)x;
  GLX_GLOBAL v4u_any* vy = (GLX_GLOBAL v4u_any*)y;
  for (uint32_t base = threadIdx.x; base < nvec; base += kBlock * U) {
    union { v4u v; S s[V]; } r[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t i = base + u * kBlock;
      if (i < nvec) r[u].v = vx[i];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t i = base + u * kBlock;
      if (i < nvec) {
#pragma unroll
        for (int e = 0; e < V; e++) r[u].s[e] = scaled(r[u].s[e], c);
        vy[i] = r[u].v;
      }
    }
  }
  const uint32_t i = nvec * V + threadIdx.x;
  if (i < g.n) y[i] = scaled(x[i], c);
}

template <int KIND>
__global__ __launch_bounds__(kBlock) void clip_kernel(const GradChunk* chunks, int nchunks,
                                                      const double* part, int nparts,
                                                      double maxNorm, void* out, int outDtype) {
  const double n = root_of<KIND>(fold_partials<KIND>(part, nparts));
  if (out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) put_scalar(out, outDtype, n);
  const double q = maxNorm / (n + 1e-6);
  const double c = q >= 1 ? 1.0 : q;  // NaN stays NaN
  for (int k = blockIdx.x; k < nchunks; k += gridDim.x) {
    const GradChunk g = chunks[k];
    if (c == 1 && g.dst == g.src) continue;  // in place, nothing to clip
    switch (g.dtype) {
      case GLX_FLOAT64: chunk_scale<F64>(g, c); break;
      case GLX_FLOAT32: chunk_scale<F32>(g, c); break;
      case GLX_FLOAT16: chunk_scale<F16>(g, c); break;
      default: chunk_scale<BF16>(g, c);
    }
  }
}

}  // namespace

hipError_t launch_power_partials(int kind, const GradChunk* chunks, int nchunks, int grid,
                                 double* part, hipStream_t s) {
  const dim3 g((unsigned)grid), b(kBlock);
  switch (kind) {
    case kGradNorm1:
      hipLaunchKernelGGL(power_partials_kernel<kGradNorm1>, g, b, 0, s, chunks, nchunks, part);
      break;
    case kGradNorm2:
      hipLaunchKernelGGL(power_partials_kernel<kGradNorm2>, g, b, 0, s, chunks, nchunks, part);
      break;
    default:
      hipLaunchKernelGGL(power_partials_kernel<kGradNormInf>, g, b, 0, s, chunks, nchunks,
                         part);
  }
  return hipGetLastError();
}

hipError_t launch_power_finish(int kind, const double* part, int nparts, bool root, void* out,
                               int outDtype, hipStream_t s) {
  const dim3 g(1), b(kBlock);
  switch (kind) {
    case kGradNorm1:
      hipLaunchKernelGGL(power_finish_kernel<kGradNorm1>, g, b, 0, s, part, nparts, root, out,
                         outDtype);
      break;
    case kGradNorm2:
      hipLaunchKernelGGL(power_finish_kernel<kGradNorm2>, g, b, 0, s, part, nparts, root, out,
                         outDtype);
      break;
    default:
      hipLaunchKernelGGL(power_finish_kernel<kGradNormInf>, g, b, 0, s, part, nparts, root,
                         out, outDtype);
  }
  return hipGetLastError();
}

hipError_t launch_clip(int kind, const GradChunk* chunks, int nchunks, int grid,
                       const double* part, int nparts, double maxNorm, void* out, int outDtype,
                       hipStream_t s) {
  const dim3 g((unsigned)grid), b(kBlock);
  switch (kind) {
    case kGradNorm1:
      hipLaunchKernelGGL(clip_kernel<kGradNorm1>, g, b, 0, s, chunks, nchunks, part, nparts,
                         maxNorm, out, outDtype);
      break;
    case kGradNorm2:
      hipLaunchKernelGGL(clip_kernel<kGradNorm2>, g, b, 0, s, chunks, nchunks, part, nparts,
                         maxNorm, out, outDtype);
      break;
    default:
      hipLaunchKernelGGL(clip_kernel<kGradNormInf>, g, b, 0, s, chunks, nchunks, part, nparts,
                         maxNorm, out, outDtype);
  }
  return hipGetLastError();
}

}  // namespace glx
