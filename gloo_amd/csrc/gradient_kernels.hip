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
// there and cannot overflow or vanish, and the loads leave the time for it
// (a widening and a double fma per element).  No atomics: workgroup b writes
// partial b, and whoever needs the sum folds the partials in one fixed order,
// so the same list gives the same bits every time.
//
// Measured on MI355X, whole calls, lists that no cache holds beforehand:
//   norm  1 GiB f32       159 us (sum 156 us, 6.9 TB/s; with plain loads 174)
//   clip  256 MiB f32 into another buffer  121 us: three streams, 6.7 TB/s
//         1 GiB and more, bf16 and f32 mixed  538 us, 6.2 TB/s
//   short lists, one launch: 160 KiB f32 norm 4.1 us (two launches 5.2)
// The sum runs 4 workgroups a CU (8, 16, 64 measured 1 to 2 % slower).  The clip
// runs one workgroup per chunk, the last chunks first; with a persistent grid
// it took 131 us.  Of what a clip will read again the sum loads the last 256 MiB
// (the Infinity Cache's size) to stay and the rest nontemporally: 256 MiB 121
// instead of 128 us, 320 MiB 151 instead of 159, 32 MiB 18 instead of 21; all of
// a 1.2 GB list loaded to stay costs 562 instead of 538 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "elem_ops.h"
#include "gradients.h"

namespace glx {
namespace {

constexpr int kShortThreads = 1024;
constexpr int kShortRounds = kGradShortChunks / (kShortThreads / 64);

// Global memory: pointers read from a table would otherwise be taken for
// generic ones and loaded with flat instructions.
#define GLX_GLOBAL __attribute__((address_space(1)))
// 16 bytes at an address that is only aligned to its elements: an output need
// not start at its gradient's distance from a 16-byte boundary.
typedef v4u __attribute__((aligned(2))) v4u_any;

// Element types, and |x| from the bits left of the sign.
struct F64 {
  using S = double;
  using Bits = uint64_t;
  static __device__ __forceinline__ double magnitude(Bits b) { return __longlong_as_double(b); }
};
struct F32 {
  using S = float;
  using Bits = uint32_t;
  static __device__ __forceinline__ double magnitude(Bits b) { return __uint_as_float(b); }
};
struct F16 {
  using S = _Float16;
  using Bits = uint16_t;
  static __device__ __forceinline__ double magnitude(Bits b) { return h2f(b); }
};
struct BF16 {
  using S = __bf16;
  using Bits = uint16_t;
  static __device__ __forceinline__ double magnitude(Bits b) { return b2f(b); }
};

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
  return acc + __builtin_fabs(x);
}

// The part of one vector (zero bits count nothing), and of one element.
template <typename T, int KIND>
struct Power {
  using S = typename T::S;
  using B = typename T::Bits;
  static constexpr int V = 16 / sizeof(S);
  static constexpr B kMagnitude = (B)~((B)1 << (8 * sizeof(B) - 1));
  double acc;
  B top = 0;  // magnitudes order as their bits do, NaN above infinity above all others
  __device__ __forceinline__ explicit Power(double a) : acc(a) {}
  __device__ __forceinline__ void add(S x) {
    if (KIND == kGradNormInf) {
      union { S s; B b; } r;
      r.s = x;
      const B m = r.b & kMagnitude;
      top = m > top ? m : top;
    } else {
      acc = power_add<KIND>(acc, (double)x);
    }
  }
  __device__ __forceinline__ void add(v4u x) {
    union { v4u v; S s[V]; } r;
    r.v = x;
#pragma unroll
    for (int e = 0; e < V; e++) add(r.s[e]);
  }
  __device__ __forceinline__ double get() const {
    return KIND == kGradNormInf ? max_nan(acc, T::magnitude(top)) : acc;
  }
};

// How a chunk lies: up to 15 bytes of elements before the first 16-byte
// boundary of src, whole vectors, up to 15 bytes after the last.  (Vectors
// loaded across 2-byte boundaries ran 16-bit sums at 5.0 instead of 6.8 TB/s.)
template <typename S>
struct Layout {
  static constexpr uint32_t V = 16 / sizeof(S);
  uint32_t head, nvec, edges;  // edges: head and tail elements together
  __device__ __forceinline__ explicit Layout(const GradChunk& g) {
    head = (uint32_t)(-(uintptr_t)g.src % 16 / sizeof(S));
    if (head > g.n) head = g.n;
    nvec = (g.n - head) / V;
    edges = g.n - nvec * V;
  }
  // where edge element i < edges is
  __device__ __forceinline__ uint32_t edge(uint32_t i) const {
    return i < head ? i : i + nvec * V;
  }
};

// One chunk's part of the sum, by a workgroup.
template <typename T, int KIND, bool NT>
__device__ __forceinline__ double chunk_power(const GradChunk& g, double acc) {
  using S = typename T::S;
  constexpr int U = 4;
  const Layout<S> at(g);
  const uint32_t nvec = at.nvec;
  const GLX_GLOBAL S* x = (const GLX_GLOBAL S*)g.src;
  const GLX_GLOBAL v4u* v = (const GLX_GLOBAL v4u*)(x + at.head);
  Power<T, KIND> sum(acc);
  for (uint32_t base = threadIdx.x; base < nvec; base += kBlock * U) {
    v4u r[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t i = base + u * kBlock;
      r[u] = (v4u)(0u);
      if (i < nvec) r[u] = NT ? __builtin_nontemporal_load(v + i) : v[i];
    }
#pragma unroll
    for (int u = 0; u < U; u++) sum.add(r[u]);
  }
  if (threadIdx.x < at.edges) sum.add((S)x[at.edge(threadIdx.x)]);
  return sum.get();
}

// The workgroup's values joined in a fixed order; the result in every thread.
template <int KIND, int THREADS>
__device__ __forceinline__ double block_join(double v) {
  __shared__ double wave[THREADS / 64];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = join<KIND>(v, __shfl_xor(v, d, 64));
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = wave[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; w++) r = join<KIND>(r, wave[w]);
  return r;
}

template <int KIND, bool NT>
__device__ __forceinline__ double any_chunk_power(const GradChunk& g, double acc) {
  switch (g.dtype) {
    case GLX_FLOAT64: return chunk_power<F64, KIND, NT>(g, acc);
    case GLX_FLOAT32: return chunk_power<F32, KIND, NT>(g, acc);
    case GLX_FLOAT16: return chunk_power<F16, KIND, NT>(g, acc);
  }
  return chunk_power<BF16, KIND, NT>(g, acc);
}

// Chunks below `streamed` are loaded nontemporally, the others to stay cached.
template <int KIND>
__global__ __launch_bounds__(kBlock) void power_partials_kernel(const GradChunk* chunks,
                                                                int nchunks, int streamed,
                                                                double* part) {
  double acc = 0;
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
    const GradChunk g = chunks[c];
    acc = c < streamed ? any_chunk_power<KIND, true>(g, acc)
                       : any_chunk_power<KIND, false>(g, acc);
  }
  acc = block_join<KIND, kBlock>(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

template <int KIND>
__device__ __forceinline__ double fold_partials(const double* part, int nparts) {
  double acc = 0;
  for (int i = threadIdx.x; i < nparts; i += kBlock) acc = join<KIND>(acc, part[i]);
  return block_join<KIND, kBlock>(acc);
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
__device__ __forceinline__ v4u scaled_vec(v4u x, double c) {
  using S = typename T::S;
  constexpr int V = 16 / sizeof(S);
  union { v4u v; S s[V]; } r;
  r.v = x;
#pragma unroll
  for (int e = 0; e < V; e++) r.s[e] = scaled(r.s[e], c);
  return r.v;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const GradChunk& g, double c) {
  using S = typename T::S;
  constexpr int U = 4;
  const Layout<S> at(g);
  const uint32_t nvec = at.nvec;
  const GLX_GLOBAL S* x = (const GLX_GLOBAL S*)g.src;
  GLX_GLOBAL S* y = (GLX_GLOBAL S*)g.dst;
  const GLX_GLOBAL v4u* vx = (const GLX_GLOBAL v4u*)(x + at.head);
  GLX_GLOBAL v4u_any* vy = (GLX_GLOBAL v4u_any*)(y + at.head);
  for (uint32_t base = threadIdx.x; base < nvec; base += kBlock * U) {
    v4u r[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t i = base + u * kBlock;
      if (i < nvec) r[u] = __builtin_nontemporal_load(vx + i);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t i = base + u * kBlock;
      if (i < nvec) __builtin_nontemporal_store((v4u_any)scaled_vec<T>(r[u], c), vy + i);
    }
  }
  if (threadIdx.x < at.edges) {
    const uint32_t i = at.edge(threadIdx.x);
    y[i] = scaled((S)x[i], c);
  }
}

__device__ __forceinline__ double coefficient(double maxNorm, double norm) {
  const double q = maxNorm / (norm + 1e-6);
  return q >= 1 ? 1.0 : q;  // NaN stays NaN
}

// One chunk per workgroup, the last chunks first (the sum read them last), each
// on the XCD that summed it: chunk and workgroup numbers agree modulo 8.  Loading
// the chunk before the partials are folded made it slower (256 MiB 127 instead of
// 121 us).
template <int KIND>
__global__ __launch_bounds__(kBlock) void clip_kernel(const GradChunk* chunks, int nchunks,
                                                      const double* part, int nparts,
                                                      double maxNorm, void* out, int outDtype) {
  const double n = root_of<KIND>(fold_partials<KIND>(part, nparts));
  if (out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) put_scalar(out, outDtype, n);
  const int last = (int)gridDim.x / 8 * 8 - 8;
  const int k = last - (int)blockIdx.x / 8 * 8 + (int)blockIdx.x % 8;
  if (k >= nchunks) return;
  const GradChunk g = chunks[k];
  const double c = coefficient(maxNorm, n);
  if (c == 1 && g.dst == g.src) return;  // in place, nothing to clip
  switch (g.dtype) {
    case GLX_FLOAT64: chunk_scale<F64>(g, c); break;
    case GLX_FLOAT32: chunk_scale<F32>(g, c); break;
    case GLX_FLOAT16: chunk_scale<F16>(g, c); break;
    default: chunk_scale<BF16>(g, c);
  }
}

// ---- short lists ----------------------------------------------------------

// One wave's part of a short list: up to kShortRounds chunks of 4 KiB, held in
// registers from the sum to the clip, all loads in flight at once.
struct ShortChunk {
  GradChunk g;
  v4u r[4];
};

template <typename S>
__device__ __forceinline__ void load_vectors(ShortChunk& h, uint32_t lane) {
  const Layout<S> at(h.g);
  const GLX_GLOBAL v4u* x = (const GLX_GLOBAL v4u*)((const GLX_GLOBAL S*)h.g.src + at.head);
#pragma unroll
  for (int u = 0; u < 4; u++) {
    h.r[u] = (v4u)(0u);
    if (lane + u * 64 < at.nvec) h.r[u] = x[lane + u * 64];
  }
}

__device__ __forceinline__ void load_short(ShortChunk& h, uint32_t lane) {
  switch (h.g.dtype) {
    case GLX_FLOAT64: load_vectors<double>(h, lane); break;
    case GLX_FLOAT32: load_vectors<float>(h, lane); break;
    default: load_vectors<_Float16>(h, lane);
  }
}

template <typename T, int KIND>
__device__ __forceinline__ double short_power(const ShortChunk& h, uint32_t lane, double acc) {
  using S = typename T::S;
  const Layout<S> at(h.g);
  Power<T, KIND> sum(acc);
#pragma unroll
  for (int u = 0; u < 4; u++) sum.add(h.r[u]);
  if (lane < at.edges) sum.add((S)((const GLX_GLOBAL S*)h.g.src)[at.edge(lane)]);
  return sum.get();
}

template <typename T>
__device__ __forceinline__ void short_scale(const ShortChunk& h, uint32_t lane, double c) {
  using S = typename T::S;
  const Layout<S> at(h.g);
  GLX_GLOBAL S* y = (GLX_GLOBAL S*)h.g.dst;
#pragma unroll
  for (int u = 0; u < 4; u++) {
    if (lane + u * 64 < at.nvec) {
      ((GLX_GLOBAL v4u_any*)(y + at.head))[lane + u * 64] = scaled_vec<T>(h.r[u], c);
    }
  }
  if (lane < at.edges) {
    const uint32_t i = at.edge(lane);
    y[i] = scaled((S)((const GLX_GLOBAL S*)h.g.src)[i], c);
  }
}

// The whole of it by one workgroup, its waves taking chunks in turn: for lists
// so short that a second launch costs more than the other CUs would save.
template <int KIND, bool CLIP>
__global__ __launch_bounds__(kShortThreads) void short_kernel(const GradChunk* chunks,
                                                              int nchunks, double maxNorm,
                                                              bool root, void* out,
                                                              int outDtype) {
  constexpr int kWaves = kShortThreads / 64;
  const uint32_t lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  ShortChunk h[kShortRounds];
#pragma unroll
  for (int q = 0; q < kShortRounds; q++) {
    const int k = wave + q * kWaves;
    h[q].g = GradChunk{nullptr, nullptr, 0, GLX_FLOAT32};
    if (k < nchunks) h[q].g = chunks[k];
  }
#pragma unroll
  for (int q = 0; q < kShortRounds; q++) load_short(h[q], lane);
  double acc = 0;
#pragma unroll
  for (int q = 0; q < kShortRounds; q++) {
    switch (h[q].g.dtype) {
      case GLX_FLOAT64: acc = short_power<F64, KIND>(h[q], lane, acc); break;
      case GLX_FLOAT32: acc = short_power<F32, KIND>(h[q], lane, acc); break;
      case GLX_FLOAT16: acc = short_power<F16, KIND>(h[q], lane, acc); break;
      default: acc = short_power<BF16, KIND>(h[q], lane, acc);
    }
  }
  acc = block_join<KIND, kShortThreads>(acc);
  const double n = root ? root_of<KIND>(acc) : acc;
  if (out != nullptr && threadIdx.x == 0) put_scalar(out, outDtype, n);
  if (!CLIP) return;
  const double c = coefficient(maxNorm, n);
#pragma unroll
  for (int q = 0; q < kShortRounds; q++) {
    if (c == 1 && h[q].g.dst == h[q].g.src) continue;
    switch (h[q].g.dtype) {
      case GLX_FLOAT64: short_scale<F64>(h[q], lane, c); break;
      case GLX_FLOAT32: short_scale<F32>(h[q], lane, c); break;
      case GLX_FLOAT16: short_scale<F16>(h[q], lane, c); break;
      default: short_scale<BF16>(h[q], lane, c);
    }
  }
}

template <int KIND>
hipError_t partials_of(const GradChunk* chunks, int nchunks, int streamed, int grid,
                       double* part, hipStream_t s) {
  hipLaunchKernelGGL(power_partials_kernel<KIND>, dim3((unsigned)grid), dim3(kBlock), 0, s,
                     chunks, nchunks, streamed, part);
  return hipGetLastError();
}

template <int KIND>
hipError_t finish_of(const double* part, int nparts, bool root, void* out, int outDtype,
                     hipStream_t s) {
  hipLaunchKernelGGL(power_finish_kernel<KIND>, dim3(1), dim3(kBlock), 0, s, part, nparts, root,
                     out, outDtype);
  return hipGetLastError();
}

template <int KIND>
hipError_t clip_of(const GradChunk* chunks, int nchunks, const double* part, int nparts,
                   double maxNorm, void* out, int outDtype, hipStream_t s) {
  const unsigned grid = ((unsigned)nchunks + 8) / 8 * 8;  // at least one, for the norm
  hipLaunchKernelGGL(clip_kernel<KIND>, dim3(grid), dim3(kBlock), 0, s, chunks, nchunks, part,
                     nparts, maxNorm, out, outDtype);
  return hipGetLastError();
}

template <int KIND>
hipError_t short_of(const GradChunk* chunks, int nchunks, bool clip, double maxNorm, bool root,
                    void* out, int outDtype, hipStream_t s) {
  if (clip) {
    hipLaunchKernelGGL((short_kernel<KIND, true>), dim3(1), dim3(kShortThreads), 0, s, chunks,
                       nchunks, maxNorm, root, out, outDtype);
  } else {
    hipLaunchKernelGGL((short_kernel<KIND, false>), dim3(1), dim3(kShortThreads), 0, s, chunks,
                       nchunks, maxNorm, root, out, outDtype);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_power_partials(int kind, const GradChunk* chunks, int nchunks, int streamed,
                                 int grid, double* part, hipStream_t s) {
  switch (kind) {
    case kGradNorm1: return partials_of<kGradNorm1>(chunks, nchunks, streamed, grid, part, s);
    case kGradNorm2: return partials_of<kGradNorm2>(chunks, nchunks, streamed, grid, part, s);
  }
  return partials_of<kGradNormInf>(chunks, nchunks, streamed, grid, part, s);
}

hipError_t launch_power_finish(int kind, const double* part, int nparts, bool root, void* out,
                               int outDtype, hipStream_t s) {
  switch (kind) {
    case kGradNorm1: return finish_of<kGradNorm1>(part, nparts, root, out, outDtype, s);
    case kGradNorm2: return finish_of<kGradNorm2>(part, nparts, root, out, outDtype, s);
  }
  return finish_of<kGradNormInf>(part, nparts, root, out, outDtype, s);
}

hipError_t launch_clip(int kind, const GradChunk* chunks, int nchunks, const double* part,
                       int nparts, double maxNorm, void* out, int outDtype, hipStream_t s) {
  switch (kind) {
    case kGradNorm1:
      return clip_of<kGradNorm1>(chunks, nchunks, part, nparts, maxNorm, out, outDtype, s);
    case kGradNorm2:
      return clip_of<kGradNorm2>(chunks, nchunks, part, nparts, maxNorm, out, outDtype, s);
  }
  return clip_of<kGradNormInf>(chunks, nchunks, part, nparts, maxNorm, out, outDtype, s);
}

hipError_t launch_short(int kind, const GradChunk* chunks, int nchunks, bool clip,
                        double maxNorm, bool root, void* out, int outDtype, hipStream_t s) {
  switch (kind) {
    case kGradNorm1:
      return short_of<kGradNorm1>(chunks, nchunks, clip, maxNorm, root, out, outDtype, s);
    case kGradNorm2:
      return short_of<kGradNorm2>(chunks, nchunks, clip, maxNorm, root, out, outDtype, s);
  }
  return short_of<kGradNormInf>(chunks, nchunks, clip, maxNorm, root, out, outDtype, s);
}

}  // namespace glx
