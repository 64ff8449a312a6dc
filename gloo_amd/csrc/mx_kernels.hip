// mx_kernels.hip -- microscaled 4-bit (MXFP4, OCP MX v1.0) messages for CDNA4
// (gfx950): gradients squeezed for the exchange, and the fold of what arrives.
//
// Block of 32 values y, A = max |y|:  the scale byte is E = max(floor(log2 A)
// + 127 - 2, 0) (2 = the exponent of E2M1's largest value, 6), and the codes are
// y / 2^(E-127) rounded to the nearest E2M1 value, ties to even, at most 6 in
// magnitude.  A block that holds an infinity or a NaN becomes a NaN block.
// Dividing by a power of two is exact, so the codes are those of y itself.
//
// Everything here is bound by HBM (17/32 byte per element and payload).  A
// lane takes 8 elements (16 bytes of bf16, 4 of codes) and four lanes a block:
// the block's maximum is two DPP exchanges away and needs no shared memory, and
// a wave's codes are one contiguous store.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "elem_ops.h"
#include "mx.h"

namespace glx {
namespace {

#define GLX_GLOBAL __attribute__((address_space(1)))
typedef v4u __attribute__((aligned(2))) v4u_any;
typedef float v2f __attribute__((ext_vector_type(2)));

constexpr int kLane = 8;   // elements of a lane
constexpr int kQuad = 4;   // lanes of a block

struct F32 { using S = float; };
struct F16 { using S = _Float16; };
struct BF16 { using S = __bf16; };

// The 8 elements from element i on; zero from n on.
template <typename T>
__device__ __forceinline__ void load8(const GLX_GLOBAL typename T::S* p, size_t i, size_t n,
                                      float (&y)[kLane]) {
  using S = typename T::S;
  constexpr int V = 16 / sizeof(S);
  if (i + kLane <= n) {
    union { v4u v[kLane / V]; S s[kLane]; } r;
#pragma unroll
    for (int q = 0; q < kLane / V; q++) {
      r.v[q] = *(const GLX_GLOBAL v4u_any*)(p + i + q * V);
    }
#pragma unroll
    for (int e = 0; e < kLane; e++) y[e] = (float)r.s[e];
  } else {
#pragma unroll
    for (int e = 0; e < kLane; e++) y[e] = i + e < n ? (float)p[i + e] : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(GLX_GLOBAL typename T::S* p, size_t i, size_t n,
                                       const float (&y)[kLane]) {
  using S = typename T::S;
  constexpr int V = 16 / sizeof(S);
  if (i + kLane <= n) {
    union { v4u v[kLane / V]; S s[kLane]; } r;
#pragma unroll
    for (int e = 0; e < kLane; e++) r.s[e] = (S)y[e];
#pragma unroll
    for (int q = 0; q < kLane / V; q++) *(GLX_GLOBAL v4u_any*)(p + i + q * V) = r.v[q];
  } else {
#pragma unroll
    for (int e = 0; e < kLane; e++) {
      if (i + e < n) p[i + e] = (S)y[e];
    }
  }
}

// The larger of v and that of the lane's partner in its group of four.
template <int PARTNER>
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  const uint32_t o =
      (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, PARTNER, 0xf, 0xf, true);
  return v > o ? v : o;
}

// A block of which this lane holds 8 values: its scale byte, and the lane's
// codes.  The block's four lanes call it together.
struct Block {
  uint32_t code, scale;
};
__device__ __forceinline__ Block encode8(const float (&y)[kLane]) {
  // bits of |y| order as the values do, NaN above infinity above all others
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < kLane; e++) {
    const uint32_t b = __float_as_uint(y[e]) & 0x7fffffffu;
    top = top > b ? top : b;
  }
  top = quad_max<0xb1>(top);  // lanes 1 0 3 2
  top = quad_max<0x4e>(top);  // lanes 2 3 0 1
  const uint32_t e = top >> 23;
  if (e == 255) return {0, 255};
  const uint32_t s = e > 2 ? e - 2 : 0;
  const float inv = __uint_as_float((254 - s) << 23);  // 2^(127 - s): s <= 252
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[0] * inv, y[1] * inv, 1.f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2] * inv, y[3] * inv, 1.f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[4] * inv, y[5] * inv, 1.f, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[6] * inv, y[7] * inv, 1.f, 3);
  return {c, s};
}

// The unscaled values of 8 codes.
__device__ __forceinline__ void decode8(uint32_t c, float (&v)[kLane]) {
  v2f p;
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0);
  v[0] = p[0], v[1] = p[1];
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1);
  v[2] = p[0], v[3] = p[1];
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2);
  v[4] = p[0], v[5] = p[1];
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3);
  v[6] = p[0], v[7] = p[1];
}

// 2^(s - 127), subnormal for s = 0, NaN for s = 255.
__device__ __forceinline__ float scale_of(uint32_t s) {
  return __uint_as_float((s << 23) | (s == 0 || s == 255 ? 0x00400000u : 0u));
}

// Codes and scale of the lane's part, and the zero bytes behind the last scale
// (up to 15: a message of fewer than four blocks has fewer lanes than that).
// g: the lane's number in the message (8 elements each), below 4 nb.
__device__ __forceinline__ void put_block(GLX_GLOBAL char* payload, size_t nb, size_t g, Block b) {
  ((GLX_GLOBAL uint32_t*)payload)[g] = b.code;
  if (g % kQuad == 0) payload[nb * 16 + g / kQuad] = (char)b.scale;
  for (size_t q = g; q < (16 - nb % 16) % 16; q += nb * kQuad) payload[nb * 17 + q] = 0;
}

template <typename T, bool RES_IN, bool RES_OUT>
__global__ __launch_bounds__(kBlock) void mx_quantize_kernel(char* payload_,
                                                             const typename T::S* x_,
                                                             const float* residual_,
                                                             float* residualOut_, size_t n,
                                                             size_t nb) {
  using S = typename T::S;
  GLX_GLOBAL char* payload = (GLX_GLOBAL char*)payload_;
  const GLX_GLOBAL S* x = (const GLX_GLOBAL S*)x_;
  const size_t step = (size_t)gridDim.x * kBlock;
  for (size_t g = (size_t)blockIdx.x * kBlock + threadIdx.x; g < nb * kQuad; g += step) {
    float y[kLane];
    load8<T>(x, g * kLane, n, y);
    if (RES_IN) {
      float r[kLane];
      load8<F32>((const GLX_GLOBAL float*)residual_, g * kLane, n, r);
#pragma unroll
      for (int e = 0; e < kLane; e++) y[e] = __fadd_rn(y[e], r[e]);
    }
    const Block b = encode8(y);
    put_block(payload, nb, g, b);
    if (RES_OUT) {
      float v[kLane];
      decode8(b.code, v);
      const float sc = scale_of(b.scale);
#pragma unroll
      for (int e = 0; e < kLane; e++) {
        v[e] = b.scale == 255 ? 0.f : __builtin_fmaf(-v[e], sc, y[e]);
      }
      store8<F32>((GLX_GLOBAL float*)residualOut_, g * kLane, n, v);
    }
  }
}

struct MxSources {
  const char* p[kMxMaxSources];
};

// acc = the left fold of the k payloads' values for lane g, times scale.
__device__ __forceinline__ void fold8(const MxSources& src, int k, size_t nb, size_t g,
                                      float scale, float (&acc)[kLane]) {
  for (int j = 0; j < k; j++) {
    const GLX_GLOBAL char* p = (const GLX_GLOBAL char*)src.p[j];
    const uint32_t c = ((const GLX_GLOBAL uint32_t*)p)[g];
    const float sc = scale_of((uint8_t)p[nb * 16 + g / kQuad]);
    float v[kLane];
    decode8(c, v);
#pragma unroll
    for (int e = 0; e < kLane; e++) {
      // v * sc is exact: the fma rounds only the sum
      acc[e] = j == 0 ? v[e] * sc : __builtin_fmaf(v[e], sc, acc[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < kLane; e++) acc[e] = __fmul_rn(acc[e], scale);
}

template <typename T>
__global__ __launch_bounds__(kBlock) void mx_reduce_n_kernel(typename T::S* dst, MxSources src,
                                                             int k, size_t n, size_t nb,
                                                             float scale) {
  using S = typename T::S;
  const size_t step = (size_t)gridDim.x * kBlock;
  const size_t lanes = (n + kLane - 1) / kLane;
  for (size_t g = (size_t)blockIdx.x * kBlock + threadIdx.x; g < lanes; g += step) {
    float acc[kLane];
    fold8(src, k, nb, g, scale, acc);
    store8<T>((GLX_GLOBAL S*)dst, g * kLane, n, acc);
  }
}

__global__ __launch_bounds__(kBlock) void mx_requantize_n_kernel(char* payload, MxSources src,
                                                                 int k, size_t n, size_t nb,
                                                                 float scale) {
  const size_t step = (size_t)gridDim.x * kBlock;
  for (size_t g = (size_t)blockIdx.x * kBlock + threadIdx.x; g < nb * kQuad; g += step) {
    float acc[kLane];
    fold8(src, k, nb, g, scale, acc);
#pragma unroll
    for (int e = 0; e < kLane; e++) {
      if (g * kLane + e >= n) acc[e] = 0.f;  // behind the end, whatever the sources hold
    }
    put_block((GLX_GLOBAL char*)payload, nb, g, encode8(acc));
  }
}

unsigned mx_grid(size_t lanes) {
  const size_t blocks = (lanes + kBlock - 1) / kBlock;
  return (unsigned)(blocks < 1 ? 1 : blocks > 16384 ? 16384 : blocks);
}

template <typename T>
hipError_t quantize_typed(void* payload, const void* x, const float* r, float* ro, size_t n,
                          hipStream_t s) {
  using S = typename T::S;
  const size_t nb = mxBlocks(n);
  const dim3 g(mx_grid(nb * kQuad)), b(kBlock);
  if (r != nullptr && ro != nullptr) {
    hipLaunchKernelGGL((mx_quantize_kernel<T, true, true>), g, b, 0, s, (char*)payload,
                       (const S*)x, r, ro, n, nb);
  } else if (r != nullptr) {
    hipLaunchKernelGGL((mx_quantize_kernel<T, true, false>), g, b, 0, s, (char*)payload,
                       (const S*)x, r, ro, n, nb);
  } else if (ro != nullptr) {
    hipLaunchKernelGGL((mx_quantize_kernel<T, false, true>), g, b, 0, s, (char*)payload,
                       (const S*)x, r, ro, n, nb);
  } else {
    hipLaunchKernelGGL((mx_quantize_kernel<T, false, false>), g, b, 0, s, (char*)payload,
                       (const S*)x, r, ro, n, nb);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t reduce_typed(void* dst, const MxSources& src, int k, size_t n, float scale,
                        hipStream_t s) {
  hipLaunchKernelGGL(mx_reduce_n_kernel<T>, dim3(mx_grid((n + kLane - 1) / kLane)), dim3(kBlock),
                     0, s, (typename T::S*)dst, src, k, n, mxBlocks(n), scale);
  return hipGetLastError();
}

MxSources sources(const void* const* payloads, int k) {
  MxSources src{};
  for (int j = 0; j < k; j++) src.p[j] = (const char*)payloads[j];
  return src;
}

}  // namespace

hipError_t launch_mx_quantize(int dtype, void* payload, const void* x, const float* residual,
                              float* residualOut, size_t n, hipStream_t s) {
  if (n == 0) return hipSuccess;
  switch (dtype) {
    case GLX_FLOAT32: return quantize_typed<F32>(payload, x, residual, residualOut, n, s);
    case GLX_FLOAT16: return quantize_typed<F16>(payload, x, residual, residualOut, n, s);
    case GLX_BFLOAT16: return quantize_typed<BF16>(payload, x, residual, residualOut, n, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_mx_reduce_n(int dtype, void* dst, const void* const* payloads, int k, size_t n,
                              float scale, hipStream_t s) {
  if (n == 0) return hipSuccess;
  if (k < 1 || k > kMxMaxSources) return hipErrorInvalidValue;
  const MxSources src = sources(payloads, k);
  switch (dtype) {
    case GLX_FLOAT32: return reduce_typed<F32>(dst, src, k, n, scale, s);
    case GLX_FLOAT16: return reduce_typed<F16>(dst, src, k, n, scale, s);
    case GLX_BFLOAT16: return reduce_typed<BF16>(dst, src, k, n, scale, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_mx_requantize_n(void* payload, const void* const* payloads, int k, size_t n,
                                  float scale, hipStream_t s) {
  if (n == 0) return hipSuccess;
  if (k < 1 || k > kMxMaxSources) return hipErrorInvalidValue;
  const size_t nb = mxBlocks(n);
  hipLaunchKernelGGL(mx_requantize_n_kernel, dim3(mx_grid(nb * kQuad)), dim3(kBlock), 0, s,
                     (char*)payload, sources(payloads, k), k, n, nb, scale);
  return hipGetLastError();
}

}  // namespace glx
