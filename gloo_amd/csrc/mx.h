// mx.h -- microscaled 4-bit (MXFP4) messages: launchers of mx_kernels.hip.
//
// A payload of n elements: nb = ceil(n / 32) blocks of 32 codes (16 bytes
// each: E2M1, two to a byte, the even element in the low half), then nb scale
// bytes (E8M0: 2^(byte - 127); 255: the block is NaN), then zero bytes up to a
// multiple of 16.  Codes behind the last element are zero.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

namespace glx {

constexpr size_t kMxBlock = 32;
constexpr int kMxMaxSources = 16;

inline size_t mxBlocks(size_t n) { return n / kMxBlock + (n % kMxBlock != 0); }
inline size_t mxPayloadBytes(size_t n) { return (mxBlocks(n) * 17 + 15) / 16 * 16; }

// y = x (+ residual); payload = the blocks of y; residual_out = y - what the
// payload stands for (0 in a NaN block).  residual / residual_out may be null.
hipError_t launch_mx_quantize(int dtype, void* payload, const void* x, const float* residual,
                              float* residualOut, size_t n, hipStream_t s);
// dst = scale * (left fold of the payloads' values in fp32), rounded once.
hipError_t launch_mx_reduce_n(int dtype, void* dst, const void* const* payloads, int k,
                              size_t n, float scale, hipStream_t s);
// The same fold, quantised again.  payload may be one of the sources.
hipError_t launch_mx_requantize_n(void* payload, const void* const* payloads, int k, size_t n,
                                  float scale, hipStream_t s);

}  // namespace glx
