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
// lane takes 16 bytes of the widest float stream -- 4 elements beside fp32, 8
// otherwise --, so that a wave's loads and stores are contiguous: lanes of 32
// bytes in two halves ran 1 GiB of f32 with feedback in 646 us instead of 535.
// The lanes of a block (8 or 4) find its maximum in two or three DPP exchanges,
// without shared memory.  One pass per lane, no loop over a capped grid: the
// loop cost 10 to 20 % everywhere (256 MiB of bf16 quantised: 65 us with 4
// workgroups a CU, 57 us with one pass).  Float loads and stores are nontemporal.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.h"
#include "elem_ops.h"
#include "mx.h"

namespace glx {
namespace {

#define GLX_GLOBAL __attribute__((address_space(1)))
typedef float v2f __attribute__((ext_vector_type(2)));

struct F32 { using S = float; };
struct F16 { using S = _Float16; };
struct BF16 { using S = __bf16; };

template <int BYTES> struct Raw;
template <> struct Raw<8> {
  typedef unsigned type __attribute__((ext_vector_type(2), aligned(2)));
};
template <> struct Raw<16> {
  typedef unsigned type __attribute__((ext_vector_type(4), aligned(2)));
};

// A lane's E elements, element i on of the `left` there are from p; FULL: all of
// them are there.  Elements behind the end read as zero and are not written.
template <typename T, int E, bool FULL>
__device__ __forceinline__ void load(const GLX_GLOBAL typename T::S* p, uint32_t i, uint32_t left,
                                     float (&y)[E]) {
  using S = typename T::S;
  using R = typename Raw<E * sizeof(S)>::type;
  if (FULL || i + E <= left) {
    union { R v; S s[E]; } r;
    r.v = __builtin_nontemporal_load((const GLX_GLOBAL R*)(p + i));
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = (float)r.s[e];
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = i + e < left ? (float)p[i + e] : 0.f;
  }
}

template <typename T, int E, bool FULL>
__device__ __forceinline__ void store(GLX_GLOBAL typename T::S* p, uint32_t i, uint32_t left,
                                      const float (&y)[E]) {
  using S = typename T::S;
  using R = typename Raw<E * sizeof(S)>::type;
  if (FULL || i + E <= left) {
    union { R v; S s[E]; } r;
#pragma unroll
    for (int e = 0; e < E; e++) r.s[e] = (S)y[e];
    __builtin_nontemporal_store(r.v, (GLX_GLOBAL R*)(p + i));
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (i + e < left) p[i + e] = (S)y[e];
    }
  }
}

// The larger of v and that of the lane's partner under a DPP permutation.
template <int DPP>
__device__ __forceinline__ uint32_t max_with(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP, 0xf, 0xf, true);
  return v > o ? v : o;
}

// The conversions take the scale as a float of which they use the exponent
// field, with E8M0's meaning throughout: 0 is 2^-127, 255 makes every value NaN
// (all 256 bytes checked, with halfway points and their neighbours).
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

template <int SEL>
__device__ __forceinline__ uint32_t two_codes(uint32_t c, float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, a, b, scale, SEL);
}

// A block of which this lane holds E values: its scale byte, and the lane's
// codes.  The block's 32 / E lanes call it together.
struct Block {
  uint32_t code, scale;
};
template <int E>
__device__ __forceinline__ Block encode(const float (&y)[E]) {
  // bits of |y| order as the values do, NaN above infinity above all others
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const uint32_t b = __float_as_uint(y[e]) & 0x7fffffffu;
    top = top > b ? top : b;
  }
  top = max_with<0xb1>(top);               // lanes 1 0 3 2 of each four
  top = max_with<0x4e>(top);               // lanes 2 3 0 1
  if (E == 4) top = max_with<0x141>(top);  // mirrored in each eight
  const uint32_t e = top >> 23;
  if (e == 255) return {0, 255};
  const uint32_t s = e > 2 ? e - 2 : 0;
  const float sc = scale_of(s);
  uint32_t c = 0;
  c = two_codes<0>(c, y[0], y[1], sc);
  c = two_codes<1>(c, y[2], y[3], sc);
  if constexpr (E == 8) {
    c = two_codes<2>(c, y[4], y[5], sc);
    c = two_codes<3>(c, y[6], y[7], sc);
  }
  return {c, s};
}

template <int SEL>
__device__ __forceinline__ void two_values(uint32_t c, float scale, float* v) {
  const v2f p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, SEL);
  v[0] = p[0];
  v[1] = p[1];
}

// The values of E codes.
template <int E>
__device__ __forceinline__ void decode(uint32_t c, float scale, float (&v)[E]) {
  two_values<0>(c, scale, v);
  two_values<1>(c, scale, v + 2);
  if constexpr (E == 8) {
    two_values<2>(c, scale, v + 4);
    two_values<3>(c, scale, v + 6);
  }
}

// E codes of a lane, as they lie in a payload.
template <int E> struct Codes;
template <> struct Codes<4> { using type = uint16_t; };
template <> struct Codes<8> { using type = uint32_t; };

// What a workgroup of N threads takes: N * U lanes' parts from lane `first` (E
// elements each) on.  Everything is addressed from there with 32 bits, from pointers
// that are the same for the whole wave.  Only the last tile is not full.  (No
// 64-bit minimum of what is left and the tile's size: beside the comparison with
// the size the compiler made of it a select on a stale condition bit, seen in
// the assembly, and the tile counted as full.)
template <int E, int U, int N>
struct Tile {
  static constexpr uint32_t kLanes = 32 / E;  // of a block
  static constexpr size_t kParts = (size_t)N * U;
  size_t first;
  bool full;
  uint32_t lanes, left;  // lanes and elements there are, of a tile that is not full
  __device__ __forceinline__ Tile(size_t tile, size_t n, size_t nb)
      : first(tile * kParts),
        full(tile < n / (kParts * E)),
        lanes((uint32_t)(nb * kLanes - first)),
        left((uint32_t)(n - first * E)) {}
};

// Codes and scale of lane t of the tile.  Plain stores, unlike those of floats:
// what sends or opens the payload next finds it in the Infinity Cache (256 MiB
// of bf16 quantised and opened 102 instead of 109 us, four payloads folded into
// one and opened 144 instead of 151; the quantisation by itself is 2 % slower).
template <int E, int U, int N>
__device__ __forceinline__ void put_block(char* payload, size_t nb, const Tile<E, U, N>& tile,
                                          uint32_t t, Block b) {
  using C = typename Codes<E>::type;
  constexpr uint32_t kLanes = Tile<E, U, N>::kLanes;
  GLX_GLOBAL C* code = (GLX_GLOBAL C*)payload + tile.first;
  GLX_GLOBAL char* scale = (GLX_GLOBAL char*)payload + nb * 16 + tile.first / kLanes;
  code[t] = (C)b.code;
  if (t % kLanes == 0) scale[t / kLanes] = (char)b.scale;
}

// The zero bytes behind the last scale, by the workgroup of the tile that is not
// full (full tiles alone hold a multiple of 16 blocks, and need none).
__device__ __forceinline__ void put_padding(char* payload, size_t nb) {
  if (threadIdx.x < (16 - nb % 16) % 16) {
    ((GLX_GLOBAL char*)payload)[nb * 17 + threadIdx.x] = 0;
  }
}

// E elements a lane, U such parts a thread (a workgroup apart).  256 MiB of
// bf16: U = 1 57 us, 2 54 us, 4 55 us; 512 MiB of f32: 103, 94, 97 us; 1 GiB of
// f32 with feedback: 525, 561, 540 us.
template <typename T, bool FEEDBACK>
struct QuantizeShape {
  static constexpr int E = FEEDBACK || sizeof(typename T::S) == 4 ? 4 : 8;
  static constexpr int U = FEEDBACK ? 1 : 2;
};

// Folds into floats, 1 GiB of f32: one payload 227, 192, 216 us with U = 1, 2,
// 4; four 285, 266, 276; eight 370, 387, 372 (into 256 MiB of bf16 128, 137, 132).
template <int K>
constexpr int kReduceParts = K <= 4 ? 2 : 1;
// ... by 512 threads: with 256 the scale bytes of a 128-byte line belong to four
// workgroups, and as many XCDs fetch it (1342 MB read for 1141 MB of eight
// payloads): 370 us; 512 threads 354, 1024 382.  One payload 190, 180, 216.
constexpr int kReduceThreads = 512;

// Folds into a payload, whose lanes do little but load: 128 Mi elements of one
// payload 29, 25, 23 us with U = 2, 4, 8; four 59, 57, 58; eight 110, 101, 107.
// From nine sources on four parts would not fit the registers.  (Both rules were
// measured at one, four and eight sources; the numbers between follow the nearest.)
template <int K>
constexpr int kRequantizeParts = K <= 8 ? 4 : 2;

template <typename T, bool RES_IN, bool RES_OUT, bool FULL, int E, int U, int N>
__device__ __forceinline__ void quantize_tile(char* payload, const typename T::S* x_,
                                              const float* residual_, float* residualOut_,
                                              size_t nb, const Tile<E, U, N>& tile) {
  const GLX_GLOBAL typename T::S* x = (const GLX_GLOBAL typename T::S*)x_ + tile.first * E;
  const GLX_GLOBAL float* residual = (const GLX_GLOBAL float*)residual_ + tile.first * E;
  GLX_GLOBAL float* residualOut = (GLX_GLOBAL float*)residualOut_ + tile.first * E;
  float y[U][E], r[U][E];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t t = threadIdx.x + u * N;
    if (!FULL && t >= tile.lanes) continue;
    load<T, E, FULL>(x, t * E, tile.left, y[u]);
    if constexpr (RES_IN) load<F32, E, FULL>(residual, t * E, tile.left, r[u]);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t t = threadIdx.x + u * N;
    if (!FULL && t >= tile.lanes) continue;
    if constexpr (RES_IN) {
#pragma unroll
      for (int e = 0; e < E; e++) y[u][e] = __fadd_rn(y[u][e], r[u][e]);
    }
    const Block b = encode<E>(y[u]);
    put_block(payload, nb, tile, t, b);
    if constexpr (RES_OUT) {
      float v[E];
      decode<E>(b.code, scale_of(b.scale), v);
#pragma unroll
      for (int e = 0; e < E; e++) v[e] = b.scale == 255 ? 0.f : y[u][e] - v[e];  // exact
      store<F32, E, FULL>(residualOut, t * E, tile.left, v);
    }
  }
}

template <typename T, bool RES_IN, bool RES_OUT>
__global__ __launch_bounds__(kBlock) void mx_quantize_kernel(char* payload,
                                                             const typename T::S* x,
                                                             const float* residual,
                                                             float* residualOut, size_t n,
                                                             size_t nb, size_t tile0) {
  using Q = QuantizeShape<T, RES_IN || RES_OUT>;
  const Tile<Q::E, Q::U, kBlock> tile(tile0 + blockIdx.x, n, nb);
  if (tile.full) {
    quantize_tile<T, RES_IN, RES_OUT, true>(payload, x, residual, residualOut, nb, tile);
  } else {
    quantize_tile<T, RES_IN, RES_OUT, false>(payload, x, residual, residualOut, nb, tile);
    put_padding(payload, nb);
  }
}

struct MxSources {
  const char* p[kMxMaxSources];
};

// What lane t of a tile reads of every source: all loads before the first use.
// NT: nontemporal (see streaming()).
template <int K, int E, bool NT>
struct Part {
  typename Codes<E>::type code[K];
  uint8_t scale[K];
  template <int U, int N>
  __device__ __forceinline__ void load(const MxSources& src, size_t nb,
                                       const Tile<E, U, N>& tile, uint32_t t) {
    using C = typename Codes<E>::type;
    constexpr uint32_t kLanes = Tile<E, U, N>::kLanes;
#pragma unroll
    for (int j = 0; j < K; j++) {
      const GLX_GLOBAL C* c = (const GLX_GLOBAL C*)src.p[j] + tile.first;
      const GLX_GLOBAL uint8_t* s =
          (const GLX_GLOBAL uint8_t*)src.p[j] + nb * 16 + tile.first / kLanes;
      code[j] = NT ? __builtin_nontemporal_load(c + t) : c[t];
      scale[j] = s[t / kLanes];
    }
  }
  // the left fold, times `by`
  __device__ __forceinline__ void fold(float by, float (&acc)[E]) const {
    decode<E>(code[0], scale_of(scale[0]), acc);
#pragma unroll
    for (int j = 1; j < K; j++) {
      float v[E];
      decode<E>(code[j], scale_of(scale[j]), v);
#pragma unroll
      for (int e = 0; e < E; e++) acc[e] = __fadd_rn(acc[e], v[e]);
    }
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] = __fmul_rn(acc[e], by);
  }
};

template <typename T, int K, bool NT, bool FULL, int E, int U, int N>
__device__ __forceinline__ void reduce_tile(typename T::S* dst, const MxSources& src, size_t nb,
                                            float scale, const Tile<E, U, N>& tile) {
  Part<K, E, NT> part[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t t = threadIdx.x + u * N;
    if (FULL || t < tile.lanes) part[u].load(src, nb, tile, t);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t t = threadIdx.x + u * N;
    if (!FULL && t >= tile.lanes) continue;
    float acc[E];
    part[u].fold(scale, acc);
    store<T, E, FULL>((GLX_GLOBAL typename T::S*)dst + tile.first * E, t * E, tile.left, acc);
  }
}

template <typename T, int K, bool NT>
__global__ __launch_bounds__(kReduceThreads) void mx_reduce_n_kernel(typename T::S* dst,
                                                                     MxSources src, size_t n,
                                                                     size_t nb, float scale,
                                                                     size_t tile0) {
  constexpr int E = 16 / sizeof(typename T::S), U = kReduceParts<K>;
  const Tile<E, U, kReduceThreads> tile(tile0 + blockIdx.x, n, nb);
  if (tile.full) {
    reduce_tile<T, K, NT, true>(dst, src, nb, scale, tile);
  } else {
    reduce_tile<T, K, NT, false>(dst, src, nb, scale, tile);
  }
}

template <int K, bool NT, bool FULL, int E, int U, int N>
__device__ __forceinline__ void requantize_tile(char* payload, const MxSources& src, size_t nb,
                                                float scale, const Tile<E, U, N>& tile) {
  Part<K, E, NT> part[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t t = threadIdx.x + u * N;
    if (FULL || t < tile.lanes) part[u].load(src, nb, tile, t);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t t = threadIdx.x + u * N;
    if (!FULL && t >= tile.lanes) continue;
    float acc[E];
    part[u].fold(scale, acc);
    if (!FULL) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (t * E + e >= tile.left) acc[e] = 0.f;  // behind the end, whatever the sources hold
      }
    }
    put_block(payload, nb, tile, t, encode<E>(acc));
  }
}

template <int K, bool NT>
__global__ __launch_bounds__(kBlock) void mx_requantize_n_kernel(char* payload, MxSources src,
                                                                 size_t n, size_t nb,
                                                                 float scale, size_t tile0) {
  constexpr int E = 8, U = kRequantizeParts<K>;
  const Tile<E, U, kBlock> tile(tile0 + blockIdx.x, n, nb);
  if (tile.full) {
    requantize_tile<K, NT, true>(payload, src, nb, scale, tile);
  } else {
    requantize_tile<K, NT, false>(payload, src, nb, scale, tile);
    put_padding(payload, nb);
  }
}

// One workgroup per tile, so many tiles a launch: a grid has fewer than 2^32
// threads.  go(grid, the launch's first tile).
constexpr size_t kTilesPerLaunch = size_t(1) << 19;

template <typename Go>
hipError_t over_tiles(size_t nb, int e, int u, int threads, Go go) {
  const size_t per = (size_t)threads * u, tiles = (nb * (32 / e) + per - 1) / per;
  for (size_t at = 0; at < tiles; at += kTilesPerLaunch) {
    go(dim3((unsigned)std::min(tiles - at, kTilesPerLaunch)), at);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

template <typename T, bool RES_IN, bool RES_OUT>
hipError_t quantize_with(void* payload, const void* x, const float* r, float* ro, size_t n,
                         hipStream_t s) {
  using Q = QuantizeShape<T, RES_IN || RES_OUT>;
  const size_t nb = mxBlocks(n);
  return over_tiles(nb, Q::E, Q::U, kBlock, [&](dim3 grid, size_t tile0) {
    hipLaunchKernelGGL((mx_quantize_kernel<T, RES_IN, RES_OUT>), grid, dim3(kBlock), 0, s,
                       (char*)payload, (const typename T::S*)x, r, ro, n, nb, tile0);
  });
}

template <typename T>
hipError_t quantize_typed(void* payload, const void* x, const float* r, float* ro, size_t n,
                          hipStream_t s) {
  if (r != nullptr) {
    return ro != nullptr ? quantize_with<T, true, true>(payload, x, r, ro, n, s)
                         : quantize_with<T, true, false>(payload, x, r, ro, n, s);
  }
  return ro != nullptr ? quantize_with<T, false, true>(payload, x, r, ro, n, s)
                       : quantize_with<T, false, false>(payload, x, r, ro, n, s);
}

// Whether a fold reads its sources with nontemporal loads: if there are several
// and each starts at a 128-byte line.  Eight payloads into 512 MiB of f32: 186
// instead of 203 us.  Where they start inside lines every wave shares its first
// and last line with its neighbours, and these want it kept: 220 instead of 200
// us.  A single payload is mostly opened right after it came, out of the cache:
// 98 instead of 86 us.
bool streaming(const MxSources& src, int k) {
  uintptr_t at = 0;
  for (int j = 0; j < k; j++) at |= (uintptr_t)src.p[j];
  return k > 1 && at % 128 == 0;
}

template <typename T, int K>
hipError_t reduce_k(void* dst, const MxSources& src, size_t n, float scale, hipStream_t s) {
  constexpr int E = 16 / sizeof(typename T::S);
  const size_t nb = mxBlocks(n);
  const bool nt = streaming(src, K);
  return over_tiles(nb, E, kReduceParts<K>, kReduceThreads, [&](dim3 grid, size_t tile0) {
    if (K > 1 && nt) {
      hipLaunchKernelGGL((mx_reduce_n_kernel<T, K, (K > 1)>), grid, dim3(kReduceThreads), 0, s,
                         (typename T::S*)dst, src, n, nb, scale, tile0);
    } else {
      hipLaunchKernelGGL((mx_reduce_n_kernel<T, K, false>), grid, dim3(kReduceThreads), 0, s,
                         (typename T::S*)dst, src, n, nb, scale, tile0);
    }
  });
}

template <int K>
hipError_t requantize_k(void* payload, const MxSources& src, size_t n, float scale,
                        hipStream_t s) {
  const size_t nb = mxBlocks(n);
  const bool nt = streaming(src, K);
  return over_tiles(nb, 8, kRequantizeParts<K>, kBlock, [&](dim3 grid, size_t tile0) {
    if (K > 1 && nt) {
      hipLaunchKernelGGL((mx_requantize_n_kernel<K, (K > 1)>), grid, dim3(kBlock), 0, s,
                         (char*)payload, src, n, nb, scale, tile0);
    } else {
      hipLaunchKernelGGL((mx_requantize_n_kernel<K, false>), grid, dim3(kBlock), 0, s,
                         (char*)payload, src, n, nb, scale, tile0);
    }
  });
}

// The number of sources as a constant, so that all of a lane's loads are in
// flight before the first is used.
template <typename T, int K = 1>
hipError_t reduce_typed(int k, void* dst, const MxSources& src, size_t n, float scale,
                        hipStream_t s) {
  if (k == K) return reduce_k<T, K>(dst, src, n, scale, s);
  if constexpr (K < kMxMaxSources) return reduce_typed<T, K + 1>(k, dst, src, n, scale, s);
  return hipErrorInvalidValue;
}

template <int K = 1>
hipError_t requantize_any(int k, void* payload, const MxSources& src, size_t n, float scale,
                          hipStream_t s) {
  if (k == K) return requantize_k<K>(payload, src, n, scale, s);
  if constexpr (K < kMxMaxSources) return requantize_any<K + 1>(k, payload, src, n, scale, s);
  return hipErrorInvalidValue;
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
    case GLX_FLOAT32: return reduce_typed<F32>(k, dst, src, n, scale, s);
    case GLX_FLOAT16: return reduce_typed<F16>(k, dst, src, n, scale, s);
    case GLX_BFLOAT16: return reduce_typed<BF16>(k, dst, src, n, scale, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_mx_requantize_n(void* payload, const void* const* payloads, int k, size_t n,
                                  float scale, hipStream_t s) {
  if (n == 0) return hipSuccess;
  if (k < 1 || k > kMxMaxSources) return hipErrorInvalidValue;
  return requantize_any(k, payload, sources(payloads, k), n, scale, s);
}

}  // namespace glx
