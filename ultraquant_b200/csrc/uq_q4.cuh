// The stored form of 4-bit weights, shared by the codec, the lookup and the
// products: w[n, k] = s e[n, k / g] q[n, k], q = u - 8 with u in 4 bits, e in
// E4M3, s a float per matrix.  Eight consecutive elements are one little-endian
// 32-bit word whose nibbles 0 .. 7 hold elements 0 2 4 6 1 3 5 7, so that
// (word >> 4 i) & 0x000f000f is the pair (2 i, 2 i + 1) in 16-bit halves.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <stdint.h>

#include "uq_common.cuh"

namespace uq {
namespace q4 {

// Launches what writes to `out` (device) what the products met since the last call,
// and clears it: [0] a wait that gave up, [1] an offset out of range (uq_q4mm.cu).
void mm_take_flags(int *out, cudaStream_t st);
inline bool group_ok(int g) { return g == 32 || g == 64 || g == 128 || g == 256; }
inline bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

#if defined(__CUDACC__)
__device__ __forceinline__ float e4m3_value(uint8_t b) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}
// Nibble of element i (0 .. 7) of a word.
__device__ __forceinline__ int nibble(uint32_t w, int i) { return int((w >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u); }

// q of element i as a float: u under the significand of 2^23, less 2^23 + 8 (a
// conversion instruction would have a quarter of the rate).
__device__ __forceinline__ float q_of(uint32_t w, int i) { return __uint_as_float(0x4b000000u | uint32_t(nibble(w, i))) - 8388616.0f; }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(double v) { return float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Eight consecutive values, 16-byte aligned, as floats and back.
template <typename T> __device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
    constexpr int N = int(sizeof(T)) / 2;   // 16-byte vectors
    union { uint4 v[N]; T t[8]; } u;
#pragma unroll
    for (int i = 0; i < N; ++i) u.v[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(u.t[i]);
}
template <typename T> __device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    constexpr int N = int(sizeof(T)) / 2;
    union { uint4 v[N]; T t[8]; } u;
#pragma unroll
    for (int i = 0; i < 8; ++i) u.t[i] = from_float<T>(x[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) __stcs(reinterpret_cast<uint4 *>(p) + i, u.v[i]);
}
#endif

}  // namespace q4
}  // namespace uq
