// elem.cuh — element types of the answer operators.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace ytm {

inline bool is_float_type(int t) { return t == YTM_F32 || t == YTM_F16 || t == YTM_BF16; }
inline bool is_sum_type(int t) { return is_float_type(t) || t == YTM_I32; }
inline int64_t type_bytes(int t) { return t == YTM_F16 || t == YTM_BF16 ? 2 : 4; }

__host__ __device__ inline int64_t q4_row_bytes(int C) { return ((int64_t)C + 31) / 32 * 16; }

__device__ __forceinline__ float to_f32(int32_t v) { return (float)v; }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ double to_f64(int32_t v) { return (double)v; }
__device__ __forceinline__ double to_f64(float v) { return (double)v; }
__device__ __forceinline__ double to_f64(__half v) { return (double)__half2float(v); }
__device__ __forceinline__ double to_f64(__nv_bfloat16 v) { return (double)__bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Bit k of a row of allowed-class words (NULL: every class is allowed).
__device__ __forceinline__ bool is_allowed(const uint32_t *row, int64_t k) {
    return !row || ((row[k >> 5] >> (k & 31)) & 1u);
}

__device__ __forceinline__ int64_t index_at(const void *p, int is64, int64_t i) {
    return is64 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

// Two fp32 operations in one instruction, on register pairs.
using F2 = unsigned long long;
__device__ __forceinline__ F2 pair(float x, float y) {
    F2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ void split(F2 a, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

}  // namespace ytm
