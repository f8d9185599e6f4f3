// vfsx_prob_device.h -- device code that vfsx_prob.hip and vfsx_f8.hip share.
#pragma once

#include <hip/hip_runtime.h>

#include "vfsx_prob.h"

namespace vfsx {
namespace {

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// exponent of block kb; `p` = the row's first dword of scales
__device__ __forceinline__ int f8_exp_of(const uint32_t *p, uint32_t kb)
{
    return (int)((p[(size_t)(kb >> 2) * 64u] >> (8u * (kb & 3u))) & 255u) - 127;
}

__device__ __forceinline__ float fma_of(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_of(double a, double b, double c) { return __builtin_fma(a, b, c); }

__device__ __forceinline__ float i8_at(uint32_t w, int i) { return (float)((int32_t)(w << (24 - 8 * i)) >> 24); }

// sum of squares of a stored chunk (4 f32 or 16 int8; the 8-bit copy's norms are those of its f32 rows)
template <int SRC>
__device__ __forceinline__ double chunk_square(uint4 v)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (SRC == kProbI8) {
        int s = 0; // exact
#pragma unroll
        for (int i = 0; i < 4; ++i)
            s = __builtin_amdgcn_sdot4((int)w[i], (int)w[i], s, false);
        return (double)s;
    } else {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double a = (double)__uint_as_float(w[i]);
            s = __builtin_fma(a, a, s);
        }
        return s;
    }
}

// acc + chunk c of a row times the same elements of q (row-major, dim elements; stored chunks are zero beyond dim)
template <int SRC, typename T>
__device__ __forceinline__ T chunk_dot(uint4 v, const float *__restrict__ q, uint32_t c, uint32_t dim, T acc)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (SRC == kProbI8) {
#pragma unroll
        for (uint32_t i = 0; i < 16u; ++i) {
            const uint32_t k = c * 16u + i;
            if (k < dim)
                acc = fma_of((T)i8_at(w[i >> 2], i & 3), (T)q[k], acc);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t k = c * 4u + i;
            if (k < dim)
                acc = fma_of((T)__uint_as_float(w[i]), (T)q[k], acc);
        }
    }
    return acc;
}

// 16 e4m3 values times 16 bf16 values
__device__ __forceinline__ double f8_chunk_dot64(uint4 u, uint4 v0, uint4 v1)
{
    const uint32_t a[4] = {u.x, u.y, u.z, u.w}, b[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x[4] = {__builtin_amdgcn_cvt_f32_fp8((int)a[i], 0), __builtin_amdgcn_cvt_f32_fp8((int)a[i], 1),
                            __builtin_amdgcn_cvt_f32_fp8((int)a[i], 2), __builtin_amdgcn_cvt_f32_fp8((int)a[i], 3)};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t w = b[2 * i + j];
            s = __builtin_fma((double)x[2 * j], (double)__uint_as_float(w << 16), s);
            s = __builtin_fma((double)x[2 * j + 1], (double)__uint_as_float(w & 0xffff0000u), s);
        }
    }
    return s;
}

// The sums of a piece are over 2^(l log2e - base), base = m log2e rounded to f32 (one fused operation per exponent); the second pass takes
// the same base.  Beyond 1e30 the product would leave the range of f32: there the sums are over 2^((l - m) log2e).
constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float piece_base(float m) { return m * kLog2e; }
__device__ __forceinline__ bool piece_is_huge(float m) { return !(fabsf(m) < 1e30f); }
// ... in f64, in units of log 2
__device__ __forceinline__ double piece_base64(float m) { return piece_is_huge(m) ? (double)m * (double)kLog2e : (double)piece_base(m); }

} // namespace
} // namespace vfsx
