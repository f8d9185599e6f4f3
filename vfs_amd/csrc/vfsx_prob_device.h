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

// acc + a whole stored chunk times the same elements of the query (q: anywhere; 16-byte loads need no more than the 4 bytes' alignment)
template <int SRC, typename T>
__device__ __forceinline__ T chunk_dot(uint4 v, const float *__restrict__ q, T acc)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    constexpr int kVec = SRC == kProbI8 ? 4 : 1;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        float a[4];
        __builtin_memcpy(a, q + 4 * j, 16);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            acc = fma_of(SRC == kProbI8 ? (T)i8_at(w[j], i) : (T)__uint_as_float(w[i]), (T)a[i], acc);
    }
    return acc;
}

// the same for chunk c when it is a row's last and not whole: the query has nothing beyond dim
template <int SRC, typename T>
__device__ __forceinline__ T chunk_dot_part(uint4 v, const float *__restrict__ q, uint32_t c, uint32_t dim, T acc)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    constexpr uint32_t per = SRC == kProbI8 ? 16u : 4u;
#pragma unroll
    for (uint32_t i = 0; i < per; ++i)
        if (c * per + i < dim)
            acc = fma_of(SRC == kProbI8 ? (T)i8_at(w[i >> 2], i & 3) : (T)__uint_as_float(w[i & 3]), (T)q[c * per + i], acc);
    return acc;
}

__device__ __forceinline__ float scaled(float v, int e) { return ldexpf(v, e); }
__device__ __forceinline__ double scaled(double v, int e) { return ldexp(v, e); }

// 16 e4m3 values times 16 bf16 values
template <typename T>
__device__ __forceinline__ T f8_chunk_dot(uint4 u, uint4 v0, uint4 v1)
{
    const uint32_t a[4] = {u.x, u.y, u.z, u.w}, b[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    T s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x[4] = {__builtin_amdgcn_cvt_f32_fp8((int)a[i], 0), __builtin_amdgcn_cvt_f32_fp8((int)a[i], 1),
                            __builtin_amdgcn_cvt_f32_fp8((int)a[i], 2), __builtin_amdgcn_cvt_f32_fp8((int)a[i], 3)};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t w = b[2 * i + j];
            s = fma_of((T)x[2 * j], (T)__uint_as_float(w << 16), s);
            s = fma_of((T)x[2 * j + 1], (T)__uint_as_float(w & 0xffff0000u), s);
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

// adds sums (s, u) over the base of m_part to sums over the base of m; s = 0: nothing there, NaN: a logit that is not finite
__device__ __forceinline__ void add_unit(float m, float m_part, double s, double u, double &S, double &U)
{
    if (s == 0.0)
        return;
    const double z = piece_base64(m_part) - piece_base64(m), e = (double)exp2f((float)z);
    S += s * e;
    U += e == 0.0 ? 0.0 : (u + z * s) * e;
}

} // namespace
} // namespace vfsx
