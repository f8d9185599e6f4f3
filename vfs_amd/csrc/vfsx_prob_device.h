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

__device__ __forceinline__ double f8_chunk_dot64(uint4 u, uint4 v)
{
    const uint32_t a[4] = {u.x, u.y, u.z, u.w}, b[4] = {v.x, v.y, v.z, v.w};
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        s += (double)(__builtin_amdgcn_cvt_f32_fp8((int)a[i], 0) * __builtin_amdgcn_cvt_f32_fp8((int)b[i], 0));
        s += (double)(__builtin_amdgcn_cvt_f32_fp8((int)a[i], 1) * __builtin_amdgcn_cvt_f32_fp8((int)b[i], 1));
        s += (double)(__builtin_amdgcn_cvt_f32_fp8((int)a[i], 2) * __builtin_amdgcn_cvt_f32_fp8((int)b[i], 2));
        s += (double)(__builtin_amdgcn_cvt_f32_fp8((int)a[i], 3) * __builtin_amdgcn_cvt_f32_fp8((int)b[i], 3));
    }
    return s;
}

// q8 . x8 of one row, one thread
__device__ __forceinline__ float f8_dot(const ProbStore &st, const ProbQueries &qs, uint32_t qi, uint32_t row)
{
    const uint4 *x = st.f8 + (size_t)(row / 64u) * st.f8_chunks * 64u + (row & 63u);
    const uint4 *q = qs.q8 + (size_t)(qi / 64u) * st.f8_chunks * 64u + (qi & 63u);
    const uint32_t *xe = st.f8_exp + (size_t)(row / 64u) * st.f8_words * 64u + (row & 63u);
    const uint32_t *qe = qs.q8_exp + (size_t)(qi / 64u) * st.f8_words * 64u + (qi & 63u);
    float sum = 0.0f;
    for (uint32_t kb = 0; kb < st.f8_chunks / kF8ChunksPerBlock; ++kb) {
        float b = 0.0f;
        for (uint32_t c = 0; c < kF8ChunksPerBlock; ++c) {
            const uint4 u = x[(size_t)(kb * kF8ChunksPerBlock + c) * 64u], v = q[(size_t)(kb * kF8ChunksPerBlock + c) * 64u];
            const uint32_t ux[4] = {u.x, u.y, u.z, u.w}, vx[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                b = __builtin_fmaf(__builtin_amdgcn_cvt_f32_fp8((int)ux[i], 0), __builtin_amdgcn_cvt_f32_fp8((int)vx[i], 0), b);
                b = __builtin_fmaf(__builtin_amdgcn_cvt_f32_fp8((int)ux[i], 1), __builtin_amdgcn_cvt_f32_fp8((int)vx[i], 1), b);
                b = __builtin_fmaf(__builtin_amdgcn_cvt_f32_fp8((int)ux[i], 2), __builtin_amdgcn_cvt_f32_fp8((int)vx[i], 2), b);
                b = __builtin_fmaf(__builtin_amdgcn_cvt_f32_fp8((int)ux[i], 3), __builtin_amdgcn_cvt_f32_fp8((int)vx[i], 3), b);
            }
        }
        sum += ldexpf(b, f8_exp_of(xe, kb) + f8_exp_of(qe, kb));
    }
    return sum;
}

} // namespace
} // namespace vfsx
