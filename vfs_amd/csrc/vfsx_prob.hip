// vfsx_prob.hip -- log probabilities over a store: softmax statistics, the most probable rows, given rows.
//
//   l_j = sim(q, x_j) / T + b_j            rows with b_j = -inf (or without a cosine) are not there at all
//   lse = log sum_j exp(l_j),  H = -sum_j p_j log p_j,  log p_j = l_j - lse
//
// First pass (the store is read once, logits are never written): for each query and PIECE of 128 rows
//   m = max l,  s = sum exp(l - m),  t = sum exp(l - m) (l - m)
// and for each GROUP of 16 rows its maximum.  Second pass, one workgroup per query: with M = max m
//   S = sum s e^(m-M),  U = sum (t + (m - M) s) e^(m-M),   lse = M + log S,   H = log S - U / S
// First-pass logits are f32 (f32-grade
// products, f32 exponentials); the joined sums are f64.
//
// Most probable rows: first-pass logits are off by at most eps (below), so a row of the true top k lies in a group whose maximum is
// at least (k-th largest group maximum) - 2 eps.  The rows of those groups, about k of them, are computed again in f64 and ordered by
// (logit descending, row ascending): the order is that of the f64 logits, whatever the first pass rounded.  Given rows are
// computed in f64 too.
//
// eps: a product of d terms accumulated in f32 in any order, from operands exact to 2^-22 (f16 pairs), is within
// (d + 64) 2^-24 |q| |x| of its value; |x| <= the largest row norm of the store.  The factor and the bias add 2^-22 |l|.
//
// A logit that is NaN or infinite makes s or t NaN (inf - inf, 0 * inf), and with it every result of its query.
#include <hip/hip_runtime.h>

#include "vfsx_internal.h"
#include "vfsx_prob.h"
#include "vfsx_prob_device.h"

#pragma clang fp contract(off)

namespace vfsx {

namespace {

// 2^a, the scale that brings vectors of norm r into the range of f16 pairs: r 2^a in (2^9, 2^10], so that elements 2^19 times smaller
// than the norm still have a normal low half.  r = 0: 1; NaN or infinite: NaN.
__device__ __forceinline__ float pair_scale(double r)
{
    if (!(r < __builtin_inf()))
        return __builtin_nanf("");
    if (r == 0.0)
        return 1.0f;
    int e;
    (void)frexp(r, &e); // r = m 2^e, m in [0.5, 1)
    e = 10 - e;
    e = e > 126 ? 126 : (e < -126 ? -126 : e);
    return __uint_as_float((uint32_t)(127 + e) << 23);
}

// ---- operands of a store: 1 / |x| per row, the largest |x| -------------------------------------------------------------------
// One thread per row.  Norms in f64: they divide every logit.  A norm whose square is zero in f32 counts as zero.
template <int SRC>
__global__ __launch_bounds__(256) void prob_rows_kernel(const uint4 *__restrict__ rows, uint32_t d_chunks, uint32_t row0, uint32_t n_rows,
                                                        float *__restrict__ row_inv, float *__restrict__ row_scale,
                                                        float *__restrict__ max_norm)
{
    const uint64_t row = (uint64_t)row0 + (uint64_t)blockIdx.x * 256u + threadIdx.x;
    float norm = 0.0f;
    if (row < n_rows) {
        const uint4 *p = rows + (size_t)(row >> 6) * d_chunks * 64u + (row & 63u);
        double s = 0.0;
        for (uint32_t c = 0; c < d_chunks; ++c)
            s += chunk_square<SRC>(p[(size_t)c * 64u]);
        const double r = __builtin_sqrt(s);
        row_inv[row] = (float)s == 0.0f ? -1.0f : (float)(1.0 / r);
        if (SRC == kProbF32)
            row_scale[row] = pair_scale(r);
        norm = (float)r;
    }
    norm = norm < __builtin_inff() ? norm : 0.0f; // (a row with a NaN or an infinity has no finite logit)
    for (int o = 32; o; o >>= 1)
        norm = fmaxf(norm, __shfl_xor(norm, o, 64));
    if ((threadIdx.x & 63u) == 0) // floats >= 0 order as their bits
        atomicMax((uint32_t *)max_norm, __float_as_uint(norm));
}

// ---- queries -------------------------------------------------------------------------------------------------------------------
// One wave per query: its norm, its factor (logit = product * factor [/ |x|] + bias) and its f16 pairs.  Pairs lie as the rows do in rb64:
// 64-query blocks of 1 KiB pieces, piece 2 c + part = elements 8 c .. 8 c + 7 of 64 queries, part 0 = hi, 1 = lo.
__global__ __launch_bounds__(64) void prob_queries_kernel(ProbStore st, const float *__restrict__ q, uint32_t nq, uint32_t pair_chunks,
                                                          float *__restrict__ fac, float *__restrict__ eps, double *__restrict__ norm,
                                                          uint4 *__restrict__ pairs)
{
    const uint32_t qi = blockIdx.x, lane = threadIdx.x;
    const bool there = qi < nq;
    const float *src = q + (size_t)qi * st.dim;
    double s = 0.0;
    if (there) {
        for (uint32_t j = lane; j < st.dim; j += 64u) {
            const double v = src[j];
            s = __builtin_fma(v, v, s);
        }
        for (int o = 32; o; o >>= 1)
            s += __shfl_xor(s, o, 64);
    }
    const double r = __builtin_sqrt(s);
    const float scale = pair_scale(r);
    if (pairs) {
        uint4 *dst = pairs + (size_t)(qi / 64u) * pair_chunks * 128u + (qi & 63u);
        for (uint32_t c = lane; c < pair_chunks; c += 64u) {
            uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
            if (there) {
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) {
                    const uint32_t k = c * 8u + i;
                    const float x = k < st.dim ? src[k] * scale : 0.0f;
                    const _Float16 h = (_Float16)x;
                    const _Float16 l = (_Float16)(x - (float)h);
                    hi[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, h) << (16u * (i & 1u));
                    lo[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, l) << (16u * (i & 1u));
                }
            }
            dst[(size_t)c * 128u] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            dst[(size_t)c * 128u + 64u] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
    if (lane || !there)
        return;
    const bool zero = (float)s == 0.0f;
    norm[qi] = zero ? 0.0 : r;
    const double by = (pairs ? (double)scale : 1.0) * st.divide;
    fac[qi] = (float)(1.0 / (st.cosine ? (zero ? by : by * r) : by));
    const double part = st.cosine ? 1.0 : r * (double)*st.max_norm;
    // 8-bit copies are up to 1 + 2^-4 times as long as their originals, each
    const double e = (double)(st.dim + 64u) * 0x1p-24 * (st.source == kProbF8 ? 1.25 : 1.0) * part / __builtin_fabs(st.divide);
    eps[qi] = (float)(e * (1.0 + 0x1p-20));
}

// ---- second pass -----------------------------------------------------------------------------------------------------------------
constexpr uint32_t kFinThreads = 256;
constexpr uint32_t kFinWaves = kFinThreads / 64;
constexpr uint32_t kFinGroups = 1024; // candidate groups kept at once
constexpr uint32_t kFinRows = 1024;   // candidate rows kept at once (64 groups)

struct FinCand {
    double l;
    uint32_t row;
    uint32_t pad;
};

// The logit of 16 rows of a group (lane & 15), in f64, on every lane; each quarter of the wave takes every fourth chunk.  Lanes whose
// row is not there get -inf.
template <int SRC>
__device__ double group_logit(const ProbStore &st, const ProbQueries &qs, uint32_t qi, uint32_t group, bool one_row, uint32_t the_row)
{
    // one_row: all 64 lanes share `the_row` and split its chunks
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t row = one_row ? the_row : group * kGroupRows + (lane & 15u);
    const uint32_t first = one_row ? lane : lane >> 4, step = one_row ? 64u : 4u;
    bool in = row < st.n_rows;
    float b = 0.0f;
    if (in) {
        b = st.bias ? st.bias[row] : 0.0f;
        in = b != neg_inf();
        if (st.cosine)
            in = in && st.row_inv[row] >= 0.0f && qs.norm[qi] > 0.0;
    }
    double dot = 0.0, sq = 0.0;
    if (in) {
        if (SRC == kProbF8) {
            const uint4 *x = st.f8 + (size_t)(row / 64u) * st.f8_chunks * 64u + (row & 63u);
            const uint4 *q = qs.operand + (size_t)(qi / 64u) * st.f8_chunks * 128u + (qi & 63u);
            const uint32_t *xe = st.f8_exp + (size_t)(row / 64u) * st.f8_words * 64u + (row & 63u);
            for (uint32_t c = first; c < st.f8_chunks; c += step) // (e4m3 times bf16 is exact in f32, their sums in f64; a power of two scales)
                dot += ldexp(f8_chunk_dot64(x[(size_t)c * 64u], q[(size_t)c * 128u], q[(size_t)c * 128u + 64u]), f8_exp_of(xe, c / kF8ChunksPerBlock));
        }
        if (SRC != kProbF8 || st.cosine) {
            const uint4 *p = st.rows + (size_t)(row >> 6) * st.d_chunks * 64u + (row & 63u);
            const float *q = qs.q + (size_t)qi * st.dim;
            for (uint32_t c = first; c < st.d_chunks; c += step) {
                const uint4 v = p[(size_t)c * 64u];
                if (SRC != kProbF8)
                    dot = chunk_dot<SRC, double>(v, q, c, st.dim, dot);
                if (st.cosine)
                    sq += chunk_square<SRC>(v);
            }
        }
    }
    if (one_row) {
        for (int o = 1; o < 16; o <<= 1) {
            dot += __shfl_xor(dot, o, 64);
            sq += __shfl_xor(sq, o, 64);
        }
    }
    for (int o = 16; o < 64; o <<= 1) {
        dot += __shfl_xor(dot, o, 64);
        sq += __shfl_xor(sq, o, 64);
    }
    if (!in)
        return -__builtin_inf();
    return (st.cosine ? dot / (qs.norm[qi] * __builtin_sqrt(sq) * st.divide) : dot / st.divide) + (double)b;
}

__device__ __forceinline__ bool cand_before(double la, uint32_t ra, double lb, uint32_t rb) { return la > lb || (la == lb && ra < rb); }

// the k-th largest of n floats in LDS (n >= k >= 1), every thread gets it: rank by counting
__device__ float kth_of(const float *v, uint32_t n, uint32_t k, float *out)
{
    for (uint32_t i = threadIdx.x; i < n; i += kFinThreads) {
        const float a = v[i];
        uint32_t before = 0;
        for (uint32_t j = 0; j < n; ++j)
            before += (v[j] > a || (v[j] == a && j < i)) ? 1u : 0u;
        if (before == k - 1u)
            *out = a;
    }
    __syncthreads();
    const float r = *out;
    __syncthreads();
    return r;
}

template <int SRC>
__global__ __launch_bounds__(kFinThreads) void prob_finish_kernel(ProbStore st, ProbQueries qs, ProbFinish f)
{
    const uint32_t qi = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const float4 *pieces = f.pieces + (size_t)qi * st.n_pieces;
    const float *groups = f.groups + (size_t)qi * st.n_pieces * kGroupsPerPiece;

    __shared__ double red[2][kFinWaves];
    __shared__ float fred[kFinWaves];
    __shared__ float lv[kFinGroups];      // maxima: of the threads' shares, then of the candidate groups
    __shared__ uint32_t lg[kFinGroups];   // candidate groups
    __shared__ FinCand cand[kFinRows + VFSX_LOG_PROBS_MAX_K];
    __shared__ FinCand best[VFSX_LOG_PROBS_MAX_K];
    __shared__ uint32_t n_lg, n_cand;
    __shared__ float kth;

    // ---- M, S, U ------------------------------------------------------------------------------------------------------------
    float m = neg_inf();
    for (uint32_t i = tid; i < st.n_pieces; i += kFinThreads)
        m = fmaxf(m, pieces[i].x);
    const float my_max = m;
    for (int o = 1; o < 64; o <<= 1)
        m = fmaxf(m, __shfl_xor(m, o, 64));
    if (lane == 0)
        fred[wave] = m;
    __syncthreads();
    m = fred[0];
    for (uint32_t w = 1; w < kFinWaves; ++w)
        m = fmaxf(m, fred[w]);
    double S = 0.0, U = 0.0; // over 2^(l log2e - base), exponents in units of log 2
    const double base = piece_base64(m), L = (double)kLog2e;
    for (uint32_t i = tid; i < st.n_pieces; i += kFinThreads) {
        const float4 p = pieces[i];
        if (p.y != 0.0f) { // (0: no row of the piece is there; NaN: a logit that is not finite)
            const double z = piece_base64(p.x) - base, e = (double)exp2f((float)z);
            S += (double)p.y * e;
            U += e == 0.0 ? 0.0 : ((double)p.z + z * (double)p.y) * e;
        }
    }
    for (int o = 1; o < 64; o <<= 1) {
        S += __shfl_xor(S, o, 64);
        U += __shfl_xor(U, o, 64);
    }
    if (lane == 0) {
        red[0][wave] = S;
        red[1][wave] = U;
    }
    __syncthreads();
    S = red[0][0], U = red[1][0];
    for (uint32_t w = 1; w < kFinWaves; ++w) {
        S += red[0][w];
        U += red[1][w];
    }
    const bool poisoned = !(S < __builtin_inf()) || U != U; // (S is about 1 or more, or 0 otherwise)
    const bool none = S == 0.0;
    const double nan = __builtin_nan("");

    // ---- the k most probable rows (one at least: it is what the sums are corrected by) -----------------------------------------------
    const uint32_t k = f.k ? f.k : 1u;
    uint32_t have = 0; // rows in best[], ordered
    if (!poisoned && !none) {
        // a first bound: the k-th largest of the threads' maxima (k <= kFinThreads pieces or more reach it)
        lv[tid] = my_max;
        __syncthreads();
        const float bound = kth_of(lv, kFinThreads, k, &kth);
        float thr = bound - 2.0f * qs.eps[qi] - 0x1p-21f * fmaxf(fabsf(bound), fabsf(m));
        if (bound == neg_inf())
            thr = neg_inf();
        if (tid == 0)
            n_lg = 0, n_cand = 0;
        __syncthreads();
        for (uint32_t i = tid; i < st.n_pieces; i += kFinThreads) {
            if (!(pieces[i].x >= thr) || pieces[i].x == neg_inf())
                continue;
            for (uint32_t g = 0; g < kGroupsPerPiece; ++g) {
                const float v = groups[(size_t)i * kGroupsPerPiece + g];
                if (v >= thr && v != neg_inf()) {
                    const uint32_t at = atomicAdd(&n_lg, 1u);
                    if (at < kFinGroups) {
                        lv[at] = v;
                        lg[at] = i * kGroupsPerPiece + g;
                    }
                }
            }
        }
        __syncthreads();
        bool whole = n_lg <= kFinGroups;
        if (whole) {
            const uint32_t n = n_lg;
            if (n > k) { // the k-th largest group maximum: a closer bound
                const float g = kth_of(lv, n, k, &kth);
                thr = fmaxf(thr, g - 2.0f * qs.eps[qi] - 0x1p-21f * fmaxf(fabsf(g), fabsf(m)));
            }
            for (uint32_t i = wave; i < n; i += kFinWaves) {
                if (!(lv[i] >= thr))
                    continue;
                const double l = group_logit<SRC>(st, qs, qi, lg[i], false, 0);
                if (lane < 16u && l >= (double)thr && l != -__builtin_inf()) {
                    const uint32_t at = atomicAdd(&n_cand, 1u);
                    if (at < kFinRows)
                        cand[at].l = l, cand[at].row = lg[i] * kGroupRows + lane;
                }
            }
            __syncthreads();
            whole = n_cand <= kFinRows;
        }
        if (whole) {
            const uint32_t n = n_cand;
            for (uint32_t i = tid; i < n; i += kFinThreads) {
                const double l = cand[i].l;
                const uint32_t r = cand[i].row;
                uint32_t before = 0;
                for (uint32_t j = 0; j < n; ++j)
                    before += cand_before(cand[j].l, cand[j].row, l, r) ? 1u : 0u;
                if (before < k)
                    best[before].l = l, best[before].row = r;
            }
            have = min(n, k);
            __syncthreads();
        } else {
            // More near ties than fit (a store that holds one vector very often): walk the groups in order, 64 at a time, and join
            // what can displace the k-th best so far.  Equal rows that come later cannot, so they cost their logits only.
            const uint32_t n_groups = st.n_pieces * kGroupsPerPiece;
            for (uint32_t g0 = 0; g0 < n_groups; g0 += 64u) {
                const float v = g0 + lane < n_groups ? groups[g0 + lane] : neg_inf();
                uint64_t todo = __ballot(v >= thr && v != neg_inf()); // the same in every wave
                if (!todo)
                    continue;
                __syncthreads();
                if (tid == 0)
                    n_cand = 0;
                __syncthreads();
                for (uint32_t i = 0; todo; ++i, todo &= todo - 1u) {
                    if (i % kFinWaves != wave)
                        continue;
                    const uint32_t group = g0 + (uint32_t)__ffsll((unsigned long long)todo) - 1u;
                    const double l = group_logit<SRC>(st, qs, qi, group, false, 0);
                    const uint32_t r = group * kGroupRows + lane;
                    if (lane < 16u && l != -__builtin_inf() && (have < k || cand_before(l, r, best[k - 1u].l, best[k - 1u].row))) {
                        const uint32_t at = atomicAdd(&n_cand, 1u); // at most 64 groups of 16 rows
                        cand[at].l = l, cand[at].row = r;
                    }
                }
                __syncthreads();
                const uint32_t fresh = n_cand;
                if (!fresh)
                    continue;
                for (uint32_t i = tid; i < have; i += kFinThreads)
                    cand[fresh + i] = best[i];
                __syncthreads();
                const uint32_t all = fresh + have;
                for (uint32_t i = tid; i < all; i += kFinThreads) {
                    const double l = cand[i].l;
                    const uint32_t r = cand[i].row;
                    uint32_t before = 0;
                    for (uint32_t j = 0; j < all; ++j)
                        before += cand_before(cand[j].l, cand[j].row, l, r) ? 1u : 0u;
                    if (before < k)
                        best[before].l = l, best[before].row = r;
                }
                have = min(all, k);
                __syncthreads();
            }
        }
    }

    // ---- lse, H ------------------------------------------------------------------------------------------------------------------
    // The sums again with the f64 logits of the best rows in place of the first pass' (a group's maximum is the first-pass logit of
    // the first of its rows in best[]): where one row has nearly all the probability, its log p is then as good as what is left
    // beside it, and never above 0.
    double lse = -__builtin_inf(), entropy = 0.0;
    if (poisoned) {
        lse = entropy = nan;
    } else if (have) {
        const double M = best[0].l, shift = base / L - M, by = exp(shift);
        double s_new = 0.0, u_new = 0.0;
        for (uint32_t j = 0; j < have; ++j) { // (every thread the same sums, in the same order)
            const uint32_t group = best[j].row / kGroupRows;
            bool first = true;
            for (uint32_t i = 0; i < j; ++i)
                first = first && best[i].row / kGroupRows != group;
            if (!first)
                continue;
            const double z = best[j].l - M, e = exp(z);
            s_new += e;
            u_new += e * z;
            // (the very terms that the sums have: where nothing else is there, nothing is left)
            const float g = groups[group], pm = pieces[group / kGroupsPerPiece].x;
            const float z1 = piece_is_huge(pm) ? (g - pm) * kLog2e : __builtin_fmaf(g, kLog2e, -piece_base(pm));
            const float e1 = __builtin_amdgcn_exp2f(z1);
            const double zp = piece_base64(pm) - base, ep = (double)exp2f((float)zp);
            S -= (double)e1 * ep;
            U -= ((double)(e1 * z1) + zp * (double)e1) * ep;
        }
        S = S > 0.0 ? S : 0.0;
        const double total = S * by + s_new, weighted = (U / L + shift * S) * by + u_new;
        lse = M + log(total);
        entropy = log(total) - weighted / total;
        entropy = entropy > 0.0 ? entropy : 0.0;
    }
    if (tid == 0) {
        if (f.lse)
            f.lse[qi] = (float)lse;
        if (f.entropy)
            f.entropy[qi] = (float)entropy;
    }

    // ---- given rows, one wave each --------------------------------------------------------------------------------------------
    if (f.log_probs) {
        for (uint32_t g = wave; g < f.n_given; g += kFinWaves) {
            const uint64_t at = f.given[(size_t)qi * f.n_given + g] - f.row_base; // (below row_base: wraps beyond n_rows)
            double l = -__builtin_inf();
            if (at < st.n_rows)
                l = group_logit<SRC>(st, qs, qi, 0, true, (uint32_t)at);
            if (lane == 0)
                f.log_probs[(size_t)qi * f.n_given + g] = poisoned ? (float)nan : (l == -__builtin_inf() ? neg_inf() : (float)(l - lse));
        }
    }
    for (uint32_t j = tid; j < f.k; j += kFinThreads) {
        vfsx_hit h;
        if (j < have) {
            const uint32_t r = best[j].row;
            h.dist = (float)(best[j].l - lse);
            h.flags = 1;
            h.row = f.row_base + r;
            h.id = f.ids ? f.ids[r] : f.id_base + r;
        } else {
            h.dist = poisoned ? (float)nan : neg_inf();
            h.flags = 0;
            h.row = ~0ull;
            h.id = ~0ull;
        }
        f.top[(size_t)qi * k + j] = h;
    }
}

} // namespace

hipError_t launch_prob_rows(const ProbStore &st, uint32_t row0, float *row_inv, float *row_scale, float *max_norm, hipStream_t s)
{
    if (st.n_rows <= row0)
        return hipSuccess;
    const uint32_t blocks = (st.n_rows - row0 + 255u) / 256u;
    if (st.source == kProbI8)
        prob_rows_kernel<kProbI8><<<blocks, 256, 0, s>>>(st.rows, st.d_chunks, row0, st.n_rows, row_inv, row_scale, max_norm);
    else
        prob_rows_kernel<kProbF32><<<blocks, 256, 0, s>>>(st.rows, st.d_chunks, row0, st.n_rows, row_inv, row_scale, max_norm);
    return hipGetLastError();
}

hipError_t launch_prob_queries(const ProbStore &st, const float *q, uint32_t nq, uint32_t nq_pad, float *fac, float *eps, double *norm,
                               uint4 *pairs, hipStream_t s)
{
    const uint32_t chunks = query_elems(st.dim) / 8u;
    prob_queries_kernel<<<pairs ? nq_pad : nq, 64, 0, s>>>(st, q, nq, chunks, fac, eps, norm, pairs);
    return hipGetLastError();
}

hipError_t launch_prob_finish(const ProbStore &st, const ProbQueries &q, const ProbFinish &f, hipStream_t s)
{
    if (st.source == kProbI8)
        prob_finish_kernel<kProbI8><<<q.nq, kFinThreads, 0, s>>>(st, q, f);
    else if (st.source == kProbF8)
        prob_finish_kernel<kProbF8><<<q.nq, kFinThreads, 0, s>>>(st, q, f);
    else
        prob_finish_kernel<kProbF32><<<q.nq, kFinThreads, 0, s>>>(st, q, f);
    return hipGetLastError();
}

} // namespace vfsx
