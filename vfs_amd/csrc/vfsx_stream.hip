// vfsx_stream.hip -- products of a batch of queries with every row of a store on the matrix cores, each row read from memory once
// per 32 NT queries, with an epilogue: softmax statistics (log probabilities) or the scores themselves.
//
// Operands
//   f32 rows   x 2^a = hi + lo in f16 (a per row, from its norm: |x| 2^a <= 2^10), q 2^b = hi + lo likewise, and
//              q.x = 2^-(a+b) (hi hi + hi lo + lo hi): three products of v_mfma_f32_32x32x16_f16 with f32 accumulators; what is left
//              out is 2^-22 of |q||x|.  Three 16-bit products at 16 times the rate of the f32 matrix instruction.
//   int8 rows  exact in f16: two products
//   f8         an e4m3 value times its power-of-two scale is exact in bf16: v_mfma_f32_32x32x16_bf16, one product
//   f8 raw     e4m3 on both sides, v_mfma_scale_f32_32x32x64_f8f6f4 with the blocks' scales as its scale operands: twice the rate.  That
//              instruction aligns eight products at a time to the largest of them and keeps about 14 bits (a product 2^14 times smaller
//              than its neighbour is lost; seen with products of powers of two), so its sums are good to 2^-13 of a group's largest
//              product (1.5e-5 of a result, by the norm): fine for scores that are rounded to bf16 (2^-9), not for f32 results.
//
// One wave owns a row-block (64 rows = two 32-row tiles of the A operand) and 32 NT queries.  Its rows go global -> VGPR (16 bytes per
// lane and load, 1 KiB contiguous per wave as rb64 has them), one K-step ahead; nobody else needs them, so they never pass
// through LDS.  The queries (B operand) are shared by the WAVES waves of a workgroup: a ring of three LDS slots filled by
// buffer_load ... lds two K-steps ahead, one barrier per K-step.
//
// Row order inside a 32-row tile: matrix row 8 a + 4 h + b holds store row 16 h + 4 a + b, so that the 16 accumulators of a lane (matrix
// rows 8 a + 4 h + b of its half h) are 16 consecutive rows of the store: a group's maximum and its share of the sums need no
// other lane, and a lane writes 16 consecutive scores.
#include <hip/hip_runtime.h>

#include "vfsx_internal.h"
#include "vfsx_prob.h"
#include "vfsx_prob_device.h"

#pragma clang fp contract(off)

namespace vfsx {

namespace {

enum { kF8Raw = 3 }; // beside ProbSource
// What one K-step is.  Rows: kLoads loads of 16 bytes per lane (two tiles, each lane half every other chunk).  Queries: kQChunks chunks of
// 16 bytes in kQParts parts (hi, lo), three slots of which leave room for two workgroups per CU.
template <int SRC, int NT>
struct Step {
    static constexpr uint32_t kElems = SRC == kProbF32 ? 32u : (SRC == kF8Raw ? 128u : (SRC == kProbI8 && NT == 4 ? 32u : 64u));
    static constexpr uint32_t kChunks = kElems / (SRC == kProbF32 ? 4u : 16u);
    static constexpr uint32_t kLoads = kChunks;
    static constexpr uint32_t kQChunks = SRC == kF8Raw ? 8u : kElems / 8u;
    static constexpr uint32_t kQParts = SRC == kProbF32 || SRC == kProbI8 ? 2u : 1u;
    static constexpr uint32_t kSlotBytes = kQChunks * kQParts * NT * 512u;
};

template <int SRC, int NT, int WAVES, int EPI>
__global__ __launch_bounds__(WAVES * 64, NT == 4 ? 2 : (NT == 2 ? 3 : 4)) void stream_kernel(ProbStore st, ProbQueries qs, StreamOut out, uint32_t n_rowtiles,
                                                                            uint32_t n_qtiles, uint32_t q_group)
{
    using S = Step<SRC, NT>;
    constexpr bool kIsF8 = SRC == kProbF8 || SRC == kF8Raw;
    constexpr uint32_t kSlots = 3, kSlotBytes = S::kSlotBytes, kPieces1k = kSlotBytes / 1024u;
    constexpr uint32_t kDma = (kPieces1k + WAVES - 1u) / WAVES; // per wave and slot (the last may be redundant)
    static_assert(NT == 1 || NT == 2 || NT == 4, "query tiles");
    __shared__ __align__(1024) uint8_t ring[kSlots][kSlotBytes];
    __shared__ __align__(16) float row_mul[WAVES][64], row_add[WAVES][64]; // epilogue: each wave its own rows

    const uint32_t lane = threadIdx.x & 63u, h = lane >> 5, r32 = lane & 31u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t perm = 16u * ((r32 >> 2) & 1u) + 4u * (r32 >> 3) + (r32 & 3u); // store row (in its tile of 32) of matrix row r32

    // Work items (row tile, query tile).  Workgroups with the same id % 8 share an XCD and its L2: they take whole groups of q_group query
    // tiles for one row tile next to one another, so the rows come from memory once per group.
    const uint32_t xcd = blockIdx.x & 7u, within = blockIdx.x >> 3;
    const uint32_t groups_q = (n_qtiles + q_group - 1u) / q_group;
    const uint32_t rt = (within / q_group / groups_q) * 8u + xcd;
    const uint32_t qt = (within / q_group % groups_q) * q_group + within % q_group;
    if (rt >= n_rowtiles || qt >= n_qtiles)
        return; // (the whole workgroup)

    const uint32_t n_rb = (st.n_rows + 63u) / 64u, rb = rt * WAVES + wave;
    const bool active = rb < n_rb;
    const uint32_t row_chunks = kIsF8 ? st.f8_chunks : st.d_chunks;
    const uint4 *a_base = (kIsF8 ? st.f8 : st.rows) + (size_t)(active ? rb : 0u) * row_chunks * 64u;
    // bounded by the row-block: chunks beyond a row's last read as zeros
    const __amdgpu_buffer_rsrc_t a_rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)a_base, 0, active ? row_chunks * 1024u : 0u, 0x00020000);
    const uint32_t n_step = (st.dim + S::kElems - 1u) / S::kElems;

    // queries: 64-query blocks of 1 KiB pieces, padded to kQueryPad elements
    const uint32_t q_block_bytes = (st.dim + kQueryPad - 1u) / kQueryPad * kQueryPad * (SRC == kF8Raw ? 64u : 128u * S::kQParts);
    const uint8_t *b_base = (const uint8_t *)qs.operand + (size_t)(NT == 4 ? qt * 2u : (NT == 2 ? qt : qt >> 1)) * q_block_bytes;
    const __amdgpu_buffer_rsrc_t b_rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)b_base, 0, 0xffffffffu, 0x00020000);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)&ring[0][0];

    // slot layout [tile nt][chunk][part][32 queries][16 B].  One DMA moves 1 KiB = two runs of 512 B: chunk * part pairs (2 j, 2 j + 1) of one
    // 32-query tile; lane >> 5 picks the pair's member.
    auto stage_queries = [&](uint32_t step, uint32_t slot) {
#pragma unroll
        for (uint32_t i = 0; i < kDma; ++i) {
            const uint32_t piece = min(wave * kDma + i, kPieces1k - 1u); // (redundant copies keep the count the same in every wave)
            constexpr uint32_t per_tile = S::kQChunks * S::kQParts / 2u;
            const uint32_t nt = piece / per_tile, pair = piece % per_tile;
            const uint32_t block = NT == 4 ? nt >> 1 : 0u, half = NT == 1 ? qt & 1u : nt & 1u;
            const uint32_t voff = h * 1024u + half * 512u + r32 * 16u;
            const uint32_t soff = block * q_block_bytes + (step * S::kQChunks * S::kQParts + 2u * pair) * 1024u;
            uint32_t dst = lds0 + slot * kSlotBytes + piece * 1024u;
            asm volatile("" : "+s"(dst)); // (the compiler must not tie this to later reads of `ring`: it would drain the ring)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(b_rsrc, (__attribute__((address_space(3))) void *)(uintptr_t)dst, 16, (int)voff, (int)soff, 0, 0);
        }
    };
    u32x4 a_next[S::kLoads];
    auto load_rows = [&](uint32_t step, u32x4 *a) {
#pragma unroll
        for (uint32_t i = 0; i < S::kLoads; ++i) {
            const uint32_t mt = i / (S::kLoads / 2u), j = i % (S::kLoads / 2u);
            // f32: chunks 4 s + 2 h, 4 s + 2 h + 1 of K-slice s (16 elements);  raw e4m3: the same of K-slice s (64 elements);
            // int8 and e4m3: chunk 2 j + h, two K-slices of 16 elements out of one 16-byte chunk per lane half
            const uint32_t c = SRC == kProbI8 || SRC == kProbF8 ? 2u * j + h : 4u * (j >> 1) + 2u * h + (j & 1u);
            const uint32_t off = (step * S::kChunks + c) * 1024u + (mt * 32u + perm) * 16u;
            a[i] = __builtin_amdgcn_raw_buffer_load_b128(a_rsrc, (int)off, 0, 0);
        }
    };

    f32x16 acc[2][NT];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                acc[mt][nt][i] = 0.0f;

    float a_scale[2] = {1.0f, 1.0f};
    if (SRC == kProbF32) {
#pragma unroll
        for (uint32_t mt = 0; mt < 2u; ++mt)
            a_scale[mt] = st.row_scale[(active ? rb : 0u) * 64u + mt * 32u + perm];
    }
    uint32_t a_exp[2] = {0, 0}, b_exp[NT] = {};
    const uint32_t *a_exp_at = nullptr, *b_exp_at = nullptr;
    if (kIsF8) {
        a_exp_at = st.f8_exp + (size_t)(active ? rb : 0u) * st.f8_words * 64u + perm;
        if (SRC == kF8Raw)
            b_exp_at = qs.q8_exp + (size_t)(NT == 4 ? qt * 2u : (NT == 2 ? qt : qt >> 1)) * st.f8_words * 64u + (NT == 1 ? (qt & 1u) * 32u : 0u) + r32;
    }

    stage_queries(0, 0);
    asm volatile("" ::: "memory");
    stage_queries(n_step > 1u ? 1u : 0u, 1);
    asm volatile("" ::: "memory");
    load_rows(0, a_next);
    asm volatile("" ::: "memory");

    uint32_t slot = 0;
    for (uint32_t step = 0; step < n_step; ++step) {
        u32x4 a[S::kLoads];
#pragma unroll
        for (uint32_t i = 0; i < S::kLoads; ++i)
            a[i] = a_next[i];
        // the queries of this step are here (all but the youngest: the next step's queries and this step's rows), for every wave;
        // and every wave is done reading the slot that is filled next
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kDma + S::kLoads) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const uint32_t fill = slot == 0u ? 2u : slot - 1u;
        stage_queries(min(step + 2u, n_step - 1u), fill);
        asm volatile("" ::: "memory");
        load_rows(min(step + 1u, n_step - 1u), a_next);
        asm volatile("" ::: "memory");
        constexpr uint32_t kStepsPerWord = 4u * kF8Block / S::kElems; // of a dword of scales
        if (kIsF8 && step % kStepsPerWord == 0u) {
            const uint32_t word = step / kStepsPerWord;
#pragma unroll
            for (uint32_t mt = 0; mt < 2u; ++mt)
                a_exp[mt] = a_exp_at[(size_t)word * 64u + mt * 32u];
            if (SRC == kF8Raw) {
#pragma unroll
                for (uint32_t nt = 0; nt < NT; ++nt)
                    b_exp[nt] = b_exp_at[((size_t)(nt >> 1) * st.f8_words + word) * 64u + (nt & 1u) * 32u];
            }
        }
        const uint8_t *q_slot = ring[slot];
        auto q_frag = [&](uint32_t nt, uint32_t chunk, uint32_t part) {
            return *(const u32x4 *)(q_slot + ((nt * S::kQChunks + chunk) * S::kQParts + part) * 512u + r32 * 16u);
        };
        if constexpr (SRC == kF8Raw) {
            const uint32_t sh = 8u * (step & 3u);
#pragma unroll
            for (uint32_t s = 0; s < 2u; ++s) {
                i32x8 fa[2];
#pragma unroll
                for (uint32_t mt = 0; mt < 2u; ++mt) {
                    const u32x4 p = a[mt * 4u + s * 2u], q = a[mt * 4u + s * 2u + 1u];
                    fa[mt] = i32x8{(int)p[0], (int)p[1], (int)p[2], (int)p[3], (int)q[0], (int)q[1], (int)q[2], (int)q[3]};
                }
#pragma unroll
                for (uint32_t nt = 0; nt < NT; ++nt) {
                    const u32x4 p = q_frag(nt, 4u * s + 2u * h, 0), q = q_frag(nt, 4u * s + 2u * h + 1u, 0);
                    const i32x8 fb = {(int)p[0], (int)p[1], (int)p[2], (int)p[3], (int)q[0], (int)q[1], (int)q[2], (int)q[3]};
#pragma unroll
                    for (uint32_t mt = 0; mt < 2u; ++mt)
                        acc[mt][nt] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[mt], fb, acc[mt][nt], 0, 0, 0,
                                                                                      (int)(a_exp[mt] >> sh), 0, (int)(b_exp[nt] >> sh));
                }
            }
        } else {
            constexpr uint32_t kSlices = S::kElems / 16u;
            float f8_scale[2] = {}; // this step's block
            if (SRC == kProbF8) {
#pragma unroll
                for (uint32_t mt = 0; mt < 2u; ++mt)
                    f8_scale[mt] = __uint_as_float(((a_exp[mt] >> (8u * (step / (kF8Block / S::kElems) & 3u))) & 255u) << 23);
            }
#pragma unroll
            for (uint32_t s = 0; s < kSlices; ++s) {
                u32x4 ah[2], al[2];
#pragma unroll
                for (uint32_t mt = 0; mt < 2u; ++mt) {
                    if constexpr (SRC == kProbF32) {
                        const u32x4 p = a[mt * 4u + s * 2u], q = a[mt * 4u + s * 2u + 1u];
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[i] = __uint_as_float(p[i]) * a_scale[mt];
                            x[i + 4] = __uint_as_float(q[i]) * a_scale[mt];
                        }
                        const HalfPair v = split8(x);
                        ah[mt] = __builtin_bit_cast(u32x4, v.hi);
                        al[mt] = __builtin_bit_cast(u32x4, v.lo);
                    } else {
                        const u32x4 p = a[mt * (S::kLoads / 2u) + (s >> 1)];
                        const uint32_t lo = p[(s & 1u) * 2u], hi = p[(s & 1u) * 2u + 1u];
                        if constexpr (SRC == kProbI8)
                            ah[mt] = __builtin_bit_cast(u32x4, halves8(lo, hi));
                        else
                            ah[mt] = bf16_of_e4m3(lo, hi, f8_scale[mt]);
                    }
                }
                // the 8 elements a lane half supplies: f32 16 s + 8 h ..;  int8, e4m3 16 (2 (s / 2) + h) + 8 (s % 2) ..
                const uint32_t qc = SRC == kProbF32 ? 2u * s + h : 4u * (s >> 1) + 2u * h + (s & 1u);
#pragma unroll
                for (uint32_t nt = 0; nt < NT; ++nt) {
                    const u32x4 bh = q_frag(nt, qc, 0);
                    u32x4 bl = bh;
                    if (S::kQParts == 2u)
                        bl = q_frag(nt, qc, 1);
#pragma unroll
                    for (uint32_t mt = 0; mt < 2u; ++mt) {
                        if (S::kQParts == 2u)
                            acc[mt][nt] = mfma16<SRC>(ah[mt], bl, acc[mt][nt]);
                        if (SRC == kProbF32)
                            acc[mt][nt] = mfma16<SRC>(al[mt], bh, acc[mt][nt]);
                        acc[mt][nt] = mfma16<SRC>(ah[mt], bh, acc[mt][nt]);
                    }
                }
            }
        }
        slot = slot == 2u ? 0u : slot + 1u;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // no copy into LDS may outlive the workgroup
    if (!active)
        return;

    // ---- epilogue: lane = query (column) r32 of tile nt; acc[mt][nt][i] = row 64 rb + 32 mt + 16 h + i ----------------------------------
    const uint32_t q0 = qt * (32u * NT) + r32;
    if constexpr (EPI == kPieces) {
        // Who is there: one row of the block per lane.  Blocks with rows that are not there, or with a bias so low that its logit leaves
        // the range of the exponent below, take the longer way (`masked`).
        const uint32_t my = rb * 64u + lane;
        bool gone = my >= st.n_rows, low = false;
        float my_mul = 1.0f, my_add = 0.0f;
        if (!gone) {
            my_add = st.bias ? st.bias[my] : 0.0f;
            my_mul = st.cosine ? st.row_inv[my] : 1.0f;
            gone = my_add == neg_inf() || (st.cosine && my_mul < 0.0f);
            low = fabsf(my_add) > 1e30f;
            if (SRC == kProbF32) // / 2^a
                my_mul *= __uint_as_float((254u << 23) - __float_as_uint(st.row_scale[my]));
        }
        row_mul[wave][lane] = my_mul;
        row_add[wave][lane] = my_add;
        const bool masked = __any(gone || low);
        const uint64_t gone_rows = __ballot(gone);
        const uint32_t gone_mine = (uint32_t)((gone_rows >> (16u * h)) & 0xffffu) | (uint32_t)((gone_rows >> (32u + 16u * h)) & 0xffffu) << 16;
#pragma unroll
        for (uint32_t nt = 0; nt < NT; ++nt) {
            const uint32_t qi = q0 + nt * 32u;
            const bool mine = qi < qs.nq;
            const float fac = mine ? qs.fac[qi] : 0.0f;
            float top[2][2] = {{neg_inf(), neg_inf()}, {neg_inf(), neg_inf()}}, s = 0.0f, t = 0.0f, m;
            auto logit = [&](uint32_t mt, uint32_t i) { // (the same address in all lanes of a half)
                const uint32_t at = mt * 32u + h * 16u + i;
                return __builtin_fmaf(acc[mt][nt][i], fac * row_mul[wave][at], row_add[wave][at]);
            };
            auto is_gone = [&](uint32_t mt, uint32_t i) { return (gone_mine >> (16u * mt + i)) & 1u; };
            if (!masked) {
#pragma unroll
                for (uint32_t mt = 0; mt < 2u; ++mt)
#pragma unroll
                    for (uint32_t i = 0; i < 16u; ++i) {
                        acc[mt][nt][i] = logit(mt, i);
                        top[mt][i >> 3] = fmaxf(top[mt][i >> 3], acc[mt][nt][i]);
                    }
                m = fmaxf(fmaxf(top[0][0], top[0][1]), fmaxf(top[1][0], top[1][1]));
                m = fmaxf(m, __shfl_xor(m, 32, 64));
                const float base = piece_base(m);
#pragma unroll
                for (uint32_t mt = 0; mt < 2u; ++mt)
#pragma unroll
                    for (uint32_t i = 0; i < 16u; ++i) {
                        const float z = __builtin_fmaf(acc[mt][nt][i], kLog2e, -base), e = __builtin_amdgcn_exp2f(z);
                        s += e;
                        t = __builtin_fmaf(e, z, t);
                    }
            } else {
#pragma unroll
                for (uint32_t mt = 0; mt < 2u; ++mt)
#pragma unroll
                    for (uint32_t i = 0; i < 16u; ++i) {
                        acc[mt][nt][i] = is_gone(mt, i) ? neg_inf() : logit(mt, i);
                        top[mt][i >> 3] = fmaxf(top[mt][i >> 3], acc[mt][nt][i]);
                    }
                m = fmaxf(fmaxf(top[0][0], top[0][1]), fmaxf(top[1][0], top[1][1]));
                m = fmaxf(m, __shfl_xor(m, 32, 64));
                const float base = piece_base(m);
                const bool huge = piece_is_huge(m);
#pragma unroll
                for (uint32_t mt = 0; mt < 2u; ++mt)
#pragma unroll
                    for (uint32_t i = 0; i < 16u; ++i) {
                        const float l = acc[mt][nt][i];
                        const float z = huge ? (l - m) * kLog2e : __builtin_fmaf(l, kLog2e, -base);
                        const float e = __builtin_amdgcn_exp2f(z);
                        // (a row there whose logit is infinite spoils the sums; a very low finite one adds nothing)
                        s += is_gone(mt, i) ? 0.0f : (fabsf(l) < __builtin_inff() ? e : __builtin_nanf(""));
                        t += is_gone(mt, i) || e == 0.0f ? 0.0f : e * z;
                    }
            }
            s += __shfl_xor(s, 32, 64);
            t += __shfl_xor(t, 32, 64);
            if (st.cosine && mine && qs.norm[qi] == 0.0) { // no cosine: no row is there
                m = top[0][0] = top[0][1] = top[1][0] = top[1][1] = neg_inf();
                s = t = 0.0f;
            }
            if (mine) {
                const size_t piece = (size_t)qi * st.n_pieces + rb;
                if (h == 0u)
                    out.pieces[piece] = make_float4(m, s, t, 0.0f);
                float2 *g = (float2 *)(out.groups + piece * kGroupsPerPiece); // groups 4 mt + 2 h, + 1
                g[h] = make_float2(top[0][0], top[0][1]);
                g[2u + h] = make_float2(top[1][0], top[1][1]);
            }
        }
    } else {
        using T = typename std::conditional<EPI == kScoresF32, float, __bf16>::type;
        {
            const uint32_t my = rb * 64u + lane;
            const float inv = st.cosine && my < st.n_rows ? st.row_inv[my] : 1.0f;
            row_mul[wave][lane] = inv < 0.0f ? __builtin_nanf("") : inv;
        }
        const uint32_t left = st.n_rows - rb * 64u; // rows of this block
#pragma unroll
        for (uint32_t nt = 0; nt < NT; ++nt) {
            const uint32_t qi = q0 + nt * 32u;
            if (qi >= qs.nq)
                continue;
            float fac = qs.fac[qi];
            if (st.cosine && qs.norm[qi] == 0.0)
                fac = __builtin_nanf("");
#pragma unroll
            for (uint32_t mt = 0; mt < 2u; ++mt) {
                const uint32_t first = mt * 32u + h * 16u;
                T *dst = (T *)out.scores + (size_t)qi * out.ld + rb * 64u + first;
                T v[16];
#pragma unroll
                for (uint32_t i = 0; i < 16u; ++i)
                    v[i] = (T)(acc[mt][nt][i] * fac * row_mul[wave][first + i]);
                if (out.aligned && first + 16u <= left) {
#pragma unroll
                    for (uint32_t i = 0; i < sizeof(T); ++i) {
                        u32x4 w;
                        __builtin_memcpy(&w, (const char *)v + 16u * i, 16);
                        __builtin_memcpy(__builtin_assume_aligned((char *)dst + 16u * i, 16), &w, 16);
                    }
                } else {
                    for (uint32_t i = 0; i < 16u; ++i)
                        if (first + i < left)
                            dst[i] = v[i];
                }
            }
        }
    }
}

template <int SRC, int NT, int EPI>
hipError_t run(const ProbStore &st, const ProbQueries &q, const StreamOut &out, hipStream_t s)
{
    constexpr uint32_t kWaves = 4;
    const uint32_t n_rb = (st.n_rows + 63u) / 64u, n_rowtiles = (n_rb + kWaves - 1u) / kWaves, n_qtiles = (q.nq + 32u * NT - 1u) / (32u * NT);
    const uint32_t q_group = n_qtiles < 8u ? n_qtiles : 8u;
    const uint64_t per_xcd = (uint64_t)((n_rowtiles + 7u) / 8u) * ((n_qtiles + q_group - 1u) / q_group) * q_group;
    if (per_xcd * 8u > 0x7fffffffull)
        return hipErrorInvalidValue;
    stream_kernel<SRC, NT, kWaves, EPI><<<(uint32_t)(per_xcd * 8u), kWaves * 64u, 0, s>>>(st, q, out, n_rowtiles, n_qtiles, q_group);
    return hipGetLastError();
}

template <int SRC, int EPI>
hipError_t run_for(const ProbStore &st, const ProbQueries &q, const StreamOut &out, hipStream_t s)
{
    if (q.nq <= 32u)
        return run<SRC, 1, EPI>(st, q, out, s);
    if (q.nq <= 64u)
        return run<SRC, 2, EPI>(st, q, out, s);
    return run<SRC, 4, EPI>(st, q, out, s);
}

} // namespace

hipError_t launch_prob_pieces(const ProbStore &st, const ProbQueries &q, float4 *pieces, float *groups, hipStream_t s)
{
    if (!st.n_pieces)
        return hipSuccess;
    const StreamOut out{pieces, groups, nullptr, 0, 0};
    if (st.source == kProbI8)
        return run_for<kProbI8, kPieces>(st, q, out, s);
    if (st.source == kProbF8)
        return run_for<kProbF8, kPieces>(st, q, out, s);
    return run_for<kProbF32, kPieces>(st, q, out, s);
}

hipError_t launch_f8_scores(const ProbStore &st, const ProbQueries &q, void *scores, uint64_t ld, int bf16, hipStream_t s)
{
    const uint32_t elem = bf16 ? 2u : 4u;
    const StreamOut out{nullptr, nullptr, scores, ld, ((uintptr_t)scores % 16u == 0 && ld * elem % 16u == 0) ? 1 : 0};
    return bf16 ? run_for<kF8Raw, kScoresBf16>(st, q, out, s) : run_for<kProbF8, kScoresF32>(st, q, out, s);
}

} // namespace vfsx
