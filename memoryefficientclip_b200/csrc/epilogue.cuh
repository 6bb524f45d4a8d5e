// The five epilogues of the tile kernels, shared by the single-CTA and the CTA-pair kernel.
// Eight warps (two per TMEM lane quadrant) work on one 128-row accumulator: warp quadrant
// q = warp % 4 owns rows 32q..32q+31, warp group wg = 0/1 owns the first / second half of the
// tile's columns.  One thread = one row (tcgen05.ld 32x32b), 32 columns per load.
#pragma once
#include "sm100_ptx.cuh"

namespace meclip {

// Value summed by the forward pass: exp2(u) for the softmax losses, softplus(a)/ln2 for the sigmoid
// loss (u = a log2(e); the loss kernel multiplies by ln2 once).
// flip: the sigmoid loss takes softplus(-a) on the diagonal (the positive pair).  It is summed in
// that form, not as softplus(a) - a, so that the many tiny off-diagonal terms of a row are never
// added to a large number.
template <bool SIG>
__device__ __forceinline__ float fwd_value(float s, float fmul, float fadd, bool flip = false) {
    float u = fmaf(s, fmul, fadd);
    if (!SIG) return ex2_approx(u);
    if (flip) u = -u;
    // log2(1 + x), x = 2^-|u| in (0, 1]: lg2.approx has an ABSOLUTE error near 1, which would dominate the
    // many tiny terms of far-apart pairs, so small x uses the series x log2(e) (1 - x/2) instead
    const float x = ex2_approx(-fabsf(u));
    const float small = x * fmaf(x, -0.72134752f, 1.44269504f);
    const float big = lg2_approx(1.f + x);
    return fmaxf(u, 0.f) + (x < 0.00390625f ? small : big);
}
// Factor of the gradient coefficient: exp2(u), or sigmoid(a) = 1 / (1 + 2^-u) with u = a log2(e)
// (relative accuracy also for the very small sigmoids of far-apart pairs).
template <bool SIG>
__device__ __forceinline__ float coef_value(float s, float fmul, float fadd) {
    const float u = fmaf(s, fmul, fadd);
    if (!SIG) return ex2_approx(u);
    return rcp_approx(1.f + ex2_approx(-u));
}

template <bool SIG>
__device__ __forceinline__ void sums_chunk(const uint32_t (&v)[32], const GemmParams& p, float fmul, float fadd,
                                           bool full_tile, bool rvalid, int col_base, bool want_cols,
                                           float (&cacc)[32], float& ra0, float& ra1, float& ra2, float& ra3, int jdc) {
    if (SIG && jdc >= -1 && __any_sync(0xffffffffu, jdc >= 0)) {      // a chunk the diagonal runs through
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            float e = fwd_value<SIG>(__uint_as_float(v[c]), fmul, fadd, c == jdc);
            if (!rvalid || col_base + c >= p.n) e = 0.f;
            ra0 += e;
        }
        return;
    }
    if (full_tile) {
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
            const float e0 = fwd_value<SIG>(__uint_as_float(v[c]), fmul, fadd);
            const float e1 = fwd_value<SIG>(__uint_as_float(v[c + 1]), fmul, fadd);
            const float e2 = fwd_value<SIG>(__uint_as_float(v[c + 2]), fmul, fadd);
            const float e3 = fwd_value<SIG>(__uint_as_float(v[c + 3]), fmul, fadd);
            ra0 += e0; ra1 += e1; ra2 += e2; ra3 += e3;
            if (want_cols) { cacc[c] += e0; cacc[c + 1] += e1; cacc[c + 2] += e2; cacc[c + 3] += e3; }
        }
    } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            float e = fwd_value<SIG>(__uint_as_float(v[c]), fmul, fadd);
            if (!rvalid || col_base + c >= p.n) e = 0.f;
            ra0 += e;
            if (want_cols) cacc[c] += e;
        }
    }
}

template <bool SIG>
__device__ __forceinline__ void coef_chunk(const uint32_t (&v)[32], float fmul, float fadd, float inv_r,
                                           const float* icol_chunk, float (&gv)[32]) {
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
        const float4 ic = *reinterpret_cast<const float4*>(icol_chunk + c);   // broadcast read
        gv[c] = coef_value<SIG>(__uint_as_float(v[c]), fmul, fadd) * (inv_r + ic.x);
        gv[c + 1] = coef_value<SIG>(__uint_as_float(v[c + 1]), fmul, fadd) * (inv_r + ic.y);
        gv[c + 2] = coef_value<SIG>(__uint_as_float(v[c + 2]), fmul, fadd) * (inv_r + ic.z);
        gv[c + 3] = coef_value<SIG>(__uint_as_float(v[c + 3]), fmul, fadd) * (inv_r + ic.w);
    }
}

// One 32-column chunk of the vocabulary statistics of a row, relative to the chunk's own maximum: u_c = S_c fmul - cm <= 0
// (up to the rounding of cm), r = sum 2^u - 1, t = sum 2^u u; nv of the 32 columns exist.  The maximum's own 1 is left out
// of the sum: where one column holds nearly all the probability its log probability is -log(1 + r), and r would drown in
// the rounding of 1 + r.  With CAND also the column of the best and a lower bound of the second best's distance: the two
// smallest of the integers |u| bits (low five cleared) | column.  Non-negative floats order like their bits and the low
// bits break ties towards the lower column, so that is one logic operation and three integer minima / maxima per element.
template <bool CAND>
__device__ __forceinline__ void stats_chunk(const uint32_t (&v)[32], float fmul, int nv, float& cm, float& r, float& t,
                                            uint32_t& second) {
    float lsum, tsum;
    int tops = 0;                                   // columns that share the maximum
    uint32_t n1 = 0x7fffffffu, n2 = 0x7fffffffu;
    if (nv >= 32) {
        float m0 = __uint_as_float(v[0]), m1 = __uint_as_float(v[1]);
#pragma unroll
        for (int c = 2; c < 30; c += 4) {
            m0 = max3(m0, __uint_as_float(v[c]), __uint_as_float(v[c + 1]));
            m1 = max3(m1, __uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
        }
        const float sm = fmaxf(m0, max3(m1, __uint_as_float(v[30]), __uint_as_float(v[31])));
        cm = sm * fmul;
        // two columns per instruction where there is one for it; `all` keeps the maxima in, to count them
        const uint64_t mul2 = f32x2(fmul, fmul), sub2 = f32x2(-cm, -cm);
        uint64_t l = 0, all = 0, t2 = 0;
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
            const float sa = __uint_as_float(v[c]), sb = __uint_as_float(v[c + 1]);
            const uint64_t u = fma_f32x2(f32x2(sa, sb), mul2, sub2);
            float ua, ub;
            f32x2_split(u, ua, ub);
            const float ea = ex2_approx(ua), eb = ex2_approx(ub);
            all = add_f32x2(all, f32x2(ea, eb));
            const uint64_t e = f32x2(sa == sm ? 0.f : ea, sb == sm ? 0.f : eb);
            l = add_f32x2(l, e);
            t2 = fma_f32x2(e, u, t2);
            if (CAND) {
                const uint32_t ka = (__float_as_uint(ua) & 0x7fffffe0u) | (uint32_t)c;
                const uint32_t kb = (__float_as_uint(ub) & 0x7fffffe0u) | (uint32_t)(c + 1);
                n2 = min(n2, max(n1, ka)); n1 = min(n1, ka);
                n2 = min(n2, max(n1, kb)); n1 = min(n1, kb);
            }
        }
        float x0, x1, y0, y1, z0, z1;
        f32x2_split(l, x0, x1);
        f32x2_split(t2, y0, y1);
        f32x2_split(all, z0, z1);
        lsum = x0 + x1;
        tsum = y0 + y1;
        tops = __float2int_rn((z0 + z1) - lsum);    // each is 1 up to the rounding of cm
    } else {
        float sm = __uint_as_float(v[0]);           // nv >= 1: column 0 exists
#pragma unroll
        for (int c = 1; c < 32; ++c)
            if (c < nv) sm = fmaxf(sm, __uint_as_float(v[c]));
        cm = sm * fmul;
        lsum = tsum = 0.f;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            if (c < nv) {
                const float s = __uint_as_float(v[c]);
                const float u = fmaf(s, fmul, -cm);
                float e = ex2_approx(u);
                if (s == sm) { e = 0.f; ++tops; }
                lsum += e;
                tsum = fmaf(e, u, tsum);
                if (CAND) {
                    const uint32_t k = (__float_as_uint(u) & 0x7fffffe0u) | (uint32_t)c;
                    n2 = min(n2, max(n1, k)); n1 = min(n1, k);
                }
            }
        }
    }
    r = lsum + (float)(tops - 1);
    t = tsum;
    second = (n2 & ~31u) | (n1 & 31u);
}

// Joins {maximum m2, sum less one r2, moment t2} to {m, r, t}: the sums are rescaled to the larger maximum and the exponents
// inside the moment shift with it.  An empty side has a finite m of -1e30, r = -1 and t = 0, so no infinities meet.
// `unit`: what the maxima are in, where they are not in base-2 units themselves.
__device__ __forceinline__ void stats_join(float& m, float& r, float& t, float m2, float r2, float t2, float unit = 1.f) {
    const float mn = fmaxf(m, m2);
    const float a = (m - mn) * unit, b = (m2 - mn) * unit;
    const float fa = ex2_approx(a), fb = ex2_approx(b);
    const float l = 1.f + r, l2 = 1.f + r2;
    t = fa * fmaf(a, l, t) + fb * fmaf(b, l2, t2);
    r = m >= m2 ? fmaf(fb, l2, r) : fmaf(fa, l, r2);
    m = mn;
}
static constexpr float STATS_EMPTY = -1e30f;

// Coefficients of a chunk over a vocabulary: 2^u (a + b u), u = log2 of the row's softmax.  Two columns per instruction: the
// pass over 2047 x 32001 x 512 takes 77 us instead of 90.
__device__ __forceinline__ void vocab_chunk(const uint32_t (&v)[32], float fmul, float lse, float a, float b,
                                            float (&gv)[32]) {
    const uint64_t mul2 = f32x2(fmul, fmul), sub2 = f32x2(-lse, -lse), a2 = f32x2(a, a), b2 = f32x2(b, b);
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
        const uint64_t u = fma_f32x2(f32x2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), mul2, sub2);
        float ua, ub;
        f32x2_split(u, ua, ub);
        f32x2_split(mul_f32x2(f32x2(ex2_approx(ua), ex2_approx(ub)), fma_f32x2(b2, u, a2)), gv[c], gv[c + 1]);
    }
}

static constexpr int COL_SLOTS = MECLIP_STRIPS ? MAX_BN / 64 : 1;   // 32-column chunks one warp group owns at most (half the tile)

struct EpiState {        // per-thread state that lives across tiles
    int stores_in_flight = 0;   // COEF: lane 0's outstanding TMA-store groups
    float gscale = 1.f;         // COEF: *grad_out (times a power of the device-resident temperature, if any)
    float fmul = 0.f, fadd = 0.f;   // the elementwise function's affine part, from the host or from device scalars
    // SUMS: column sums of this thread's row, kept in registers over a strip of tiles that share
    // their columns; reduced across rows (shuffles, shared memory, atomics) once per strip
    float cacc[COL_SLOTS][32] = {};
    int strip_n0 = -1;          // first column of the tiles accumulated so far, -1 = nothing pending
    int strip_m0 = 0;           // first row of the last tile accumulated (the slot of a deterministic flush)
};

// Per-thread set-up of the epilogue state: the affine part of the elementwise function and the
// coefficient scale, from the host values or from scalars that live on the device.
template <int EPI>
__device__ __forceinline__ void epilogue_init(const GemmParams& p, EpiState& st) {
    st.fmul = p.fmul;
    st.fadd = p.fadd;
    float gfac = 1.f;
    if (p.t_dev != nullptr) {
        const float t = __ldg(p.t_dev);
        if (p.sigmoid) {
            st.fmul = t * 1.4426950408889634f;
            if (p.b_dev != nullptr) st.fadd = __ldg(p.b_dev) * 1.4426950408889634f;
        } else {
            st.fmul = 1.4426950408889634f / t;
            st.fadd = -st.fmul;
        }
        gfac = p.g_rule == 1 ? 1.f / t : p.g_rule == 2 ? rsqrtf(t) : p.g_rule == 3 ? t : 1.f;
    }
    if (EPI == EPI_COEF) st.gscale = (p.grad_out ? __ldg(p.grad_out) : 1.f) * gfac;
}

// SUMS: add the pending column accumulators of all eight warps into col_sum and clear them.
// Every epilogue thread must call this at the same point (it uses the epilogue named barrier).
__device__ __forceinline__ void flush_column_sums(const GemmParams& p, SharedTail* tail, EpiState& st, int warp, int lane) {
    if (!MECLIP_STRIPS || st.strip_n0 < 0) return;
    const int q = warp & 3;
    const int wg = (warp - 2) >> 2;
    const int et = (int)threadIdx.x - 64;
    const int units = p.bn >> 5;
    const int u_split = (units + 1) >> 1;
    const int u_begin = wg == 0 ? 0 : u_split;
    const int u_end = wg == 0 ? u_split : units;
    float (*colpart)[MAX_BN] = reinterpret_cast<float (*)[MAX_BN]>(tail->scratch + sizeof(tail->scratch) - 4 * MAX_BN * 4);
#pragma unroll
    for (int k = 0; k < COL_SLOTS; ++k) {
        if (u_begin + k < u_end) {
            const float cs = warp_transpose_reduce32(st.cacc[k], lane);
            colpart[q][(u_begin + k) * 32 + lane] = cs;
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) st.cacc[k][c] = 0.f;
    }
    named_bar_sync(1, EPI_THREADS);
    for (int j = et; j < p.bn; j += EPI_THREADS)
        if (st.strip_n0 + j < p.n) {
            const float v = (colpart[0][j] + colpart[1][j]) + (colpart[2][j] + colpart[3][j]);
            if (p.col_part != nullptr) p.col_part[(long long)(st.strip_m0 >> 7) * p.part_ld_cols + st.strip_n0 + j] = v;
            else atomicAdd(p.col_sum + st.strip_n0 + j, v);
        }
    named_bar_sync(1, EPI_THREADS);
    st.strip_n0 = -1;
}

// `release()` is called by every thread once its last tcgen05.ld of the tile has completed; it must
// tell the MMA issuer that this thread is done with the accumulator.
template <int EPI, class Release>
__device__ __forceinline__ void epilogue_tile(const GemmParams& p, const OutDesc od, const CUtensorMap* tmap_c,
                                              SharedTail* tail, EpiState& st, uint32_t taddr, int m0, int n0,
                                              int tile_bn, int warp, int lane, Release release) {
    const int q = warp & 3;
    const int wg = EPI_WARPS == 8 ? (warp - 2) >> 2 : 0;
    const int et = (int)threadIdx.x - 64;                 // index within the epilogue group
    const int grow = m0 + q * 32 + lane;
    const bool rvalid = grow < od.m;          // od.m == p.m except for the second problem of a dual launch
    const bool full_tile = (m0 + BM <= od.m) && (n0 + p.bn <= p.n);
    // column (tile-local) on which this row meets the diagonal, -1 if outside the tile
    const long long jd_ll = (long long)grow + p.diag_shift - n0;
    const int jd = (jd_ll >= 0 && jd_ll < p.bn && n0 + jd_ll < p.n && rvalid) ? (int)jd_ll : -1;
    // this warp group's share of the columns, in units of 32 (SUMS, OUT) or 64 (COEF) columns
    // tile_bn differs from p.bn only for the narrower last column tile of a contraction (EPI_OUT)
    const int units = epi_is_coef(EPI) ? (p.bn >> 6) : (EPI == EPI_OUT ? (tile_bn >> 5) : (p.bn >> 5));
    const int u_split = EPI_WARPS == 8 ? (units + 1) >> 1 : units;
    const int u_begin = wg == 0 ? 0 : u_split;
    const int u_end = wg == 0 ? u_split : units;

    if (EPI == EPI_SUMS && !MECLIP_STRIPS) {
        // per-tile reduction of the column sums: butterfly per 32x32 block, combine the quadrants in shared memory
        float (*colpart)[MAX_BN] = reinterpret_cast<float (*)[MAX_BN]>(tail->scratch + sizeof(tail->scratch) - 4 * MAX_BN * 4);
        const bool want_cols = p.col_sum != nullptr;
        float ra0 = 0.f, ra1 = 0.f, ra2 = 0.f, ra3 = 0.f;
        float sdiag = 0.f;
        const bool diag_here = __any_sync(0xffffffffu, jd >= 0);
        for (int ch = u_begin; ch < u_end; ++ch) {
            uint32_t v[32];
            tmem_ld32(taddr + ch * 32, v);
            tmem_ld_wait();
            if (diag_here) {
                const int jdc = (jd >= 0 && (jd >> 5) == ch) ? (jd & 31) : -1;
#pragma unroll
                for (int c = 0; c < 32; ++c) sdiag = (c == jdc) ? __uint_as_float(v[c]) : sdiag;
            }
            float e[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) e[c] = 0.f;
            const int jdc_s = (diag_here && jd >= 0 && (jd >> 5) == ch) ? (jd & 31) : -1;
            if (p.sigmoid) sums_chunk<true>(v, p, st.fmul, st.fadd, full_tile, rvalid, n0 + ch * 32, want_cols, e, ra0, ra1, ra2, ra3, jdc_s);
            else           sums_chunk<false>(v, p, st.fmul, st.fadd, full_tile, rvalid, n0 + ch * 32, want_cols, e, ra0, ra1, ra2, ra3, -1);
            if (want_cols) {
                const float cs = warp_transpose_reduce32(e, lane);
                colpart[q][ch * 32 + lane] = cs;
            }
        }
        tc_fence_before();
        release();
        if (rvalid && u_end > u_begin) atomicAdd(p.row_sum + grow, (ra0 + ra1) + (ra2 + ra3));
        if (jd >= 0 && (jd >> 5) >= u_begin && (jd >> 5) < u_end) p.diag[grow] = sdiag;
        if (want_cols) {
            named_bar_sync(1, EPI_THREADS);
            for (int j = et; j < p.bn; j += EPI_THREADS)
                if (n0 + j < p.n)
                    atomicAdd(p.col_sum + n0 + j, (colpart[0][j] + colpart[1][j]) + (colpart[2][j] + colpart[3][j]));
            named_bar_sync(1, EPI_THREADS);
        }
    } else if (EPI == EPI_SUMS) {
        const bool want_cols = p.col_sum != nullptr;
        if (want_cols && st.strip_n0 != n0) {       // the columns change: hand in what was accumulated
            flush_column_sums(p, tail, st, warp, lane);
            st.strip_n0 = n0;
        }
        st.strip_m0 = m0;
        float ra0 = 0.f, ra1 = 0.f, ra2 = 0.f, ra3 = 0.f;
        float sdiag = 0.f;
        const bool diag_here = __any_sync(0xffffffffu, jd >= 0);   // warp-uniform: most tiles miss the diagonal
#pragma unroll
        for (int k = 0; k < COL_SLOTS; ++k) {
            const int ch = u_begin + k;
            if (ch < u_end) {
                uint32_t v[32];
                tmem_ld32(taddr + ch * 32, v);
                tmem_ld_wait();
                if (diag_here) {
                    const int jdc = (jd >= 0 && (jd >> 5) == ch) ? (jd & 31) : -1;
#pragma unroll
                    for (int c = 0; c < 32; ++c) sdiag = (c == jdc) ? __uint_as_float(v[c]) : sdiag;
                }
                const int jdc_s = (diag_here && jd >= 0 && (jd >> 5) == ch) ? (jd & 31) : -1;
                if (p.sigmoid) sums_chunk<true>(v, p, st.fmul, st.fadd, full_tile, rvalid, n0 + ch * 32, want_cols, st.cacc[k], ra0, ra1, ra2, ra3, jdc_s);
                else           sums_chunk<false>(v, p, st.fmul, st.fadd, full_tile, rvalid, n0 + ch * 32, want_cols, st.cacc[k], ra0, ra1, ra2, ra3, -1);
            }
        }
        tc_fence_before();
        release();
        if (rvalid && u_end > u_begin) {
            const float rs = (ra0 + ra1) + (ra2 + ra3);
            if (p.row_part != nullptr) p.row_part[(long long)(2 * (n0 / p.bn) + wg) * p.part_ld_rows + grow] = rs;
            else atomicAdd(p.row_sum + grow, rs);
        }
        if (jd >= 0 && (jd >> 5) >= u_begin && (jd >> 5) < u_end) p.diag[grow] = sdiag;
        // deterministic mode: one slot per tile, so the column partials are handed in after every tile
        if (want_cols && p.col_part != nullptr) flush_column_sums(p, tail, st, warp, lane);
    } else if (epi_is_coef(EPI)) {
        // g / c_j for the tile's columns, staged once per tile for all eight warps
        constexpr bool VOCAB = EPI == EPI_VCOEF;   // softmax over a vocabulary: row factors only, no diagonal
        if (!VOCAB) {
            named_bar_sync(1, EPI_THREADS);        // previous tile's readers of icol are done
            for (int j = et; j < p.bn; j += EPI_THREADS) {
                float v = 0.f;
                if (p.c != nullptr && n0 + j < p.n) v = p.coef * st.gscale / __ldg(p.c + n0 + j);
                tail->icol[j] = v;
            }
        }
        // row factor: g / r_i for the softmax losses, plain g when there are no row sums (sigmoid loss)
        const float inv_r = (VOCAB || !rvalid) ? 0.f : (p.r != nullptr ? p.coef * st.gscale / __ldg(p.r + grow) : p.coef * st.gscale);
        float v_lse = 1e30f, v_a = 0.f, v_b = 0.f;          // a row past the edge: 2^-huge = 0
        int v_col[VOCAB_TILE_ENTRIES];                      // tile columns of the row's entries, -1: none here
        float v_val[VOCAB_TILE_ENTRIES];
#pragma unroll
        for (int e = 0; e < VOCAB_TILE_ENTRIES; ++e) { v_col[e] = -1; v_val[e] = 0.f; }
        bool v_here = false;
        if (VOCAB) {
            if (rvalid) {
                const float4 f = __ldg(p.row_factors + grow);
                const float g_scale = pow2(row_exponent(f.w));
                v_lse = f.x;
                v_a = f.y * g_scale;
                v_b = f.z * g_scale;
                if (p.row_entries != nullptr) {
                    const float4 en = __ldg(p.row_entries + grow);
                    const float cols[2] = {en.x, en.z}, vals[2] = {en.y, en.w};
#pragma unroll
                    for (int e = 0; e < VOCAB_TILE_ENTRIES; ++e) {
                        const long long col = (long long)__float_as_int(cols[e]) - p.panel_col0 - n0;
                        if (__float_as_int(cols[e]) >= 0 && col >= 0 && col < p.bn && n0 + col < p.n) {
                            v_col[e] = (int)col;
                            v_val[e] = vals[e] * g_scale;
                        }
                    }
                }
            }
            bool any = false;
#pragma unroll
            for (int e = 0; e < VOCAB_TILE_ENTRIES; ++e) any |= v_col[e] >= 0;
            v_here = __any_sync(0xffffffffu, any);
        } else {
            named_bar_sync(1, EPI_THREADS);
        }
        // Each warp turns 32 rows x 64 columns into a 128-byte-swizzled shared tile and one lane
        // TMA-stores it (full 128-byte lines; rows and chunks outside the panel are clipped by the
        // tensor map).
        const float dsub = p.dcoef * st.gscale;
        const bool diag_here = !VOCAB && __any_sync(0xffffffffu, jd >= 0);
        const bool want_sg = !VOCAB && p.sg_acc != nullptr;      // sum of G_ij * S_ij for the temperature gradient
        float sg = 0.f, sg1 = 0.f;
        uint8_t* buf = tail->scratch + (size_t)(warp - 2) * STORE_BUF_BYTES;
        for (int u = u_begin; u < u_end; ++u) {
            if (lane == 0 && st.stores_in_flight > 0) {     // the previous store has finished reading `buf`
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                st.stores_in_flight = 0;
            }
            __syncwarp();
            uint32_t lo[VOCAB ? 32 : 1];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int ch = u * 2 + half;
                uint32_t v[32];
                tmem_ld32(taddr + ch * 32, v);
                tmem_ld_wait();
                float gv[32];
                if (VOCAB) vocab_chunk(v, st.fmul, v_lse, v_a, v_b, gv);
                else if (p.sigmoid) coef_chunk<true>(v, st.fmul, st.fadd, inv_r, &tail->icol[ch * 32], gv);
                else           coef_chunk<false>(v, st.fmul, st.fadd, inv_r, &tail->icol[ch * 32], gv);
                if (diag_here) {      // warp-uniform: only tiles that cross the diagonal pay for the correction
                    const int jdc = (jd >= 0 && (jd >> 5) == ch) ? (jd & 31) : -1;
                    if (p.sigmoid) {
                        // sigmoid(a) - 1 = -1 / (1 + 2^u), computed in that form: no cancellation for a confident pair
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            const float u = fmaf(__uint_as_float(v[c]), st.fmul, st.fadd);
                            gv[c] = (c == jdc) ? -dsub * rcp_approx(1.f + ex2_approx(u)) : gv[c];
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; ++c) gv[c] -= (c == jdc) ? dsub : 0.f;
                    }
                }
                if (VOCAB && v_here) {
#pragma unroll
                    for (int e = 0; e < VOCAB_TILE_ENTRIES; ++e) {
                        const int jc = (v_col[e] >> 5) == ch ? (v_col[e] & 31) : -1;
#pragma unroll
                        for (int c = 0; c < 32; ++c) gv[c] = (c == jc) ? v_val[e] : gv[c];
                    }
                }
                if (!full_tile) {     // columns past the panel edge share a stored chunk with valid ones: zero them
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (n0 + ch * 32 + c >= p.n) gv[c] = 0.f;
                }
                if (want_sg && rvalid) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) { sg = fmaf(gv[c], __uint_as_float(v[c]), sg); sg1 += gv[c]; }
                }
#pragma unroll
                for (int pc = 0; pc < 4; ++pc) {         // 16-byte piece index within the 128-byte row
                    uint4 pk;
                    if (VOCAB && p.panel_f16) {
                        pk.x = pack_f16x2(gv[pc * 8 + 0], gv[pc * 8 + 1]);
                        pk.y = pack_f16x2(gv[pc * 8 + 2], gv[pc * 8 + 3]);
                        pk.z = pack_f16x2(gv[pc * 8 + 4], gv[pc * 8 + 5]);
                        pk.w = pack_f16x2(gv[pc * 8 + 6], gv[pc * 8 + 7]);
                    } else {
                        pk.x = pack_bf16x2(gv[pc * 8 + 0], gv[pc * 8 + 1]);
                        pk.y = pack_bf16x2(gv[pc * 8 + 2], gv[pc * 8 + 3]);
                        pk.z = pack_bf16x2(gv[pc * 8 + 4], gv[pc * 8 + 5]);
                        pk.w = pack_bf16x2(gv[pc * 8 + 6], gv[pc * 8 + 7]);
                    }
                    const int piece = half * 4 + pc;
                    *reinterpret_cast<uint4*>(buf + lane * 128 + ((piece ^ (lane & 7)) << 4)) = pk;
                    if (VOCAB && p.lo_chunk > 0) {       // what the rounding left, for the second panel
                        const uint32_t hi[4] = {pk.x, pk.y, pk.z, pk.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float a = gv[pc * 8 + 2 * i] - __uint_as_float(hi[i] << 16);
                            const float b = gv[pc * 8 + 2 * i + 1] - __uint_as_float(hi[i] & 0xffff0000u);
                            lo[half * 16 + pc * 4 + i] = pack_bf16x2(a, b);
                        }
                    }
                }
            }
            fence_proxy_async();
            __syncwarp();
            // with a second panel behind the first, chunks past the last column must not be stored into it
            const bool store = !VOCAB || p.lo_chunk == 0 || (n0 >> 6) + u < (p.n + 63) >> 6;
            if (lane == 0 && store) {
                tma_store_3d(tmap_c, smem_u32(buf), 0, m0 + q * 32, (n0 >> 6) + u);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                st.stores_in_flight = 1;
            }
            if (VOCAB && p.lo_chunk > 0 && store) {
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
#pragma unroll
                for (int piece = 0; piece < 8; ++piece)
                    *reinterpret_cast<uint4*>(buf + lane * 128 + ((piece ^ (lane & 7)) << 4)) =
                        make_uint4(lo[piece * 4], lo[piece * 4 + 1], lo[piece * 4 + 2], lo[piece * 4 + 3]);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    tma_store_3d(tmap_c, smem_u32(buf), 0, m0 + q * 32, (n0 >> 6) + u + p.lo_chunk);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
        }
        tc_fence_before();
        release();
        if (want_sg) {
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) {
                sg += __shfl_xor_sync(0xffffffffu, sg, o);
                sg1 += __shfl_xor_sync(0xffffffffu, sg1, o);
            }
            if (lane == 0) { atomicAdd(p.sg_acc, sg); atomicAdd(p.sg_acc + 1, sg1); }
        }
    } else if (EPI == EPI_STATS) {
        // A row's part of the tile stays in registers: nothing but 16 bytes per row and half tile leaves the SM, and 8 per 32
        // columns with candidates.  4096 x 32768 x 1024: 202 us, 1360 TFLOP/s or 83 % of a measured library product (213 us with
        // candidates); the tensor pipe is active 63 % of that time, between K loops of 16 steps it waits for the next operands.
        float m = STATS_EMPTY, r = -1.f, t = 0.f;
        const bool cand = p.chunk_max != nullptr;
        for (int ch = u_begin; ch < u_end; ++ch) {
            uint32_t v[32];
            tmem_ld32(taddr + ch * 32, v);
            tmem_ld_wait();
            const int col0 = n0 + ch * 32;
            const int nv = p.n - col0;
            if (nv > 0) {                      // the same for the whole warp
                float cm, cr, ct;
                uint32_t second;
                if (cand) stats_chunk<true>(v, st.fmul, nv, cm, cr, ct, second);
                else      stats_chunk<false>(v, st.fmul, nv, cm, cr, ct, second);
                stats_join(m, r, t, cm, cr, ct);
                if (cand && rvalid) {
                    const long long at = (long long)grow * p.chunk_ld + (col0 >> 5);
                    p.chunk_max[at] = cm;
                    p.chunk_second[at] = second;
                }
            }
        }
        tc_fence_before();
        release();
        if (rvalid) p.stats[(long long)grow * p.stats_ld + 2 * (n0 / p.bn) + wg] = make_float4(m, r, t, 0.f);
    } else {   // EPI_OUT
        // Wide tiles (two MMAs per K step, see GemmParams::wide): the first MMA's 256 accumulator columns hold the
        // first 128 B rows of CTA 0 and of CTA 1, the second MMA's columns (from TMEM column 256) the remaining rows
        // of each, so accumulator chunk ch maps to tile columns through the four pieces below.  For tiles of up
        // to 256 columns the map is the identity.
        const bool scaled = od.scale.rows != nullptr || od.scale.total != nullptr;
        float unscale_g = 1.f, unscale_b = 1.f;
        if (od.scale.rows != nullptr) {
            if (rvalid) unscale_g = pow2(-row_exponent(__ldg(&od.scale.rows[grow].w)));
            unscale_b = pow2(-pow2_exponent(od.scale.operand, OPERAND_TARGET));
        } else if (od.scale.total != nullptr) {      // two factors: one could leave fp32's range (below 2^-252 all is zero)
            const int e = -total_exponent(od.scale.total);
            unscale_g = pow2(::max(e >> 1, -126));
            unscale_b = pow2(::max(e - (e >> 1), -126));
        }
        if (p.tile_out) {
            // 32 rows x 128 bytes per warp and store: 64 bf16 or 32 fp32 columns (two or one accumulator chunks).  The map's
            // third dimension is the part of K; rows and columns outside the output are clipped.
            const int per_unit = od.out_bf16 ? 2 : 1;
            const int chunks = tile_bn >> 5, tu = (chunks + per_unit - 1) / per_unit, tu_split = (tu + 1) >> 1;
            uint8_t* buf = tail->scratch + (size_t)(warp - 2) * STORE_BUF_BYTES;
            for (int u = wg == 0 ? 0 : tu_split; u < (wg == 0 ? tu_split : tu); ++u) {
                if (lane == 0 && st.stores_in_flight > 0) {
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    st.stores_in_flight = 0;
                }
                __syncwarp();
                for (int h = 0; h < per_unit; ++h) {
                    uint32_t v[32];
                    tmem_ld32(taddr + (u * per_unit + h) * 32, v);
                    tmem_ld_wait();
                    if (scaled) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * unscale_g * unscale_b);
                    }
                    if (od.out_bf16) {
#pragma unroll
                        for (int pc = 0; pc < 4; ++pc) {
                            uint4 pk;
                            pk.x = pack_bf16x2(__uint_as_float(v[pc * 8 + 0]), __uint_as_float(v[pc * 8 + 1]));
                            pk.y = pack_bf16x2(__uint_as_float(v[pc * 8 + 2]), __uint_as_float(v[pc * 8 + 3]));
                            pk.z = pack_bf16x2(__uint_as_float(v[pc * 8 + 4]), __uint_as_float(v[pc * 8 + 5]));
                            pk.w = pack_bf16x2(__uint_as_float(v[pc * 8 + 6]), __uint_as_float(v[pc * 8 + 7]));
                            *reinterpret_cast<uint4*>(buf + lane * 128 + (((h * 4 + pc) ^ (lane & 7)) << 4)) = pk;
                        }
                    } else {
#pragma unroll
                        for (int pc = 0; pc < 8; ++pc)
                            *reinterpret_cast<uint4*>(buf + lane * 128 + ((pc ^ (lane & 7)) << 4)) =
                                make_uint4(v[pc * 4], v[pc * 4 + 1], v[pc * 4 + 2], v[pc * 4 + 3]);
                    }
                }
                fence_proxy_async();
                __syncwarp();
                const int col = n0 + u * per_unit * 32;
                if (lane == 0 && col < p.n && m0 + q * 32 < od.m) {
                    tma_store_3d(&p.out_map[od.problem], smem_u32(buf), col, m0 + q * 32, od.part);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    st.stores_in_flight = 1;
                }
            }
            tc_fence_before();
            release();
            return;
        }
        const int n1 = tile_bn < MAX_BN ? tile_bn : MAX_BN, n2 = tile_bn - n1, h1 = n1 >> 1, half = tile_bn >> 1;
        for (int ch = u_begin; ch < u_end; ++ch) {
            const int c = ch * 32;
            int tcol = c, gcol = c;
            if (p.wide && tile_bn > MAX_BN) {
                if (c < n1) {
                    gcol = c < h1 ? c : half + (c - h1);
                } else {
                    const int c2 = c - n1;
                    tcol = MAX_BN + c2;
                    gcol = c2 < (n2 >> 1) ? h1 + c2 : half + h1 + (c2 - (n2 >> 1));
                }
            }
            uint32_t v[32];
            tmem_ld32(taddr + tcol, v);
            tmem_ld_wait();
            if (scaled) {             // two factors: their product could leave fp32's range
#pragma unroll
                for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * unscale_g * unscale_b);
            }
            if (rvalid) {
                const int col0 = n0 + gcol;
                if (od.acc_in != nullptr) {
                    const float* ap = od.acc_in + (long long)grow * od.ld_acc + col0;
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        if (col0 + c < p.n) {
                            const float4 a = *reinterpret_cast<const float4*>(ap + c);
                            v[c] = __float_as_uint(__uint_as_float(v[c]) + a.x);
                            v[c + 1] = __float_as_uint(__uint_as_float(v[c + 1]) + a.y);
                            v[c + 2] = __float_as_uint(__uint_as_float(v[c + 2]) + a.z);
                            v[c + 3] = __float_as_uint(__uint_as_float(v[c + 3]) + a.w);
                        }
                    }
                }
                if (od.out_bf16) {
                    __nv_bfloat16* op = reinterpret_cast<__nv_bfloat16*>(od.out) + (long long)grow * od.ld_out + col0;
#pragma unroll
                    for (int c = 0; c < 32; c += 8) {
                        if (col0 + c < p.n) {
                            uint4 pk;
                            pk.x = pack_bf16x2(__uint_as_float(v[c]), __uint_as_float(v[c + 1]));
                            pk.y = pack_bf16x2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
                            pk.z = pack_bf16x2(__uint_as_float(v[c + 4]), __uint_as_float(v[c + 5]));
                            pk.w = pack_bf16x2(__uint_as_float(v[c + 6]), __uint_as_float(v[c + 7]));
                            *reinterpret_cast<uint4*>(op + c) = pk;
                        }
                    }
                } else {
                    float* op = reinterpret_cast<float*>(od.out) + (long long)grow * od.ld_out + col0;
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        if (col0 + c < p.n) {
                            float4 o;
                            o.x = __uint_as_float(v[c]);
                            o.y = __uint_as_float(v[c + 1]);
                            o.z = __uint_as_float(v[c + 2]);
                            o.w = __uint_as_float(v[c + 3]);
                            *reinterpret_cast<float4*>(op + c) = o;
                        }
                    }
                }
            }
        }
        tc_fence_before();
        release();
    }
}

// Called once per epilogue thread before the CTA ends: panel stores must have been written.
// (Pending column sums are flushed by the kernels, which know whether the tile loop ended cleanly.)
template <int EPI>
__device__ __forceinline__ void epilogue_drain(const EpiState& st, int lane) {
    if ((epi_is_coef(EPI) || EPI == EPI_OUT) && lane == 0 && st.stores_in_flight > 0) {
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
}

}  // namespace meclip
