// Softmax over a vocabulary: the row kernels around the tile passes EPI_STATS and EPI_VCOEF.
//
//   z_ij = <x_i, y_j> / T over a table of V rows y_j,  p_ij = exp(z_ij - lse_i)
//
// The tile pass leaves, per row and half column tile, {maximum, sum, first moment} in base-2 units, and per 32 columns
// the maximum; nothing of size rows x V is stored.  vocab_rows_kernel joins those, and forms from the operands
// themselves the few scores that are wanted one by one: those of given tokens, of a teacher's entries, of the best.
// Base 2: s2 = <x, y> log2(e)/T, lse2 = log2 sum_j 2^s2_j, so log p = (s2 - lse2) ln 2.
#pragma once
#include <cuda_fp16.h>

namespace meclip {

static constexpr int VOCAB_THREADS = 256;
static constexpr int VOCAB_MAX_ENTRIES = 256;      // given tokens or teacher entries of one row
static constexpr int VOCAB_MAX_TOP = 32;           // top alternatives: one per lane
static constexpr int VOCAB_EXTRA = 32;             // chunks beyond the K best that rounding may have kept apart

// Entries (given tokens, teacher entries) of a backward, and the row factors of the dense part.
struct VocabGrad {
    const float* row_lse;
    const float* row_a;
    const float* row_b;               // null: no log2 p term
    const long long* tokens;          // [rows, k]
    const float* token_s2;            // [rows, k], saved by the forward
    int k;
    const float* entry;               // [rows, k] and
    const float* entry_scale;         // [rows] or null: the entry's own term is entry * entry_scale * entry_mul
    float entry_mul;
    const __nv_bfloat16* x_f16;       // fp16 operands for the scores (typed as 16-bit words), null: the bf16 ones
    long long ldx_f16;
    const __nv_bfloat16* y_f16;
    long long ldy_f16;
};

struct VocabRows {
    const float4* stats; int slots; long long stats_ld;
    const float* chunk_max; const uint32_t* chunk_second; int chunks; long long chunk_ld;
    const void* x; const void* y; long long ldx, ldy; int d;
    long long rows, vocab;
    float fmul;                       // log2(e) / T
    const long long* tokens; int k;
    float* row_lse;                   // base 2, may be null
    float* entropy;                   // nats, may be null
    float* token_s2;                  // may be null
    float* log_probs;                 // [rows, k], token scoring
    int top_k; float* top_log_probs; long long* top_tokens; int list_cap;
    // distillation
    const void* teacher_logits; int teacher_dtype; float inv_teacher_t;
    float* teacher_probs;             // [rows, k]
    float* row_loss;                  // [rows]
    float* row_has;                   // [rows], 1 where the teacher says anything
};

__device__ __forceinline__ void half8(const __nv_bfloat16* p, float (&v)[8]) { load8(p, v); }
__device__ __forceinline__ void half8(const __half* p, float (&v)[8]) { load8(p, v); }

// Dot products of x with four rows of the table by one warp, in fp32: the products are exact (8 or 11 bits each),
// a lane adds d / 32 of them.  Operand rows are padded to 16 bytes and 8 elements.
template <typename T>
__device__ __forceinline__ void warp_dot4(const T* __restrict__ x, const T* const (&y)[4], int d, int lane, float (&out)[4]) {
    float acc[4][2] = {};
    for (int c = lane * 8; c < d; c += 256) {
        float xv[8], yv[4][8];
        half8(x + c, xv);
#pragma unroll
        for (int r = 0; r < 4; ++r) half8(y[r] + c, yv[r]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[r][i & 1] = fmaf(xv[i], yv[r][i], acc[r][i & 1]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) out[r] = warp_sum(acc[r][0] + acc[r][1]);
}

// The same in fp64: which of two close alternatives comes first has to be right, and products are exact in fp32.
template <typename T>
__device__ __forceinline__ void warp_dot4(const T* __restrict__ x, const T* const (&y)[4], int d, int lane, double (&out)[4]) {
    double acc[4] = {};
    for (int c = lane * 8; c < d; c += 256) {
        float xv[8], yv[4][8];
        half8(x + c, xv);
#pragma unroll
        for (int r = 0; r < 4; ++r) half8(y[r] + c, yv[r]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[r] += (double)(xv[i] * yv[r][i]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
        out[r] = acc[r];
    }
}

// (value, index) order of alternatives: larger value first, then the lower index.
template <typename V, typename I>
__device__ __forceinline__ bool comes_first(V a, I ia, V b, I ib) { return a > b || (a == b && ia < ib); }

// A warp's sorted list, one element per lane: inserts (z, j), the last lane's element falls off.
__device__ __forceinline__ void list_insert(double& lz, long long& lj, double z, long long j, int lane) {
    const unsigned ahead = __ballot_sync(0xffffffffu, comes_first(lz, lj, z, j));
    const int pos = __popc(ahead);               // the list is sorted: the lanes ahead are the first ones
    const double pz = __shfl_up_sync(0xffffffffu, lz, 1);
    const long long pj = __shfl_up_sync(0xffffffffu, lj, 1);
    if (lane > pos) { lz = pz; lj = pj; }
    if (lane == pos) { lz = z; lj = j; }
}

template <int G> __device__ __forceinline__ void group_sync() {
    if (G == 32) __syncwarp();
    else __syncthreads();
}

// Shared memory of one row, in bytes (a multiple of 16).
__host__ __device__ constexpr int vocab_row_smem(int k, int top_k, int list_cap, int warps) {
    return 64 * 8 +                                                       // reductions across warps
           (k * 4 + 15) / 16 * 16 +                                       // scores of the entries
           (top_k > 0 ? (VOCAB_MAX_TOP + VOCAB_EXTRA) * 4 + list_cap * 4 + warps * VOCAB_MAX_TOP * 16 : 0);
}

// Sum / maximum over the G threads of a row, the same on all of them.
template <int G, bool MAX>
__device__ __forceinline__ float group_reduce(float v, float* red, int gt) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmaxf(v, w) : v + w;
    }
    if (G > 32) {
        __syncthreads();
        if ((gt & 31) == 0) red[gt >> 5] = v;
        __syncthreads();
        v = red[0];
        for (int i = 1; i < G / 32; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
    }
    return v;
}

// The top alternatives of one row.  The K largest elements lie in the K chunks that come first by (maximum, index),
// and the tile pass knows each chunk's best column and its second best value up to rounding.  So: take chunks in that
// order until the K-th is found, go on while rounding could still matter, score in fp64 the best column of each taken
// chunk - all 32 columns where the second best might be among the K too - and sort.  By warp 0 up to the list of
// columns, by all warps of the row from there.
template <int G, typename T>
__device__ __forceinline__ void row_top(const VocabRows& p, long long row, int gt, uint8_t* smem, float m, float log2l) {
    constexpr int W = G / 32;
    const int lane = gt & 31, w = gt >> 5;
    int* sel = reinterpret_cast<int*>(smem);                                 // taken chunks
    int* list = sel + VOCAB_MAX_TOP + VOCAB_EXTRA;                           // columns to score
    double* lz_s = reinterpret_cast<double*>(list + p.list_cap);
    long long* lj_s = reinterpret_cast<long long*>(lz_s + W * VOCAB_MAX_TOP);
    __shared__ int count_s[VOCAB_THREADS / G];
    int* count_p = &count_s[threadIdx.x / G];
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
    const T* y = reinterpret_cast<const T*>(p.y);
    const float* cmax = p.chunk_max + row * p.chunk_ld;
    const uint32_t* csec = p.chunk_second + row * p.chunk_ld;
    const int K = p.top_k;
    if (w == 0) {
        // each lane owns every 32nd chunk and keeps its first one that has not been taken
        auto rescan = [&](float tv, int tc, float& bv, int& bc) {
            bv = -INFINITY; bc = 0x7fffffff;
#pragma unroll 8
            for (int c = lane; c < p.chunks; c += 32) {
                const float v = cmax[c];
                if (comes_first(tv, tc, v, c) && comes_first(v, c, bv, bc)) { bv = v; bc = c; }
            }
        };
        float bv; int bc;
        rescan(INFINITY, -1, bv, bc);
        int taken = 0;
        float theta = -INFINITY, eps = 0.f;
        while (taken < K + VOCAB_EXTRA) {
            float v = bv; int c = bc;
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) {
                const float ov = __shfl_xor_sync(0xffffffffu, v, o);
                const int oc = __shfl_xor_sync(0xffffffffu, c, o);
                if (comes_first(ov, oc, v, c)) { v = ov; c = oc; }
            }
            if (c == 0x7fffffff) break;                                      // no chunk left
            if (taken >= K && !(v >= theta - 2.f * eps)) break;
            if (lane == 0) sel[taken] = c;
            if (bc == c) rescan(v, c, bv, bc);
            if (++taken == K) {
                theta = v;
                // how far the tile pass may be off: d / 16 accumulation steps that each drop up to an ulp of a partial
                // sum, which stays below |x| |y|; the best alternative's |y| stands for those of its rivals, doubled
                __syncwarp();
                const long long c1 = (long long)sel[0] * 32 + (csec[sel[0]] & 31u);
                const T* const rows4[4] = {y + c1 * p.ldy, x, x, x};
                float yy = 0.f, xx = 0.f;
                for (int i = lane * 8; i < p.d; i += 256) {
                    float a[8], b[8];
                    half8(rows4[0] + i, a);
                    half8(rows4[1] + i, b);
#pragma unroll
                    for (int j = 0; j < 8; ++j) { yy = fmaf(a[j], a[j], yy); xx = fmaf(b[j], b[j], xx); }
                }
                yy = warp_sum(yy); xx = warp_sum(xx);
                eps = 2.f * 1.1920929e-7f * ((float)p.d * 0.0625f + 4.f) * p.fmul * sqrtf(yy) * sqrtf(xx) +
                      4.f * 1.1920929e-7f * fabsf(theta);
            }
        }
        if (taken < K) theta = -INFINITY;
        __syncwarp();
        int n = 0;
        for (int i = 0; i < taken; ++i) {
            const int c = sel[i];
            const uint32_t sec = csec[c];
            const bool whole = cmax[c] - __uint_as_float(sec & ~31u) >= theta - 2.f * eps;   // false for "no second" (NaN)
            if (n + (whole ? 32 : 1) > p.list_cap) break;
            if (whole) {
                const int left = (int)min(32ll, p.vocab - (long long)c * 32);
                if (lane < left) list[n + lane] = c * 32 + lane;
                n += left;
            } else {
                if (lane == 0) list[n] = c * 32 + (int)(sec & 31u);
                ++n;
            }
        }
        if (lane == 0) *count_p = n;
    }
    group_sync<G>();
    const int n = *count_p;
    double lz = -INFINITY;
    long long lj = 0x7fffffffffffffffll;
    for (int i = w * 4; i < n; i += W * 4) {
        const T* r4[4];
        long long j4[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) { j4[r] = list[min(i + r, n - 1)]; r4[r] = y + j4[r] * p.ldy; }
        double z[4];
        const T* const rr[4] = {r4[0], r4[1], r4[2], r4[3]};
        warp_dot4<T>(x, rr, p.d, lane, z);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (i + r < n) list_insert(lz, lj, z[r], j4[r], lane);
    }
    if (W > 1) {
        lz_s[w * VOCAB_MAX_TOP + lane] = lz;
        lj_s[w * VOCAB_MAX_TOP + lane] = lj;
        group_sync<G>();
        if (w == 0)
            for (int i = 1; i < W; ++i)
                for (int e = 0; e < K; ++e) {
                    const long long j = lj_s[i * VOCAB_MAX_TOP + e];
                    if (j == 0x7fffffffffffffffll) break;
                    list_insert(lz, lj, lz_s[i * VOCAB_MAX_TOP + e], j, lane);
                }
    }
    if (w == 0 && lane < K) {
        const bool any = lj != 0x7fffffffffffffffll;       // false only where a row's scores are not numbers
        p.top_tokens[row * K + lane] = any ? lj : -1;
        p.top_log_probs[row * K + lane] =
            any ? (float)((lz * (double)p.fmul - (double)m - (double)log2l) * 0.6931471805599453) : NAN;
    }
}

// One row per G threads.  Bound by memory latency: a row reads its 2 V / 256 partial sums, V / 32 chunk maxima (with
// alternatives) and one table row per entry; many rows in flight per SM hide that (G = 32), and a few rows are spread
// over a block each (G = 256).
template <int G, typename T, bool DISTILL>
__global__ void __launch_bounds__(VOCAB_THREADS)
vocab_rows_kernel(const __grid_constant__ VocabRows p) {
    extern __shared__ __align__(16) uint8_t smem_all[];
    constexpr int W = G / 32;
    const int gt = (int)threadIdx.x % G, lane = gt & 31, w = gt >> 5;
    const long long row = (long long)blockIdx.x * (VOCAB_THREADS / G) + threadIdx.x / G;
    if (row >= p.rows) return;                    // whole warps (G = 32) or whole blocks (G = 256)
    uint8_t* smem = smem_all + (size_t)(threadIdx.x / G) * vocab_row_smem(p.k, p.top_k, p.list_cap, W);
    float* red = reinterpret_cast<float*>(smem);
    float* s2 = reinterpret_cast<float*>(smem + 64 * 8);
    uint8_t* top_smem = smem + 64 * 8 + (p.k * 4 + 15) / 16 * 16;

    // (1) the row's statistics
    float m = STATS_EMPTY, l = 0.f, t = 0.f;
    const float4* st = p.stats + row * p.stats_ld;
    for (int i = gt; i < p.slots; i += G) {
        const float4 v = st[i];
        stats_join(m, l, t, v.x, v.y, v.z);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o),
                    t2 = __shfl_xor_sync(0xffffffffu, t, o);
        stats_join(m, l, t, m2, l2, t2);
    }
    if (W > 1) {
        if (lane == 0) { red[w * 4] = m; red[w * 4 + 1] = l; red[w * 4 + 2] = t; }
        __syncthreads();
        m = red[0]; l = red[1]; t = red[2];
        for (int i = 1; i < W; ++i) stats_join(m, l, t, red[i * 4], red[i * 4 + 1], red[i * 4 + 2]);
        __syncthreads();
    }
    const float log2l = log2f(l);
    if (gt == 0) {
        if (p.row_lse != nullptr) p.row_lse[row] = m + log2l;
        if (p.entropy != nullptr) p.entropy[row] = 0.6931471805599453f * (log2l - t / l);
    }

    // (2) the scores of the row's entries
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
    const T* y = reinterpret_cast<const T*>(p.y);
    const long long* tok = p.tokens + row * p.k;
    for (int e = w * 4; e < p.k; e += W * 4) {
        const T* r4[4];
        bool any = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const long long j = e + r < p.k ? tok[e + r] : -1;
            const bool in = j >= 0 && j < p.vocab;
            any |= in;
            r4[r] = y + (in ? j : 0) * p.ldy;
        }
        float z[4] = {0.f, 0.f, 0.f, 0.f};
        const T* const rr[4] = {r4[0], r4[1], r4[2], r4[3]};
        if (any) warp_dot4<T>(x, rr, p.d, lane, z);
        if (lane < 4 && e + lane < p.k) {
            const float zz = lane == 0 ? z[0] : lane == 1 ? z[1] : lane == 2 ? z[2] : z[3];
            s2[e + lane] = zz * p.fmul;
        }
    }
    group_sync<G>();

    // (3) what is made of them
    if (!DISTILL) {
        for (int e = gt; e < p.k; e += G) {
            const long long j = tok[e];
            // a token below 0 is padding: 0; one behind the table is a mistake that shows
            const float lp = (float)(((double)s2[e] - (double)m - (double)log2l) * 0.6931471805599453);
            p.log_probs[row * p.k + e] = j < 0 ? 0.f : j >= p.vocab ? NAN : lp;
            if (p.token_s2 != nullptr) p.token_s2[row * p.k + e] = s2[e];
        }
    } else {
        // q = softmax of the teacher's logits over the entries that are there; KL = sum q (log q - log p)
        auto logit = [&](int e) -> float {
            const long long at = row * p.k + e;
            const float v = p.teacher_dtype == 1 ? reinterpret_cast<const float*>(p.teacher_logits)[at]
                            : p.teacher_dtype == 0 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.teacher_logits)[at])
                                                   : __half2float(reinterpret_cast<const __half*>(p.teacher_logits)[at]);
            return v * p.inv_teacher_t;
        };
        auto there = [&](int e) -> bool { return tok[e] >= 0 && !(logit(e) == -INFINITY); };
        float um = -INFINITY, seen = 0.f;
        for (int e = gt; e < p.k; e += G)
            if (there(e)) { um = fmaxf(um, logit(e)); seen = 1.f; }
        um = group_reduce<G, true>(um, red, gt);
        seen = group_reduce<G, true>(seen, red, gt);
        float sum = 0.f;
        for (int e = gt; e < p.k; e += G)
            if (there(e)) sum += expf(logit(e) - um);
        sum = group_reduce<G, false>(sum, red, gt);
        const float inv = 1.f / sum, log_sum = logf(sum);
        double kl = 0.0;
        for (int e = gt; e < p.k; e += G) {
            const long long at = row * p.k + e;
            float q = 0.f;
            if (there(e)) {
                const float u = logit(e) - um;
                q = expf(u) * inv;
                const double lp = ((double)s2[e] - (double)m - (double)log2l) * 0.6931471805599453;
                if (tok[e] >= p.vocab) q = NAN;
                if (q != 0.f) kl += (double)q * ((double)u - (double)log_sum - lp);
            }
            p.teacher_probs[at] = q;
            p.token_s2[at] = s2[e];
        }
        // the terms are few and of one row: fp64 costs nothing and keeps the difference of two logarithms exact
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) kl += __shfl_xor_sync(0xffffffffu, kl, o);
        if (W > 1) {
            double* red64 = reinterpret_cast<double*>(red);
            __syncthreads();
            if (lane == 0) red64[w] = kl;
            __syncthreads();
            kl = red64[0];
            for (int i = 1; i < W; ++i) kl += red64[i];
        }
        if (gt == 0) {
            p.row_loss[row] = seen > 0.f ? (float)kl : 0.f;
            p.row_has[row] = seen;
        }
    }
    if (!DISTILL && p.top_k > 0) {
        group_sync<G>();
        row_top<G, T>(p, row, gt, top_smem, m, log2l);
    }
}

// loss = sum of the rows' losses, divided by the number of rows that have one when `mean`; inv_count gets the factor.
// One block, fixed order.  No row at all: loss 0, factor 0.
__global__ void __launch_bounds__(1024)
distill_reduce_kernel(const float* __restrict__ row_loss, const float* __restrict__ row_has, long long n, int mean,
                      float* __restrict__ loss, float* __restrict__ inv_count) {
    __shared__ double part[1024];
    __shared__ double cnt[1024];
    double a = 0.0, c = 0.0;
#pragma unroll 4
    for (long long i = threadIdx.x; i < n; i += 1024) {
        a += (double)row_loss[i];
        c += (double)row_has[i];
    }
    part[threadIdx.x] = a;
    cnt[threadIdx.x] = c;
    __syncthreads();
    for (int s = 512; s >= 1; s >>= 1) {
        if ((int)threadIdx.x < s) { part[threadIdx.x] += part[threadIdx.x + s]; cnt[threadIdx.x] += cnt[threadIdx.x + s]; }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double f = mean ? (cnt[0] > 0.0 ? 1.0 / cnt[0] : 0.0) : 1.0;
        *loss = (float)(part[0] * f);
        *inv_count = (float)f;
    }
}

// Row factors of the backward, dz_ij = p_ij (a + b log2 p_ij) + entries, divided by T (in `inv_t`).
//   token scoring: a = -(sum_k g_k + h H), b = -h ln 2, g_k over the tokens inside the table
__global__ void __launch_bounds__(ROW_KERNEL_THREADS)
token_grad_rows_kernel(const float* __restrict__ grad_log_probs, const float* __restrict__ grad_entropy,
                       const float* __restrict__ entropy, const long long* __restrict__ tokens, int k, long long rows,
                       long long vocab, float inv_t, float* __restrict__ row_a, float* __restrict__ row_b) {
    const long long row = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= rows) return;
    float g = 0.f;
    if (grad_log_probs != nullptr)
        for (int e = lane; e < k; e += 32) {
            const long long j = tokens[row * k + e];
            if (j >= 0 && j < vocab) g += grad_log_probs[row * k + e];
        }
    g = warp_sum(g);
    if (lane == 0) {
        const float h = grad_entropy != nullptr ? grad_entropy[row] : 0.f;
        // h = 0 takes no part, whatever the row's entropy is
        row_a[row] = -(g + (h != 0.f ? h * entropy[row] : 0.f)) * inv_t;
        if (row_b != nullptr) row_b[row] = -h * 0.6931471805599453f * inv_t;
    }
}

//   distillation: a = w = grad_out * factor / T for the rows that have a teacher, b = 0
__global__ void __launch_bounds__(256)
distill_grad_rows_kernel(const float* __restrict__ grad_out, int per_row, const float* __restrict__ factor,
                         const float* __restrict__ row_has, long long rows, float inv_t, float* __restrict__ row_a) {
    const long long row = (long long)blockIdx.x * 256 + threadIdx.x;
    if (row >= rows) return;
    const float f = factor != nullptr ? __ldg(factor) : 1.f;
    row_a[row] = row_has[row] > 0.f ? grad_out[per_row ? row : 0] * f * inv_t : 0.f;
}

// Puts the entries' own terms into a coefficient panel: G_ij = p_ij (a + b log2 p_ij) + sum of the row's terms at j,
// formed in fp32 from the saved scores and rounded to bf16 once, over what the tile pass stored there.  One warp per
// row; of entries with the same token the first writes and adds the others' terms.
__global__ void __launch_bounds__(ROW_KERNEL_THREADS)
vocab_entries_kernel(const __grid_constant__ VocabGrad g, long long r0, long long nr, long long c0, long long nc,
                     __nv_bfloat16* __restrict__ panel, long long rows_alloc) {
    const long long i = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= nr) return;
    const long long row = r0 + i;
    const long long* tok = g.tokens + row * g.k;
    const float scale = (g.entry_scale != nullptr ? g.entry_scale[row] : 1.f) * g.entry_mul;
    for (int e = lane; e < g.k; e += 32) {
        const long long j = tok[e];
        if (j < c0 || j >= c0 + nc) continue;          // absent, outside the table or in another panel
        bool first = true;
        float term = 0.f;
        for (int o = 0; o < g.k; ++o)
            if (tok[o] == j) {
                if (o < e) { first = false; break; }
                if (g.entry != nullptr) term += g.entry[row * g.k + o];
            }
        if (!first) continue;
        const float u = g.token_s2[row * g.k + e] - g.row_lse[row];
        const float b = g.row_b != nullptr ? g.row_b[row] : 0.f;
        const float v = fmaf(exp2f(u), fmaf(b, u, g.row_a[row]), scale != 0.f ? term * scale : 0.f);
        const long long col = j - c0;
        panel[((col >> 6) * rows_alloc + i) * 64 + (col & 63)] = __float2bfloat16_rn(v);
    }
}

static int launch_vocab_entries(const VocabGrad& g, long long r0, long long nr, long long c0, long long nc, long long,
                                __nv_bfloat16* panel, long long rows_alloc, cudaStream_t s) {
    if (g.k == 0 || g.entry == nullptr) return MECLIP_OK;
    const int wpb = ROW_KERNEL_THREADS / 32;
    ScopedTiming timing(s, TAG_ROW, (double)nr * g.k * 18.0);
    vocab_entries_kernel<<<(unsigned)((nr + wpb - 1) / wpb), ROW_KERNEL_THREADS, 0, s>>>(g, r0, nr, c0, nc, panel, rows_alloc);
    MECLIP_CUDA(cudaGetLastError());
    return MECLIP_OK;
}

}  // namespace meclip
