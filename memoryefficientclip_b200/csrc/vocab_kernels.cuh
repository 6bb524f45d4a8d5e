// Softmax over a vocabulary: the row kernels around the tile passes EPI_STATS and EPI_VCOEF.
//
//   z_ij = <x_i, y_j> / T over a table of V rows y_j,  p_ij = exp(z_ij - lse_i)
//
// The tile pass leaves, per row and half column tile, {maximum, sum, first moment} in base-2 units, and per 32 columns
// the maximum; nothing of size rows x V is stored.  vocab_rows_kernel joins those, and forms from the operands
// themselves the few scores that are wanted one by one: those of given tokens, of a teacher's entries, of the best.
// Base 2: s2 = <x, y> log2(e)/T, lse2 = log2 sum_j 2^s2_j = m + log2(1 + r), log2 p = s2 - lse2.
#pragma once
#include <cuda_fp16.h>

namespace meclip {

static constexpr int VOCAB_THREADS = 256;
static constexpr int VOCAB_MAX_ENTRIES = 256;      // given tokens or teacher entries of one row
static constexpr int VOCAB_MAX_TOP = 32;           // top alternatives: one per lane

// Coefficients of a softmax over a vocabulary, dz_ij / T = p_ij (a_i + b_i log2 p_ij) + sum of the terms of the row's
// entries at j; what a_i, b_i and the terms are follows from the loss.
struct VocabCoef {
    const float* row_lse;             // base 2
    const float* token_lp2;           // [rows, k] base-2 log probabilities of the entries, saved by the forward
    const long long* tokens;          // [rows, k]
    int k;
    int distill;
    long long vocab;
    float inv_t;
    // token scoring: a = -(sum of g over the tokens inside the table + h H) / T, b = -h ln 2 / T, terms g / T
    const float *grad_log_probs, *grad_entropy, *entropy;        // g [rows, k], h, H [rows]; g, h may be null
    // distillation: a = w = grad_out * factor / T where there is a teacher, b = 0, terms -w q
    const float *grad_out, *factor, *row_has, *probs;            // probs = q [rows, k]; factor may be null
    int grad_per_row;
};

// Coefficient at entry e of a row: the dense part from the saved log probability, and the terms of all entries that name the
// same token.  Entries but the first of a token return false.
__device__ __forceinline__ bool vocab_entry(const VocabCoef& v, long long row, int e, float a, float b, float& value) {
    const long long* tok = v.tokens + row * v.k;
    const float* term = v.distill ? v.probs : v.grad_log_probs;
    float sum = 0.f;
    for (int o = 0; o < v.k; ++o)
        if (tok[o] == tok[e]) {
            if (o < e) return false;
            if (term != nullptr) sum += term[row * v.k + o];
        }
    const float u = v.token_lp2[row * v.k + e];
    const float scale = v.distill ? -a : v.inv_t;
    value = fmaf(exp2f(u), fmaf(b, u, a), scale != 0.f ? sum * scale : 0.f);     // (no teacher: whatever q is)
    return true;
}

// A backward: the coefficients, the type of the operands, and which form the panel takes.
struct VocabGrad {
    VocabCoef coef;
    float4 *row_factors, *row_entries;          // see GemmParams; entries null: vocab_entries_kernel stores them
    int f16;                          // operands are fp16, and so is the panel
    float tile_fmul;
    long long widest;                 // columns of a coefficient panel at most
    int two_panels;                   // bf16 panel and a second one with its remainders
    unsigned int* total;              // see OutScale; it and table_max behind it are cleared by grad_impl
    float* table_max;
    __half* features;                 // [rows, d] scaled features where no transposed copies are made of an fp16 problem
    float *split_buf, *split_buf2;    // parts of contractions that are cut along K: dX's own when both run at a time
    size_t split_bytes;               // of each
};

// The tensor cores cut what does not fit into an fp32 accumulator instead of rounding it, once every 16 products, so a
// score comes out too small in magnitude, on average by a part of the partial sums it ran through.  For a score that
// grows steadily that is 0.09 ulp-of-itself per step (half of the 2^-24 .. 2^-25 that a cut at one guard bit costs, over
// a triangle); for the scores that carry a softmax 0.11 to 0.13 was measured (D = 64 .. 1152).  The tile passes scale by
// that much more, which leaves their log-sum-exp unbiased: at D = 1024 and scores up to 20 its error fell from 1.1e-5
// to 2e-6 (root of the mean square, base 2).
static constexpr double VOCAB_KAPPA = 0.12;
static float vocab_tile_fmul(float temperature, long long d) {
    return (float)(1.4426950408889634 / (double)temperature * (1.0 + VOCAB_KAPPA * (double)((d + 15) / 16) * 0x1p-23));
}

struct VocabRows {
    const float4* stats; int slots; long long stats_ld;
    float unit;                       // of the maxima in stats: fmul for plain scores, 1 for base 2
    const float* chunk_max; const uint32_t* chunk_second; int chunks; long long chunk_ld;
    const void* x; const void* y; long long ldx, ldy; int d;
    long long rows, vocab;
    float fmul;                       // log2(e) / T
    const long long* tokens; int k;
    float* row_lse;                   // base 2, may be null
    float* entropy;                   // nats, may be null
    float* token_lp2;                 // may be null
    float* log_probs;                 // [rows, k], token scoring
    int top_k; float* top_log_probs; long long* top_tokens; int rank_cap;
    // distillation
    const void* teacher_logits; int teacher_dtype; float inv_teacher_t;
    float* teacher_probs;             // [rows, k]
    float* row_loss;                  // [rows]
    float* row_has;                   // [rows], 1 where the teacher says anything
    // sum over the rows by the last block, for the last block of rows of the problem: loss null otherwise
    unsigned int* blocks_done;        // the unused fourth word of stats[0], which the tile pass has stored as zero
    const float *all_loss, *all_has;  // of all rows, all_rows of them
    long long all_rows;
    int mean;
    float *loss, *inv_count;
};

// log2 p of a score z that was formed from the operands, in a row with maximum m (in p.unit) and sum 1 + r of the tile pass.
// The maximum itself takes the pass's score: its log probability is then -log2(1 + r), exact however small r is, and what
// the pass is off by cancels.  Another column can be mistaken for the maximum only where the pass cannot tell them apart (an
// ulp for every 64 columns of d).
__device__ __forceinline__ double vocab_lp2(const VocabRows& p, double z, float m, float r, float log2l) {
    const double below = p.unit == 1.f ? z * (double)p.fmul - (double)m : (z - (double)m) * (double)p.unit;
    const float off = fabsf((float)below);
    const bool is_max = off <= 1.2e-7f * ((float)p.d * 0.015625f + 1.f) * (fabsf(m * p.unit) + 8.f) || (r < 0.25f && off < 0.5f);
    return (is_max ? 0.0 : below) - (double)log2l;
}

__device__ __forceinline__ void half8(const __nv_bfloat16* p, float (&v)[8]) { load8(p, v); }
__device__ __forceinline__ void half8(const __half* p, float (&v)[8]) { load8(p, v); }

// Dot products of x with four rows of the table by one warp.  The products are exact in fp32 (8 or 11 bits each); a
// lane adds d / 32 of them, in fp32 for a score and in fp64 to tell two close alternatives apart.  Two column steps are
// loaded before the first is used: the rows come from anywhere in the table, so what counts is loads in flight.  Operand
// rows are padded to 16 bytes and 8 elements.
template <typename T, typename A>
__device__ __forceinline__ void dot_step(const uint4& xr, const uint4 (&yr)[4], A (&acc)[4][2]) {
    float xv[8];
    half8(reinterpret_cast<const T*>(&xr), xv);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float yv[8];
        half8(reinterpret_cast<const T*>(&yr[r]), yv);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (sizeof(A) == 4) acc[r][i & 1] = fmaf(xv[i], yv[i], acc[r][i & 1]);
            else                acc[r][i & 1] += (A)(xv[i] * yv[i]);
        }
    }
}
template <typename T, typename A>
__device__ __forceinline__ void warp_dot4(const T* __restrict__ x, const T* const (&y)[4], int d, int lane, A (&out)[4]) {
    A acc[4][2] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int c = lane * 8; c < d; c += 512) {
        const bool more = c + 256 < d;
        const uint4 xa = *reinterpret_cast<const uint4*>(x + c), xb = more ? *reinterpret_cast<const uint4*>(x + c + 256) : zero;
        uint4 ya[4], yb[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) ya[r] = __ldg(reinterpret_cast<const uint4*>(y[r] + c));
#pragma unroll
        for (int r = 0; r < 4; ++r) yb[r] = more ? __ldg(reinterpret_cast<const uint4*>(y[r] + c + 256)) : zero;
        dot_step<T, A>(xa, ya, acc);
        dot_step<T, A>(xb, yb, acc);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        A v = acc[r][0] + acc[r][1];
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        out[r] = v;
    }
}

// The statistics of a few rows (a token at a time is answered like that) without the tensor cores, whose tile would be empty
// but for these rows: a pass over the table at the memory's rate, with fp32 multiplications and additions that round instead
// of cutting.  A block takes chunks of 32 columns, a warp eight of them, 256 elements of each at a time.  A lane copies what
// it will read itself into a ring in shared memory, so nothing but its own copies has to be waited for, and the ring runs on
// into the next chunk.  Then a warp looks at the chunk for a row: a lane per column.  Leaves what EPI_STATS leaves, with one
// partial sum per block and its maximum as a plain score, whose difference to another is exact where the difference of
// scaled ones carries the rounding of both.
// 1 x 250000 x 1152: 91 us, 6.3 TB/s (the tile pass 93.5, loads through registers instead of the ring 118); 1 x 32768 x 1024
// 15 us (18), 1 x 4099 x 512 9 us (14), events included.  Two rows take as long as the tile pass takes from large tables, four
// 10 % longer and eight twice as long: the arithmetic shows then.
static constexpr int VOCAB_FEW_THREADS = 128;
static constexpr int VOCAB_FEW_BLOCKS = 3;         // per SM
static constexpr int VOCAB_FEW_ROWS = 2;
static constexpr int VOCAB_FEW_STAGES = 4;
static constexpr int VOCAB_FEW_RING = VOCAB_FEW_STAGES * VOCAB_FEW_THREADS * 8 * 16;      // bytes
static constexpr int VOCAB_FEW_X = 64 * 1024;      // bytes of features at most

struct VocabFew {
    const void *x, *y; long long ldx, ldy; int d, d_smem, rows;      // d_smem: d rounded up to 256
    long long vocab, chunks;
    float fmul;
    float4* stats; long long stats_ld;
    float* chunk_max; uint32_t* chunk_second; long long chunk_ld;
};

__device__ __forceinline__ void wide8(const __nv_bfloat16*, const uint4& w, uint64_t (&v)[4]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f32x2(__uint_as_float(a[i] << 16), __uint_as_float(a[i] & 0xffff0000u));
}
__device__ __forceinline__ void wide8(const __half*, const uint4& w, uint64_t (&v)[4]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
        v[i] = f32x2(f.x, f.y);
    }
}

template <typename T, int R>
__global__ void __launch_bounds__(VOCAB_FEW_THREADS, VOCAB_FEW_BLOCKS)
vocab_few_kernel(const __grid_constant__ VocabFew p) {
    constexpr int S = VOCAB_FEW_STAGES;
    static_assert(R <= VOCAB_FEW_THREADS / 32, "a warp per row");
    extern __shared__ __align__(16) uint8_t few_smem[];
    __shared__ float scores[2][R][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    uint4* ring = reinterpret_cast<uint4*>(few_smem) + threadIdx.x;       // [S][8] of the lane's own, VOCAB_FEW_THREADS apart
    T* xs = reinterpret_cast<T*>(few_smem + VOCAB_FEW_RING);
    // what is copied next: 256 elements of eight columns
    long long next_ch = blockIdx.x;
    int next_c = lane * 8, next_slot = 0;
    auto copy = [&]() {
        if (next_ch < p.chunks) {
            long long col = min(next_ch * 32 + w * 8, p.vocab - 1);
            const T* src = reinterpret_cast<const T*>(p.y) + col * p.ldy;
            const bool in = next_c < p.d;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring + (next_slot * 8 + j) * VOCAB_FEW_THREADS);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src + (in ? next_c : 0)), "r"(in ? 16 : 0) : "memory");
                if (++col < p.vocab) src += p.ldy;                        // columns behind the last repeat it
            }
            next_c += 256;
            if (next_c >= p.d_smem) { next_c = lane * 8; next_ch += gridDim.x; }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        next_slot = next_slot + 1 == S ? 0 : next_slot + 1;
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) copy();
    for (int i = threadIdx.x * 8; i < R * p.d_smem; i += VOCAB_FEW_THREADS * 8) {
        const int r = i / p.d_smem, c = i % p.d_smem;
        *reinterpret_cast<uint4*>(xs + i) = r < p.rows && c < p.d
            ? *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.x) + r * p.ldx + c) : make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    float m = STATS_EMPTY, l = -1.f, t = 0.f;          // of the lane's columns in the warp's row: maximum, sum less one, moment
    int buf = 0, slot = 0;
    for (long long ch = blockIdx.x; ch < p.chunks; ch += gridDim.x, buf ^= 1) {
        uint64_t acc[8][R] = {};
#pragma unroll 1
        for (int c = lane * 8; c < p.d_smem; c += 256) {
            asm volatile("cp.async.wait_group %0;" :: "n"(S - 2) : "memory");
            copy();                    // into the slot that the step before this one has read
#pragma unroll
            for (int h = 0; h < 8; h += 4) {
                uint64_t yv[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) wide8(xs, ring[(slot * 8 + h + j) * VOCAB_FEW_THREADS], yv[j]);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    uint64_t xv[4];
                    wide8(xs, *reinterpret_cast<const uint4*>(xs + r * p.d_smem + c), xv);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[h + j][r] = fma_f32x2(xv[i], yv[j][i], acc[h + j][r]);
                }
            }
            slot = slot + 1 == S ? 0 : slot + 1;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            // eight sums over 32 lanes: halves change hands until a lane holds one column, then the rest is added up
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float a, b;
                f32x2_split(acc[j][r], a, b);
                v[j] = a + b;
            }
#pragma unroll
            for (int h = 4; h >= 1; h >>= 1)
#pragma unroll
                for (int j = 0; j < h; ++j) {
                    const bool up = (lane & h) != 0;
                    const float keep = up ? v[j + h] : v[j], give = up ? v[j] : v[j + h];
                    v[j] = keep + __shfl_xor_sync(0xffffffffu, give, h);
                }
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], 8);
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], 16);
            if (lane < 8) scores[buf][r][w * 8 + lane] = v[0];
        }
        __syncthreads();               // the other buffer is written next, this one again only behind the next barrier
        if (w < p.rows) {
            const float score = scores[buf][w < R ? w : 0][lane];
            const bool in = ch * 32 + lane < p.vocab;
            // one column: sum less one is 0 (NaN for a score that is not a number, which the maximum would hide)
            if (in) stats_join(m, l, t, score, score - score, 0.f, p.fmul);
            if (p.chunk_max != nullptr) {          // see stats_chunk
                float cm = in ? score * p.fmul : -INFINITY;
#pragma unroll
                for (int o = 16; o >= 1; o >>= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, o));
                const uint32_t key = in ? (__float_as_uint(fmaf(score, p.fmul, -cm)) & 0x7fffffe0u) | (uint32_t)lane : 0x7fffffffu;
                const uint32_t n1 = __reduce_min_sync(0xffffffffu, key);
                const uint32_t n2 = __reduce_min_sync(0xffffffffu, key == n1 ? 0x7fffffffu : key);
                if (lane == 0) {
                    p.chunk_max[w * p.chunk_ld + ch] = cm;
                    p.chunk_second[w * p.chunk_ld + ch] = (n2 & ~31u) | (n1 & 31u);
                }
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (w >= p.rows) return;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o),
                    t2 = __shfl_xor_sync(0xffffffffu, t, o);
        stats_join(m, l, t, m2, l2, t2, p.fmul);
    }
    if (lane == 0) p.stats[w * p.stats_ld + blockIdx.x] = make_float4(m, l, t, 0.f);
}

// (value, index) order of alternatives: larger value first, then the lower index.
template <typename V, typename I>
__device__ __forceinline__ bool comes_first(V a, I ia, V b, I ib) { return a > b || (a == b && ia < ib); }

// A warp's sorted list, one element per lane: inserts (z, j), the last lane's element falls off.
__device__ __forceinline__ void list_insert(double& lz, int& lj, double z, int j, int lane) {
    const unsigned ahead = __ballot_sync(0xffffffffu, comes_first(lz, lj, z, j));
    const int pos = __popc(ahead);               // the list is sorted: the lanes ahead are the first ones
    const double pz = __shfl_up_sync(0xffffffffu, lz, 1);
    const int pj = __shfl_up_sync(0xffffffffu, lj, 1);
    if (lane > pos) { lz = pz; lj = pj; }
    if (lane == pos) { lz = z; lj = j; }
}

template <int G> __device__ __forceinline__ void group_sync() {
    if (G == 32) __syncwarp();
    else __syncthreads();
}

// Shared memory of one row, in bytes (a multiple of 16).
__host__ __device__ constexpr int vocab_row_smem(int k, int top_k, int rank_cap) {
    return 64 * 8 +                                                            // reductions across warps
           (k * 4 + 15) / 16 * 16 +                                            // scores of the entries
           (top_k > 0 ? rank_cap * 16 + 64 * 8 + 16 : 0);                      // see RowTopShared
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

// The top alternatives.  The K largest elements of a row lie in the K chunks that come first by (maximum, index), and the
// tile pass knows each chunk's best column and, from below, the distance of its second best.  Per row:
//  (a) every lane keeps the two largest maxima of its share of the chunks; the K-th largest of those 64 is a bound that
//      K chunks reach, and few others do;
//  (b) the chunks that reach it, less what rounding may hide, are collected: K and a few;
//  (c) their K-th largest value decides which of them stay, and where the second best may be among the K too (one row
//      in fifty at K = 8 of 32768) all 32 columns are looked at.
// From here on the warps of a block share the work of its rows, since a row that looks at 40 columns would otherwise keep
// one warp busy long after the others are done:
//  (d) the columns are scored from the operands in fp32, those that come closer to another than that is exact in fp64;
//  (e) every column counts who comes before it.
// Crowds (many scores that are equal or nearly so: a row of zeros, repeated table rows) do not fit (b) or (c) and are taken
// chunk by chunk instead.
static constexpr int VOCAB_LIST = 64;              // chunks collected in (b)
// Columns scored in (d), a multiple of 4: K whole chunks and a few where a block has one row or the table is small; else K
// chunks of which a few as a whole, and shared memory for more warps (a row in a million has more, from 32768 columns).
__host__ __device__ constexpr int vocab_rank_cap(int top_k, bool all) { return all ? 32 * top_k + 64 : 128 + 4 * top_k; }

struct RowTopShared {
    double* z;                                     // [rank_cap] scores
    int* chunk;                                    // [VOCAB_LIST] collected, then the chunks taken
    float* value;                                  // [VOCAB_LIST]
    int* again;                                    // [rank_cap] which columns to score again
    int* count;                                    // [4]: chunks collected, columns, columns again
    int* list;                                     // [rank_cap] columns to score
};

__device__ __forceinline__ RowTopShared row_top_shared(uint8_t* smem, int rank_cap) {
    RowTopShared sh;
    sh.z = reinterpret_cast<double*>(smem);
    sh.chunk = reinterpret_cast<int*>(sh.z + rank_cap);
    sh.value = reinterpret_cast<float*>(sh.chunk + VOCAB_LIST);
    sh.again = reinterpret_cast<int*>(sh.value + VOCAB_LIST);
    sh.count = sh.again + rank_cap;
    sh.list = sh.count + 4;
    return sh;
}

// 32 values, one per lane, sorted in descending order.
__device__ __forceinline__ float warp_sort_desc(float v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const float o = __shfl_xor_sync(0xffffffffu, v, j);
            const bool keep_max = ((lane & j) == 0) == ((lane & k) == 0);
            v = keep_max ? fmaxf(v, o) : fminf(v, o);
        }
    return v;
}

// The K-th largest (K <= 32) of 64 values, two per lane, and the largest: both halves are sorted, and i come from the first
// and K - i from the second for the best split.
__device__ __forceinline__ float warp_kth(float b1, float b2, int K, int lane, float& best) {
    const float s1 = warp_sort_desc(b1, lane), s2 = warp_sort_desc(b2, lane);
    const float other = __shfl_sync(0xffffffffu, s2, max(K - lane - 2, 0));
    float bound = lane >= K ? -INFINITY : lane == K - 1 ? s1 : fminf(s1, other);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, o));
    best = __shfl_sync(0xffffffffu, s1, 0);
    return bound;
}

__device__ __forceinline__ void row_top_write(const VocabRows& p, long long row, int at, double z, long long j, float m, float r, float log2l) {
    p.top_tokens[row * p.top_k + at] = j;
    p.top_log_probs[row * p.top_k + at] = (float)(vocab_lp2(p, z, m, r, log2l) * 0.6931471805599453);
}

// A crowd, by the warps of its row: of the chunks that reach red[0] every column that the tile pass cannot rule out is scored in
// fp64 and inserted into the K best so far, whose last one rules out more as it grows.  However many columns are close to one
// another, all are looked at; of equal scores the first K are (a row of zeros, where the pass is exact, reads the maxima and
// scores a chunk a warp).  Bound by the latency of the table's rows, four at a time per warp: K = 8 from a table whose rows are
// all equal, 1 x 32768 x 1024 3.7 ms, 4096 rows 50 ms (a quarter of the features zero 0.32 ms; no crowd 0.30).
template <int G, typename T>
__device__ __forceinline__ void row_top_crowd(const VocabRows& p, long long row, int gt, const RowTopShared& sh, float m, float r,
                                              float log2l, const float* red) {
    constexpr int W = G / 32;
    constexpr int NONE = 0x7fffffff;
    const int lane = gt & 31, w = gt >> 5, K = p.top_k;
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
    const T* y = reinterpret_cast<const T*>(p.y);
    const float* cmax = p.chunk_max + row * p.chunk_ld;
    const uint32_t* csec = p.chunk_second + row * p.chunk_ld;
    const float floor_v = red[0], slack = red[1];
    double lz = -INFINITY, kth = -INFINITY;
    int lj = NONE;
    float ruled_out = -INFINITY;                   // a score of the tile pass up to here is not among the K
    for (int c0 = w * 32; c0 < p.chunks; c0 += W * 32) {
        const float v = c0 + lane < p.chunks ? cmax[c0 + lane] : -INFINITY;
        unsigned who = __ballot_sync(0xffffffffu, c0 + lane < p.chunks && v >= floor_v && v > ruled_out);
        for (; who != 0; who &= who - 1) {
            const int src = __ffs(who) - 1, c = c0 + src;
            const float vc = __shfl_sync(0xffffffffu, v, src);
            if (!(vc > ruled_out)) continue;
            const uint32_t sec = csec[c];
            const float second = vc - __uint_as_float(sec & ~31u);           // NaN: there is none
            const bool whole = second >= floor_v && second > ruled_out;
            const int first = c * 32 + (whole ? 0 : (int)(sec & 31u));
            const int n = whole ? (int)min(32ll, p.vocab - first) : 1;
            for (int i = 0; i < n; i += 4) {
                const T* r4[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) r4[q] = y + (long long)(first + min(i + q, n - 1)) * p.ldy;
                const T* const rr[4] = {r4[0], r4[1], r4[2], r4[3]};
                double z[4];
                warp_dot4<T, double>(x, rr, p.d, lane, z);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (i + q < n && z[q] > kth) {  // a later column has a higher index: equal is not enough
                        list_insert(lz, lj, z[q], first + i + q, lane);
                        kth = __shfl_sync(0xffffffffu, lz, K - 1);
                    }
            }
            ruled_out = (float)(kth * (double)p.fmul) - slack;
        }
    }
    if (W > 1) {                                   // the first warp takes in the others' lists
        if (lane < K) { sh.z[w * K + lane] = lz; sh.list[w * K + lane] = lj; }
        __syncthreads();
        if (w > 0) return;
        for (int i = K; i < W * K; ++i) {
            const double z = sh.z[i];
            const int j = sh.list[i];
            if (j != NONE) list_insert(lz, lj, z, j, lane);
        }
    }
    if (lane >= K) return;
    if (lj != NONE) row_top_write(p, row, lane, lz, lj, m, r, log2l);
    else { p.top_tokens[row * K + lane] = -1; p.top_log_probs[row * K + lane] = NAN; }     // scores that are not numbers
}

// (a) to (c): leaves the columns in sh.list, their number in sh.count[1] (-1 for a crowd) and 2 |x| |y| in red[3].
template <int G, typename T>
__device__ __forceinline__ void row_top_select(const VocabRows& p, long long row, int gt, const RowTopShared& sh, float* red) {
    constexpr int W = G / 32;
    const int lane = gt & 31, w = gt >> 5;
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
    const T* y = reinterpret_cast<const T*>(p.y);
    const float* cmax = p.chunk_max + row * p.chunk_ld;
    const uint32_t* csec = p.chunk_second + row * p.chunk_ld;
    const int K = p.top_k;

    // (a)
    float b1 = -INFINITY, b2 = -INFINITY; int bc = 0x7fffffff;
#pragma unroll 8
    for (int c = gt; c < p.chunks; c += G) {
        const float v = cmax[c];
        b2 = fmaxf(b2, fminf(b1, v));
        if (v > b1) { b1 = v; bc = c; }
    }
    if (W > 1) {
        int* red_c = reinterpret_cast<int*>(sh.z);          // 128 words each, free until (b) and (d)
        float* red_2 = reinterpret_cast<float*>(sh.chunk);  // (chunk and value)
#pragma unroll
        for (int k = W / 2; k >= 1; k >>= 1) {              // the upper half of the warps hands its maxima to the lower
            __syncthreads();
            if (w >= k && w < 2 * k) {
                red[(w - k) * 32 + lane] = b1; red_2[(w - k) * 32 + lane] = b2; red_c[(w - k) * 32 + lane] = bc;
            }
            __syncthreads();
            if (w < k) {
                const float o1 = red[w * 32 + lane], o2 = red_2[w * 32 + lane];
                b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
                if (o1 > b1) { b1 = o1; bc = red_c[w * 32 + lane]; }
            }
        }
        __syncthreads();
    }
    float floor_v = -INFINITY, slack = 0.f, size = 0.f;
    if (w == 0) {
        float best;
        const float bound = warp_kth(b1, b2, K, lane, best);
        const unsigned who = __ballot_sync(0xffffffffu, b1 == best && bc != 0x7fffffff);
        if (who != 0) {
            // How far the tile pass may be off: d / 16 accumulation steps that each drop up to an ulp of a partial sum,
            // which stays below |x| |y|; the best alternative's |y| stands for those of its rivals, doubled.
            const int c0 = __shfl_sync(0xffffffffu, bc, __ffs(who) - 1);
            const T* y0 = y + ((long long)c0 * 32 + (csec[c0] & 31u)) * p.ldy;
            float yy = 0.f, xx = 0.f;
            for (int i = lane * 8; i < p.d; i += 256) {
                float a[8], b[8];
                half8(y0 + i, a);
                half8(x + i, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) { yy = fmaf(a[j], a[j], yy); xx = fmaf(b[j], b[j], xx); }
            }
            size = 2.f * sqrtf(warp_sum(yy)) * sqrtf(warp_sum(xx));
            slack = 2.f * 1.1920929e-7f * (((float)p.d * 0.0625f + 4.f) * p.fmul * size +
                                           2.f * fabsf(best) + 2.f * fabsf(bound == -INFINITY ? 0.f : bound));
        }
        floor_v = bound - slack;
        if (lane == 0) { sh.count[0] = 0; red[0] = floor_v; red[1] = slack; red[3] = size; }
    }
    group_sync<G>();
    floor_v = red[0];
    slack = red[1];
    // (b)
#pragma unroll 8
    for (int c = gt; c < p.chunks; c += G) {
        const float v = cmax[c];
        if (v >= floor_v) {
            const int at = atomicAdd(sh.count, 1);
            if (at < VOCAB_LIST) { sh.chunk[at] = c; sh.value[at] = v; }
        }
    }
    group_sync<G>();
    // (c)
    if (w == 0) {
        const int taken = sh.count[0];
        float theta = -INFINITY;
        if (taken <= VOCAB_LIST) {
            for (int i = lane; i < taken; i += 32) {
                const float v = sh.value[i];
                const int c = sh.chunk[i];
                int before = 0;
#pragma unroll 8
                for (int j = 0; j < taken; ++j) before += comes_first(sh.value[j], sh.chunk[j], v, c) ? 1 : 0;
                if (before == K - 1) red[2] = v;
            }
            __syncwarp();
            if (taken >= K) theta = red[2];
        }
        int n = 0;
        bool crowd = taken > VOCAB_LIST;
        if (!crowd) {
#pragma unroll
            for (int h = 0; h < VOCAB_LIST; h += 32) {
                const int i = h + lane;
                int c = 0, size = 0, best = 0;
                if (i < taken && sh.value[i] >= theta - slack) {
                    c = sh.chunk[i];
                    const uint32_t sec = csec[c];
                    best = (int)(sec & 31u);
                    const bool whole = sh.value[i] - __uint_as_float(sec & ~31u) >= theta - slack;   // false for "no second" (NaN)
                    size = whole ? (int)min(32ll, p.vocab - (long long)c * 32) : 1;
                }
                int upto = size;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int t = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += t;
                }
                const int all = __shfl_sync(0xffffffffu, upto, 31);
                if (n + all > p.rank_cap) { crowd = true; break; }
                const int at = n + upto - size;
                if (size == 1) sh.list[at] = c * 32 + best;
                for (unsigned big = __ballot_sync(0xffffffffu, size > 1); big != 0; big &= big - 1) {
                    const int src = __ffs(big) - 1;
                    const int bc_ = __shfl_sync(0xffffffffu, c, src), ba = __shfl_sync(0xffffffffu, at, src),
                              bs = __shfl_sync(0xffffffffu, size, src);
                    if (lane < bs) sh.list[ba + lane] = bc_ * 32 + lane;
                }
                n += all;
            }
        }
        if (lane == 0) { sh.count[1] = crowd ? -1 : n; sh.count[2] = 0; }
    }
}

// (d) for all rows of a block: warp `bw` of the block takes every eighth group of four columns, of all columns in fp32 or
// of those marked in sh.again in fp64.
template <int G, typename T, typename A>
__device__ __forceinline__ void rows_top_score(const VocabRows& p, uint8_t* top_base, int stride, int bw, int lane) {
    constexpr int R = VOCAB_THREADS / G, WARPS = VOCAB_THREADS / 32;
    constexpr bool AGAIN = sizeof(A) == 8;
    int turn = 0;
#pragma unroll 1
    for (int r = 0; r < R; ++r) {
        const RowTopShared sh = row_top_shared(top_base + (size_t)r * stride, p.rank_cap);
        const int n = AGAIN ? sh.count[2] : sh.count[1];
        const T* x = reinterpret_cast<const T*>(p.x) + ((long long)blockIdx.x * R + r) * p.ldx;
        const T* y = reinterpret_cast<const T*>(p.y);
#pragma unroll 1
        for (int i = 0; i < n; i += 4, ++turn) {
            if (turn % WARPS != bw) continue;
            int at[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) at[q] = AGAIN ? sh.again[min(i + q, n - 1)] : min(i + q, n - 1);
            const T* const r4[4] = {y + (long long)sh.list[at[0]] * p.ldy, y + (long long)sh.list[at[1]] * p.ldy,
                                    y + (long long)sh.list[at[2]] * p.ldy, y + (long long)sh.list[at[3]] * p.ldy};
            A z[4];
            warp_dot4<T, A>(x, r4, p.d, lane, z);
            if (lane < 4) sh.z[lane == 0 ? at[0] : lane == 1 ? at[1] : lane == 2 ? at[2] : at[3]] =
                (double)(lane == 0 ? z[0] : lane == 1 ? z[1] : lane == 2 ? z[2] : z[3]);
        }
    }
}

// Between (d) and (e), by one warp: of many columns those stay that reach the K-th largest of the lanes' two best, less what is
// unclear; K and a few.
__device__ __forceinline__ void row_top_prune(const RowTopShared& sh, int K, double unclear, int lane) {
    const int n = sh.count[1];
    if (n <= 64) return;
    float b1 = -INFINITY, b2 = -INFINITY, best;
    for (int i = lane; i < n; i += 32) {
        const float v = (float)sh.z[i];            // fp32 scores: exact
        b2 = fmaxf(b2, fminf(b1, v));
        b1 = fmaxf(b1, v);
    }
    const double bound = (double)warp_kth(b1, b2, K, lane, best) - unclear;
    int kept = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int i = i0 + lane;
        const double z = i < n ? sh.z[i] : 0.0;
        const int j = i < n ? sh.list[i] : 0;
        const bool keep = i < n && z >= bound;
        const unsigned who = __ballot_sync(0xffffffffu, keep);       // (all have read before one writes)
        const int at = kept + __popc(who & ((1u << lane) - 1u));
        if (keep) { sh.z[at] = z; sh.list[at] = j; }
        kept += __popc(who);
        __syncwarp();
    }
    if (lane == 0) sh.count[1] = kept;
}

// (e) of column i among the n of its row: how many come before it, and whether another one is closer than `unclear`.
__device__ __forceinline__ int row_top_rank(const RowTopShared& sh, int n, int i, double unclear, bool& near) {
    const double z = sh.z[i];
    const int j = sh.list[i];
    int before = 0;
    near = false;
#pragma unroll 8
    for (int o = 0; o < n; ++o) {
        const double zo = sh.z[o];
        before += comes_first(zo, sh.list[o], z, j) ? 1 : 0;
        near |= o != i && fabs(zo - z) <= unclear;
    }
    return before;
}

// loss = sum of the rows' losses, divided by the number of rows that have one when `mean`; inv_count gets the factor.
// By the block that is done last, in a fixed order over the rows.  No row at all: loss 0, factor 0.
__device__ __forceinline__ void distill_reduce(const VocabRows& p) {
    __shared__ double part[VOCAB_THREADS], cnt[VOCAB_THREADS];
    __shared__ bool last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(p.blocks_done, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    double a = 0.0, c = 0.0;
#pragma unroll 8
    for (long long i = threadIdx.x; i < p.all_rows; i += VOCAB_THREADS) {
        a += (double)__ldcg(p.all_loss + i);           // other blocks wrote these: not from this SM's L1
        c += (double)__ldcg(p.all_has + i);
    }
    part[threadIdx.x] = a;
    cnt[threadIdx.x] = c;
    __syncthreads();
    for (int s = VOCAB_THREADS / 2; s >= 1; s >>= 1) {
        if ((int)threadIdx.x < s) { part[threadIdx.x] += part[threadIdx.x + s]; cnt[threadIdx.x] += cnt[threadIdx.x + s]; }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double f = p.mean ? (cnt[0] > 0.0 ? 1.0 / cnt[0] : 0.0) : 1.0;
        *p.loss = (float)(part[0] * f);
        *p.inv_count = (float)f;
    }
}

// One row per G threads.  Bound by memory latency: a row reads its 2 V / 256 partial sums, V / 32 chunk maxima (with
// alternatives) and one table row per entry; many rows in flight per SM hide that (G = 32), and a few rows are spread
// over a block each (G = 256).  4096 x 32768 x 1024: 14 us, with alternatives 49 (K = 8, 90 MB from DRAM) and 107 to 150 us
// (K = 32); one row 8 and 15 us; events included.
template <int G, typename T, bool DISTILL, bool TOP>
__global__ void __launch_bounds__(VOCAB_THREADS, 4)
vocab_rows_kernel(const __grid_constant__ VocabRows p) {
    extern __shared__ __align__(16) uint8_t smem_all[];
    constexpr int W = G / 32;
    const int gt = (int)threadIdx.x % G, lane = gt & 31, w = gt >> 5;
    const long long row = (long long)blockIdx.x * (VOCAB_THREADS / G) + threadIdx.x / G;
    const bool active = row < p.rows;             // the same for the row's threads
    if (!TOP && !DISTILL && !active) return;      // (a block of G = 256 has one row, warps of G = 32 do not meet)
    uint8_t* smem = smem_all + (size_t)(threadIdx.x / G) * vocab_row_smem(p.k, p.top_k, p.rank_cap);
    float* red = reinterpret_cast<float*>(smem);
    float* z_of = reinterpret_cast<float*>(smem + 64 * 8);
    uint8_t* top_smem = smem + 64 * 8 + (p.k * 4 + 15) / 16 * 16;

    // (1) the row's statistics
    float m = STATS_EMPTY, r = -1.f, t = 0.f, log2l = 0.f;
    if (active) {
        const float4* st = p.stats + row * p.stats_ld;
        for (int i = gt; i < p.slots; i += G) {
            const float4 v = st[i];
            stats_join(m, r, t, v.x, v.y, v.z, p.unit);
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), r2 = __shfl_xor_sync(0xffffffffu, r, o),
                        t2 = __shfl_xor_sync(0xffffffffu, t, o);
            stats_join(m, r, t, m2, r2, t2, p.unit);
        }
        if (W > 1) {
            if (lane == 0) { red[w * 4] = m; red[w * 4 + 1] = r; red[w * 4 + 2] = t; }
            __syncthreads();
            m = red[0]; r = red[1]; t = red[2];
            for (int i = 1; i < W; ++i) stats_join(m, r, t, red[i * 4], red[i * 4 + 1], red[i * 4 + 2], p.unit);
            __syncthreads();
        }
        log2l = log1pf(r) * 1.4426950408889634f;
        if (gt == 0) {
            if (p.row_lse != nullptr) p.row_lse[row] = m * p.unit + log2l;
            if (p.entropy != nullptr) p.entropy[row] = 0.6931471805599453f * (log2l - t / (1.f + r));
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
            if (any) warp_dot4<T, float>(x, rr, p.d, lane, z);
            if (lane < 4 && e + lane < p.k) {
                const float zz = lane == 0 ? z[0] : lane == 1 ? z[1] : lane == 2 ? z[2] : z[3];
                z_of[e + lane] = zz;
            }
        }
        group_sync<G>();

        // (3) what is made of them
        if (!DISTILL) {
            for (int e = gt; e < p.k; e += G) {
                const long long j = tok[e];
                // a token below 0 is padding: 0; one behind the table is a mistake that shows
                const double lp2 = vocab_lp2(p, (double)z_of[e], m, r, log2l);
                p.log_probs[row * p.k + e] = j < 0 ? 0.f : j >= p.vocab ? NAN : (float)(lp2 * 0.6931471805599453);
                if (p.token_lp2 != nullptr) p.token_lp2[row * p.k + e] = (float)lp2;
            }
        } else {
            // q = softmax of the teacher's logits over the entries that are there; KL = sum q (log q - log p)
            auto logit = [&](int e) -> float {
                const long long at = row * p.k + e;
                return p.teacher_dtype == 1 ? reinterpret_cast<const float*>(p.teacher_logits)[at]
                       : p.teacher_dtype == 0 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.teacher_logits)[at])
                                              : __half2float(reinterpret_cast<const __half*>(p.teacher_logits)[at]);
            };
            // differences are taken before the temperature divides them: the type's lowest value, which masks carry, stays
            // finite and so does a row of nothing else
            auto below = [&](int e, float most) -> float { return (logit(e) - most) * p.inv_teacher_t; };
            auto there = [&](int e) -> bool { return tok[e] >= 0 && !(logit(e) == -INFINITY); };
            float um = -INFINITY, seen = 0.f;
            for (int e = gt; e < p.k; e += G)
                if (there(e)) { um = fmaxf(um, logit(e)); seen = 1.f; }
            um = group_reduce<G, true>(um, red, gt);
            seen = group_reduce<G, true>(seen, red, gt);
            float sum = 0.f;
            for (int e = gt; e < p.k; e += G)
                if (there(e)) sum += expf(below(e, um));
            sum = group_reduce<G, false>(sum, red, gt);
            const float inv = 1.f / sum, log_sum = logf(sum);
            double kl = 0.0;
            for (int e = gt; e < p.k; e += G) {
                const long long at = row * p.k + e;
                float q = 0.f;
                // of every entry that names a row, also an impossible one: the backward stores a coefficient at each
                const double lp2 = vocab_lp2(p, (double)z_of[e], m, r, log2l);
                if (there(e)) {
                    const float u = below(e, um);
                    q = expf(u) * inv;
                    if (tok[e] >= p.vocab) q = NAN;
                    if (q != 0.f) kl += (double)q * ((double)u - (double)log_sum - lp2 * 0.6931471805599453);
                }
                p.teacher_probs[at] = q;
                p.token_lp2[at] = (float)lp2;
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
    }
    if (DISTILL && p.loss != nullptr) distill_reduce(p);
    if (TOP) {
        const RowTopShared sh = row_top_shared(top_smem, p.rank_cap);
        const int stride = vocab_row_smem(p.k, p.top_k, p.rank_cap), bw = threadIdx.x >> 5;
        uint8_t* top_base = smem_all + (top_smem - smem);
        group_sync<G>();
        if (active) row_top_select<G, T>(p, row, gt, sh, red);
        else if (gt == 0) sh.count[1] = sh.count[2] = 0;
        __syncthreads();
        rows_top_score<G, T, float>(p, top_base, stride, bw, lane);
        __syncthreads();
        // In fp32 an order counts only when it is clear: d / 64 products in a row and a tree of 6, each off by half an ulp
        // (2^-24) of at most |x| |y|, on both sides.
        const double unclear = active ? (double)(1.1920929e-7f * ((float)p.d * 0.015625f + 6.f) * red[3]) : 0.0;
        if (w == 0) row_top_prune(sh, p.top_k, unclear, lane);
        group_sync<G>();
        const int n = sh.count[1];
        for (int i0 = w * 32; i0 < n; i0 += G) {
            const int i = i0 + lane;
            bool near = false;
            if (i < n) row_top_rank(sh, n, i, unclear, near);
            const unsigned who = __ballot_sync(0xffffffffu, near);
            int at = 0;
            if (lane == 0 && who != 0) at = atomicAdd(sh.count + 2, __popc(who));
            at = __shfl_sync(0xffffffffu, at, 0);
            if (near) sh.again[at + __popc(who & ((1u << lane) - 1u))] = i;
        }
        __syncthreads();
        rows_top_score<G, T, double>(p, top_base, stride, bw, lane);
        __syncthreads();
        if (!active) return;
        if (n < 0) { row_top_crowd<G, T>(p, row, gt, sh, m, r, log2l, red); return; }
        for (int i = gt; i < n; i += G) {
            bool ignored;
            const int place = row_top_rank(sh, n, i, 0.0, ignored);
            if (place < p.top_k) row_top_write(p, row, place, sh.z[i], sh.list[i], m, r, log2l);
        }
        // only where a row's scores are not numbers are there fewer than K
        if (w == 0 && lane < p.top_k && lane >= n) { p.top_tokens[row * p.top_k + lane] = -1; p.top_log_probs[row * p.top_k + lane] = NAN; }
    }
}

// Row factors and, for rows of few entries, their coefficients, so that a tile pass loads two vectors per row; one warp per
// row.  With `scale` also the row's exponent (see OutScale), from a bound on its coefficients' magnitude, |a| + 0.5308 |b| +
// sum |terms| (p |log2 p| <= log2(e) / e).  Bound by latency: 7 us at 2047 rows.
__global__ void __launch_bounds__(ROW_KERNEL_THREADS)
vocab_prepare_kernel(const __grid_constant__ VocabCoef v, long long rows, float4* __restrict__ factors,
                     float4* __restrict__ entries, int scale) {
    const long long row = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= rows) return;
    float m, a, b = 0.f;
    if (v.distill) {
        a = v.row_has[row] > 0.f ? v.grad_out[v.grad_per_row ? row : 0] * (v.factor != nullptr ? __ldg(v.factor) : 1.f) * v.inv_t : 0.f;
        m = 2.f * fabsf(a);                                  // sum q <= 1
    } else {
        float g = 0.f, size = 0.f;
        if (v.grad_log_probs != nullptr)
            for (int e = lane; e < v.k; e += 32) {
                const long long j = v.tokens[row * v.k + e];
                if (j >= 0 && j < v.vocab) { const float x = v.grad_log_probs[row * v.k + e]; g += x; size += fabsf(x); }
            }
        g = warp_sum(g);
        size = warp_sum(size);
        const float h = v.grad_entropy != nullptr ? v.grad_entropy[row] : 0.f;
        a = -(g + (h != 0.f ? h * v.entropy[row] : 0.f)) * v.inv_t;      // h = 0 takes no part, whatever the entropy is
        b = -h * 0.6931471805599453f * v.inv_t;
        m = fabsf(a) + 0.5308f * fabsf(b) + size * v.inv_t;
    }
    if (lane == 0) {
        int e = 0;                               // also where the bound is no number: the row's coefficients are none either
        if (scale && m == 0.f) e = ROW_EMPTY;
        else if (scale && m < INFINITY) e = min(126, PANEL_TARGET + 127 - (int)(__float_as_uint(m) >> 23));   // (subnormal: 126)
        factors[row] = make_float4(v.row_lse[row], a, b, __int_as_float(e));
    }
    if (entries != nullptr && lane < VOCAB_TILE_ENTRIES) {
        float value = 0.f;
        int col = -1;
        if (lane < v.k) {
            const long long j = v.tokens[row * v.k + lane];
            if (j >= 0 && j < v.vocab && vocab_entry(v, row, lane, a, b, value)) col = (int)j;
        }
        reinterpret_cast<float2*>(entries + row)[lane] = make_float2(__int_as_float(col), value);
    }
}

__device__ __forceinline__ unsigned int max_bits8(const uint16_t* p, unsigned int best) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
    return __vmaxu2(best, __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
}

// Largest magnitude of a bf16 table, the integer maximum of bits without the sign (blockIdx.y + first = 0), and the heaviest
// row's part M of the table's gradient (1; see OutScale): maxima, so the order of the atomics does not matter.
// Bound by HBM; it and the transposition after it read the matrices from L2 the second time (34048 x 512: 15 us each).
__global__ void __launch_bounds__(256)
operand_max_kernel(const uint16_t* __restrict__ table, long long ldt, long long vocab, const uint16_t* __restrict__ x, long long ldx,
                   long long rows, int d, int first, int f16, const float4* __restrict__ factors, float* __restrict__ table_max,
                   unsigned int* __restrict__ total) {
    const int lane = threadIdx.x & 31;
    if (blockIdx.y + first == 1) {
        unsigned int most = 0;
        for (long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (long long)gridDim.x * 8) {
            unsigned int best = 0;
#pragma unroll 4
            for (int c = lane * 8; c < d; c += 256) best = max_bits8(x + r * ldx + c, best);
            const unsigned int top = __reduce_max_sync(0xffffffffu, max(best & 0xffffu, best >> 16));
            const int e = __float_as_int(__ldg(&factors[r].w));
            const float size = f16 ? __half2float(__ushort_as_half((unsigned short)top)) : __uint_as_float(top << 16);
            if (e != ROW_EMPTY && size > 0.f && size < INFINITY)
                most = max(most, (unsigned int)(PANEL_TARGET - e + max((int)(__float_as_uint(size) >> 23), 1) - 127) + TOTAL_BIAS);
        }
        if (lane == 0 && most != 0) atomicMax(total, most);
        return;
    }
    // rows that follow one another are one long row
    const long long per_row = ldt == d ? vocab * d / 8 : d / 8, lines = ldt == d ? 1 : vocab;
    const long long all = lines * per_row, step = (long long)gridDim.x * 256;
    unsigned int best = 0;
#pragma unroll 8
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += step)
        best = max_bits8(table + (lines == 1 ? i * 8 : i / per_row * ldt + i % per_row * 8), best);
    const unsigned int top = __reduce_max_sync(0xffffffffu, max(best & 0xffffu, best >> 16)) << 16;      // as fp32 bits
    if (lane == 0 && top != 0) atomicMax(reinterpret_cast<unsigned int*>(table_max), top);
}

// The two factors that row r of the features is multiplied by (one could leave fp32's range).
struct FeatureScale { float f, g; };
__device__ __forceinline__ FeatureScale feature_scale(const float4* factors, const unsigned int* total, long long r) {
    const int e = __float_as_int(__ldg(&factors[r].w));
    if (e == ROW_EMPTY) return FeatureScale{0.f, 0.f};       // its coefficients are zero: any finite number will do
    const int t = max(-200, min(200, total_exponent(total) - e));         // (below -200 all is zero in fp16, above all was zero)
    return FeatureScale{pow2(t >> 1), pow2(t - (t >> 1))};
}

// out[c][r] = in[r][c] scaled, as fp16: transpose_bf16_kernel (same tiles, same shared-memory layout) with a conversion.
// FEATURES: rows of features, each by its own factor; else a table, by one.  bf16's 8 bits fit fp16's 11; what is far below
// the largest magnitude loses bits (see OutScale).
template <typename T, bool FEATURES>
__global__ void __launch_bounds__(256)
transpose_scaled_f16_kernel(const T* __restrict__ in, long long ld_in, long long rows, int cols, const float* __restrict__ largest,
                            const float4* __restrict__ factors, const unsigned int* __restrict__ total,
                            __half* __restrict__ out, long long ld_out) {
    __shared__ __align__(16) uint32_t tile[64][32];
    const long long r0 = (long long)blockIdx.x * 64;
    const int c0 = blockIdx.y * 64;
    const int t = threadIdx.x;
    {
        const int k = t & 7, rp = t >> 3;
        const long long r = r0 + 2 * rp;
        const int c = c0 + 8 * k;
        float a[8] = {}, b[8] = {};
        FeatureScale sa = {1.f, 1.f}, sb = {1.f, 1.f};
        if (!FEATURES) sa.f = sb.f = pow2(pow2_exponent(largest, OPERAND_TARGET));
        if (c < cols) {
            if (r < rows) { load8(in + r * ld_in + c, a); if (FEATURES) sa = feature_scale(factors, total, r); }
            if (r + 1 < rows) { load8(in + (r + 1) * ld_in + c, b); if (FEATURES) sb = feature_scale(factors, total, r + 1); }
        }
        const int pw = rp ^ (k << 2);
#pragma unroll
        for (int m = 0; m < 8; ++m)
            tile[8 * k + m][pw] = FEATURES ? pack_f16x2(a[m] * sa.f * sa.g, b[m] * sb.f * sb.g) : pack_f16x2(a[m] * sa.f, b[m] * sb.f);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int oc = (t >> 3) + h * 32, g = t & 7;
        if (c0 + oc < cols && r0 + 8 * g < rows) {
            const uint4 v = *reinterpret_cast<const uint4*>(&tile[oc][4 * (g ^ ((oc >> 3) & 7))]);
            *reinterpret_cast<uint4*>(out + (long long)(c0 + oc) * ld_out + r0 + 8 * g) = v;
        }
    }
}

// The same without the transposition, for an fp16 problem whose contractions read the operands as they lie: [rows, d].
__global__ void __launch_bounds__(ROW_KERNEL_THREADS)
scale_features_f16_kernel(const __half* __restrict__ in, long long ld_in, long long rows, int d, const float4* __restrict__ factors,
                          const unsigned int* __restrict__ total, __half* __restrict__ out) {
    const long long row = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    if (row >= rows) return;
    const FeatureScale s = feature_scale(factors, total, row);
    for (int c = (threadIdx.x & 31) * 8; c < d; c += 256) {
        float v[8];
        load8(in + row * ld_in + c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * s.f * s.g;
        *reinterpret_cast<uint4*>(out + row * d + c) =
            make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
    }
}

// Puts the entries' own terms into a coefficient panel: formed in fp32 from the saved log probabilities and rounded once,
// over what the tile pass stored there.  One warp per row.
__global__ void __launch_bounds__(ROW_KERNEL_THREADS)
vocab_entries_kernel(const __grid_constant__ VocabCoef v, const float4* __restrict__ factors, long long r0, long long nr,
                     long long c0, long long nc, __nv_bfloat16* __restrict__ panel, long long rows_alloc, int lo_chunk,
                     int f16) {
    const long long i = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= nr) return;
    const float4 f = factors[r0 + i];
    const float g_scale = pow2(row_exponent(f.w));
    for (int e = lane; e < v.k; e += 32) {
        const long long j = v.tokens[(r0 + i) * v.k + e];
        if (j < c0 || j >= c0 + nc) continue;          // absent, outside the table or in another panel
        float value;
        if (!vocab_entry(v, r0 + i, e, f.y, f.z, value)) continue;
        const long long col = j - c0, at = ((col >> 6) * rows_alloc + i) * 64 + (col & 63);
        if (f16) {
            reinterpret_cast<__half*>(panel)[at] = __float2half_rn(value * g_scale);
            continue;
        }
        const __nv_bfloat16 hi = __float2bfloat16_rn(value);
        panel[at] = hi;
        if (lo_chunk > 0) panel[at + (long long)lo_chunk * rows_alloc * 64] = __float2bfloat16_rn(value - __bfloat162float(hi));
    }
}

static int launch_vocab_entries(const VocabGrad& g, long long r0, long long nr, long long c0, long long nc, __nv_bfloat16* panel,
                                long long rows_alloc, int lo_chunk, int f16, cudaStream_t s) {
    const VocabCoef& v = g.coef;
    if (v.k == 0 || g.row_entries != nullptr || (!v.distill && v.grad_log_probs == nullptr)) return MECLIP_OK;
    const int wpb = ROW_KERNEL_THREADS / 32;
    ScopedTiming timing(s, TAG_ROW, (double)nr * v.k * 18.0);
    vocab_entries_kernel<<<(unsigned)((nr + wpb - 1) / wpb), ROW_KERNEL_THREADS, 0, s>>>(
        v, g.row_factors, r0, nr, c0, nc, panel, rows_alloc, lo_chunk, f16);
    MECLIP_CUDA(cudaGetLastError());
    return MECLIP_OK;
}

}  // namespace meclip
