// Rows of a table looked up by token and scaled, and the table's gradient by sorted tokens (include/meclip.h).
//
//   out_i = s table[t_i]          dtable_v = s sum_{i: t_i = v} g_i
//
// Both move each byte once; the sum has to be the same from run to run, so there are no floating-point atomics: the
// positions are sorted by token (stable radix sort of (token, position) pairs), every row of the table then knows its
// run of positions and adds their gradients in ascending order.  Runs of common tokens are thousands of positions long:
// aligned chunks of 32, and of 1024, positions that lie inside one run are added up beforehand, each by its own warp,
// so that the longest row of the table adds at most 4 x 31 + n / 1024 vectors instead of n.
#pragma once
#include <cuda_fp16.h>

namespace meclip {

static constexpr int EMB_SORT_THREADS = 1024;
static constexpr int EMB_MAX_BITS = 10;              // bits per sorting pass: 1024 bins, one per thread
static constexpr int EMB_MAX_BLOCKS = 128;           // blocks of a sorting pass
static constexpr long long EMB_ONE_BLOCK = 4096;     // up to here one block does all passes in one launch
static constexpr int EMB_CHUNK = 32;                 // positions per first-level sum, first-level sums per second-level one

// Eight elements from column c on; vec: 16-byte accesses are possible and d is a multiple of 8.
template <typename T>
__device__ __forceinline__ void load8_any(const T* p, int c, int d, int vec, float (&v)[8]) {
    if (vec) { load8(p + c, v); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < d ? load1(p + c + i) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store8_any(T* p, int c, int d, int vec, const float (&v)[8]) {
    if (vec) { store8(p + c, v); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < d) store1(p + c + i, v[i]);
}

// One warp per looked-up row; a token below 0 gives zeros, one behind the table NaN.
template <typename T>
__global__ void __launch_bounds__(ROW_KERNEL_THREADS)
embed_kernel(const long long* __restrict__ tokens, long long n, const T* __restrict__ table, long long ldt, long long vocab,
             int d, float scale, int vec, T* __restrict__ out, long long ldo) {
    const long long i = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= n) return;
    const long long t = tokens[i];
    const bool in = t >= 0 && t < vocab;
    const T* src = table + (in ? t : 0) * ldt;
    T* dst = out + i * ldo;
    const float fill = t < 0 ? 0.f : NAN;
#pragma unroll 4
    for (int c = lane * 8; c < d; c += 256) {
        float v[8];
        if (in) load8_any(src, c, d, vec, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = in ? v[k] * scale : fill;
        store8_any(dst, c, d, vec, v);
    }
}

struct EmbSort {
    const long long* tokens;          // pass 0 reads these; a token outside the table becomes the key `vocab`
    const uint32_t *keys_in, *pos_in;
    uint32_t *keys_out, *pos_out;
    long long n, vocab, per_block;    // per_block: a multiple of EMB_SORT_THREADS
    int shift, bits, blocks;
    uint32_t* hist;                   // [1 << bits][blocks]
};

__device__ __forceinline__ uint32_t emb_key(const EmbSort& s, long long i) {
    if (s.tokens == nullptr) return s.keys_in[i];
    const long long t = s.tokens[i];
    return (uint32_t)(t >= 0 && t < s.vocab ? t : s.vocab);
}

// How often each digit occurs in the block's share.
__global__ void __launch_bounds__(EMB_SORT_THREADS) emb_hist_kernel(const __grid_constant__ EmbSort s) {
    __shared__ uint32_t h[1 << EMB_MAX_BITS];
    const int bins = 1 << s.bits;
    for (int b = threadIdx.x; b < bins; b += EMB_SORT_THREADS) h[b] = 0;
    __syncthreads();
    const long long first = blockIdx.x * s.per_block, last = min(s.n, first + s.per_block);
    for (long long i = first + threadIdx.x; i < last; i += EMB_SORT_THREADS)
        atomicAdd(&h[(emb_key(s, i) >> s.shift) & (bins - 1)], 1u);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += EMB_SORT_THREADS) s.hist[(long long)b * s.blocks + blockIdx.x] = h[b];
}

// Exclusive prefix sum over the block's 1024 threads.
__device__ __forceinline__ uint32_t emb_block_scan(uint32_t v, uint32_t* warp_sums) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == 31) warp_sums[w] = inc;
    __syncthreads();
    if (w == 0) {
        uint32_t t = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += u;
        }
        warp_sums[lane] = t;
    }
    __syncthreads();
    const uint32_t before = w > 0 ? warp_sums[w - 1] : 0u;
    __syncthreads();
    return before + inc - v;
}

// Stable scatter of the positions [first, last): offs[bin] is where the block's next key of that bin goes.  1024 keys
// at a time: equal digits find each other inside a warp (match), the warps' counts are added up per bin.
__device__ __forceinline__ void emb_scatter(const EmbSort& s, long long first, long long last, uint32_t* offs, uint16_t* cnt) {
    const int bins = 1 << s.bits, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (long long at = first; at < last; at += EMB_SORT_THREADS) {
        for (int b = lane; b < bins; b += 32) cnt[w * bins + b] = 0;
        __syncwarp();
        const long long i = at + threadIdx.x;
        const bool in = i < last;
        const uint32_t key = in ? emb_key(s, i) : 0u;
        const uint32_t pos = in ? (s.tokens != nullptr ? (uint32_t)i : s.pos_in[i]) : 0u;
        const uint32_t digit = in ? (key >> s.shift) & (bins - 1) : 0xffffffffu;
        const uint32_t same = __match_any_sync(0xffffffffu, digit);
        const int rank = __popc(same & ((1u << lane) - 1u));
        if (in && rank == 0) cnt[w * bins + digit] = (uint16_t)__popc(same);
        __syncthreads();
        uint32_t sum = 0;
        if ((int)threadIdx.x < bins) {
#pragma unroll 8
            for (int k = 0; k < EMB_SORT_THREADS / 32; ++k) {
                const uint32_t c = cnt[k * bins + threadIdx.x];
                cnt[k * bins + threadIdx.x] = (uint16_t)sum;
                sum += c;
            }
        }
        __syncthreads();
        if (in) {
            const uint32_t dst = offs[digit] + cnt[w * bins + digit] + rank;
            s.keys_out[dst] = key;
            s.pos_out[dst] = pos;
        }
        __syncthreads();
        if ((int)threadIdx.x < bins) offs[threadIdx.x] += sum;
        __syncthreads();
    }
}

// One pass: where each bin starts for this block (bins of lower digits everywhere, this bin in earlier blocks), scatter.
__global__ void __launch_bounds__(EMB_SORT_THREADS) emb_scatter_kernel(const __grid_constant__ EmbSort s) {
    extern __shared__ __align__(16) uint8_t emb_smem[];
    __shared__ uint32_t offs[1 << EMB_MAX_BITS];
    __shared__ uint32_t warp_sums[32];
    uint32_t total = 0, before = 0;
    if ((int)threadIdx.x < (1 << s.bits)) {
        const uint32_t* h = s.hist + (long long)threadIdx.x * s.blocks;
#pragma unroll 8
        for (int b = 0; b < s.blocks; ++b) {
            const uint32_t c = h[b];
            total += c;
            before += b < (int)blockIdx.x ? c : 0u;
        }
    }
    const uint32_t start = emb_block_scan(total, warp_sums);
    offs[threadIdx.x] = start + before;
    __syncthreads();
    const long long first = blockIdx.x * s.per_block;
    emb_scatter(s, first, min(s.n, first + s.per_block), offs, reinterpret_cast<uint16_t*>(emb_smem));
}

// All passes of a short list by one block (a launch each would cost more than the work).
__global__ void __launch_bounds__(EMB_SORT_THREADS)
emb_sort_small_kernel(EmbSort s, int passes, uint32_t* keys_a, uint32_t* pos_a, uint32_t* keys_b, uint32_t* pos_b) {
    extern __shared__ __align__(16) uint8_t emb_smem[];
    __shared__ uint32_t offs[1 << EMB_MAX_BITS];
    __shared__ uint32_t warp_sums[32];
    const int bins = 1 << s.bits;
    for (int p = 0; p < passes; ++p) {
        s.shift = p * s.bits;
        s.keys_out = (p & 1) ? keys_b : keys_a;
        s.pos_out = (p & 1) ? pos_b : pos_a;
        offs[threadIdx.x] = 0;
        __syncthreads();
        for (long long i = threadIdx.x; i < s.n; i += EMB_SORT_THREADS) atomicAdd(&offs[(emb_key(s, i) >> s.shift) & (bins - 1)], 1u);
        __syncthreads();
        const uint32_t start = emb_block_scan(offs[threadIdx.x], warp_sums);
        offs[threadIdx.x] = start;
        __syncthreads();
        emb_scatter(s, 0, s.n, offs, reinterpret_cast<uint16_t*>(emb_smem));
        s.tokens = nullptr;
        s.keys_in = s.keys_out;
        s.pos_in = s.pos_out;
    }
}

// start[v] = first sorted place whose key is >= v, for v = 0 .. vocab (start[vocab]: how many tokens are in the table).
__global__ void __launch_bounds__(256)
emb_start_kernel(const uint32_t* __restrict__ keys, long long n, long long vocab, uint32_t* __restrict__ start) {
    const long long v = (long long)blockIdx.x * 256 + threadIdx.x;
    if (v > vocab) return;
    long long lo = 0, hi = n;
    while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (keys[mid] < (uint32_t)v) lo = mid + 1;
        else hi = mid;
    }
    start[v] = (uint32_t)lo;
}

static constexpr int EMB_COLS = 4;                   // 256-column pieces a warp keeps in registers

// acc += the gradients at the sorted places [a, b)
template <typename T>
__device__ __forceinline__ void emb_add_places(const T* __restrict__ g, long long ldg, const uint32_t* __restrict__ pos,
                                               long long a, long long b, int c0, int d, int vec, int lane,
                                               float (&acc)[EMB_COLS][8]) {
    for (long long at = a; at < b; at += 32) {
        const int m = (int)min(32ll, b - at);
        const uint32_t mine = lane < m ? pos[at + lane] : 0u;
#pragma unroll 2
        for (int e = 0; e < m; ++e) {
            const T* row = g + (long long)__shfl_sync(0xffffffffu, mine, e) * ldg;
#pragma unroll
            for (int k = 0; k < EMB_COLS; ++k) {
                const int c = c0 + k * 256 + lane * 8;
                if (c < d) {
                    float v[8];
                    load8_any(row, c, d, vec, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[k][i] += v[i];
                }
            }
        }
    }
}
// acc += rows [a, b) of fp32 sums with a pitch of dp (a multiple of 8)
__device__ __forceinline__ void emb_add_sums(const float* __restrict__ sums, long long dp, long long a, long long b, int c0,
                                             int lane, float (&acc)[EMB_COLS][8]) {
#pragma unroll 2
    for (long long r = a; r < b; ++r) {
#pragma unroll
        for (int k = 0; k < EMB_COLS; ++k) {
            const int c = c0 + k * 256 + lane * 8;
            if (c < dp) {
                float v[8];
                load8(sums + r * dp + c, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[k][i] += v[i];
            }
        }
    }
}

// First and second level: chunk b of 32 (1024) sorted places, if all of them belong to one row of the table.
template <typename T, bool SECOND>
__global__ void __launch_bounds__(ROW_KERNEL_THREADS)
emb_chunk_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, const uint32_t* __restrict__ start,
                 long long vocab, const T* __restrict__ g, long long ldg, int d, int vec, const float* __restrict__ level1,
                 float* __restrict__ sums, long long dp, long long chunks) {
    const long long b = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (b >= chunks) return;
    const long long size = SECOND ? EMB_CHUNK * EMB_CHUNK : EMB_CHUNK;
    if ((b + 1) * size > (long long)start[vocab] || keys[b * size] != keys[(b + 1) * size - 1]) return;
    for (int c0 = 0; c0 < d; c0 += 256 * EMB_COLS) {
        float acc[EMB_COLS][8] = {};
        if (SECOND) emb_add_sums(level1, dp, b * EMB_CHUNK, (b + 1) * EMB_CHUNK, c0, lane, acc);
        else        emb_add_places<T>(g, ldg, pos, b * EMB_CHUNK, (b + 1) * EMB_CHUNK, c0, d, vec, lane, acc);
#pragma unroll
        for (int k = 0; k < EMB_COLS; ++k) {
            const int c = c0 + k * 256 + lane * 8;
            if (c < dp) store8(sums + b * dp + c, acc[k]);
        }
    }
}

// One warp per row of the table: its run of sorted places, whole chunks from the sums of the levels before; rows that
// no token names are written as zeros, so the gradient needs no clearing pass.
template <typename T>
__global__ void __launch_bounds__(ROW_KERNEL_THREADS)
emb_rows_kernel(const uint32_t* __restrict__ pos, const uint32_t* __restrict__ start, long long vocab,
                const T* __restrict__ g, long long ldg, int d, int vec, const float* __restrict__ level1,
                const float* __restrict__ level2, long long dp, float scale, int vec_out, T* __restrict__ out, long long ldo) {
    const long long v = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (v >= vocab) return;
    const long long a = start != nullptr ? start[v] : 0, b = start != nullptr ? start[v + 1] : 0;
    // whole chunks [f1, l1) and among them whole second-level ones [f2, l2)
    long long f1 = (a + EMB_CHUNK - 1) / EMB_CHUNK, l1 = b / EMB_CHUNK;
    const bool use1 = level1 != nullptr && l1 > f1;
    long long f2 = (f1 + EMB_CHUNK - 1) / EMB_CHUNK, l2 = l1 / EMB_CHUNK;
    const bool use2 = use1 && level2 != nullptr && l2 > f2;
    T* row = out + v * ldo;
    for (int c0 = 0; c0 < d; c0 += 256 * EMB_COLS) {
        float acc[EMB_COLS][8] = {};
        if (!use1) {
            emb_add_places<T>(g, ldg, pos, a, b, c0, d, vec, lane, acc);
        } else {
            emb_add_places<T>(g, ldg, pos, a, f1 * EMB_CHUNK, c0, d, vec, lane, acc);
            if (use2) {
                emb_add_sums(level1, dp, f1, f2 * EMB_CHUNK, c0, lane, acc);
                emb_add_sums(level2, dp, f2, l2, c0, lane, acc);
                emb_add_sums(level1, dp, l2 * EMB_CHUNK, l1, c0, lane, acc);
            } else {
                emb_add_sums(level1, dp, f1, l1, c0, lane, acc);
            }
            emb_add_places<T>(g, ldg, pos, l1 * EMB_CHUNK, b, c0, d, vec, lane, acc);
        }
#pragma unroll
        for (int k = 0; k < EMB_COLS; ++k) {
            const int c = c0 + k * 256 + lane * 8;
            if (c < d) {
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[k][i] *= scale;
                store8_any(row, c, d, vec_out, acc[k]);
            }
        }
    }
}

struct EmbPlan {
    int bits, passes, blocks;
    long long per_block, chunks1, chunks2, dp;
    size_t list_bytes, hist_bytes, start_bytes, level1_bytes, level2_bytes;
    size_t total() const { return 4 * list_bytes + hist_bytes + start_bytes + level1_bytes + level2_bytes; }
};
static EmbPlan plan_embed_grad(long long n, long long vocab, long long d) {
    EmbPlan p;
    int bits = 1;
    while (bits < 32 && (vocab >> bits) != 0) ++bits;            // keys are 0 .. vocab
    p.passes = (bits + EMB_MAX_BITS - 1) / EMB_MAX_BITS;
    p.bits = (bits + p.passes - 1) / p.passes;
    const long long rounds = (n + EMB_SORT_THREADS - 1) / EMB_SORT_THREADS;
    const long long per = (rounds + EMB_MAX_BLOCKS - 1) / EMB_MAX_BLOCKS;
    p.per_block = (per < 1 ? 1 : per) * EMB_SORT_THREADS;
    p.blocks = (int)((n + p.per_block - 1) / p.per_block);
    p.dp = (d + 7) / 8 * 8;
    // the levels only pay when a run can be longer than a warp adds in the time of another launch
    p.chunks1 = n >= 512 ? n / EMB_CHUNK : 0;
    p.chunks2 = n >= 8192 ? n / (EMB_CHUNK * EMB_CHUNK) : 0;
    p.list_bytes = round_up((size_t)n * 4, 256);
    p.hist_bytes = round_up((size_t)(p.blocks < 1 ? 1 : p.blocks) * 4 << p.bits, 256);
    p.start_bytes = round_up((size_t)(vocab + 1) * 4, 256);
    p.level1_bytes = round_up((size_t)p.chunks1 * p.dp * 4, 256);
    p.level2_bytes = round_up((size_t)p.chunks2 * p.dp * 4, 256);
    return p;
}

template <typename T>
static int embed_grad_t(const long long* tokens, long long n, const T* g, long long vocab, int d, long long ldg, float scale,
                        T* out, long long ldo, uint8_t* ws, const EmbPlan& pl, cudaStream_t s) {
    constexpr int elt = (int)sizeof(T), wpb = ROW_KERNEL_THREADS / 32;
    const int vec = d % 8 == 0 && aligned16(g) && (ldg * elt) % 16 == 0;
    const int vec_out = d % 8 == 0 && aligned16(out) && (ldo * elt) % 16 == 0;
    uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(ws), reinterpret_cast<uint32_t*>(ws + pl.list_bytes)};
    uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(ws + 2 * pl.list_bytes), reinterpret_cast<uint32_t*>(ws + 3 * pl.list_bytes)};
    uint32_t* hist = reinterpret_cast<uint32_t*>(ws + 4 * pl.list_bytes);
    uint32_t* start = reinterpret_cast<uint32_t*>(ws + 4 * pl.list_bytes + pl.hist_bytes);
    float* level1 = reinterpret_cast<float*>(ws + 4 * pl.list_bytes + pl.hist_bytes + pl.start_bytes);
    float* level2 = reinterpret_cast<float*>(ws + 4 * pl.list_bytes + pl.hist_bytes + pl.start_bytes + pl.level1_bytes);
    const unsigned row_grid = (unsigned)((vocab + wpb - 1) / wpb);
    if (n == 0) {
        ScopedTiming timing(s, TAG_ROW, (double)vocab * d * elt);
        emb_rows_kernel<T><<<row_grid, ROW_KERNEL_THREADS, 0, s>>>(nullptr, nullptr, vocab, g, ldg, d, 0, nullptr, nullptr,
                                                                  pl.dp, scale, vec_out, out, ldo);
        MECLIP_CUDA(cudaGetLastError());
        return MECLIP_OK;
    }
    EmbSort st{};
    st.tokens = tokens; st.n = n; st.vocab = vocab; st.per_block = pl.per_block; st.bits = pl.bits; st.blocks = pl.blocks;
    st.hist = hist;
    const int smem = (EMB_SORT_THREADS / 32) * 2 << pl.bits;
    if (n <= EMB_ONE_BLOCK) {
        MECLIP_CUDA(cudaFuncSetAttribute(emb_sort_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        ScopedTiming timing(s, TAG_ROW, 16.0 * (double)n * pl.passes);
        emb_sort_small_kernel<<<1, EMB_SORT_THREADS, smem, s>>>(st, pl.passes, keys[0], pos[0], keys[1], pos[1]);
        MECLIP_CUDA(cudaGetLastError());
    } else {
        MECLIP_CUDA(cudaFuncSetAttribute(emb_scatter_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        for (int p = 0; p < pl.passes; ++p) {
            st.shift = p * pl.bits;
            st.keys_out = keys[p & 1];
            st.pos_out = pos[p & 1];
            {
                ScopedTiming timing(s, TAG_ROW, (p == 0 ? 8.0 : 4.0) * (double)n);
                emb_hist_kernel<<<pl.blocks, EMB_SORT_THREADS, 0, s>>>(st);
            }
            {
                ScopedTiming timing(s, TAG_ROW, 16.0 * (double)n);
                emb_scatter_kernel<<<pl.blocks, EMB_SORT_THREADS, smem, s>>>(st);
            }
            MECLIP_CUDA(cudaGetLastError());
            st.tokens = nullptr;
            st.keys_in = st.keys_out;
            st.pos_in = st.pos_out;
        }
    }
    const uint32_t* ks = keys[(pl.passes - 1) & 1];
    const uint32_t* ps = pos[(pl.passes - 1) & 1];
    {
        ScopedTiming timing(s, TAG_ROW, 4.0 * (double)vocab);
        emb_start_kernel<<<(unsigned)((vocab + 256) / 256), 256, 0, s>>>(ks, n, vocab, start);
    }
    if (pl.chunks1 > 0) {
        ScopedTiming timing(s, TAG_ROW, 0.0);
        emb_chunk_kernel<T, false><<<(unsigned)((pl.chunks1 + wpb - 1) / wpb), ROW_KERNEL_THREADS, 0, s>>>(
            ks, ps, start, vocab, g, ldg, d, vec, nullptr, level1, pl.dp, pl.chunks1);
    }
    if (pl.chunks2 > 0) {
        ScopedTiming timing(s, TAG_ROW, 0.0);
        emb_chunk_kernel<T, true><<<(unsigned)((pl.chunks2 + wpb - 1) / wpb), ROW_KERNEL_THREADS, 0, s>>>(
            ks, ps, start, vocab, g, ldg, d, vec, level1, level2, pl.dp, pl.chunks2);
    }
    MECLIP_CUDA(cudaGetLastError());
    ScopedTiming timing(s, TAG_ROW, ((double)vocab + (double)n) * d * elt);
    emb_rows_kernel<T><<<row_grid, ROW_KERNEL_THREADS, 0, s>>>(ps, start, vocab, g, ldg, d, vec, pl.chunks1 > 0 ? level1 : nullptr,
                                                              pl.chunks2 > 0 ? level2 : nullptr, pl.dp, scale, vec_out, out, ldo);
    MECLIP_CUDA(cudaGetLastError());
    return MECLIP_OK;
}

static int check_embed(const char* what, const void* tokens, int64_t n, const void* a, int dtype, int64_t vocab, int64_t d,
                       int64_t lda, const void* b, int64_t ldb) {
    if ((tokens == nullptr && n > 0) || (a == nullptr && n > 0) || b == nullptr) return fail(MECLIP_EINVAL, "%s: null pointer", what);
    if (dtype != MECLIP_BF16 && dtype != MECLIP_F32 && dtype != MECLIP_F16) return fail(MECLIP_EINVAL, "%s: bad dtype %d", what, dtype);
    if (n < 0 || n > 0x7fffffffLL || vocab < 1 || vocab > 0x7fffffffLL || d < 1 || d > 0x7fffffffLL - 1024 || lda < d || ldb < d)
        return fail(MECLIP_EINVAL, "%s: need 0 <= n < 2^31, vocab and d in [1, 2^31), pitches >= d", what);
    return MECLIP_OK;
}

}  // namespace meclip

extern "C" {

int meclip_embed(const int64_t* tokens, int64_t n, const void* table, int dtype, int64_t vocab, int64_t d, int64_t ldt,
                 float scale, void* out, int64_t ldo, void* stream) {
    NvtxRange range("meclip_embed");
    if (n == 0) return MECLIP_OK;
    int rc = check_embed("embed", tokens, n, table, dtype, vocab, d, ldt, out, ldo);
    if (rc) return rc;
    rc = check_device();
    if (rc) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    const int elt = dtype == MECLIP_F32 ? 4 : 2, wpb = ROW_KERNEL_THREADS / 32;
    const int vec = d % 8 == 0 && aligned16(table) && aligned16(out) && (ldt * elt) % 16 == 0 && (ldo * elt) % 16 == 0;
    const unsigned grid = (unsigned)((n + wpb - 1) / wpb);
    const long long* t = reinterpret_cast<const long long*>(tokens);
    ScopedTiming timing(s, TAG_ROW, (double)n * (8.0 + 2.0 * d * elt));
    if (dtype == MECLIP_F32)
        embed_kernel<float><<<grid, ROW_KERNEL_THREADS, 0, s>>>(t, n, (const float*)table, ldt, vocab, (int)d, scale, vec, (float*)out, ldo);
    else if (dtype == MECLIP_BF16)
        embed_kernel<__nv_bfloat16><<<grid, ROW_KERNEL_THREADS, 0, s>>>(t, n, (const __nv_bfloat16*)table, ldt, vocab, (int)d, scale, vec, (__nv_bfloat16*)out, ldo);
    else
        embed_kernel<__half><<<grid, ROW_KERNEL_THREADS, 0, s>>>(t, n, (const __half*)table, ldt, vocab, (int)d, scale, vec, (__half*)out, ldo);
    MECLIP_CUDA(cudaGetLastError());
    return MECLIP_OK;
}

size_t meclip_embed_grad_workspace_bytes(int64_t n, int64_t vocab, int64_t d) {
    if (n < 0 || vocab < 1 || d < 1) return 0;
    return plan_embed_grad(n, vocab, d).total();
}

int meclip_embed_grad(const int64_t* tokens, int64_t n, const void* grad, int dtype, int64_t vocab, int64_t d, int64_t ldg,
                      float scale, void* dtable, int64_t ldd, void* workspace, size_t workspace_bytes, void* stream) {
    NvtxRange range("meclip_embed_grad");
    int rc = check_embed("embed_grad", tokens, n, grad, dtype, vocab, d, ldg, dtable, ldd);
    if (rc) return rc;
    const EmbPlan pl = plan_embed_grad(n, vocab, d);
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return fail(MECLIP_EINVAL, "embed_grad: workspace must be 256-byte aligned");
    if (workspace_bytes < pl.total()) return fail(MECLIP_ENOSPC, "embed_grad: workspace %zu < %zu bytes", workspace_bytes, pl.total());
    rc = check_device();
    if (rc) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    const long long* t = reinterpret_cast<const long long*>(tokens);
    uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
    if (dtype == MECLIP_F32) return embed_grad_t<float>(t, n, (const float*)grad, vocab, (int)d, ldg, scale, (float*)dtable, ldd, ws, pl, s);
    if (dtype == MECLIP_BF16) return embed_grad_t<__nv_bfloat16>(t, n, (const __nv_bfloat16*)grad, vocab, (int)d, ldg, scale, (__nv_bfloat16*)dtable, ldd, ws, pl, s);
    return embed_grad_t<__half>(t, n, (const __half*)grad, vocab, (int)d, ldg, scale, (__half*)dtable, ldd, ws, pl, s);
}

}  // extern "C"
