// Rows of a table looked up by token and scaled, and the table's gradient by sorted tokens (include/meclip.h).
//
//   out_i = s table[t_i]          dtable_v = s sum_{i: t_i = v} g_i
//
// Both move each byte once; the sum has to be the same from run to run, so there are no floating-point atomics: the
// positions are sorted by token (stable radix sort of (token, position) pairs) and added in ascending order.
//   sort     few blocks, bound by latency; further blocks of the same launches clear the table's gradient meanwhile
//   chunks   one warp per 32 sorted places and 256 columns adds what it finds; a run of one token that lies inside the
//            chunk is a finished row, a run that goes on leaves a partial sum: in `head` if it fills the chunk from its
//            first place on, in `tail` otherwise.  Every warp has the same work, however common a token is.
//   level 2  32 chunks that lie inside one run, added up (the run of a common token is thousands of places long)
//   join     runs over several chunks: tail + heads, whole level-2 sums in place of 32 heads
#pragma once
#include <cuda_fp16.h>

namespace meclip {

static constexpr int EMB_SORT_THREADS = 1024;
static constexpr int EMB_MAX_BITS = 10;              // bits per sorting pass: 1024 bins, one per thread
static constexpr int EMB_MAX_BLOCKS = 128;           // blocks of a sorting pass
static constexpr long long EMB_ONE_BLOCK = 4096;     // up to here one block does all passes in one launch
static constexpr int EMB_CHUNK = 32;                 // places per chunk, chunks per second-level sum

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

// One warp per looked-up row; a token below 0 gives zeros, one behind the table NaN.  Bound by HBM: 131072 x 1152 bf16 from
// a table of 49999 rows 59 us (302 MB written, the table read once and further on from L2).
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
    uint32_t* hist;                   // [blocks][1 << bits]
    // the gradient's rows, cleared by the blocks behind `blocks`: part `part` of `parts` of them per launch
    void* out;
    long long ldo;
    int d, elt, flat, part, parts;
};

// flat: the rows follow one another and start on 16 bytes, as one run of vocab * d * elt bytes (a multiple of 16)
__device__ __forceinline__ void emb_clear(const EmbSort& s) {
    const long long who = (long long)(blockIdx.x - s.blocks) * EMB_SORT_THREADS + threadIdx.x;
    const long long step = (long long)(gridDim.x - s.blocks) * EMB_SORT_THREADS;
    const long long all = s.flat ? s.vocab * s.d * s.elt / 16 : s.vocab * s.d;
    const long long first = all * s.part / s.parts, last = all * (s.part + 1) / s.parts;
    if (s.flat) {
        uint4* o = reinterpret_cast<uint4*>(s.out);
        for (long long i = first + who; i < last; i += step) o[i] = make_uint4(0, 0, 0, 0);
    } else {
        for (long long i = first + who; i < last; i += step) {
            const long long at = i / s.d * s.ldo + i % s.d;
            if (s.elt == 4) reinterpret_cast<uint32_t*>(s.out)[at] = 0;
            else            reinterpret_cast<uint16_t*>(s.out)[at] = 0;
        }
    }
}

__device__ __forceinline__ uint32_t emb_key(const EmbSort& s, long long i) {
    if (s.tokens == nullptr) return s.keys_in[i];
    const long long t = s.tokens[i];
    return (uint32_t)(t >= 0 && t < s.vocab ? t : s.vocab);
}

// How often each digit occurs in the block's share.  131072 keys and a quarter of a 115 MB gradient to clear: 11 us, the
// scatter 12.5; the clearing is what takes the time.
__global__ void __launch_bounds__(EMB_SORT_THREADS) emb_hist_kernel(const __grid_constant__ EmbSort s) {
    __shared__ uint32_t h[1 << EMB_MAX_BITS];
    if ((int)blockIdx.x >= s.blocks) { emb_clear(s); return; }
    const int bins = 1 << s.bits;
    for (int b = threadIdx.x; b < bins; b += EMB_SORT_THREADS) h[b] = 0;
    __syncthreads();
    const long long first = blockIdx.x * s.per_block, last = min(s.n, first + s.per_block);
    for (long long i = first + threadIdx.x; i < last; i += EMB_SORT_THREADS)
        atomicAdd(&h[(emb_key(s, i) >> s.shift) & (bins - 1)], 1u);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += EMB_SORT_THREADS) s.hist[((long long)blockIdx.x << s.bits) + b] = h[b];
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
    if ((int)blockIdx.x >= s.blocks) { emb_clear(s); return; }
    // a bin's counts, one per block, are read by 1024 >> bits threads: the reads are a chain of L2 latencies otherwise
    __shared__ uint32_t total[1 << EMB_MAX_BITS], before[1 << EMB_MAX_BITS];
    total[threadIdx.x] = 0;
    before[threadIdx.x] = 0;
    __syncthreads();
    {
        const int bin = threadIdx.x & ((1 << s.bits) - 1), part = threadIdx.x >> s.bits, parts = EMB_SORT_THREADS >> s.bits;
        uint32_t t = 0, u = 0;
#pragma unroll 16
        for (int b = part; b < s.blocks; b += parts) {
            const uint32_t c = s.hist[((long long)b << s.bits) + bin];
            t += c;
            u += b < (int)blockIdx.x ? c : 0u;
        }
        if (t != 0) atomicAdd(&total[bin], t);
        if (u != 0) atomicAdd(&before[bin], u);
    }
    __syncthreads();
    const uint32_t start = emb_block_scan(total[threadIdx.x], warp_sums);
    offs[threadIdx.x] = start + before[threadIdx.x];
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
    if (blockIdx.x > 0) { emb_clear(s); return; }            // s.blocks is 1 here
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

// A warp works on 256 columns, eight per lane, and keeps several rows' loads in flight: the sums are bound by memory
// latency unless enough of it overlaps (131072 x 1152 bf16, a fifth of it padding: 242 MB in 50 us, 64 % of the DRAM
// rate).
static constexpr int EMB_COLS = 256;

// Eight elements of a row as loaded, widened when they are added.
template <typename T, bool VEC> struct EmbRaw;
template <typename T> struct EmbRaw<T, true> {
    static constexpr int U = sizeof(T) == 4 ? 4 : 8;
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p, int, int) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void add(float (&acc)[8]) const {
        float v[8];
        load8(reinterpret_cast<const T*>(w), v);
#pragma unroll
        for (int i = 0; i < 8; i += 2) f32x2_split(add_f32x2(f32x2(acc[i], acc[i + 1]), f32x2(v[i], v[i + 1])), acc[i], acc[i + 1]);
    }
};
template <typename T> struct EmbRaw<T, false> {
    static constexpr int U = 4;
    T w[8];
    __device__ __forceinline__ void load(const T* p, int c, int d) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < d) w[i] = p[i];
    }
    __device__ __forceinline__ void add(float (&acc)[8]) const {     // columns past d hold anything and are not stored
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += load1(&w[i]);
    }
};

template <typename T>
__device__ __forceinline__ void emb_finish(float (&acc)[8], float scale, T* out, long long ldo, long long v, int c, int d, int vec_out) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= scale;
    store8_any(out + v * ldo, c, d, vec_out, acc);
}

struct EmbLevels { float *head, *tail, *level2; long long dp; };     // dp: pitch of the sums, a multiple of 8

template <typename T, bool VEC>
__global__ void __launch_bounds__(ROW_KERNEL_THREADS, 3)
emb_chunk_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, long long n, long long vocab,
                 const T* __restrict__ g, long long ldg, int d, EmbLevels lv, float scale, int vec_out, T* __restrict__ out,
                 long long ldo, long long chunks, int pieces) {
    constexpr int U = EmbRaw<T, VEC>::U;
    const long long unit = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    const long long b = unit / pieces;
    const int lane = threadIdx.x & 31, c = (int)(unit % pieces) * EMB_COLS + lane * 8;
    if (b >= chunks) return;
    const long long first = b * EMB_CHUNK;
    const int m = (int)min((long long)EMB_CHUNK, n - first);
    const uint32_t none = 0xffffffffu;                               // no key: keys are at most vocab < 2^31
    const uint32_t key = lane < m ? keys[first + lane] : none;
    const uint32_t mine = lane < m ? pos[first + lane] : 0u;
    const uint32_t before = first > 0 ? keys[first - 1] : none;
    const uint32_t after = first + m < n ? keys[first + m] : none;
    // places where another run begins, and how many places hold tokens of the table (padding sorts last)
    const uint32_t prev = __shfl_up_sync(0xffffffffu, key, 1);
    const uint32_t begins = __ballot_sync(0xffffffffu, lane > 0 && key != prev);
    const int valid = __popc(__ballot_sync(0xffffffffu, (long long)key < vocab));
    if (valid == 0) return;
    const bool here = c < d;
    bool from_start = true;                                          // the current run began at the chunk's first place
    float acc[8] = {};
    auto hand_in = [&](int e) {                                      // the run that ends before place e
        const uint32_t cur = __shfl_sync(0xffffffffu, key, e - 1);
        const bool goes_on = e == m && after == cur, came_in = from_start && before == cur;
        if (goes_on || came_in) {
            if (c < lv.dp) store8((from_start ? lv.head : lv.tail) + b * lv.dp + c, acc);
        } else if (here) {
            emb_finish(acc, scale, out, ldo, cur, c, d, vec_out);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.f;
        from_start = false;
    };
#pragma unroll 1
    for (int e0 = 0; e0 < valid; e0 += U) {
        EmbRaw<T, VEC> raw[U];
        const int live = min(U, valid - e0);
#pragma unroll
        for (int r = 0; r < U; ++r) {
            const long long row = __shfl_sync(0xffffffffu, mine, (e0 + r) & 31);
            if (r < live && here) raw[r].load(g + row * ldg + c, c, d);
        }
        const uint32_t marks = (begins >> e0) & ((1u << U) - 1u);    // the same for the whole warp
        if (marks == 0 && live == U) {
#pragma unroll
            for (int r = 0; r < U; ++r) raw[r].add(acc);
        } else {
#pragma unroll
            for (int r = 0; r < U; ++r) {
                if (r >= live) break;
                if ((marks >> r) & 1u) hand_in(e0 + r);
                raw[r].add(acc);
            }
        }
    }
    hand_in(valid);
}

// acc += rows [a, b) of fp32 sums
__device__ __forceinline__ void emb_add_sums(const float* __restrict__ sums, long long dp, long long a, long long b, int c,
                                             float (&acc)[8]) {
    constexpr int U = 8;
    if (c >= dp) return;
    for (long long r0 = a; r0 < b; r0 += U) {
        float v[U][8];
#pragma unroll
        for (int r = 0; r < U; ++r) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[r][i] = 0.f;
            if (r0 + r < b) load8(sums + (r0 + r) * dp + c, v[r]);
        }
#pragma unroll
        for (int r = 0; r < U; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] += v[r][i];
    }
}

__global__ void __launch_bounds__(ROW_KERNEL_THREADS)
emb_level2_kernel(const uint32_t* __restrict__ keys, long long vocab, EmbLevels lv, long long groups, int pieces) {
    const long long unit = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    const long long b = unit / pieces;
    const int lane = threadIdx.x & 31, c = (int)(unit % pieces) * EMB_COLS + lane * 8;
    if (b >= groups) return;
    const long long size = EMB_CHUNK * EMB_CHUNK;
    const uint32_t k = keys[b * size];
    if ((long long)k >= vocab || k != keys[(b + 1) * size - 1]) return;
    float acc[8] = {};
    emb_add_sums(lv.head, lv.dp, b * EMB_CHUNK, (b + 1) * EMB_CHUNK, c, acc);
    if (c < lv.dp) store8(lv.level2 + b * lv.dp + c, acc);
}

// One warp per chunk and 256 columns: the run that starts in it and goes on behind it.  Bound by latency: the longest run
// is a chain of loads (131072 tokens, the common ones thousands of times as frequent as the rare: 26 us, level 2 13 us).
template <typename T>
__global__ void __launch_bounds__(ROW_KERNEL_THREADS)
emb_join_kernel(const uint32_t* __restrict__ keys, long long n, long long vocab, int d, EmbLevels lv, float scale, int vec_out,
                T* __restrict__ out, long long ldo, long long chunks, int pieces) {
    const long long unit = (long long)blockIdx.x * (ROW_KERNEL_THREADS / 32) + (threadIdx.x >> 5);
    const long long b = unit / pieces;
    const int lane = threadIdx.x & 31, c = (int)(unit % pieces) * EMB_COLS + lane * 8;
    if (b + 1 >= chunks) return;
    const long long first = b * EMB_CHUNK, next = first + EMB_CHUNK;
    const uint32_t k = keys[next - 1];
    if ((long long)k >= vocab || keys[next] != k) return;
    const bool from_start = keys[first] == k;
    if (from_start && first > 0 && keys[first - 1] == k) return;     // it started earlier
    long long lo = next, hi = n;                                     // where the run ends: 32 probes at a time
    while (lo < hi) {
        const long long step = (hi - lo + 31) / 32, at = lo + lane * step;
        const uint32_t in_run = __ballot_sync(0xffffffffu, at < hi && keys[min(at, hi - 1)] <= k);
        if (in_run == 0) { hi = lo; break; }
        const long long last = lo + (31 - __clz(in_run)) * step;     // the last probe inside the run
        hi = min(hi, last + step);
        lo = last + 1;
    }
    const long long h0 = from_start ? b : b + 1, h1 = (lo + EMB_CHUNK - 1) / EMB_CHUNK;      // heads [h0, h1)
    // whole groups of 32 full chunks: [g0, g1) lies inside the run
    const long long g0 = (h0 + EMB_CHUNK - 1) / EMB_CHUNK, g1 = lo / (EMB_CHUNK * EMB_CHUNK);
    float acc[8] = {};
    if (!from_start) emb_add_sums(lv.tail, lv.dp, b, b + 1, c, acc);
    if (lv.level2 != nullptr && g1 > g0) {
        emb_add_sums(lv.head, lv.dp, h0, g0 * EMB_CHUNK, c, acc);
        emb_add_sums(lv.level2, lv.dp, g0, g1, c, acc);
        emb_add_sums(lv.head, lv.dp, g1 * EMB_CHUNK, h1, c, acc);
    } else {
        emb_add_sums(lv.head, lv.dp, h0, h1, c, acc);
    }
    if (c < d) emb_finish(acc, scale, out, ldo, k, c, d, vec_out);
}

struct EmbPlan {
    int bits, passes, blocks;
    long long per_block, chunks, groups, dp;
    size_t list_bytes, hist_bytes, chunk_bytes, group_bytes;
    size_t total() const { return 4 * list_bytes + hist_bytes + 2 * chunk_bytes + group_bytes; }
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
    p.chunks = (n + EMB_CHUNK - 1) / EMB_CHUNK;
    // a warp adds 64 heads in about the time that another launch takes
    p.groups = n >= 2 * EMB_CHUNK * EMB_CHUNK ? n / (EMB_CHUNK * EMB_CHUNK) : 0;
    p.list_bytes = round_up((size_t)n * 4, 256);
    p.hist_bytes = round_up((size_t)(p.blocks < 1 ? 1 : p.blocks) * 4 << p.bits, 256);
    p.chunk_bytes = round_up((size_t)p.chunks * p.dp * 4, 256);
    p.group_bytes = round_up((size_t)p.groups * p.dp * 4, 256);
    return p;
}

template <typename T>
static int embed_grad_t(const long long* tokens, long long n, const T* g, long long vocab, int d, long long ldg, float scale,
                        T* out, long long ldo, uint8_t* ws, const EmbPlan& pl, cudaStream_t s) {
    constexpr int elt = (int)sizeof(T), wpb = ROW_KERNEL_THREADS / 32;
    const int vec = d % 8 == 0 && aligned16(g) && (ldg * elt) % 16 == 0;
    const int vec_out = d % 8 == 0 && aligned16(out) && (ldo * elt) % 16 == 0;
    const int pieces = (d + EMB_COLS - 1) / EMB_COLS;
    if ((pl.chunks * pieces + wpb - 1) / wpb > 0x7fffffffLL) return fail(MECLIP_EINVAL, "embed_grad: too much for one launch");
    uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(ws), reinterpret_cast<uint32_t*>(ws + pl.list_bytes)};
    uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(ws + 2 * pl.list_bytes), reinterpret_cast<uint32_t*>(ws + 3 * pl.list_bytes)};
    uint8_t* rest = ws + 4 * pl.list_bytes;
    EmbLevels lv;
    lv.head = reinterpret_cast<float*>(rest + pl.hist_bytes);
    lv.tail = reinterpret_cast<float*>(rest + pl.hist_bytes + pl.chunk_bytes);
    lv.level2 = pl.groups > 0 ? reinterpret_cast<float*>(rest + pl.hist_bytes + 2 * pl.chunk_bytes) : nullptr;
    lv.dp = pl.dp;
    EmbSort st{};
    st.tokens = tokens; st.n = n; st.vocab = vocab; st.per_block = pl.per_block; st.bits = pl.bits; st.blocks = pl.blocks;
    st.hist = reinterpret_cast<uint32_t*>(rest);
    st.out = out; st.ldo = ldo; st.d = d; st.elt = elt;
    st.flat = ldo == d && aligned16(out) && ((size_t)vocab * d * elt) % 16 == 0;
    const int smem = (EMB_SORT_THREADS / 32) * 2 << pl.bits, most_smem = (EMB_SORT_THREADS / 32) * 2 << EMB_MAX_BITS;
    static std::atomic<unsigned long long> smem_small{0}, smem_scatter{0};
    const int clear_blocks = sm_count();       // beside the sort's blocks: two blocks of 1024 threads fit an SM
    if (n <= EMB_ONE_BLOCK) {
        st.blocks = 1;
        st.parts = 1;
        const int rc = allow_all_smem(emb_sort_small_kernel, smem_small, most_smem);
        if (rc) return rc;
        ScopedTiming timing(s, TAG_ROW, 16.0 * (double)n * pl.passes + (double)vocab * d * elt);
        emb_sort_small_kernel<<<1 + 2 * clear_blocks, EMB_SORT_THREADS, smem, s>>>(st, pl.passes, keys[0], pos[0], keys[1], pos[1]);
        MECLIP_CUDA(cudaGetLastError());
        if (n == 0) return MECLIP_OK;
    } else {
        const int rc = allow_all_smem(emb_scatter_kernel, smem_scatter, most_smem);
        if (rc) return rc;
        st.parts = 2 * pl.passes;
        const double clear_bytes = (double)vocab * d * elt / st.parts;
        for (int p = 0; p < pl.passes; ++p) {
            st.shift = p * pl.bits;
            st.keys_out = keys[p & 1];
            st.pos_out = pos[p & 1];
            st.part = 2 * p;
            {
                ScopedTiming timing(s, TAG_ROW, (p == 0 ? 8.0 : 4.0) * (double)n + clear_bytes);
                emb_hist_kernel<<<pl.blocks + clear_blocks, EMB_SORT_THREADS, 0, s>>>(st);
            }
            st.part = 2 * p + 1;
            {
                ScopedTiming timing(s, TAG_ROW, 16.0 * (double)n + clear_bytes);
                emb_scatter_kernel<<<pl.blocks + clear_blocks, EMB_SORT_THREADS, smem, s>>>(st);
            }
            MECLIP_CUDA(cudaGetLastError());
            st.tokens = nullptr;
            st.keys_in = st.keys_out;
            st.pos_in = st.pos_out;
        }
    }
    const uint32_t* ks = keys[(pl.passes - 1) & 1];
    const uint32_t* ps = pos[(pl.passes - 1) & 1];
    const unsigned grid = (unsigned)((pl.chunks * pieces + wpb - 1) / wpb);
    {
        ScopedTiming timing(s, TAG_ROW, (double)n * d * elt);
        if (vec) emb_chunk_kernel<T, true><<<grid, ROW_KERNEL_THREADS, 0, s>>>(ks, ps, n, vocab, g, ldg, d, lv, scale, vec_out, out, ldo, pl.chunks, pieces);
        else     emb_chunk_kernel<T, false><<<grid, ROW_KERNEL_THREADS, 0, s>>>(ks, ps, n, vocab, g, ldg, d, lv, scale, vec_out, out, ldo, pl.chunks, pieces);
        MECLIP_CUDA(cudaGetLastError());
    }
    if (pl.chunks < 2) return MECLIP_OK;
    if (pl.groups > 0) {
        ScopedTiming timing(s, TAG_ROW, 0.0);
        emb_level2_kernel<<<(unsigned)((pl.groups * pieces + wpb - 1) / wpb), ROW_KERNEL_THREADS, 0, s>>>(ks, vocab, lv, pl.groups, pieces);
        MECLIP_CUDA(cudaGetLastError());
    }
    ScopedTiming timing(s, TAG_ROW, 0.0);
    emb_join_kernel<T><<<grid, ROW_KERNEL_THREADS, 0, s>>>(ks, n, vocab, d, lv, scale, vec_out, out, ldo, pl.chunks, pieces);
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
