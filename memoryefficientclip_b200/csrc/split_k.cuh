// Contractions with few output tiles and a long K, cut into parts of K (GemmParams::splits): rules and the sum of the parts.
//
// A gradient of `rows` features against a vocabulary has rows / 256 x d / 256 tiles of K = vocab for dX: 16 tiles of 500
// K steps at 2047 x 32001 x 512 on 74 CTA pairs.  Cut so that no tile is longer than a quarter of what a pair has to do in
// all, the launch ends when the work does.  The parts are fp32, written once and read once, and added in order.  Both
// contractions in one launch, whole tiles or parts of at most a half, of a quarter of a pair's share (their sum, 10 to
// 19 us, included where there are parts): 2047 x 32001 x 512 - / 149 / 139 us, 4096 x 32768 x 768 - / 384 / 340,
// x 1152 630 / 630 / 566 (half leaves them whole), x 1536 716 / 716 / 655, 4736 x 32768 x 1024 632 / 632 / 561.
#pragma once

namespace meclip {

static constexpr int SPLIT_MAX = 32;               // parts of a contraction
static constexpr int SPLIT_MIN_STEPS = 8;          // K steps of a part: shorter ones are all prologue and epilogue

struct SplitK {
    int parts = 1;
    const float* buf = nullptr;
    long long stride = 0, m = 0, n = 0;
    void* out = nullptr;
    long long ld_out = 0;
    int out_bf16 = 0;
    const float* acc_in = nullptr;
    long long ld_acc = 0;
};

// out = acc_in + part 0 + part 1 + ..., four columns per thread (n is a multiple of 8)
__global__ void __launch_bounds__(256)
split_sum_kernel(const __grid_constant__ SplitK s) {
    const long long n4 = s.n / 4, all = s.m * n4, step = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += step) {
        const long long r = i / n4, c = i % n4 * 4;
        float4 a = s.acc_in != nullptr ? *reinterpret_cast<const float4*>(s.acc_in + r * s.ld_acc + c) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int q = 0; q < s.parts; ++q) {
            const float4 v = __ldcs(reinterpret_cast<const float4*>(s.buf + q * s.stride + i * 4));
            a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
        }
        if (s.out_bf16) {
            uint2 o;
            o.x = pack_bf16x2(a.x, a.y);
            o.y = pack_bf16x2(a.z, a.w);
            *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(s.out) + r * s.ld_out + c) = o;
        } else {
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(s.out) + r * s.ld_out + c) = a;
        }
    }
}

static int launch_split_sum(const SplitK& s, cudaStream_t stream) {
    if (s.parts < 2) return MECLIP_OK;
    long long blocks = (s.m * (s.n / 4) + 255) / 256;
    if (blocks > 16LL * sm_count()) blocks = 16LL * sm_count();
    ScopedTiming timing(stream, TAG_ACCUM, (double)s.m * s.n * (4.0 * s.parts + 4.0));
    split_sum_kernel<<<(unsigned)blocks, 256, 0, stream>>>(s);
    MECLIP_CUDA(cudaGetLastError());
    return MECLIP_OK;
}

// Redirects a contraction of m x n outputs to `parts` partial sums in buf, as far as `bytes` allow.
static SplitK split_into(GemmParams& p, long long m, long long n, long long k_steps, long long parts, float* buf, size_t bytes) {
    SplitK s;
    const long long room = buf == nullptr ? 0 : (long long)(bytes / ((size_t)m * n * 4));
    if (parts > room) parts = room;
    if (parts > SPLIT_MAX) parts = SPLIT_MAX;
    if (parts > k_steps / SPLIT_MIN_STEPS) parts = k_steps / SPLIT_MIN_STEPS;
    if (parts < 2) return s;
    p.k_part = (int)((k_steps + parts - 1) / parts);
    p.splits = (int)((k_steps + p.k_part - 1) / p.k_part);       // every part has steps
    p.split_stride = m * n;
    s.parts = p.splits; s.buf = buf; s.stride = m * n; s.m = m; s.n = n;
    s.out = p.out; s.ld_out = p.ld_out; s.out_bf16 = p.out_bf16; s.acc_in = p.acc_in; s.ld_acc = p.ld_acc;
    p.out = buf; p.ld_out = n; p.out_bf16 = 0; p.acc_in = nullptr; p.ld_acc = 0;
    return s;
}

// Tile width of a contraction that may be cut: 256 columns where K is long, since parts fill the SMs then and every column
// tile reads the panel again (dX of 64 x 50000 x 1152: 18 tiles of 64 columns 78 us, 5 of 256 42 us); else as for others.
static int split_tile_width(long long m, long long n, long long k, bool shares_gpu, bool b_k_major) {
    return n >= 256 && k >= 64 * BK ? 256 : pick_contraction_bn(m, n, shares_gpu, b_k_major);
}

// A contraction that has the GPU to itself: as many parts as SMs have no tile.
static long long split_parts_alone(long long m, long long n, long long k_steps, int bn) {
    const long long tiles = ((m + BM - 1) / BM) * ((n + bn - 1) / bn);
    long long parts = sm_count() / tiles;
    if (parts > k_steps / SPLIT_MIN_STEPS) parts = k_steps / SPLIT_MIN_STEPS;
    return parts > SPLIT_MAX ? SPLIT_MAX : parts;
}
static SplitK split_alone(GemmParams& p, long long m, long long n, long long k, int bn, float* buf, size_t bytes) {
    const long long k_steps = (k + BK - 1) / BK * (p.lo_chunk > 0 ? 2 : 1);
    return split_into(p, m, n, k_steps, split_parts_alone(m, n, k_steps, bn), buf, bytes);
}

// Both contractions of a block in one launch: parts for tiles that are longer than a quarter of a pair's share of all steps.
static void split_parts_dual(long long rows, long long cols, long long d, long long& parts_y, long long& parts_x) {
    const long long nt = (d + 255) / 256, my = (cols + PAIR_BM - 1) / PAIR_BM, mx = (rows + PAIR_BM - 1) / PAIR_BM;
    const long long ky = (rows + BK - 1) / BK, kx = (cols + BK - 1) / BK, pairs = sm_count() / 2;
    long long limit = (nt * (my * ky + mx * kx) + 4 * pairs - 1) / (4 * pairs);
    if (limit < 2 * SPLIT_MIN_STEPS) limit = 2 * SPLIT_MIN_STEPS;
    parts_y = (ky + limit - 1) / limit;
    parts_x = (kx + limit - 1) / limit;
}
static void split_dual(GemmParams& py, GemmParams& px, long long rows, long long cols, long long d, float* buf, size_t bytes,
                       SplitK& sy, SplitK& sx) {
    long long parts_y, parts_x;
    split_parts_dual(rows, cols, d, parts_y, parts_x);
    if (parts_y > 1) sy = split_into(py, cols, d, (rows + BK - 1) / BK, parts_y, buf, bytes);
    const size_t used = sy.parts > 1 ? (size_t)sy.parts * cols * d * 4 : 0;
    if (parts_x > 1) sx = split_into(px, rows, d, (cols + BK - 1) / BK, parts_x, buf + used / 4, bytes - used);
}

// Bytes that the parts of one rows x cols block want at most.
static size_t split_bytes(long long rows, long long cols, long long d, bool dual, bool two_panels) {
    if (dual) {
        long long py, px;
        split_parts_dual(rows, cols, d, py, px);
        if (py > SPLIT_MAX) py = SPLIT_MAX;
        if (px > SPLIT_MAX) px = SPLIT_MAX;
        return round_up((size_t)(py > 1 ? py : 0) * cols * d * 4 + (size_t)(px > 1 ? px : 0) * rows * d * 4, 256);
    }
    size_t most = 0;
    for (int which = 0; which < 2; ++which) {
        const long long m = which ? rows : cols, k = which ? cols : rows;
        const long long parts = split_parts_alone(m, d, (k + BK - 1) / BK * (two_panels ? 2 : 1), 256);
        // narrower tiles mean more of them and fewer parts, so this is the most
        if (parts > 1) { const size_t b = (size_t)parts * m * d * 4; if (b > most) most = b; }
    }
    return round_up(most, 256);
}

}  // namespace meclip
