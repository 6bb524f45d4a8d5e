// Host side of the vocabulary softmax: meclip_token_log_probs, meclip_distill and their gradients (include/meclip.h).
#pragma once

namespace meclip {

// Rows handled by one tile pass: the partial results (1/8 byte per score, 3/8 with alternatives) stay a bounded
// workspace however many rows there are, and 16384 rows fill the GPU many times over.
static constexpr long long VOCAB_ROW_BLOCK = 16384;

// Column-tile width of the statistics pass.  Up to 128 rows there is one row tile, the pass is bound by reading the table,
// and what counts is that every SM gets the same share of it: the fewest waves x width, in steps of 32 columns (V = 32768:
// 147 tiles of 224 columns instead of 128 of 256).  With more rows 256: a narrower tile costs more per column than a
// fuller last wave brings.
static int pick_stats_bn(long long rows, long long vocab) {
    if (rows > BM) return vocab >= 256 ? 256 : (int)((vocab + 63) / 64 * 64);
    int best = 256;
    long long best_t = -1;
    for (int bn = 256; bn >= 64; bn -= 32) {
        const long long tiles = (vocab + bn - 1) / bn;
        const long long t = (tiles + sm_count() - 1) / sm_count() * (bn + 8);      // + 8: a tile's own overhead
        if (best_t < 0 || t < best_t) { best_t = t; best = bn; }
    }
    return best;
}

struct VocabPlan {
    long long row_block, slots, chunks, chunk_ld, few_blocks;      // slots: room for the partial sums of either pass
    long long tile_slots;                                           // those that the tile pass writes
    int bn;
    size_t stats_bytes, chunk_bytes, total;
};
static VocabPlan plan_vocab(long long rows, long long vocab, int top_k) {
    VocabPlan v;
    v.row_block = rows < VOCAB_ROW_BLOCK ? rows : VOCAB_ROW_BLOCK;
    v.bn = pick_stats_bn(v.row_block, vocab);
    v.slots = v.tile_slots = 2 * ((vocab + v.bn - 1) / v.bn);
    v.chunks = (vocab + 31) / 32;
    v.few_blocks = v.chunks < VOCAB_FEW_BLOCKS * sm_count() ? v.chunks : VOCAB_FEW_BLOCKS * sm_count();
    if (rows <= VOCAB_FEW_ROWS && v.slots < v.few_blocks) v.slots = v.few_blocks;
    v.chunk_ld = (long long)round_up((size_t)v.chunks, 4);
    v.stats_bytes = round_up((size_t)v.row_block * v.slots * 16, 256);
    v.chunk_bytes = top_k > 0 ? round_up((size_t)v.row_block * v.chunk_ld * 4, 256) : 0;
    v.total = v.stats_bytes + 2 * v.chunk_bytes;
    return v;
}

static constexpr int VOCAB_ROWS_SMEM = 200 * 1024;      // dynamic shared memory of a block of the row kernel at most

template <int G, bool DISTILL, bool TOP>
static int launch_vocab_rows_t(const VocabRows& p, int f16, cudaStream_t s) {
    const int per_block = VOCAB_THREADS / G;
    const size_t smem = (size_t)per_block * vocab_row_smem(p.k, p.top_k, p.rank_cap);
    const unsigned grid = (unsigned)((p.rows + per_block - 1) / per_block);
    const double bytes = (double)p.rows * (16.0 * p.slots + (p.top_k > 0 ? 8.0 * p.chunks : 0.0) +
                                           2.0 * p.d * (1 + p.k + p.top_k));
    ScopedTiming timing(s, TAG_ROW, bytes);
    auto kern = f16 ? vocab_rows_kernel<G, __half, DISTILL, TOP> : vocab_rows_kernel<G, __nv_bfloat16, DISTILL, TOP>;
    // (once to the most: a limit that follows the call could shrink between another thread's setting and its launch)
    static_assert(VOCAB_THREADS / 32 * vocab_row_smem(VOCAB_MAX_ENTRIES, VOCAB_MAX_TOP, vocab_rank_cap(VOCAB_MAX_TOP, true)) <= VOCAB_ROWS_SMEM, "shared memory of a block");
    static std::atomic<unsigned long long> smem_allowed[2] = {{0}, {0}};
    const int rc = allow_all_smem(kern, smem_allowed[f16 ? 1 : 0], VOCAB_ROWS_SMEM);
    if (rc) return rc;
    kern<<<grid, VOCAB_THREADS, smem, s>>>(p);
    MECLIP_CUDA(cudaGetLastError());
    return MECLIP_OK;
}

template <typename T, int R>
static int launch_vocab_few_r(const VocabFew& p, unsigned blocks, cudaStream_t s) {
    const int smem = VOCAB_FEW_RING + R * p.d_smem * 2;
    static std::atomic<unsigned long long> smem_allowed{0};
    const int rc = allow_all_smem(vocab_few_kernel<T, R>, smem_allowed, VOCAB_FEW_RING + VOCAB_FEW_X);
    if (rc) return rc;
    vocab_few_kernel<T, R><<<blocks, VOCAB_FEW_THREADS, smem, s>>>(p);
    MECLIP_CUDA(cudaGetLastError());
    return MECLIP_OK;
}
template <typename T>
static int launch_vocab_few(const VocabFew& p, unsigned blocks, cudaStream_t s) {
    ScopedTiming timing(s, TAG_SUMS, 2.0 * (double)p.rows * (double)p.vocab * (double)p.d);
    return p.rows == 1 ? launch_vocab_few_r<T, 1>(p, blocks, s) : launch_vocab_few_r<T, 2>(p, blocks, s);
}

// What both forwards ask of their operands.
static int check_vocab(const char* what, const void* x, const void* table, int dtype, int64_t rows, int64_t vocab,
                       int64_t d, int64_t ldx, int64_t ldt, float temperature, const void* tokens, int64_t k) {
    if (x == nullptr || table == nullptr || (tokens == nullptr && k > 0)) return fail(MECLIP_EINVAL, "%s: null pointer", what);
    if (dtype != MECLIP_BF16 && dtype != MECLIP_F16) return fail(MECLIP_EINVAL, "%s: operands are bf16 or fp16", what);
    if (rows < 1 || vocab < 1 || rows > 0x7fffffffLL || vocab > 0x7fffffffLL || d < 8 || d % 8 != 0 || d > 0x7fffffffLL ||
        ldx < d || ldt < d || ldx % 8 != 0 || ldt % 8 != 0 || !aligned16(x) || !aligned16(table))
        return fail(MECLIP_EINVAL, "%s: need rows, vocab in [1, 2^31), d and pitches multiples of 8, 16-byte alignment", what);
    if (!(temperature > 0.f) || std::isinf(temperature) || std::isinf(1.4426950408889634f / temperature))
        return fail(MECLIP_EINVAL, "%s: temperature must be positive, and its inverse finite", what);
    if (k < 0 || k > VOCAB_MAX_ENTRIES) return fail(MECLIP_EINVAL, "%s: at most %d entries per row", what, VOCAB_MAX_ENTRIES);
    return MECLIP_OK;
}

// Statistics pass and row kernel over blocks of rows.  `r` holds the per-row arguments of the whole problem.
template <bool DISTILL>
static int vocab_forward(VocabRows r, float temperature, int dtype, void* workspace, size_t workspace_bytes, int* status, cudaStream_t s) {
    int rc = check_device();
    if (rc) return rc;
    const long long rows = r.rows;
    const VocabPlan plan = plan_vocab(rows, r.vocab, r.top_k);
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
        return fail(MECLIP_EINVAL, "vocabulary pass: the workspace must be 256-byte aligned");
    if (workspace_bytes < plan.total) return fail(MECLIP_ENOSPC, "vocabulary pass: workspace %zu < %zu bytes", workspace_bytes, plan.total);
    uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
    r.stats = reinterpret_cast<const float4*>(ws);
    r.slots = (int)plan.tile_slots;
    r.stats_ld = plan.slots;
    r.unit = 1.f;
    r.chunk_max = r.top_k > 0 ? reinterpret_cast<const float*>(ws + plan.stats_bytes) : nullptr;
    r.chunk_second = r.top_k > 0 ? reinterpret_cast<const uint32_t*>(ws + plan.stats_bytes + plan.chunk_bytes) : nullptr;
    r.chunks = (int)plan.chunks;
    r.chunk_ld = plan.chunk_ld;
    for (long long r0 = 0; r0 < rows; r0 += plan.row_block) {
        VocabRows b = r;
        b.rows = rows - r0 < plan.row_block ? rows - r0 : plan.row_block;
        b.x = reinterpret_cast<const uint16_t*>(r.x) + r0 * r.ldx;
        if (r.tokens != nullptr) b.tokens = r.tokens + r0 * r.k;
        if (r.row_lse != nullptr) b.row_lse = r.row_lse + r0;
        if (r.entropy != nullptr) b.entropy = r.entropy + r0;
        if (r.token_lp2 != nullptr) b.token_lp2 = r.token_lp2 + r0 * r.k;
        if (r.log_probs != nullptr) b.log_probs = r.log_probs + r0 * r.k;
        if (r.top_k > 0) { b.top_log_probs = r.top_log_probs + r0 * r.top_k; b.top_tokens = r.top_tokens + r0 * r.top_k; }
        if (DISTILL) {
            b.teacher_logits = reinterpret_cast<const uint8_t*>(r.teacher_logits) + (size_t)r0 * r.k * (r.teacher_dtype == MECLIP_F32 ? 4 : 2);
            b.teacher_probs = r.teacher_probs + r0 * r.k;
            b.row_loss = r.row_loss + r0;
            b.row_has = r.row_has + r0;
        }
        GemmParams p;
        std::memset(&p, 0, sizeof(p));
        p.fmul = vocab_tile_fmul(temperature, r.d);
        p.stats = const_cast<float4*>(r.stats);
        p.stats_ld = r.stats_ld;
        p.chunk_max = const_cast<float*>(r.chunk_max);
        p.chunk_second = const_cast<uint32_t*>(r.chunk_second);
        p.chunk_ld = r.chunk_ld;
        p.status = status;
        if (DISTILL && r.loss != nullptr) {
            b.blocks_done = reinterpret_cast<unsigned int*>(ws) + 3;
            if (r0 + plan.row_block < rows) b.loss = nullptr;      // only behind the last block of rows
        }
        const bool f16 = dtype == MECLIP_F16;
        const long long d_smem = (r.d + 255LL) / 256 * 256;
        // (an empty partial sum's -1e30 has to stay finite in base 2)
        const bool by_lines = rows <= VOCAB_FEW_ROWS && d_smem * 2 * VOCAB_FEW_ROWS <= VOCAB_FEW_X && r.fmul < 1e8f;
        if (by_lines) {
            b.slots = (int)plan.few_blocks;
            b.unit = r.fmul;
            VocabFew f{};
            f.x = b.x; f.y = r.y; f.ldx = r.ldx; f.ldy = r.ldy; f.d = r.d; f.d_smem = (int)d_smem; f.rows = (int)rows;
            f.vocab = r.vocab; f.chunks = plan.chunks; f.fmul = r.fmul;
            f.stats = p.stats; f.stats_ld = p.stats_ld;
            f.chunk_max = p.chunk_max; f.chunk_second = p.chunk_second; f.chunk_ld = p.chunk_ld;
            rc = f16 ? launch_vocab_few<__half>(f, (unsigned)plan.few_blocks, s) : launch_vocab_few<__nv_bfloat16>(f, (unsigned)plan.few_blocks, s);
            if (rc) return rc;
        }
        Operand a{b.x, r.ldx, false, 0, false, f16}, t{r.y, r.ldy, false, 0, false, f16};
        t_tag = TAG_SUMS;
        if (!by_lines) rc = launch_gemm(EPI_STATS, a, t, b.rows, r.vocab, r.d, plan.bn, p, s);
        if (rc) return rc;
        // A few rows: a block each; many: a warp each.  Where the table has hardly more chunks than alternatives are wanted, most
        // columns are candidates and a block takes a row too (4096 x 1000 x 512, K = 32: 523 us instead of 1250; 2000 columns
        // 247 instead of 519; K = 8 of 1000 100 instead of 71, so not there).
        const bool few = b.rows <= 2 * sm_count() || plan.chunks <= 2 * r.top_k;
        b.rank_cap = r.top_k > 0 ? vocab_rank_cap(b.top_k, few || plan.chunks <= 4 * r.top_k) : 0;
        if (!DISTILL && r.top_k > 0) rc = few ? launch_vocab_rows_t<256, false, true>(b, f16, s) : launch_vocab_rows_t<32, false, true>(b, f16, s);
        else                         rc = few ? launch_vocab_rows_t<256, DISTILL, false>(b, f16, s) : launch_vocab_rows_t<32, DISTILL, false>(b, f16, s);
        if (rc) return rc;
    }
    return MECLIP_OK;
}

// Up to this many rows the contractions read bf16 operands as they are, and two panels keep the coefficients' bits; beyond
// it scaled fp16 copies of the operands (a pass over the table and its transposition) cost less than walking K twice.  What
// the second panel adds to a gradient: 128 x 32768 x 1024 72 -> 84 us, 256 x 50000 x 1152 136 -> 185 us.
static constexpr long long VOCAB_TWO_PANEL_ROWS = 256;
// From here on side streams pay for their events, for an fp16 problem transposed copies of the operands too.
static constexpr long long VOCAB_OVERLAP_ROWS = 1024;

struct VocabGradPlan {
    size_t rows_bytes, features_bytes, split_bytes, grad_bytes;
    long long widest;
    int split_bufs;
    bool transposed, two_panels, overlap;
    size_t total() const { return rows_bytes + 256 + features_bytes + split_bufs * split_bytes + grad_bytes; }
};
static VocabGradPlan plan_vocab_grad(int dtype, long long rows, long long vocab, long long d) {
    VocabGradPlan g;
    const bool f16 = dtype == MECLIP_F16;
    g.rows_bytes = round_up((size_t)rows * 2 * sizeof(float4), 256);
    g.overlap = rows >= VOCAB_OVERLAP_ROWS;
    g.transposed = transposes_allowed() && (f16 ? g.overlap : rows > VOCAB_TWO_PANEL_ROWS);
    g.features_bytes = f16 && !g.transposed ? round_up((size_t)rows * d * 2, 256) : 0;
    // The rounding of a coefficient to bf16 (2^-9 on average) does not average out where a row's gradient is carried by one
    // coefficient: its whole gradient is off by that much, as much as the output's own rounding.
    g.two_panels = !f16 && !g.transposed;
    g.widest = vocab;           // the panel's bytes are limit enough; every further panel is three launches
    const GradPlan plan = plan_grad(rows, vocab, d, g.transposed, true, g.two_panels ? 2 : 1, g.widest);
    g.grad_bytes = plan.total();
    const bool dual = g.transposed && d >= 256 && dual_allowed() && pair_mode() != 0 && !wide_allowed();
    g.split_bytes = split_bytes(plan.row_block, plan.panel_w, d, dual, g.two_panels);
    g.split_bufs = g.overlap && !dual ? 2 : 1;          // the two contractions on two streams
    return g;
}

static int check_vocab_grad(const char* what, const void* ws, size_t ws_bytes, const VocabGradPlan& plan) {
    if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 255u) != 0) return fail(MECLIP_EINVAL, "%s: workspace must be 256-byte aligned", what);
    if (ws_bytes < plan.total()) return fail(MECLIP_ENOSPC, "%s: workspace %zu < %zu bytes", what, ws_bytes, plan.total());
    return MECLIP_OK;
}

static int vocab_grad(const VocabCoef& coef, int dtype, const void* x, const void* t, int64_t rows, int64_t vocab, int64_t d,
                      int64_t ldx, int64_t ldt, float temperature, void* dx, int dx_mode, int64_t lddx, void* dt,
                      int dt_mode, int64_t lddt, uint8_t* ws, const VocabGradPlan& plan, int* status, cudaStream_t s) {
    VocabGrad vg;
    vg.coef = coef;
    vg.row_factors = reinterpret_cast<float4*>(ws);
    vg.row_entries = coef.k <= VOCAB_TILE_ENTRIES ? vg.row_factors + rows : nullptr;
    vg.f16 = dtype == MECLIP_F16;
    vg.tile_fmul = vocab_tile_fmul(temperature, d);
    vg.two_panels = plan.two_panels;
    vg.widest = plan.widest;
    vg.total = reinterpret_cast<unsigned int*>(ws + plan.rows_bytes);
    vg.table_max = reinterpret_cast<float*>(vg.total + 1);
    vg.features = reinterpret_cast<__half*>(ws + plan.rows_bytes + 256);
    uint8_t* split = ws + plan.rows_bytes + 256 + plan.features_bytes;
    vg.split_buf = reinterpret_cast<float*>(split);
    vg.split_buf2 = reinterpret_cast<float*>(split + (plan.split_bufs > 1 ? plan.split_bytes : 0));
    vg.split_bytes = plan.split_bytes;
    return grad_impl(MECLIP_SIGLIP, x, t, rows, vocab, d, ldx, ldt, temperature, 0, 0, nullptr, nullptr, nullptr, 1.f, dx,
                     dx_mode, lddx, dt, dt_mode, lddt, split + plan.split_bufs * plan.split_bytes, plan.grad_bytes, status, s,
                     plan.overlap && overlap_allowed(), plan.transposed, nullptr, 0.f, 0.f, 0, false, DeviceScalars(), true,
                     nullptr, 0, nullptr, 0, &vg);
}

}  // namespace meclip

extern "C" {

size_t meclip_vocab_workspace_bytes(int64_t rows, int64_t vocab, int top_k) {
    if (rows < 1 || vocab < 1 || top_k < 0) return 0;
    return plan_vocab(rows, vocab, top_k).total;
}

size_t meclip_vocab_grad_workspace_bytes(int dtype, int64_t rows, int64_t vocab, int64_t d) {
    if (rows < 1 || vocab < 1 || d < 1) return 0;
    return plan_vocab_grad(dtype, rows, vocab, d).total();
}

int meclip_token_log_probs(const void* x, const void* table, int dtype, int64_t rows, int64_t vocab, int64_t d,
                           int64_t ldx, int64_t ldt, float temperature, const int64_t* tokens, int64_t per_row,
                           float* log_probs, float* entropy, int top_k, float* top_log_probs, int64_t* top_tokens,
                           float* row_lse, float* token_scores, void* workspace, size_t workspace_bytes, int* status,
                           void* stream) {
    NvtxRange range("meclip_token_log_probs");
    int rc = check_vocab("token_log_probs", x, table, dtype, rows, vocab, d, ldx, ldt, temperature, tokens, per_row);
    if (rc) return rc;
    if (per_row > 0 && log_probs == nullptr) return fail(MECLIP_EINVAL, "token_log_probs: log_probs is null");
    if (top_k < 0 || top_k > VOCAB_MAX_TOP || top_k > vocab)
        return fail(MECLIP_EINVAL, "token_log_probs: top_k must be in [0, min(%d, vocab)]", VOCAB_MAX_TOP);
    if (top_k > 0 && (top_log_probs == nullptr || top_tokens == nullptr)) return fail(MECLIP_EINVAL, "token_log_probs: top outputs are null");
    VocabRows r;
    std::memset(&r, 0, sizeof(r));
    r.x = x; r.y = table; r.ldx = ldx; r.ldy = ldt; r.d = (int)d; r.rows = rows; r.vocab = vocab;
    r.fmul = 1.4426950408889634f / temperature;
    r.tokens = reinterpret_cast<const long long*>(tokens); r.k = (int)per_row;
    r.row_lse = row_lse; r.entropy = entropy; r.token_lp2 = token_scores; r.log_probs = log_probs;
    r.top_k = top_k; r.top_log_probs = top_log_probs; r.top_tokens = reinterpret_cast<long long*>(top_tokens);
    return vocab_forward<false>(r, temperature, dtype, workspace, workspace_bytes, status, (cudaStream_t)stream);
}

int meclip_token_log_probs_grad(const void* x, const void* table, int dtype, int64_t rows, int64_t vocab, int64_t d,
                                int64_t ldx, int64_t ldt, float temperature, const int64_t* tokens, int64_t per_row,
                                const float* row_lse, const float* entropy, const float* token_scores,
                                const float* grad_log_probs, const float* grad_entropy, void* dx, int dx_mode, int64_t lddx,
                                void* dtable, int dtable_mode, int64_t lddt, void* workspace, size_t workspace_bytes,
                                int* status, void* stream) {
    NvtxRange range("meclip_token_log_probs_grad");
    int rc = check_vocab("token_log_probs_grad", x, table, dtype, rows, vocab, d, ldx, ldt, temperature, tokens, per_row);
    if (rc) return rc;
    if (row_lse == nullptr || (per_row > 0 && token_scores == nullptr) || (grad_entropy != nullptr && entropy == nullptr))
        return fail(MECLIP_EINVAL, "token_log_probs_grad: null pointer");
    const VocabGradPlan plan = plan_vocab_grad(dtype, rows, vocab, d);
    rc = check_vocab_grad("token_log_probs_grad", workspace, workspace_bytes, plan);
    if (rc) return rc;
    VocabCoef c{};
    c.row_lse = row_lse; c.token_lp2 = token_scores; c.tokens = reinterpret_cast<const long long*>(tokens); c.k = (int)per_row;
    c.vocab = vocab; c.inv_t = 1.f / temperature;
    c.grad_log_probs = grad_log_probs; c.grad_entropy = grad_entropy; c.entropy = entropy;
    return vocab_grad(c, dtype, x, table, rows, vocab, d, ldx, ldt, temperature, dx, dx_mode, lddx, dtable, dtable_mode, lddt,
                      reinterpret_cast<uint8_t*>(workspace), plan, status, (cudaStream_t)stream);
}

int meclip_distill(const void* x, const void* table, int dtype, int64_t rows, int64_t vocab, int64_t d, int64_t ldx,
                   int64_t ldt, float temperature, const int64_t* teacher_tokens, const void* teacher_logits,
                   int teacher_dtype, int64_t per_row, float teacher_temperature, int mean, float* row_loss, float* row_has,
                   float* loss, float* inv_count, float* row_lse, float* token_scores, float* teacher_probs,
                   void* workspace, size_t workspace_bytes, int* status, void* stream) {
    NvtxRange range("meclip_distill");
    int rc = check_vocab("distill", x, table, dtype, rows, vocab, d, ldx, ldt, temperature, teacher_tokens, per_row);
    if (rc) return rc;
    if (per_row < 1) return fail(MECLIP_EINVAL, "distill: at least one teacher entry per row");
    if (teacher_logits == nullptr || row_loss == nullptr || row_has == nullptr || row_lse == nullptr || token_scores == nullptr ||
        teacher_probs == nullptr || (loss == nullptr) != (inv_count == nullptr))
        return fail(MECLIP_EINVAL, "distill: null pointer");
    if (teacher_dtype != MECLIP_BF16 && teacher_dtype != MECLIP_F32 && teacher_dtype != MECLIP_F16)
        return fail(MECLIP_EINVAL, "distill: bad teacher dtype %d", teacher_dtype);
    if (!(teacher_temperature > 0.f) || std::isinf(teacher_temperature) || std::isinf(1.f / teacher_temperature))
        return fail(MECLIP_EINVAL, "distill: teacher temperature must be positive, and its inverse finite");
    VocabRows r;
    std::memset(&r, 0, sizeof(r));
    r.x = x; r.y = table; r.ldx = ldx; r.ldy = ldt; r.d = (int)d; r.rows = rows; r.vocab = vocab;
    r.fmul = 1.4426950408889634f / temperature;
    r.tokens = reinterpret_cast<const long long*>(teacher_tokens); r.k = (int)per_row;
    r.row_lse = row_lse; r.token_lp2 = token_scores;
    r.teacher_logits = teacher_logits; r.teacher_dtype = teacher_dtype; r.inv_teacher_t = 1.f / teacher_temperature;
    r.teacher_probs = teacher_probs; r.row_loss = row_loss; r.row_has = row_has;
    r.all_loss = row_loss; r.all_has = row_has; r.all_rows = rows; r.mean = mean; r.loss = loss; r.inv_count = inv_count;
    return vocab_forward<true>(r, temperature, dtype, workspace, workspace_bytes, status, (cudaStream_t)stream);
}

int meclip_distill_grad(const void* x, const void* table, int dtype, int64_t rows, int64_t vocab, int64_t d, int64_t ldx,
                        int64_t ldt, float temperature, const int64_t* teacher_tokens, int64_t per_row, const float* row_lse,
                        const float* token_scores, const float* teacher_probs, const float* row_has, const float* grad_out,
                        int grad_per_row, const float* inv_count, void* dx, int dx_mode, int64_t lddx, void* dtable,
                        int dtable_mode, int64_t lddt, void* workspace, size_t workspace_bytes, int* status, void* stream) {
    NvtxRange range("meclip_distill_grad");
    int rc = check_vocab("distill_grad", x, table, dtype, rows, vocab, d, ldx, ldt, temperature, teacher_tokens, per_row);
    if (rc) return rc;
    if (per_row < 1 || row_lse == nullptr || token_scores == nullptr || teacher_probs == nullptr || row_has == nullptr || grad_out == nullptr)
        return fail(MECLIP_EINVAL, "distill_grad: null pointer");
    const VocabGradPlan plan = plan_vocab_grad(dtype, rows, vocab, d);
    rc = check_vocab_grad("distill_grad", workspace, workspace_bytes, plan);
    if (rc) return rc;
    VocabCoef c{};
    c.row_lse = row_lse; c.token_lp2 = token_scores; c.tokens = reinterpret_cast<const long long*>(teacher_tokens);
    c.k = (int)per_row; c.distill = 1; c.vocab = vocab; c.inv_t = 1.f / temperature;
    c.grad_out = grad_out; c.grad_per_row = grad_per_row; c.factor = inv_count; c.row_has = row_has; c.probs = teacher_probs;
    return vocab_grad(c, dtype, x, table, rows, vocab, d, ldx, ldt, temperature, dx, dx_mode, lddx, dtable, dtable_mode, lddt,
                      reinterpret_cast<uint8_t*>(workspace), plan, status, (cudaStream_t)stream);
}

}  // extern "C"
