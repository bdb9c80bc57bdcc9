// rb200k_linear_ce: softmax cross entropy of x W^T + b, forward and backward, without the rows x classes matrix.
//   forward   one product whose epilogue keeps, for every row and tile of classes, the largest score and the sum
//             of exp(score - largest); ce_merge_kernel joins them (and makes the loss). The scores stay on the chip.
//   backward  piece by piece: the product again, its epilogue turning scores into (softmax - target) in the element type, then
//             that piece times W and transposed times x. Pieces are cut along the longer of classes and rows; the
//             gradient that sums over pieces is accumulated in 32 bits.
// Pieces hold (softmax - target) * c_i * 2^15 with |c_i| <= 1, so that a probability of 2^-29 is still a normal fp16;
// the common factor (2^-15, the loss gradient, 1 / count) is applied to the 32-bit sums. They are rounded to the element type once, as
// operands of two products have to be. What fp16 loses of a row far below the largest is half of its least
// step, 2^-25, for each class: 2^-40 G times the norm of a feature's weights in dx, with the common factor G. For G up to 2^15 that is about
// half of dx' own least step; larger gradients of single rows' losses (reduction NONE) are named in rb200_kernels.h.
// Few classes and features take one sweep over x each way instead (narrow_loss.cuh).
#include "narrow_loss.cuh"

namespace rb200 {

constexpr size_t kStatBytes = 128u << 20;    // partial maxima and sums of one launch (about)
constexpr size_t kPieceBytes = 256u << 20;   // scores' gradients of one piece

// ---- forward: joining the partial statistics ----------------------------------------------------------------
struct MergeArgs {
    const float* part;      // [parts][rows] maxima, sums, sums of z / classes
    int parts, want_zsum;
    const void* labels;
    int label_bytes, classes, rows, reduction;
    long long ignore_index;
    float smoothing;
    int first, last;        // piece of the classes: the first starts the statistics, the last makes the loss
    float* stats;           // [3][rows]: maximum, sum, the label's z
    float* zsum;            // [rows], between pieces
    float* loss;
    int* info;
    double* block_sums;
};

__device__ __forceinline__ void join(RunningSoftmax& a, float m, float s) {
    const float top = fmaxf(a.m, m), base = finite_max(top);
    a.s = a.s * exp_diff(a.m - base) + s * exp_diff(m - base);
    a.m = top;
}

// A block takes 256 / SUBS rows at a time; SUBS threads share a row's parts.
template <int SUBS>
__global__ void __launch_bounds__(256) ce_merge_kernel(MergeArgs a) {
    constexpr int ROWS = 256 / SUBS;
    __shared__ float sm[SUBS][ROWS], ss[SUBS][ROWS], sz[SUBS][ROWS];
    __shared__ double sums[256];
    __shared__ int counts[8], dirts[8], last_block;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x % ROWS, sub = threadIdx.x / ROWS;
    const long long plane = (long long)a.parts * a.rows;
    double mine = 0.0;
    int counts_mine = 0, dirty_mine = 0;
    for (long long row0 = (long long)blockIdx.x * ROWS; row0 < a.rows; row0 += (long long)gridDim.x * ROWS) {
        const long long row = row0 + lane;
        RunningSoftmax r = {-INFINITY, 0.0f};
        float z = 0.0f, at_label = 0.0f;
        int label = -1;
        bool counted = false;
        if (row < a.rows && sub == 0 && a.last) {   // on their way while the parts are joined
            label = load_label(a.labels, a.label_bytes, row, a.ignore_index, a.classes, &counted);
            at_label = a.stats[2ll * a.rows + row];
        }
        if (row < a.rows) {
#pragma unroll 4
            for (int p = sub; p < a.parts; p += SUBS) {
                const long long at = (long long)p * a.rows + row;
                join(r, a.part[at], a.part[plane + at]);
                if (a.want_zsum) z += a.part[2 * plane + at];
            }
        }
        if (SUBS > 1) {
            __syncthreads();
            sm[sub][lane] = r.m;
            ss[sub][lane] = r.s;
            sz[sub][lane] = z;
            __syncthreads();
            if (sub) continue;
#pragma unroll
            for (int i = 1; i < SUBS; i++) {
                join(r, sm[i][lane], ss[i][lane]);
                z += sz[i][lane];
            }
        }
        if (row >= a.rows) continue;
        if (!a.first) {
            join(r, a.stats[row], a.stats[a.rows + row]);
            if (a.want_zsum) z += a.zsum[row];
        }
        if (!a.last) {
            if (a.want_zsum) a.zsum[row] = z;
        } else {
            float loss = 0.0f;
            if (counted) {
                counts_mine++;
                if (label < 0) {
                    r.m = r.s = loss = nanf("");
                } else {
                    const float lse = logf(r.s);   // above the maximum
                    loss = (1.0f - a.smoothing) * (lse + (r.m - at_label));
                    if (a.want_zsum) loss += a.smoothing * (lse + (r.m - z));
                }
            } else {
                dirty_mine |= !(isfinite(r.m) && isfinite(r.s));
            }
            mine += loss;
            if (a.reduction == RB200_REDUCE_NONE) a.loss[row] = loss;
        }
        a.stats[row] = r.m;
        a.stats[a.rows + row] = r.s;
    }
    if (!a.last) return;
    // the block's counts and sum, then one atomic each (whole numbers: their order does not matter)
    const int warp_count = __reduce_add_sync(0xFFFFFFFFu, counts_mine), warp_dirt = __any_sync(0xFFFFFFFFu, dirty_mine);
    if ((threadIdx.x & 31) == 0) {
        counts[threadIdx.x >> 5] = warp_count;
        dirts[threadIdx.x >> 5] = warp_dirt;
    }
    auto block_sum = [&](double s) {   // in thread 0; always in the same order
        __syncthreads();
        sums[threadIdx.x] = s;
        __syncthreads();
        for (int d = 128; d; d >>= 1) {
            if (threadIdx.x < d) sums[threadIdx.x] += sums[threadIdx.x + d];
            __syncthreads();
        }
        return sums[0];
    };
    const double block = a.reduction != RB200_REDUCE_NONE ? block_sum(mine) : 0.0;
    __syncthreads();
    if (threadIdx.x == 0) {
        int n = 0, any = 0;
        for (int i = 0; i < 8; i++) {
            n += counts[i];
            any |= dirts[i];
        }
        if (n) atomicAdd(a.info, n);
        if (any) atomicOr(a.info + 1, 1);
        if (a.reduction != RB200_REDUCE_NONE) {
            a.block_sums[blockIdx.x] = block;
            __threadfence();
            last_block = atomicAdd(a.info + 2, 1) == (int)gridDim.x - 1;
        }
    }
    if (a.reduction == RB200_REDUCE_NONE) return;
    __syncthreads();
    if (!last_block) return;
    // the block that finished last adds the others' sums
    __threadfence();
    double s = 0.0;
    for (unsigned b = threadIdx.x; b < gridDim.x; b += 256) s += __ldcg(a.block_sums + b);
    s = block_sum(s);
    if (threadIdx.x == 0) {
        const int count = atomicAdd(a.info, 0);
        *a.loss = (float)(a.reduction == RB200_REDUCE_MEAN ? s / (double)max(1, count) : s);
    }
}

constexpr int kMergeBlocks = 148 * 2;   // every block ends with atomics on the same words
static int merge_launch(const MergeArgs& m, cudaStream_t stream, const char* what) {
    // as many threads a row as there are parts for them to share, while the rows alone do not fill the GPU
    const int subs = m.parts >= 32 && m.rows <= 4096 ? 32 : m.parts >= 8 ? 8 : m.parts >= 4 ? 4 : m.parts >= 2 && m.rows < 148 * 256 ? 2 : 1;
    const long long blocks = ((long long)m.rows + 256 / subs - 1) / (256 / subs);
    const unsigned grid = (unsigned)(blocks < kMergeBlocks ? blocks : kMergeBlocks);
    auto* kernel = subs == 32 ? ce_merge_kernel<32> : subs == 8 ? ce_merge_kernel<8> : subs == 4 ? ce_merge_kernel<4> : subs == 2 ? ce_merge_kernel<2> : ce_merge_kernel<1>;
    int rc = check_cuda(launch_overlapped(kernel, dim3(grid), dim3(256), 0, stream, m), what);
    if (rc) return rc;
    count_launch();
    return RB200_OK;
}

// ---- backward: per-row factors --------------------------------------------------------------------------------
// NONE: c_i = g_i / G and the common factor G, the power of two above the largest finite |g_i| of a counted row (so
// the division is exact). Two launches where there are many rows: the blocks' largest (ce_tops_kernel), then the factors, for which
// every block looks at all of those. (One block for all rows took 330 us for 279424 of them.)
__device__ __forceinline__ float largest(float top) {   // of a block of 256 threads, in all of them
    __shared__ float tops[8];
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int i = 0; i < 8; i++) top = fmaxf(top, tops[i]);
    return top;
}
__device__ __forceinline__ float counted_top(const float* dloss, const void* labels, int label_bytes, int classes, long long ignore_index, int rows) {
    float top = 0.0f;
#pragma unroll 4
    for (int i = blockIdx.x * 256 + threadIdx.x; i < rows; i += gridDim.x * 256) {
        bool counted;
        load_label(labels, label_bytes, i, ignore_index, classes, &counted);
        const float g = fabsf(dloss[i]);
        if (counted && g <= 3.4028235e38f) top = fmaxf(top, g);
    }
    return largest(top);
}
__global__ void __launch_bounds__(256) ce_tops_kernel(const float* __restrict__ dloss, const void* labels, int label_bytes, int classes,
                                                      long long ignore_index, int rows, float* tops) {
    pdl_launch_dependents();
    pdl_wait();
    const float top = counted_top(dloss, labels, label_bytes, classes, ignore_index, rows);
    if (threadIdx.x == 0) tops[blockIdx.x] = top;
}
// blocks: the entries of `tops`, or 0 if this one block finds the largest itself.
__global__ void __launch_bounds__(256) ce_factors_kernel(const float* __restrict__ dloss, const void* labels, int label_bytes, int classes,
                                                         long long ignore_index, int rows, const float* tops, int blocks, float* coef, float* factor) {
    pdl_launch_dependents();
    pdl_wait();
    float top;
    if (blocks) {
        top = 0.0f;
        for (int i = threadIdx.x; i < blocks; i += 256) top = fmaxf(top, tops[i]);
        top = largest(top);
    } else {
        top = counted_top(dloss, labels, label_bytes, classes, ignore_index, rows);
    }
    // both the factor and its inverse stay normal: exponents -100 .. 100
    int e = top > 0.0f ? ilogbf(top) + 1 : 0;
    e = max(-100, min(100, e));
    if (blockIdx.x == 0 && threadIdx.x == 0) *factor = ldexpf(1.0f, e);
    const float inv = ldexpf(1.0f, -e);
    for (int i = blockIdx.x * 256 + threadIdx.x; i < rows; i += gridDim.x * 256) coef[i] = dloss[i] * inv;
}
constexpr int kFactorBlocks = 296;
static int factors_launch(const rb200_linear_ce_params& p, float* tops, float* coef, float* factor, cudaStream_t stream, const char* what) {
    const int rows = (int)p.rows, wanted = (rows + 2047) / 2048, blocks = wanted < kFactorBlocks ? wanted : kFactorBlocks;
    int rc;
    if (blocks > 1) {
        if ((rc = check_cuda(launch_overlapped(ce_tops_kernel, dim3(blocks), dim3(256), 0, stream, p.dloss, p.labels, p.label_bytes, (int)p.classes,
                                               (long long)p.ignore_index, rows, tops),
                             what)))
            return rc;
        count_launch();
    }
    if ((rc = check_cuda(launch_overlapped(ce_factors_kernel, dim3(blocks), dim3(256), 0, stream, p.dloss, p.labels, p.label_bytes, (int)p.classes,
                                           (long long)p.ignore_index, rows, (const float*)tops, blocks > 1 ? blocks : 0, coef, factor),
                         what)))
        return rc;
    count_launch();
    return RB200_OK;
}

// ---- argument checks --------------------------------------------------------------------------------------------
static int check_sizes(const char* what, const rb200_linear_ce_params& p) {
    int rc = check_dtype(what, p.dtype);
    if (rc) return rc;
    if (p.reduction < RB200_REDUCE_NONE || p.reduction > RB200_REDUCE_SUM) {
        set_error("%s: reduction %d is not one of RB200_REDUCE_*", what, p.reduction);
        return RB200_E_INVALID;
    }
    if (p.label_bytes != 4 && p.label_bytes != 8) {
        set_error("%s: labels of %d bytes (4 or 8)", what, p.label_bytes);
        return RB200_E_INVALID;
    }
    if (!(p.label_smoothing >= 0.0f && p.label_smoothing <= 1.0f)) {
        set_error("%s: label_smoothing %g outside [0, 1]", what, p.label_smoothing);
        return RB200_E_INVALID;
    }
    return check_extents(what, p.rows, "features", p.features, "classes", p.classes);
}

static int check_common(const char* what, const rb200_linear_ce_params& p) {
    int rc;
    if ((rc = check_matrix(what, "x", p.x, p.ldx, p.rows, p.features))) return rc;
    if ((rc = check_matrix(what, "weight", p.weight, p.ldw, p.classes, p.features))) return rc;
    if (p.bias && (rc = check_matrix(what, "bias", p.bias, 0, 1, p.classes))) return rc;
    if (!p.labels || !p.stats || !p.info) {
        set_error("%s: labels, stats or info is null", what);
        return RB200_E_INVALID;
    }
    if (((uintptr_t)p.labels & (p.label_bytes - 1)) || (((uintptr_t)p.stats | (uintptr_t)p.info) & 3)) {
        set_error("%s: labels, stats or info is not aligned to its elements", what);
        return RB200_E_INVALID;
    }
    return RB200_OK;
}

static EpiArgs label_args(const rb200_linear_ce_params& p) {
    EpiArgs e = {};
    e.labels = p.labels;
    e.label_bytes = p.label_bytes;
    e.classes = (int)p.classes;
    e.ignore_index = p.ignore_index;
    e.smooth_on = 1.0f - p.label_smoothing;
    e.smooth_off = p.label_smoothing / (float)p.classes;
    e.inv_classes = 1.0f / (float)p.classes;
    return e;
}
static NarrowArgs narrow_args(const rb200_linear_ce_params& p, const GemmWait& wait) {
    NarrowArgs g = {};
    g.bias = p.bias;
    g.labels = p.labels;
    g.label_bytes = p.label_bytes;
    g.ignore_index = p.ignore_index;
    g.smoothing = p.label_smoothing;
    g.smooth_on = 1.0f - p.label_smoothing;
    g.smooth_off = p.label_smoothing / (float)p.classes;
    g.inv_classes = 1.0f / (float)p.classes;
    g.stats = p.stats;
    g.status = p.status;
    g.wait_cycles = wait.cycles;
    g.skip_chunk = wait.skip_block;
    return g;
}
static const uint8_t* at_row(const void* p, long long ld, long long row) { return (const uint8_t*)p + row * ld * 2; }

// ---- forward ------------------------------------------------------------------------------------------------------
struct StatsPlan {
    Packed x, w;
    bool narrow;
    int* counts;            // narrow, with block_sums
    int piece;              // classes of one launch
    size_t part_bytes;
    float *part, *zsum;
    double* block_sums;
    size_t bytes;
};
// The loss is made of 32-bit scores, which drift with the length of one accumulator's sum (gemm.cuh). The border is where the loss comes
// off 64 bits by some 1e-6 of itself: with scores of spread 2 (8192 rows, 16384 classes, fp16) it is off by 0.45e-6 at 1024 features,
// 0.87e-6 at 2048, 1.7e-6 at 4096; a loss that is small beside its scores by more, 1.2e-6 with 227 classes at 1875. Longer sums take
// tiles that leave TMEM columns for a second accumulator: 0.85e-6 at 4096, for 12 to 17% of time (714 -> 838 us). A border at 1024 would
// halve the error at 2048 (0.44e-6), for 4.5% of a training step (8192 x 2048, 128000 classes: 13.3 -> 13.9 ms) and 16% of an evaluation
// (64 x 2048, 21841 classes: 25.1 -> 29.2 us); four accumulators beyond 4096 that at 8192 (1.7e-6 -> 0.83e-6), for 55% of the forward pass.
constexpr int kLongSum = 2048;
static GemmPlan stats_gemm(const rb200_linear_ce_params& p, const DeviceInfo& dev, int classes) {
    return gemm_plan(dev, (int)p.rows, classes, (int)p.features, false, false, p.features > kLongSum ? kTileNMax / 2 : kTileNMax);
}
static StatsPlan plan_stats(const rb200_linear_ce_params& p, const DeviceInfo& dev, void* ws) {
    StatsPlan s = {};
    Carver c(ws);
    s.x = plan_pack(operand(p.x, p.ldx, p.rows, p.features, false), &c);
    s.w = plan_pack(operand(p.weight, p.ldw, p.classes, p.features, false), &c);
    s.narrow = narrow_fits(p.classes, p.features);
    if (s.narrow) {
        const int ctas = narrow_ctas(p.rows, dev.sms);
        s.block_sums = (double*)c.take(ctas * sizeof(double));
        s.counts = (int*)c.take(2 * ctas * sizeof(int));
        s.bytes = c.used;
        return s;
    }
    // two parts a tile, as wide as the tiles of the whole product (those of a piece may be cut anew)
    const size_t per_part = (size_t)p.rows * 3 * sizeof(float);
    const long long parts = (long long)(kStatBytes / per_part);
    long long piece = parts / 2 * stats_gemm(p, dev, (int)p.classes).bn / kTileNMax * kTileNMax;
    if (piece < kTileNMax) piece = kTileNMax;
    s.piece = (int)(piece < p.classes ? piece : p.classes);
    const long long most = 2ll * stats_gemm(p, dev, s.piece).tiles_n;
    const long long rest = p.classes % s.piece ? 2ll * stats_gemm(p, dev, (int)(p.classes % s.piece)).tiles_n : 0;
    s.part_bytes = (size_t)(most > rest ? most : rest) * per_part;
    s.part = (float*)c.take(s.part_bytes);
    s.zsum = (float*)c.take((size_t)p.rows * sizeof(float));
    s.block_sums = (double*)c.take(kMergeBlocks * sizeof(double));
    s.bytes = c.used;
    return s;
}

static int ce_forward(const rb200_linear_ce_params* p, cudaStream_t stream, GemmWait wait) {
    const char* what = "rb200k_linear_ce";
    if (!p) {
        set_error("%s: params is null", what);
        return RB200_E_INVALID;
    }
    int rc = check_sizes(what, *p);
    if (rc) return rc;
    if (p->rows == 0) {
        if (p->info && (rc = check_cuda(cudaMemsetAsync(p->info, 0, 16, stream), what))) return rc;
        if (p->loss && p->reduction != RB200_REDUCE_NONE) return check_cuda(cudaMemsetAsync(p->loss, 0, 4, stream), what);
        return RB200_OK;
    }
    if ((rc = check_common(what, *p))) return rc;
    if (!p->loss || ((uintptr_t)p->loss & 3)) {
        set_error("%s: loss is null or not aligned", what);
        return RB200_E_INVALID;
    }
    DeviceInfo dev;
    if ((rc = device_info(&dev))) return rc;
    const StatsPlan s = plan_stats(*p, dev, p->workspace);
    if ((rc = check_workspace(what, p->workspace, p->workspace_bytes, s.bytes))) return rc;
    const bool bf16 = p->dtype == RB200_BF16;
    if ((rc = pack_operands(&s.x, &s.w, stream, what))) return rc;
    if (s.narrow) {
        NarrowArgs g = narrow_args(*p, wait);
        g.loss = p->loss;
        g.none = p->reduction == RB200_REDUCE_NONE;
        g.sums = s.block_sums;
        g.counts = s.counts;
        if ((rc = narrow_launch(g, false, bf16, s.x.use, s.w.use, dev, stream, what))) return rc;
        rc = check_cuda(launch_overlapped(ce_total_kernel, dim3(1), dim3(256), 0, stream, (const double*)s.block_sums, (const int*)s.counts,
                                          narrow_ctas(p->rows, dev.sms), p->reduction, p->loss, p->info),
                        what);
        if (rc) return rc;
        count_launch();
        return RB200_OK;
    }
    wait.status = p->status;
    for (long long c0 = 0; c0 < p->classes; c0 += s.piece) {
        const int classes = (int)(p->classes - c0 < s.piece ? p->classes - c0 : s.piece);
        const GemmPlan plan = stats_gemm(*p, dev, classes);
        EpiArgs e = label_args(*p);
        e.bias = p->bias ? at_row(p->bias, 1, c0) : nullptr;
        e.class0 = (int)c0;
        e.part = s.part;
        e.parts = 2 * plan.tiles_n;
        e.want_zsum = p->label_smoothing > 0.0f;
        e.zlabel = p->stats + 2 * p->rows;
        e.clear = p->info;
        const Operand w = operand(at_row(s.w.use.data, s.w.use.ld, c0), s.w.use.ld, classes, p->features, false);
        if ((rc = gemm_launch<EPI_CE_STATS, false, false>(bf16, s.x.use, w, nullptr, nullptr, plan, e, wait, stream, what))) return rc;
        MergeArgs m = {};
        m.part = s.part;
        m.parts = e.parts;
        m.want_zsum = e.want_zsum;
        m.labels = p->labels;
        m.label_bytes = p->label_bytes;
        m.classes = (int)p->classes;
        m.rows = (int)p->rows;
        m.reduction = p->reduction;
        m.ignore_index = p->ignore_index;
        m.smoothing = p->label_smoothing;
        m.first = c0 == 0;
        m.last = c0 + classes == p->classes;
        m.stats = p->stats;
        m.zsum = s.zsum;
        m.loss = p->loss;
        m.info = p->info;
        m.block_sums = s.block_sums;
        if ((rc = merge_launch(m, stream, what))) return rc;
    }
    return RB200_OK;
}

// ---- backward -----------------------------------------------------------------------------------------------------
struct GradPlan {
    Packed x, w;
    bool narrow;
    float* dw_part;             // narrow: [CTAs][classes][ldpart]
    long long ldpart;
    Operand clean;              // x without the rows that do not count
    bool by_rows;               // pieces are cut along the rows
    int piece, pieces;
    long long ldd;              // of the piece's gradients
    void* dz;
    float *coef, *factor, *tops;
    float* sum;                 // 32-bit sums over pieces: dx (pieces of classes) or dweight (pieces of rows)
    long long ldsum;
    void *px, *pw;              // partial products
    float* col_part;            // [rows / 32][ldcol] column sums
    long long ldcol;
    size_t bytes;
};
static int piece_rows(const rb200_linear_ce_params& p, const GradPlan& g, int i) {
    if (!g.by_rows) return (int)p.rows;
    const long long left = p.rows - (long long)i * g.piece;
    return (int)(left < g.piece ? left : g.piece);
}
static int piece_classes(const rb200_linear_ce_params& p, const GradPlan& g, int i) {
    if (g.by_rows) return (int)p.classes;
    const long long left = p.classes - (long long)i * g.piece;
    return (int)(left < g.piece ? left : g.piece);
}
static GradPlan plan_grad(const rb200_linear_ce_params& p, const DeviceInfo& dev, void* ws) {
    GradPlan g = {};
    Carver c(ws);
    const int k = (int)p.features;
    g.x = plan_pack(operand(p.x, p.ldx, p.rows, k, false), &c);
    g.w = plan_pack(operand(p.weight, p.ldw, p.classes, k, false), &c);
    if (p.reduction == RB200_REDUCE_NONE) {
        g.coef = (float*)c.take((size_t)p.rows * sizeof(float));
        g.factor = (float*)c.take(sizeof(float));
        g.tops = (float*)c.take(kFactorBlocks * sizeof(float));
    }
    g.narrow = narrow_fits(p.classes, p.features);
    if (g.narrow) {
        g.ldpart = round_up(k + 1, 4);
        if (p.dweight || p.dbias) g.dw_part = (float*)c.take((size_t)narrow_ctas(p.rows, dev.sms) * p.classes * g.ldpart * sizeof(float));
        g.bytes = c.used;
        return g;
    }
    g.by_rows = p.rows > p.classes;
    const long long longer = g.by_rows ? p.rows : p.classes, shorter = g.by_rows ? p.classes : p.rows;
    long long piece = (long long)(kPieceBytes / 2) / shorter / kTileNMax * kTileNMax;
    if (piece < kTileNMax) piece = kTileNMax;
    if (piece < longer) {   // pieces of about one size
        const long long pieces = (longer + piece - 1) / piece;
        piece = round_up((longer + pieces - 1) / pieces, kTileNMax);
    }
    g.piece = (int)(piece < longer ? piece : longer);
    g.pieces = (int)((longer + g.piece - 1) / g.piece);
    g.ldd = round_up(piece_classes(p, g, 0), 8);
    g.dz = c.take((size_t)g.ldd * piece_rows(p, g, 0) * 2);
    if (p.dweight) {
        g.clean = operand(nullptr, round_up(k, 8), p.rows, k, true);
        g.clean.data = c.take((size_t)g.clean.ld * p.rows * 2);
    }
    g.ldsum = round_up(k, 4);
    if (g.pieces > 1 && (g.by_rows ? p.dweight : p.dx)) g.sum = (float*)c.take((size_t)shorter * g.ldsum * sizeof(float));
    // the last piece is the only one of another size
    size_t px = 0, pw = 0;
    for (int i = 0; i < g.pieces; i += g.pieces > 1 ? g.pieces - 1 : 1) {
        const int rows = piece_rows(p, g, i), classes = piece_classes(p, g, i);
        const size_t bx = gemm_partial_bytes(gemm_plan(dev, rows, k, classes, true, true), rows, k);
        const size_t bw = gemm_partial_bytes(gemm_plan(dev, classes, k, rows, true, true), classes, k);
        if (bx > px) px = bx;
        if (bw > pw) pw = bw;
    }
    if (p.dx) g.px = c.take(px);
    if (p.dweight) g.pw = c.take(pw);
    g.ldcol = round_up(piece_classes(p, g, 0), 32);
    if (p.dbias) g.col_part = (float*)c.take((size_t)((p.rows + 31) / 32) * g.ldcol * sizeof(float));
    g.bytes = c.used;
    return g;
}

template <typename T>
static int narrow_join(const NarrowArgs& a, const rb200_linear_ce_params& p, const DeviceInfo& dev, cudaStream_t stream, const char* what) {
    const dim3 grid((unsigned)((a.features + (p.dbias ? 1 : 0) + 31) / 32), (unsigned)a.classes);
    const int rc = check_cuda(launch_overlapped(narrow_join_kernel<T>, grid, dim3(256), 0, stream, (const float*)a.dw_part,
                                                narrow_ctas(a.rows, dev.sms), a.classes, a.features, a.ldpart, (T*)p.dweight, (long long)p.lddw,
                                                (T*)p.dbias, a.scale),
                              what);
    if (rc) return rc;
    count_launch();
    return RB200_OK;
}
static int ce_backward(const rb200_linear_ce_params* p, cudaStream_t stream, GemmWait wait) {
    const char* what = "rb200k_linear_ce_backward";
    if (!p) {
        set_error("%s: params is null", what);
        return RB200_E_INVALID;
    }
    int rc = check_sizes(what, *p);
    if (rc) return rc;
    const long long n = p->rows, v = p->classes, k = p->features;
    if (p->dweight && (rc = check_matrix(what, "dweight", p->dweight, p->lddw, v, k))) return rc;
    if (p->dbias && (rc = check_matrix(what, "dbias", p->dbias, 0, 1, v))) return rc;
    if (n == 0) {
        if (p->dweight && (rc = clear_matrix(p->dweight, p->lddw, v, k, stream, what))) return rc;
        if (p->dbias && (rc = clear_matrix(p->dbias, 0, 1, v, stream, what))) return rc;
        return RB200_OK;
    }
    if (!p->dx && !p->dweight && !p->dbias) return RB200_OK;
    if ((rc = check_common(what, *p))) return rc;
    if (p->dx && (rc = check_matrix(what, "dx", p->dx, p->lddx, n, k))) return rc;
    if (!p->dloss || ((uintptr_t)p->dloss & 3)) {
        set_error("%s: dloss is null or not aligned", what);
        return RB200_E_INVALID;
    }
    DeviceInfo dev;
    if ((rc = device_info(&dev))) return rc;
    const GradPlan g = plan_grad(*p, dev, p->workspace);
    if ((rc = check_workspace(what, p->workspace, p->workspace_bytes, g.bytes))) return rc;
    const bool bf16 = p->dtype == RB200_BF16;
    wait.status = p->status;
    if ((rc = pack_operands(&g.x, &g.w, stream, what))) return rc;
    const bool none = p->reduction == RB200_REDUCE_NONE;
    if (none && (rc = factors_launch(*p, g.tops, g.coef, g.factor, stream, what))) return rc;
    const Scale scale(1.0f / 32768.0f, none ? g.factor : p->dloss, p->reduction == RB200_REDUCE_MEAN ? p->info : nullptr);
    if (g.narrow) {
        NarrowArgs a = narrow_args(*p, wait);
        a.coef = none ? g.coef : nullptr;
        a.dirty = p->info + 1;
        a.dx = p->dx;
        a.lddx = p->lddx;
        a.vec_dx = ((uintptr_t)p->dx & 15) == 0 && (n == 1 || (p->lddx & 7) == 0);
        a.scale = scale;
        a.dw_part = g.dw_part;
        a.ldpart = g.ldpart;
        a.want_dw = p->dweight != nullptr;
        a.want_db = p->dbias != nullptr;
        if ((rc = narrow_launch(a, true, bf16, g.x.use, g.w.use, dev, stream, what)) || !g.dw_part) return rc;
        return bf16 ? narrow_join<__nv_bfloat16>(a, *p, dev, stream, what) : narrow_join<__half>(a, *p, dev, stream, what);
    }
    for (int i = 0; i < g.pieces; i++) {
        const int rows = piece_rows(*p, g, i), classes = piece_classes(*p, g, i);
        const long long r0 = g.by_rows ? (long long)i * g.piece : 0, c0 = g.by_rows ? 0 : (long long)i * g.piece;
        const Operand x = operand(at_row(g.x.use.data, g.x.use.ld, r0), g.x.use.ld, rows, k, false);
        const Operand w = operand(at_row(g.w.use.data, g.w.use.ld, c0), g.w.use.ld, classes, k, false);
        Operand dz = operand(g.dz, g.ldd, rows, classes, false);
        EpiArgs e = label_args(*p);
        e.labels = (const uint8_t*)p->labels + r0 * p->label_bytes;
        e.bias = p->bias ? at_row(p->bias, 1, c0) : nullptr;
        e.class0 = (int)c0;
        e.stats = p->stats + r0;
        e.stats_stride = n;
        e.coef = none ? g.coef + r0 : nullptr;
        if (p->dbias) {   // pieces of the rows keep their sums until the last one
            e.col_part = g.col_part + (r0 >> 5) * g.ldcol;
            e.ldcol = g.ldcol;
        }
        e.out = g.dz;
        e.ldo = g.ldd;
        // Rows that do not count but hold inf or NaN would reach dweight as 0 * NaN: if the forward pass found any, the
        // first launch also makes a copy of x with those rows zeroed.
        if (p->dweight && i == 0) {
            e.clean = const_cast<void*>(g.clean.data);
            e.ldclean = g.clean.ld;
            e.clean_src = p->x;
            e.ldsrc = p->ldx;
            e.clean_rows = n;
            e.clean_labels = p->labels;
            e.dirty = p->info + 1;
        }
        const GemmPlan plan = gemm_plan(dev, rows, classes, (int)k, false, false);
        if ((rc = gemm_launch<EPI_CE_GRAD, false, false>(bf16, x, w, nullptr, nullptr, plan, e, wait, stream, what))) return rc;
        const bool first = i == 0, last = i == g.pieces - 1;
        if (p->dx) {
            EpiArgs o = {};
            Operand wt = w;
            wt.transposed = true;
            if (g.by_rows || g.pieces == 1) {
                o.out = const_cast<uint8_t*>(at_row(p->dx, p->lddx, r0));
                o.ldo = p->lddx;
            } else {   // a piece of the classes gives a summand of dx
                o.acc_in = first ? nullptr : g.sum;
                o.acc_out = last ? nullptr : g.sum;
                o.ldacc = g.ldsum;
                o.out = p->dx;
                o.ldo = p->lddx;
            }
            o.scale = scale;
            if ((rc = gemm_store_joined(GEMM_KN, bf16, dz, wt, nullptr, nullptr, gemm_plan(dev, rows, (int)k, classes, true, true), o, g.px, wait,
                                        stream, what)))
                return rc;
        }
        if (p->dweight) {
            EpiArgs o = {};
            Operand xt = x, clean = g.clean, dzt = dz;
            xt.transposed = dzt.transposed = true;
            clean.data = at_row(clean.data, clean.ld, r0);
            clean.rows = rows;
            if (!g.by_rows || g.pieces == 1) {
                o.out = const_cast<uint8_t*>(at_row(p->dweight, p->lddw, c0));
                o.ldo = p->lddw;
            } else {
                o.acc_in = first ? nullptr : g.sum;
                o.acc_out = last ? nullptr : g.sum;
                o.ldacc = g.ldsum;
                o.out = p->dweight;
                o.ldo = p->lddw;
            }
            o.scale = scale;
            if ((rc = gemm_store_joined(GEMM_NN, bf16, dzt, xt, &clean, p->info + 1, gemm_plan(dev, classes, (int)k, rows, true, true), o, g.pw,
                                        wait, stream, what)))
                return rc;
        }
        if (p->dbias && (!g.by_rows || last)) {
            const int planes = (int)((r0 + rows + 31) / 32);   // a piece of the rows starts on a multiple of 256
            if ((rc = sum_planes(bf16, g.col_part, g.ldcol, planes, classes, const_cast<uint8_t*>(at_row(p->dbias, 1, c0)), scale, stream, what)))
                return rc;
        }
    }
    return RB200_OK;
}

}  // namespace rb200

using namespace rb200;

static const GemmWait kNoProbe = {nullptr, 0, -1};

extern "C" uint64_t rb200k_linear_ce_workspace_bytes(const rb200_linear_ce_params* p) {
    DeviceInfo dev;
    if (!p || check_sizes("rb200k_linear_ce_workspace_bytes", *p) || p->rows == 0 || device_info(&dev)) return 0;
    return plan_stats(*p, dev, nullptr).bytes;
}
extern "C" int rb200k_linear_ce(const rb200_linear_ce_params* p, void* stream) { return ce_forward(p, (cudaStream_t)stream, kNoProbe); }
extern "C" uint64_t rb200k_linear_ce_backward_workspace_bytes(const rb200_linear_ce_params* p) {
    DeviceInfo dev;
    if (!p || check_sizes("rb200k_linear_ce_backward_workspace_bytes", *p) || p->rows == 0 || device_info(&dev)) return 0;
    return plan_grad(*p, dev, nullptr).bytes;
}
extern "C" int rb200k_linear_ce_backward(const rb200_linear_ce_params* p, void* stream) { return ce_backward(p, (cudaStream_t)stream, kNoProbe); }
extern "C" int rb200k_linear_ce_probe(const rb200_linear_ce_params* p, void* stream, int backward, uint64_t wait_cycles, int skip_block) {
    const GemmWait wait = {nullptr, wait_cycles, skip_block};
    return backward ? ce_backward(p, (cudaStream_t)stream, wait) : ce_forward(p, (cudaStream_t)stream, wait);
}
