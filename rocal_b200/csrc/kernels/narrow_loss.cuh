// Softmax cross entropy of x W^T + b for few classes and features (a detection head: tens of classes for every anchor of a
// batch), in one sweep over x each way. The rows are all of the data, so what counts is that x is read once:
//   W lies in shared memory for the whole launch; a CTA takes tiles of 128 rows, x arriving in chunks of 64 features,
//   forward   scores into TMEM, a thread per row makes maximum, sum of exponentials and loss,
//   backward  scores again, a thread per row turns them into (softmax - target) in the element type, written to shared memory as the
//             tensor cores read it; then dx = dz W leaves at once, and W's gradient stays in TMEM over all of the CTA's tiles,
//             with the same chunks of x as its other operand. CTAs' sums are joined by narrow_join_kernel in a fixed
//             order, with the column sums for the bias.
// Against the general way (scores' gradients through memory, x read for each product), 279424 x 256, 81 classes, bf16: forward
// 31 us (43), backward 74 us (156). Forward it is bound by the read of x (143 MB at 5 TB/s). Backwards a tile takes 7100 clocks, most
// of them one after another, since shared memory has no room for a third tile of x: scores 1300, softmax 2000, the other two products
// 3000, handshakes 800. The products are bound by the read of their operands (some 64 bytes a clock: 128 clocks for 128 x 128 x 16, so
// W's gradient is made 256 columns at a time: 79 us with 128). Tried and slower: sixteen softmax warps (91 us), the next scores ahead of
// dx with the softmax holding its results until dz is read (93 us), column sums by shuffles for every tile (2 us).
// Warps: 0 copies, 1 issues products, 2 allocates TMEM, 4-11 softmax (forward: two groups take turns; backward: two warps share a
// row), 12-15 dx. Rows that do not count but hold inf or NaN (the forward pass found some) are zeroed in shared memory before W's gradient.
#pragma once

#include "matrix_args.cuh"

namespace rb200 {

constexpr int kNarrowClasses = 128, kNarrowFeatures = 256;
constexpr int kNarrowSlots = 8;
constexpr int narrow_threads(bool grad) { return grad ? 512 : 384; }
constexpr uint32_t kChunkBytes = kTileM * kTileK * 2;   // 128 rows x 64 features
constexpr uint32_t kNarrowSmem = 232448 - 2048;         // 227 KB, without the kernel's own KB and what aligning the start may take
enum { kNarrowDw = 128, kNarrowDx = 384 };              // TMEM columns: scores at 0 (forward: and at 128)

struct NarrowArgs {
    CUtensorMap x, w;
    int rows, features, classes;
    int vb;                   // classes in whole strips of 32
    int chunks;               // of a tile and of W; backwards an even number (the last may be zeros)
    int slots;                // of the ring: a multiple of chunks
    uint32_t idesc_s, idesc_x, idesc_w;
    const void* bias;         // T[classes] or null
    const void* labels;
    int label_bytes;
    long long ignore_index;
    float smoothing, smooth_on, smooth_off, inv_classes;   // s, 1 - s, s / classes, 1 / classes
    int none;                 // forward: a loss for every row
    float* stats;             // [3][rows]
    float* loss;              // forward, none: [rows]
    double* sums;             // forward: [CTAs] losses
    int* counts;              // forward: [2][CTAs] rows that count, and whether a row that does not holds inf or NaN
    const float* coef;        // backward: [rows] or null
    const int* dirty;         // backward
    void* dx;                 // backward: T[rows][lddx] or null
    long long lddx;
    int vec_dx;
    Scale scale;
    float* dw_part;           // backward: [CTAs][classes][ldpart]; column `features` takes the bias's sum
    long long ldpart;
    int want_dw, want_db;
    int* status;
    unsigned long long wait_cycles;   // 0: the ordinary limit
    int skip_chunk;           // copies of x's chunks from this one on are left out (-1: none)
};

static __host__ __device__ inline uint32_t narrow_smem(int vb, int chunks, int slots, bool grad) {
    return (uint32_t)chunks * vb * 128 + slots * kChunkBytes + (grad ? 2 * kChunkBytes + 4 * kStageBytes : 0);
}

// Sums of 16 columns over the warp's lanes: at every step a lane keeps the half of its columns that its own number's next bit names
// and hands the other half to its partner. Lanes l and l + 16 end with column l.
__device__ __forceinline__ float column_sums(float (&v)[16], int lane) {
#pragma unroll
    for (int w = 8; w; w >>= 1) {
        const bool upper = lane & w;
#pragma unroll
        for (int i = 0; i < w; i++) {
            const float keep = upper ? v[i + w] : v[i], send = upper ? v[i] : v[i + w];
            v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, send, w);
        }
    }
    return v[0] + __shfl_xor_sync(0xFFFFFFFFu, v[0], 16);
}

template <typename T, bool GRAD>
__global__ void __launch_bounds__(narrow_threads(GRAD), 1) ce_narrow_kernel(const __grid_constant__ NarrowArgs g) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kNarrowSlots + 9];
    __shared__ uint32_t tmem_addr_s;
    __shared__ int gave_up_s;
    __shared__ __align__(16) float bias_s[kNarrowClasses];
    __shared__ double sums_s[8];
    __shared__ int counts_s[2][8];

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t w0 = (tc::smem_u32(smem_raw) + 1023u) & ~1023u, w_chunk = (uint32_t)g.vb * 128, x0 = w0 + g.chunks * w_chunk;
    const uint32_t dz0 = x0 + g.slots * kChunkBytes, stage0 = dz0 + 2 * kChunkBytes;
    const uint32_t bar0 = tc::smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (kNarrowSlots + s); };
    auto s_full = [&](int b) { return bar0 + 8u * (2 * kNarrowSlots + b); };
    auto s_empty = [&](int b) { return bar0 + 8u * (2 * kNarrowSlots + 2 + b); };   // backward: 0 = dz written, 1 = dz read
    const uint32_t dx_full = bar0 + 8u * (2 * kNarrowSlots + 4), dx_empty = dx_full + 8, w_full = dx_full + 16, done = dx_full + 24,
                   drained = dx_full + 32;
    const uint32_t dz_full = s_empty(0), dz_empty = s_empty(1);

    if (threadIdx.x == 0) {
        gave_up_s = 0;
        for (int s = 0; s < kNarrowSlots; s++) {
            tc::bar_init(full(s), 1);
            tc::bar_init(empty(s), 1);
        }
        tc::bar_init(s_full(0), 1);
        tc::bar_init(s_full(1), 1);
        tc::bar_init(s_empty(0), GRAD ? 8 : 4);
        tc::bar_init(s_empty(1), GRAD ? 1 : 4);
        tc::bar_init(dx_full, 1);
        tc::bar_init(dx_empty, 4);
        tc::bar_init(w_full, 1);
        tc::bar_init(done, 1);
        tc::bar_init(drained, 1);
        tc::bar_init_fence();
        tc::prefetch_map(&g.x);
        tc::prefetch_map(&g.w);
    }
    if (warp == 2) tc::tmem_alloc<1>(tc::smem_u32(&tmem_addr_s));
    pdl_launch_dependents();
    pdl_wait();   // everything above touches this CTA's own state only
    if (threadIdx.x < kNarrowClasses)
        bias_s[threadIdx.x] = g.bias && threadIdx.x < g.classes ? Elem<T>::to_float(reinterpret_cast<const T*>(g.bias)[threadIdx.x]) : 0.0f;
    if (threadIdx.x < 8) {
        sums_s[threadIdx.x] = 0.0;
        counts_s[0][threadIdx.x] = counts_s[1][threadIdx.x] = 0;
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_addr_s;
    const tc::Patience patience = {&gave_up_s, g.status, g.wait_cycles};
    const int tiles = (g.rows + kTileM - 1) / kTileM;   // rows up to 2^30
    const int real = (g.features + kTileK - 1) / kTileK, halves = (g.features + 127) / 128;
    const bool want_dx = GRAD && g.dx, want_dw = GRAD && g.want_dw;

    if (warp == 0) {
        if (tc::elect_one()) {
            int s = 0;
            uint32_t phase = 0;
            long long filled = 0;
            tc::bar_expect(w_full, g.chunks * w_chunk);
            for (int c = 0; c < g.chunks; c++) tc::tma_load<1>(w0 + c * w_chunk, &g.w, c * kTileK, 0, w_full);
            bool ok = true;
            for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                for (int c = 0; c < g.chunks; c++) {
                    ok = tc::bar_wait(empty(s), phase ^ 1, patience);
                    if (!ok) break;
                    tc::bar_expect(full(s), kChunkBytes);
                    if (g.skip_chunk < 0 || c < g.skip_chunk) tc::tma_load<1>(x0 + s * kChunkBytes, &g.x, c * kTileK, t * kTileM, full(s));
                    filled++;
                    if (++s == g.slots) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
            // Copies still on their way into this CTA. The products wait for every one of them, but may have given up, also when this
            // warp is through.
            tc::bar_drain(w_full, 0, g.wait_cycles);
            for (int i = 0; i < g.slots && i < filled; i++) {
                if (s == 0) {
                    s = g.slots;
                    phase ^= 1;
                }
                s--;
                tc::bar_drain(full(s), phase, g.wait_cycles);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (tc::elect_one()) {
            bool ok = true;
            int s = 0, it = 0, pieces = 0;   // the ring's next chunk; tiles; pieces of dx
            uint32_t phase = 0;
            // scores of the tile whose chunks come next, as they come
            auto scores = [&](uint32_t d, uint32_t bar) {
                for (int c = 0; c < g.chunks; c++) {
                    if (!tc::bar_wait(full(s), phase, patience)) return false;
                    tc::fence_after();
                    if (c < real) {
                        const uint64_t a = tc::operand_desc(x0 + s * kChunkBytes, false, 0), b = tc::operand_desc(w0 + c * w_chunk, false, 0);
#pragma unroll
                        for (int k = 0; k < 4; k++) tc::mma_f16<1>(d, a + k * 2, b + k * 2, g.idesc_s, c > 0 || k > 0);
                    }
                    if (!GRAD) tc::mma_commit<1>(empty(s));
                    if (++s == g.slots) {
                        s = 0;
                        phase ^= 1;
                    }
                }
                tc::mma_commit<1>(bar);
                return true;
            };
            ok = tc::bar_wait(w_full, 0, patience);
            if constexpr (!GRAD) {
                for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, it++) {
                    ok = tc::bar_wait(s_empty(it & 1), (it >> 1 & 1) ^ 1, patience);
                    if (!ok) break;
                    tc::fence_after();
                    ok = scores(tmem + (it & 1) * 128, s_full(it & 1));
                }
            } else {
                int first = 0;   // slot of the tile's first chunk
                if (ok) ok = scores(tmem, s_full(0));
                for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, it++) {
                    ok = tc::bar_wait(dz_full, it & 1, patience);
                    if (!ok) break;
                    tc::fence_after();
                    auto gradient_of_x = [&](int h) {
                        if (!tc::bar_wait(dx_empty, (pieces & 1) ^ 1, patience)) return false;
                        pieces++;
                        tc::fence_after();
                        const uint64_t b = tc::operand_desc(w0 + 2 * h * w_chunk, true, w_chunk);
                        for (int k = 0; k < g.vb / 16; k++) {
                            const uint64_t a = tc::operand_desc(dz0 + (k >> 2) * kChunkBytes, false, 0);
                            tc::mma_f16<1>(tmem + kNarrowDx, a + (k & 3) * 2, b + k * 128, g.idesc_x, k > 0);
                        }
                        tc::mma_commit<1>(dx_full);
                        return true;
                    };
                    if (want_dx && !(ok = gradient_of_x(0))) break;
                    if (want_dw) {
                        const uint64_t a = tc::operand_desc(dz0, true, kChunkBytes), b = tc::operand_desc(x0 + first * kChunkBytes, true, kChunkBytes);
#pragma unroll
                        for (int k = 0; k < 8; k++) tc::mma_f16<1>(tmem + kNarrowDw, a + k * 128, b + k * 128, g.idesc_w, it > 0 || k > 0);
                    }
                    for (int c = 0; c < g.chunks; c++) tc::mma_commit<1>(empty(first + c));
                    first = first + g.chunks == g.slots ? 0 : first + g.chunks;
                    if (want_dx && halves > 1 && !(ok = gradient_of_x(1))) break;
                    tc::mma_commit<1>(dz_empty);
                    if (t + (int)gridDim.x < tiles) ok = scores(tmem, s_full(0));   // dz says that the scores before have been read
                }
                if (ok) tc::mma_commit<1>(done);
            }
            tc::mma_commit<1>(drained);   // products still running: the other warps wait for all of them, but may have given up
            tc::bar_drain(drained, 0, g.wait_cycles);
        }
        __syncwarp();
    } else if (GRAD && warp >= 4 && warp < 12) {   // softmax - target; two warps share a row's classes
        const int quarter = warp & 3, share = warp - 4 >> 2, half = g.vb / 2, line = quarter * 32 + lane;
        const uint32_t acc = tmem + share * half + ((uint32_t)(quarter * 32) << 16);
        constexpr int kStrips = kNarrowClasses / 32, kKept = 3;   // of 16 classes
        // Column sums: a lane adds up what it has of every tile, and the lanes join theirs at the end; of a fourth strip, for which there
        // are no registers left, after every tile.
        float2 kept[kKept][8] = {};
        float last = 0.0f;
        const bool dirty = *g.dirty, zero_rows = want_dw && dirty;
        int it = 0, first = 0;
        // what does not depend on the products is on its way a tile ahead
        struct {
            int label;
            bool counted;
            float m, s, zl, coef;
        } next;
        auto fetch = [&](int t) {
            const int row = t * kTileM + line;
            next.label = -1;
            next.counted = false;
            next.m = next.zl = 0.0f;
            next.s = next.coef = 1.0f;
            if (t < tiles && row < g.rows) {
                next.label = load_label(g.labels, g.label_bytes, row, g.ignore_index, g.classes, &next.counted);
                next.m = g.stats[row];
                next.s = g.stats[(long long)g.rows + row];
                next.zl = g.stats[2ll * g.rows + row];
                if (g.coef) next.coef = g.coef[row];
            }
        };
        fetch(blockIdx.x);
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, it++) {
            const bool counted = next.counted;
            const int label = counted ? next.label : -1;
            // (softmax - target) * factor = exp(z - top) * mul + add, and at the label
            // rows that do not count: exp(z - inf) * 0 + 0, except where z may be inf or NaN (behind the last row: 0 times W)
            const float factor = counted ? next.coef * 32768.0f : 0.0f, top = counted ? finite_max(next.m) : INFINITY;
            const float mul = counted ? factor / next.s : 0.0f, add = -g.smooth_off * factor;
            const float at_label = exp_diff(next.zl - top) * mul + add - g.smooth_on * factor;
            const bool clear = !counted && (dirty || t * kTileM + line >= g.rows);
            fetch(t + gridDim.x);
            // the lanes leave together: what follows needs whole warps
            if (!__all_sync(0xFFFFFFFFu, tc::bar_wait(s_full(0), it & 1, patience) && tc::bar_wait(dz_empty, (it & 1) ^ 1, patience))) break;
            tc::fence_after();
            const float2 off = make_float2(-top, -top), unit = make_float2(kLog2e, kLog2e);
            const float2 mul_v = make_float2(mul, mul), add_v = make_float2(add, add);
#pragma unroll
            for (int c = 0; c < kStrips; c++) {
                if (c * 16 >= half) break;
                const int col = share * half + c * 16, count = clear ? 0 : g.classes - col, l = label - col;
                uint32_t raw[16];
                tc::tmem_load16(acc + c * 16, raw);
                tc::tmem_wait();
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 b = *reinterpret_cast<const float4*>(bias_s + col + i);
                    const float2 z[2] = {add2(make_float2(__uint_as_float(raw[i]), __uint_as_float(raw[i + 1])), make_float2(b.x, b.y)),
                                         add2(make_float2(__uint_as_float(raw[i + 2]), __uint_as_float(raw[i + 3])), make_float2(b.z, b.w))};
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float2 d = mul2(add2(z[j], off), unit);
                        const float2 p = fma2(make_float2(exp2_fast(d.x), exp2_fast(d.y)), mul_v, add_v);
                        v[i + 2 * j] = p.x;
                        v[i + 2 * j + 1] = p.y;
                    }
                }
                if (l >= 0 && l < 16) {
#pragma unroll
                    for (int i = 0; i < 16; i++) v[i] = i == l ? at_label : v[i];
                }
                if (count < 16) {   // beyond the classes; rows that may hold anything
#pragma unroll
                    for (int i = 0; i < 16; i++) v[i] = i < count ? v[i] : 0.0f;
                }
                // rounded to the element type: an operand of two products (column sums are made of what it was before)
#pragma unroll
                for (int i = 0; i < 2; i++) {   // piece j of line r lies at j ^ (r % 8): the 128-byte swizzle
                    const int piece = col / 8 + i;
                    st_shared16(dz0 + (piece >> 3) * kChunkBytes + line * 128 + (((piece & 7) ^ (line & 7)) << 4), pack8<T>(v + 8 * i));
                }
                if (g.want_db) {
                    if (c < kKept) {
#pragma unroll
                        for (int i = 0; i < 8; i++) kept[c < kKept ? c : 0][i] = add2(kept[c < kKept ? c : 0][i], make_float2(v[2 * i], v[2 * i + 1]));
                    } else {
                        last += column_sums(v, lane);
                    }
                }
            }
            tc::fence_before();
            if (zero_rows && !counted && share == 0) {
                for (int c = 0; c < g.chunks; c++)
#pragma unroll
                    for (int i = 0; i < 8; i++) st_shared16(x0 + (first + c) * kChunkBytes + line * 128 + i * 16, make_uint4(0, 0, 0, 0));
            }
            first = first + g.chunks == g.slots ? 0 : first + g.chunks;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the tensor cores read what was written
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(dz_full) : "memory");
        }
        if (g.want_db && __all_sync(0xFFFFFFFFu, tc::bar_wait(done, 0, patience))) {   // nothing reads dz any more: [4][128] column sums
#pragma unroll
            for (int c = 0; c < kStrips; c++) {
                float s = last;
                if (c < kKept) {
                    float v[16];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        v[2 * i] = kept[c < kKept ? c : 0][i].x;
                        v[2 * i + 1] = kept[c < kKept ? c : 0][i].y;
                    }
                    s = column_sums(v, lane);
                }
                if (c * 16 < half && lane < 16)
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(dz0 + (quarter * kNarrowClasses + share * half + c * 16 + lane) * 4), "f"(s) : "memory");
            }
        }
    } else if (!GRAD && warp >= 4 && warp < 12) {   // a group of four takes every other tile
        const int quarter = warp & 3, group = warp - 4 >> 2;
        const uint32_t acc = tmem + group * 128 + ((uint32_t)(quarter * 32) << 16);
        double mine = 0.0;
        int counts = 0, dirts = 0, it = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, it++) {
            if ((it & 1) != group) continue;
            const int row = t * kTileM + quarter * 32 + lane;
            const bool row_ok = row < g.rows;
            bool counted = false;
            int label = -1;
            if (row_ok) label = load_label(g.labels, g.label_bytes, row, g.ignore_index, g.classes, &counted);
            // the lanes leave together: what follows needs whole warps
            if (!__all_sync(0xFFFFFFFFu, tc::bar_wait(s_full(group), it >> 1 & 1, patience))) break;
            tc::fence_after();
            RunningSoftmax run = {-INFINITY, 0.0f};
            float z_label = 0.0f, zsum = 0.0f;
#pragma unroll
            for (int c = 0; c < kNarrowClasses / 32; c++) {
                const int count = g.classes - c * 32;
                if (count <= 0) break;
                uint32_t raw[32];
                tc::tmem_load32(acc + c * 32, raw);
                tc::tmem_wait();
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 b = *reinterpret_cast<const float4*>(bias_s + c * 32 + i);
                    v[i] = __uint_as_float(raw[i]) + b.x;
                    v[i + 1] = __uint_as_float(raw[i + 1]) + b.y;
                    v[i + 2] = __uint_as_float(raw[i + 2]) + b.z;
                    v[i + 3] = __uint_as_float(raw[i + 3]) + b.w;
                }
                const int l = label - c * 32;
                if (l >= 0 && l < 32) {   // element l of the strip, by its bits
                    float a[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) a[i] = l & 16 ? v[i + 16] : v[i];
#pragma unroll
                    for (int w = 8; w; w >>= 1)
#pragma unroll
                        for (int i = 0; i < w; i++) a[i] = l & w ? a[i + w] : a[i];
                    z_label = a[0];
                }
                if (g.smoothing > 0.0f) {   // four sums, not one chain of 32; of z / classes, as in gemm.cuh
                    const float2 inv = make_float2(g.inv_classes, g.inv_classes);
                    float2 sum[2] = {};
                    if (count >= 32) {
#pragma unroll
                        for (int i = 0; i < 32; i += 2) sum[i >> 1 & 1] = fma2(make_float2(v[i], v[i + 1]), inv, sum[i >> 1 & 1]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 2)
                            sum[i >> 1 & 1] = fma2(make_float2(i < count ? v[i] : 0.0f, i + 1 < count ? v[i + 1] : 0.0f), inv, sum[i >> 1 & 1]);
                    }
                    zsum += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                }
                if (count < 32) {
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (i >= count) v[i] = -INFINITY;
                }
                float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int i = 4; i < 32; i += 4)
#pragma unroll
                    for (int j = 0; j < 4; j++) m[j] = fmaxf(m[j], v[i + j]);
                const float now = fmaxf(run.m, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]))), base = finite_max(now);
                run.s *= exp_diff(run.m - base);
                run.m = now;
                float2 sum[2] = {};
                const float2 off = make_float2(-base, -base), unit = make_float2(kLog2e, kLog2e);
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 d = mul2(add2(make_float2(v[i], v[i + 1]), off), unit);
                    sum[i >> 1 & 1] = add2(sum[i >> 1 & 1], make_float2(exp2_fast(d.x), exp2_fast(d.y)));
                }
                run.s += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::bar_arrive_relaxed(s_empty(group));
            if (row_ok) {
                float loss = 0.0f;
                if (counted) {
                    counts++;
                    if (label < 0) {
                        run.m = run.s = loss = nanf("");
                    } else {
                        const float lse = logf(run.s);   // above the maximum
                        loss = g.smooth_on * (lse + (run.m - z_label));
                        if (g.smoothing > 0.0f) loss += g.smoothing * (lse + (run.m - zsum));
                    }
                } else {
                    dirts |= !(isfinite(run.m) && isfinite(run.s));
                }
                mine += loss;
                if (g.none) g.loss[row] = loss;
                g.stats[row] = run.m;
                g.stats[(long long)g.rows + row] = run.s;
                g.stats[2ll * g.rows + row] = z_label;
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) mine += __shfl_xor_sync(0xFFFFFFFFu, mine, d);
        counts = __reduce_add_sync(0xFFFFFFFFu, counts);
        dirts = __any_sync(0xFFFFFFFFu, dirts);
        if (lane == 0) {
            sums_s[warp - 4] = mine;
            counts_s[0][warp - 4] = counts;
            counts_s[1][warp - 4] = dirts;
        }
    } else if (GRAD && warp >= 12) {
        const int quarter = warp & 3;
        const uint32_t area = stage0 + quarter * kStageBytes, lanes = (uint32_t)(quarter * 32) << 16;
        const float scale = g.scale.value();
        int pieces = 0;
        bool ok = true;
        for (int t = blockIdx.x; want_dx && t < tiles && ok; t += gridDim.x) {
            const int row0 = t * kTileM + quarter * 32;
            for (int h = 0; h < halves; h++, pieces++) {
                ok = __all_sync(0xFFFFFFFFu, tc::bar_wait(dx_full, pieces & 1, patience));
                if (!ok) break;
                tc::fence_after();
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    uint32_t raw[2][32];
                    tc::tmem_load32(tmem + kNarrowDx + q * 64 + lanes, raw[0]);
                    tc::tmem_load32(tmem + kNarrowDx + q * 64 + 32 + lanes, raw[1]);
                    tc::tmem_wait();
                    if (q == 1) {   // the accumulator is in registers
                        tc::fence_before();
                        __syncwarp();
                        if (lane == 0) tc::bar_arrive_relaxed(dx_empty);
                    }
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const int col = h * 128 + q * 64 + s * 32, count = g.features - col;
                        if (count <= 0 || row0 >= g.rows) continue;
                        float v[32];
#pragma unroll
                        for (int i = 0; i < 32; i++) v[i] = __uint_as_float(raw[s][i]) * scale;
                        __syncwarp();   // the staging area is free: the strip before has been read
#pragma unroll
                        for (int i = 0; i < 4; i++) st_shared16(staged(area, lane, i), pack8<T>(v + 8 * i));
                        __syncwarp();
                        copy_strip(area, reinterpret_cast<T*>(g.dx), g.lddx, g.vec_dx, col, min(32, count), row0, g.rows - row0, lane);
                    }
                }
            }
        }
        if (want_dw && ok && __all_sync(0xFFFFFFFFu, tc::bar_wait(done, 0, patience))) {   // the CTA's sums: lanes are classes
            tc::fence_after();
            const int c = quarter * 32 + lane;
            float* out = g.dw_part + ((long long)blockIdx.x * g.classes + c) * g.ldpart;
            for (int f = 0; f < g.features && quarter * 32 < g.classes; f += 32) {
                uint32_t raw[32];
                tc::tmem_load32(tmem + kNarrowDw + f + lanes, raw);
                tc::tmem_wait();
#pragma unroll
                for (int i = 0; i < 32; i += 4)   // rows padded to four; the column behind the features is the bias's and written later
                    if (c < g.classes && f + i < g.features)
                        *reinterpret_cast<uint4*>(out + f + i) = make_uint4(raw[i], raw[i + 1], raw[i + 2], raw[i + 3]);
            }
        }
        __syncwarp();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 2) tc::tmem_free<1>(tmem);
    if constexpr (GRAD) {
        const int c = threadIdx.x;
        if (g.want_db && c < g.classes) {
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(s[i]) : "r"(dz0 + (i * kNarrowClasses + c) * 4) : "memory");
            g.dw_part[((long long)blockIdx.x * g.classes + c) * g.ldpart + g.features] = (s[0] + s[1]) + (s[2] + s[3]);
        }
    } else if (threadIdx.x == 0) {
        double s = 0.0;
        int n = 0, any = 0;
        for (int i = 0; i < 8; i++) {
            s += sums_s[i];
            n += counts_s[0][i];
            any |= counts_s[1][i];
        }
        g.sums[blockIdx.x] = s;
        g.counts[blockIdx.x] = n;
        g.counts[gridDim.x + blockIdx.x] = any;
    }
}

// Forward: the CTAs' losses and counts, in order. One block.
__global__ void __launch_bounds__(256) ce_total_kernel(const double* __restrict__ sums, const int* __restrict__ counts, int ctas, int reduction,
                                                       float* loss, int* info) {
    __shared__ double sum_s[256];
    pdl_launch_dependents();
    pdl_wait();
    double s = 0.0;
    int n = 0, any = 0;
    for (int i = threadIdx.x; i < ctas; i += 256) {
        s += sums[i];
        n += counts[i];
        any |= counts[ctas + i];
    }
    sum_s[threadIdx.x] = s;
    any = __syncthreads_or(any);
    __shared__ int counts_s[8];
    n = __reduce_add_sync(0xFFFFFFFFu, n);
    if ((threadIdx.x & 31) == 0) counts_s[threadIdx.x >> 5] = n;
    for (int d = 128; d; d >>= 1) {
        __syncthreads();
        if (threadIdx.x < d) sum_s[threadIdx.x] += sum_s[threadIdx.x + d];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        n = 0;
        for (int i = 0; i < 8; i++) n += counts_s[i];
        info[0] = n;
        info[1] = any != 0;
        info[2] = info[3] = 0;
        if (reduction != RB200_REDUCE_NONE) *loss = (float)(reduction == RB200_REDUCE_MEAN ? sum_s[0] / (double)max(1, n) : sum_s[0]);
    }
}

// Backward: gradient of W (and, in the column behind it, of the bias): the sum over CTAs, scaled. 32 columns of a class a block, CTAs
// spread over 8 threads a column.
template <typename T>
__global__ void __launch_bounds__(256) narrow_join_kernel(const float* __restrict__ part, int ctas, int classes, int features, long long ldpart,
                                                          T* dw, long long lddw, T* db, Scale scale) {
    __shared__ float sums[8][32];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, c = blockIdx.y;
    const bool there = col < features ? dw != nullptr : col == features && db;
    float s = 0.0f;
    if (there) {
#pragma unroll 4
        for (int p = sub; p < ctas; p += 8) s += part[((long long)p * classes + c) * ldpart + col];
    }
    sums[sub][lane] = s;
    __syncthreads();
    if (sub || !there) return;
#pragma unroll
    for (int i = 1; i < 8; i++) s += sums[i][lane];
    const T v = Elem<T>::from_float(s * scale.value());
    if (col < features)
        dw[c * lddw + col] = v;
    else
        db[c] = v;
}

// ---- host side --------------------------------------------------------------------------------------------------
// Backwards W, two tiles of x, dz and the staging areas have to fit, and the gradient of W in TMEM.
static inline bool narrow_fits(long long classes, long long features) {
    if (classes > kNarrowClasses || features > kNarrowFeatures) return false;
    const int chunks = (int)((features + 127) / 128) * 2;
    return narrow_smem((int)round_up(classes, 32), chunks, 2 * chunks, true) <= kNarrowSmem;
}
// One for every SM - or as many as it takes for none to add up more than 32768 rows: sums on the tensor cores drift (gemm.cuh; 2^25 rows of
// one sign over 148 CTAs: 1.1e-3).
constexpr int kNarrowTiles = 32768 / kTileM;
static inline int narrow_ctas(long long rows, int sms) {
    const long long tiles = (rows + kTileM - 1) / kTileM, least = (tiles + kNarrowTiles - 1) / kNarrowTiles, most = tiles < sms ? tiles : sms;
    return (int)(least > most ? least : most);
}

template <typename T, bool GRAD>
static int narrow_launch_as(const NarrowArgs& g, const DeviceInfo& dev, cudaStream_t stream, const char* what) {
    auto* kernel = ce_narrow_kernel<T, GRAD>;
    static unsigned long long ready;   // a bit for each device whose kernel has its shared-memory limit
    int rc;
    if (!(__atomic_load_n(&ready, __ATOMIC_RELAXED) >> dev.index & 1)) {
        rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kNarrowSmem + 1024)), what);
        if (rc) return rc;
        __atomic_fetch_or(&ready, 1ull << dev.index, __ATOMIC_RELAXED);
    }
    rc = check_cuda(launch_overlapped(kernel, dim3(narrow_ctas(g.rows, dev.sms)), dim3(narrow_threads(GRAD)),
                                      narrow_smem(g.vb, g.chunks, g.slots, GRAD) + 1024, stream, g),
                    what);
    if (rc) return rc;
    count_launch();
    return RB200_OK;
}

// Fills what both directions share and launches. x and w are map_ready.
static int narrow_launch(NarrowArgs& g, bool grad, bool bf16, const Operand& x, const Operand& w, const DeviceInfo& dev, cudaStream_t stream,
                         const char* what) {
    g.rows = x.rows;
    g.features = x.cols;
    g.classes = w.rows;
    g.vb = (int)round_up(g.classes, 32);
    g.chunks = grad ? (g.features + 127) / 128 * 2 : (g.features + 63) / 64;
    g.slots = grad ? 2 * g.chunks : kNarrowSlots / g.chunks * g.chunks;
    g.idesc_s = tc::instr_desc(bf16, false, false, kTileM, g.vb);
    g.idesc_x = tc::instr_desc(bf16, false, true, kTileM, 128);
    g.idesc_w = tc::instr_desc(bf16, true, true, kTileM, 64 * g.chunks);
    int rc = make_map(&g.x, x, bf16, kTileM, what);
    if (rc) return rc;
    if ((rc = make_map(&g.w, w, bf16, g.vb, what))) return rc;
    if (!g.status) g.status = dev.status;
    if (!g.wait_cycles) g.wait_cycles = kDefaultWaitCycles;
    if (grad) return bf16 ? narrow_launch_as<__nv_bfloat16, true>(g, dev, stream, what) : narrow_launch_as<__half, true>(g, dev, stream, what);
    return bf16 ? narrow_launch_as<__nv_bfloat16, false>(g, dev, stream, what) : narrow_launch_as<__half, false>(g, dev, stream, what);
}

}  // namespace rb200
