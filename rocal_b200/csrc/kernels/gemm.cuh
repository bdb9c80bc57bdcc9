// Matrix products C[m][n] = sum_k A[m][k] B[n][k] of 16-bit operands with fp32 accumulation on the fifth-generation
// tensor cores, and what is done with the accumulators before they leave the chip (EPI_*). One persistent kernel:
//   warps 0, 3  copy the tiles of A and of B (128-byte swizzle) into a ring of shared-memory stages,
//   warp 2      allocates TMEM (and has one rare task, EpiArgs::dirty),
//   warp 1      issues the products of a stage (64 contracted elements, 128 of small tiles: the handshakes of a stage cost
//               some 300 clocks, 234 on this side, which is more than a small tile's products) into one of two TMEM accumulators,
//   warps 4-19  two groups of eight; each group reads its own accumulator, 32 columns at a time (thread = row, two
//               warps share a row's strips), and runs the epilogue of every other tile, so that the epilogues of two tiles
//               overlap each other's latency and the products of the tiles behind them. Results cross over in shared
//               memory from threads that hold rows to lanes that write whole pieces of rows.
//               An epilogue strip is some 150 to 400 instructions of a warp, mostly in chains: with 8 warps instead of 16
//               it took 900 to 2500 clocks and bounded products of up to 1024 contracted elements.
// CG = 2: two CTAs (a cluster) work on one tile of 256 rows; each holds its 128 rows of A and half of the B tile, so a
// tile of 256 columns takes 128 bytes of operands per SM and clock at the full rate of the tensor cores instead of 192.
// The tensor cores cut the sums they add to where they do not fit 32 bits, always towards zero, so a long sum drifts (measured, one
// accumulator, relative to the root mean square of the sums: 0.7e-6 after 2048 products of normal numbers, 1.4e-6 after 4096, 3.0e-6
// after 8192, 26e-6 after 65536; of numbers of one sign 1.7e-6, 4.3e-6, 11e-6 and 0.19e-3, and 3e-3 after 524288). Up to 32768 products, which
// is where sums are split (gemm_plan), that is well below a 16-bit result's rounding, but not below an fp32 loss': where that is made, tiles of up to 128 columns, which leave TMEM columns free, spread the contracted axis over several
// accumulators, 512 elements at least in each, and the epilogue adds them with correct rounding. And a sum near zero may come out on
// its other side: a relu then passes or stops a gradient that it should not, for 0.3e-6 of the elements at 2048 products and 0.7e-6 at
// 4096 (sums rounded to nearest: 0.1e-6 and 0.2e-6).
// Either operand may have the contracted axis contiguous (K-major) or the other one (MN-major): the backward products
// need no transposed copies. Rows and columns beyond the matrices arrive as zeros and are not stored.
#pragma once

#include "tensor_core.cuh"

namespace rb200 {

constexpr int kTileM = 128, kTileK = 64, kTileNMax = 256;
constexpr int kEpiWarps = 16, kGemmThreads = 128 + 32 * kEpiWarps;
constexpr int kStageBytes = 2048;            // of an epilogue warp: 32 lines of 64 bytes
constexpr int kRingBytes = 196608;           // of the 227 KB: operand stages

enum { EPI_LINEAR = 0, EPI_STORE = 1, EPI_CE_STATS = 2, EPI_CE_GRAD = 3, EPI_LINEAR_ADD = 4 };   // ADD: with a residual
enum { ACT_NONE = RB200_ACT_NONE, ACT_RELU = RB200_ACT_RELU, ACT_GELU = RB200_ACT_GELU, ACT_SILU = RB200_ACT_SILU };

// A factor that is partly known on the device only: constant * *scalar / max(1, *count).
struct Scale {
    float constant;
    const float* scalar;   // or null (= 1)
    const int* count;      // or null (= 1)
    __host__ __device__ Scale(float c = 1.0f, const float* s = nullptr, const int* n = nullptr) : constant(c), scalar(s), count(n) {}
    __device__ float value() const { return constant * (scalar ? *scalar : 1.0f) / (count ? (float)max(1, *count) : 1.0f); }
};

// What the epilogues read and write; the fields an epilogue does not name are unused.
struct EpiArgs {
    void* out;                // LINEAR, STORE (final): T[m][ldo]; CE_GRAD: T[m][ldo]
    long long ldo;
    const void* bias;         // LINEAR, CE_*: T[n] or null
    const void* residual;     // LINEAR: T[residual_rows][ldr], row i % residual_rows, or null
    long long ldr;
    int residual_rows;
    void* preact;             // LINEAR: T[m][ldp] or null
    long long ldp;
    int act;
    int vec_out, vec_res, vec_pre;   // 1: the rows of that array start on 16-byte boundaries
    // STORE: value = acc + acc_in; to acc_out (fp32) if that is set, else scale * value to out.
    const float* acc_in;
    float* acc_out;
    long long ldacc, acc_split_stride;
    Scale scale;
    // CE: labels of the rows (4- or 8-byte integers), all classes and the first one of this launch, the ignored label.
    const void* labels;
    int label_bytes, classes, class0;
    long long ignore_index;
    float smooth_on, smooth_off;   // 1 - smoothing, smoothing / classes
    float inv_classes;
    float* part;              // STATS: [parts][m] maxima, then [parts][m] sums, then (smoothing) [parts][m] sums of z / classes;
                              // two parts a tile
    int parts, want_zsum;
    float* zlabel;            // STATS: [m] the label's z
    int* clear;               // STATS: four words to be zeroed, or null
    const float* stats;       // GRAD: maxima; stats_stride further the sums, twice that the labels' z
    long long stats_stride;
    const float* coef;        // GRAD: [m] per-row factor or null (= 1)
    float* col_part;          // GRAD: [m / 32][ldcol] sums over 32 rows of what is written, before its rounding, or null
    long long ldcol;
    // GRAD: if *dirty, clean[clean_rows][k] = clean_src with the rows that do not count zeroed, made on the side; or null.
    const int* dirty;
    const void* clean_src;
    void* clean;
    long long ldsrc, ldclean, clean_rows;
    const void* clean_labels;
};

struct GemmArgs {
    CUtensorMap a, b, b_alt;   // b_alt replaces b when *b_select is not 0
    const int* b_select;
    int m, n, k;
    int bn;                    // columns of a tile
    int tiles_m, tiles_n, splits;
    int kblocks, kblocks_per_split;
    int kblocks_per_sum;       // contracted blocks that go into one accumulator of a tile
    int a_box_rows;            // rows of a K-major A copy
    int stage_blocks;          // contracted blocks of a stage
    uint32_t idesc, block_bytes, stages;
    int* status;
    unsigned long long wait_cycles;
    int skip_block;            // copies of the k-blocks from this one on are left out (-1: none)
    EpiArgs e;
};

// ---- 16-bit elements ---------------------------------------------------------------------------------
template <typename T>
struct Elem;
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
};

// Eight elements, `count` of them there (the others are zeros).
template <typename T>
__device__ __forceinline__ uint4 load8(const T* p, int count, bool vec) {
    if (vec && count >= 8) return __ldg(reinterpret_cast<const uint4*>(p));
    uint32_t w[4] = {};
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < count) w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = Elem<T>::unpack(u[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// W words that start SHIFT words and `bits` bits into two neighbouring vectors of W words.
template <int W, int SHIFT>
__device__ __forceinline__ void window(const uint32_t (&w)[2 * W], uint32_t (&out)[W], int bits) {
#pragma unroll
    for (int k = 0; k < W; k++) out[k] = __funnelshift_r(w[SHIFT + k], w[(SHIFT + k + 1) % (2 * W)], bits);
}

// Upper tail of the normal distribution over its density shape: R(a) = Q(a) exp(a^2 / 2) for a in [0, 14]. Q falls like
// 1 / a times the density, so R is smooth in t = 1 / (1 + p a): a polynomial t, ..., t^7, fitted here together with p for the least
// relative error (1.0e-6 evaluated in fp32, and the reciprocal's 1e-7). Beyond 13.2 the exponential that it goes with is flushed to zero.
// (A polynomial in a takes degree 12 for 2e-6 up to 6, and in packed pairs its coefficients sit in 26 registers: the epilogues
// spilled, and the spills took half of the L1's stores.)
constexpr float kTailEnd = 14.0f, kTailScale = 0.264f;
__device__ constexpr float tail_term(int i) {   // of t^(i + 1); folded where the loops below are unrolled
    constexpr float c[7] = {0.105179973f, 0.107738927f, 0.0808872133f, 0.147553459f, -0.0746941119f, 0.202287167f, -0.0689526573f};
    return c[i];
}
__device__ __forceinline__ float tail_ratio(float a) {
    float t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(a, kTailScale, 1.0f)));
    float r = tail_term(6);
#pragma unroll
    for (int i = 5; i >= 0; i--) r = fmaf(r, t, tail_term(i));
    return r * t;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// z Phi(z) = max(z, 0) - |z| Q(|z|): one exponential and one reciprocal, accurate down the whole negative tail.
// Infinities give 0 and inf (the exponential is 0 there), NaN stays.
__device__ __forceinline__ float gelu(float z) {
    const float a = fminf(fabsf(z), kTailEnd), e = exp2_fast(z * (z * -0.72134752f));
    return (z < 0.0f ? 0.0f : z) - a * e * tail_ratio(a);
}
// Phi(z) + z phi(z), two at a time (fma.f32x2: the sweep over a gradient that this is for is bound by issue as much as by memory;
// 8192 x 4096 with gelu 47 -> 39 us). |z| is held at 40, where the exponential is 0, so that infinities give 0 and 1; NaN passes.
__device__ __forceinline__ float2 gelu_slopes(float2 z) {
    float2 a, t;
    asm("min.NaN.f32 %0, %1, 0f42200000;" : "=f"(a.x) : "f"(fabsf(z.x)));
    asm("min.NaN.f32 %0, %1, 0f42200000;" : "=f"(a.y) : "f"(fabsf(z.y)));
    const float2 x = mul2(a, mul2(a, make_float2(-0.72134752f, -0.72134752f))), e = make_float2(exp2_fast(x.x), exp2_fast(x.y));
    const float2 b = fma2(make_float2(fminf(a.x, kTailEnd), fminf(a.y, kTailEnd)), make_float2(kTailScale, kTailScale), make_float2(1.0f, 1.0f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(b.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(b.y));
    auto both = [](float c) { return make_float2(c, c); };
    float2 r = both(-tail_term(6));   // -R: tail_ratio's polynomial
#pragma unroll
    for (int i = 5; i >= 0; i--) r = fma2(r, t, both(-tail_term(i)));
    // |z| phi - Q, which the sign of z turns into the distance from 1 or from 0
    const float2 d = mul2(e, fma2(a, both(0.39894228f), mul2(r, t)));
    auto turn = [](float v, float dist) {
        const uint32_t sign = __float_as_uint(v) & 0x80000000u;
        return (sign ? 0.0f : 1.0f) + __uint_as_float(__float_as_uint(dist) ^ sign);
    };
    return make_float2(turn(z.x, d.x), turn(z.y, d.y));
}
// sigmoid(z) = h (h r) and 1 - sigmoid(z) = r from h = exp(z / 2), r = 1 / (1 + h^2): the root, because exp(z) itself and its reciprocal
// leave the range of normal numbers while z sigmoid(z) is still a number of the result's type. z is held at 60, where
// sigmoid is 1; NaN passes.
struct Sigmoid {
    float z, h, r;
    __device__ __forceinline__ explicit Sigmoid(float v) {
        asm("min.NaN.f32 %0, %1, 0f42700000;" : "=f"(z) : "f"(v));
        h = exp2_fast(z * 0.72134752f);
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(h, h, 1.0f)));
    }
};

// N values at a time: one branch on the activation, and N independent chains of operations behind it.
template <int N>
__device__ __forceinline__ void act_values(float* v, int act) {
    if (act == ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = v[i] < 0.0f ? 0.0f : v[i];   // NaN stays
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = gelu(v[i]);
    } else if (act == ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const Sigmoid g(v[i]);
            v[i] = v[i] * g.h * (g.h * g.r);
        }
    }
}
template <int N>
__device__ __forceinline__ void act_slopes(float* v, int act) {   // z -> slope
    if (act == ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = v[i] > 0.0f ? 1.0f : v[i] <= 0.0f ? 0.0f : v[i];   // NaN stays
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 s = gelu_slopes(make_float2(v[i], v[i + 1]));
            v[i] = s.x;
            v[i + 1] = s.y;
        }
    } else if (act == ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const Sigmoid g(v[i]);
            v[i] = fmaf(g.z, g.r, 1.0f) * g.h * (g.h * g.r);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = 1.0f;
    }
}

// ---- results through shared memory -----------------------------------------------------------------------
// Threads hold rows; memory wants whole pieces of rows. A warp's strip crosses over in its staging area, 32 lines of 64
// bytes: each thread writes its own line, then 16-byte pieces are read back so that four neighbouring lanes hold the pieces of a
// line. Piece j of line r lies at place j ^ (r / 2 & 3), so that neither side has bank conflicts.
__device__ __forceinline__ uint32_t staged(uint32_t area, int line, int piece) { return area + line * 64 + ((piece ^ (line >> 1 & 3)) << 4); }
__device__ __forceinline__ void st_shared16(uint32_t addr, const uint4& w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
    uint4 w;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(addr) : "memory");
    return w;
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* v) {
    return make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]), Elem<T>::pack(v[6], v[7]));
}
// The staged strip to rows [row0, row0 + rows) and columns [col, col + cols) of out.
template <typename T>
__device__ __forceinline__ void copy_strip(uint32_t area, T* out, long long ld, bool vec, int col, int cols, int row0, int rows, int lane) {
    rows = min(rows, 32);
    if (vec && (cols & 7) == 0) {
        const int piece = lane & 3;
        T* o = out + (long long)(row0 + (lane >> 2)) * ld + col + piece * 8;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = (lane >> 2) + 8 * i;
            const uint4 w = ld_shared16(staged(area, r, piece));
            if (r < rows && piece * 8 < cols) *reinterpret_cast<uint4*>(o) = w;
            o += 8 * ld;
        }
    } else {   // odd boundaries: a row at a time, an element a lane
#pragma unroll 4
        for (int r = 0; r < rows; r++) {
            uint16_t w;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(staged(area, r, lane >> 3) + (lane & 7) * 2) : "memory");
            if (lane < cols) reinterpret_cast<uint16_t*>(out + (long long)(row0 + r) * ld + col)[lane] = w;
        }
    }
}
// 32-bit sums: the strip in two halves of 16 columns, added to `in` if that is set. out and in point at the strip's first
// element, cols counts the padding of the rows (a multiple of 4).
__device__ __forceinline__ void leave_sums(uint32_t area, const float (&v)[32], float* out, const float* in, long long ld, int cols, int rows,
                                           int lane) {
    const int piece = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float* q = v + 16 * h + 4 * i;
            st_shared16(staged(area, lane, i), make_uint4(__float_as_uint(q[0]), __float_as_uint(q[1]), __float_as_uint(q[2]), __float_as_uint(q[3])));
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = (lane >> 2) + 8 * i;
            const long long at = r * ld + 16 * h + piece * 4;
            const uint4 w = ld_shared16(staged(area, r, piece));
            if (r < rows && 16 * h + piece * 4 < cols) {
                float4 f = make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
                if (in) {
                    const float4 s = *reinterpret_cast<const float4*>(in + at);
                    f.x += s.x;
                    f.y += s.y;
                    f.z += s.z;
                    f.w += s.w;
                }
                *reinterpret_cast<float4*>(out + at) = f;
            }
        }
    }
}

// Running maximum and sum of exp(z - maximum) of one row. A maximum of -inf (every class masked so far) is replaced by
// 0 in the differences, so that masked classes add exp(-inf) = 0 and no -inf - -inf arises. NaN reaches the sum.
struct RunningSoftmax {
    float m, s;
};
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }
constexpr float kLog2e = 1.4426950408889634f;
// exp(d) for a difference d <= 0 (or NaN): one special-function operation, 2^-22 relative, and the rounding of its argument,
// |d| 2^-24 relative (a term that weighs exp(d) in a sum with one of 1).
__device__ __forceinline__ float exp_diff(float d) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * kLog2e));
    return r;
}

// The class of a row and whether it counts; -1 for a label that is no class.
__device__ __forceinline__ int load_label(const void* labels, int bytes, long long row, long long ignore_index, int classes, bool* counted) {
    const long long v = bytes == 8 ? reinterpret_cast<const long long*>(labels)[row] : reinterpret_cast<const int32_t*>(labels)[row];
    *counted = v != ignore_index;
    return v >= 0 && v < classes ? (int)v : -1;
}

template <typename T, bool A_MN, bool B_MN, int EPI, int CG>
__global__ void __launch_bounds__(kGemmThreads, 1) gemm_kernel(const __grid_constant__ GemmArgs g) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * 16 + 2 * 2 + 1];
    __shared__ uint32_t tmem_addr_s;
    __shared__ int gave_up_s;

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? tc::cta_rank() : 0;
    const uint32_t smem0 = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bar0 = tc::smem_u32(bars);
    const int S = (int)g.stages;
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (16 + s); };
    auto acc_full = [&](int b) { return bar0 + 8u * (32 + b); };
    auto acc_empty = [&](int b) { return bar0 + 8u * (34 + b); };
    const uint32_t drained = bar0 + 8u * 36;

    if (threadIdx.x == 0) {
        gave_up_s = 0;
        for (int s = 0; s < S; s++) {
            tc::bar_init(full(s), 2);   // what A and what B have to bring
            tc::bar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; b++) {
            tc::bar_init(acc_full(b), 1);
            tc::bar_init(acc_empty(b), kEpiWarps / 2 * CG);
        }
        tc::bar_init(drained, 1);
        tc::bar_init_fence();
        tc::prefetch_map(&g.a);
        tc::prefetch_map(&g.b);
    }
    if (warp == 2) tc::tmem_alloc<CG>(tc::smem_u32(&tmem_addr_s));
    tc::fence_before();
    if constexpr (CG == 2)
        tc::cluster_sync();
    else
        __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_addr_s;
    pdl_launch_dependents();
    pdl_wait();   // everything above touches this CTA's own state only
    if (EPI == EPI_CE_STATS && g.e.clear && blockIdx.x == 0 && threadIdx.x < 4) g.e.clear[threadIdx.x] = 0;
    const tc::Patience patience = {&gave_up_s, g.status, g.wait_cycles};

    const uint32_t tiles = (uint32_t)g.tiles_m * g.tiles_n * g.splits;   // below 2^31 (gemm_args)
    const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;
    // Tiles in bands of 8 tile rows, row fastest: the tiles in flight share their operands in L2.
    auto place = [&](uint32_t t, int& mb, int& nb, int& sp) {
        const uint32_t per = (uint32_t)g.tiles_m * g.tiles_n;
        sp = g.splits == 1 ? 0 : (int)(t / per);
        const uint32_t r = t - sp * per, whole = 8u * g.tiles_n, band = r / whole, q = r - band * whole;
        const uint32_t rows = min(8u, g.tiles_m - band * 8u);
        const uint32_t col = rows == 8 ? q >> 3 : q / rows;
        nb = (int)col;
        mb = (int)(band * 8 + q - col * rows);
    };
    const int bn_cta = g.bn / CG;

    if (warp == 0 || warp == 3) {
        const bool loads_a = warp == 0;
        if (tc::elect_one()) {
            const CUtensorMap* map_b = (!loads_a && g.b_select && *g.b_select) ? &g.b_alt : &g.b;
            const uint32_t block_bytes = loads_a ? (A_MN ? kTileM : g.a_box_rows) * kTileK * 2 : bn_cta * kTileK * 2;
            int s = 0;
            uint32_t phase = 0;
            long long filled = 0;
            bool ok = true;
            for (uint32_t t = first; t < tiles && ok; t += step) {
                int mb, nb, sp;
                place(t, mb, nb, sp);
                const int m0 = mb * (kTileM * CG) + (int)rank * kTileM, n0 = nb * g.bn + (int)rank * bn_cta;
                const int k_end = min(g.kblocks, (sp + 1) * g.kblocks_per_split);
                for (int k0 = sp * g.kblocks_per_split; k0 < k_end; k0 += g.stage_blocks) {
                    ok = tc::bar_wait(empty(s), phase ^ 1, patience);
                    if (!ok) break;
                    const int blocks = min(g.stage_blocks, k_end - k0);
                    uint32_t bar = full(s);
                    if constexpr (CG == 2) bar = tc::map_to_rank(bar, 0);
                    if (rank == 0) tc::bar_expect(full(s), CG * blocks * block_bytes);
                    for (int i = 0; i < blocks; i++) {
                        const int kb = k0 + i;
                        if (g.skip_block >= 0 && kb >= g.skip_block) break;
                        const uint32_t sa = smem0 + (s * g.stage_blocks + i) * g.block_bytes, sb = sa + kTileM * kTileK * 2;
                        if (loads_a) {
                            if constexpr (A_MN) {
                                tc::tma_load<CG>(sa, &g.a, m0, kb * kTileK, bar);
                                tc::tma_load<CG>(sa + 64 * kTileK * 2, &g.a, m0 + 64, kb * kTileK, bar);
                            } else {
                                tc::tma_load<CG>(sa, &g.a, kb * kTileK, m0, bar);
                            }
                        } else {
                            if constexpr (B_MN) {
                                for (int j = 0; j < bn_cta; j += 64) tc::tma_load<CG>(sb + j * kTileK * 2, map_b, n0 + j, kb * kTileK, bar);
                            } else {
                                tc::tma_load<CG>(sb, map_b, kb * kTileK, n0, bar);
                            }
                        }
                    }
                    filled++;
                    if (++s == S) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
            // Copies still on their way into this CTA's (and its peer's) stages. The products wait for every one of them, but may have
            // given up, also when this warp is through.
            if (rank == 0) {
                for (int i = 0; i < S && i < filled; i++) {
                    if (s == 0) {
                        s = S;
                        phase ^= 1;
                    }
                    s--;
                    tc::bar_drain(full(s), phase, g.wait_cycles);
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && tc::elect_one()) {
            int s = 0, buf = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true, issued = false;
            for (uint32_t t = first; t < tiles && ok; t += step) {
                int mb, nb, sp;
                place(t, mb, nb, sp);
                const int k_begin = sp * g.kblocks_per_split, k_end = min(g.kblocks, (sp + 1) * g.kblocks_per_split);
                ok = tc::bar_wait(acc_empty(buf), acc_phase ^ 1, patience);
                if (!ok) break;
                tc::fence_after();
                uint32_t d = tmem + buf * kTileNMax - g.bn;
                int left = 0;   // blocks that still go into accumulator d
                for (int k0 = k_begin; k0 < k_end; k0 += g.stage_blocks) {
                    ok = tc::bar_wait(full(s), phase, patience);
                    if (!ok) break;
                    tc::fence_after();
                    for (int i = 0; i < g.stage_blocks && k0 + i < k_end; i++) {
                        const bool fresh = left == 0;
                        if (fresh) {
                            d += g.bn;
                            left = g.kblocks_per_sum;
                        }
                        left--;
                        const uint32_t sa = smem0 + (s * g.stage_blocks + i) * g.block_bytes, sb = sa + kTileM * kTileK * 2;
                        const uint64_t da = tc::operand_desc(sa, A_MN, 64 * kTileK * 2), db = tc::operand_desc(sb, B_MN, 64 * kTileK * 2);
#pragma unroll
                        for (int k = 0; k < kTileK / 16; k++)
                            tc::mma_f16<CG>(d, da + k * (A_MN ? 2048 >> 4 : 32 >> 4), db + k * (B_MN ? 2048 >> 4 : 32 >> 4), g.idesc,
                                            (!fresh || k > 0) ? 1u : 0u);
                    }
                    issued = true;
                    tc::mma_commit<CG>(empty(s));
                    if (++s == S) {
                        s = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                tc::mma_commit<CG>(acc_full(buf));
                buf ^= 1;
                acc_phase ^= buf == 0;
            }
            if (issued) {   // products still running: the epilogues wait for all of them, but may have given up
                tc::mma_commit<CG>(drained);
                tc::bar_drain(drained, 0, g.wait_cycles);
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        if constexpr (EPI == EPI_CE_GRAD) {
            if (g.e.dirty && *g.e.dirty) {
                const int cols = g.k;
                for (long long r = blockIdx.x; r < g.e.clean_rows; r += gridDim.x) {
                    bool counted;
                    load_label(g.e.clean_labels, g.e.label_bytes, r, g.e.ignore_index, g.e.classes, &counted);
                    const T* src = reinterpret_cast<const T*>(g.e.clean_src) + r * g.e.ldsrc;
                    T* dst = reinterpret_cast<T*>(g.e.clean) + r * g.e.ldclean;   // rows padded to whole pieces
                    for (int c = lane * 8; c < cols; c += 256)
                        *reinterpret_cast<uint4*>(dst + c) = counted ? load8(src + c, cols - c, false) : make_uint4(0, 0, 0, 0);
                }
            }
        }
    } else if (warp >= 4) {
        // group 0: even tiles and accumulator 0; share 0: even strips
        const int ew = warp - 4, quarter = warp & 3, group = ew >> 3, share = ew >> 2 & 1;
        const uint32_t area = smem0 + kRingBytes + ew * kStageBytes;
        const uint32_t acc = tmem + group * kTileNMax + ((uint32_t)(quarter * 32) << 16);
        uint32_t acc_phase = 0;
        float scale = 1.0f;
        if constexpr (EPI == EPI_STORE) scale = g.e.scale.value();
        for (uint32_t t = first + group * step; t < tiles; t += 2 * step) {
            int mb, nb, sp;
            place(t, mb, nb, sp);
            const int row0 = mb * (kTileM * CG) + (int)rank * kTileM + quarter * 32, row = row0 + lane;
            const bool row_ok = row < g.m;
            const int n0 = nb * g.bn, n1 = min(n0 + g.bn, g.n);

            // what does not depend on the products is fetched before the wait for them
            int label = -1;
            bool counted = false;
            float top = 0.0f, zsum = 0.0f, mul = 0.0f, add = 0.0f, at_label = 0.0f;
            RunningSoftmax run = {-INFINITY, 0.0f};
            if constexpr (EPI == EPI_CE_STATS || EPI == EPI_CE_GRAD) {
                if (row_ok) {
                    label = load_label(g.e.labels, g.e.label_bytes, row, g.e.ignore_index, g.e.classes, &counted);
                    label = label < g.e.class0 ? -1 : label - g.e.class0;
                }
            }
            if constexpr (EPI == EPI_CE_GRAD) {
                if (counted) {   // (softmax - target) * factor = exp(z - top) * mul + add, and at the label
                    const float zl = g.e.stats[2 * g.e.stats_stride + row], factor = (g.e.coef ? g.e.coef[row] : 1.0f) * 32768.0f;
                    top = finite_max(g.e.stats[row]);
                    mul = factor / g.e.stats[g.e.stats_stride + row];
                    add = -g.e.smooth_off * factor;
                    at_label = exp_diff(zl - top) * mul + add - g.e.smooth_on * factor;
                } else {
                    label = -1;
                }
            }

            int res_row[4];   // the residual's rows of this lane (below), -1: none
            if constexpr (EPI == EPI_LINEAR_ADD) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = row0 + (lane >> 2) + 8 * i;
                    res_row[i] = r < g.m ? r % g.e.residual_rows : -1;
                }
            }
            // A strip of the residual: lane l takes piece l % 4 of the rows l / 4 + 8 i. The tile's first one is on its way
            // before the products are done, the others from the strip before (50176 x 768 -> 1024 with a residual of as many rows: 116 -> 104 us).
            uint4 res[4];
            auto fetch_residual = [&](int c) {
                if constexpr (EPI == EPI_LINEAR_ADD) {
                    const int col = n0 + c, left = n1 - col - (lane & 3) * 8;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        res[i] = make_uint4(0, 0, 0, 0);
                        if (res_row[i] >= 0 && left > 0)
                            res[i] = load8(reinterpret_cast<const T*>(g.e.residual) + res_row[i] * g.e.ldr + col + (lane & 3) * 8, left, g.e.vec_res);
                    }
                }
            };
            fetch_residual(share * 32);

            // the lanes leave together: what follows needs whole warps
            if (!__all_sync(0xFFFFFFFFu, tc::bar_wait(acc_full(group), acc_phase, patience))) break;
            acc_phase ^= 1;
            tc::fence_after();

            const int in_sum = min(g.kblocks, (sp + 1) * g.kblocks_per_split) - sp * g.kblocks_per_split;
            const int sums = (in_sum + g.kblocks_per_sum - 1) / g.kblocks_per_sum;
            auto release = [&] {   // this warp's part of the accumulator is in registers
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::bar_arrive_relaxed(CG == 2 ? tc::map_to_rank(acc_empty(group), 0) : acc_empty(group));
            };
            for (int c = share * 32; c < g.bn; c += 64) {
                const int col = n0 + c, count = n1 - col;   // columns of this strip inside the matrix (may be <= 0)
                const bool work = count > 0 && row0 < g.m;
                uint32_t raw[32];
                if (work) tc::tmem_load32(acc + c, raw);
                float own_bias = 0.0f;   // of column `lane`
                if constexpr (EPI != EPI_STORE) {
                    if (work && g.e.bias && lane < count) own_bias = Elem<T>::to_float(reinterpret_cast<const T*>(g.e.bias)[col + lane]);
                }
                tc::tmem_wait();
                if (!work) {
                    if (c + 64 >= g.bn) release();
                    continue;
                }
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; i++) v[i] = __uint_as_float(raw[i]);
                for (int s = 1; EPI == EPI_CE_STATS && s < sums; s++) {   // the tile's other accumulators
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint32_t more[8];
                        tc::tmem_load8(acc + s * g.bn + c + i, more);
                        tc::tmem_wait();
#pragma unroll
                        for (int j = 0; j < 8; j++) v[i + j] += __uint_as_float(more[j]);
                    }
                }
                if (c + 64 >= g.bn) release();
                __syncwarp();   // the staging area is free: the strip before has been read
                if constexpr (EPI != EPI_STORE) {
                    if (g.e.bias) {
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"(area + lane * 4), "f"(own_bias) : "memory");
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const uint4 w = ld_shared16(area + i * 4);
                            const float2 s = add2(make_float2(v[i], v[i + 1]), make_float2(__uint_as_float(w.x), __uint_as_float(w.y)));
                            const float2 u = add2(make_float2(v[i + 2], v[i + 3]), make_float2(__uint_as_float(w.z), __uint_as_float(w.w)));
                            v[i] = s.x;
                            v[i + 1] = s.y;
                            v[i + 2] = u.x;
                            v[i + 3] = u.y;
                        }
                        __syncwarp();
                    }
                }
                auto leave = [&](void* out, long long ld, bool vec) {
#pragma unroll
                    for (int i = 0; i < 4; i++) st_shared16(staged(area, lane, i), pack8<T>(v + 8 * i));
                    __syncwarp();
                    copy_strip(area, reinterpret_cast<T*>(out), ld, vec, col, min(32, count), row0, g.m - row0, lane);
                };
                if constexpr (EPI == EPI_LINEAR || EPI == EPI_LINEAR_ADD) {
                    if (g.e.preact) {   // in the element type: kept in 32 bits, z would add 4 bytes a value each way to a pass bound by memory
                        leave(g.e.preact, g.e.ldp, g.e.vec_pre);
                        __syncwarp();
                    }
                    if (g.e.act != ACT_NONE) {
                        act_values<8>(v, g.e.act);
                        act_values<8>(v + 8, g.e.act);
                        act_values<8>(v + 16, g.e.act);
                        act_values<8>(v + 24, g.e.act);
                    }
                    if constexpr (EPI == EPI_LINEAR_ADD) {   // the other way round: whole pieces of rows in, a row a thread out
#pragma unroll
                        for (int i = 0; i < 4; i++) st_shared16(staged(area, (lane >> 2) + 8 * i, lane & 3), res[i]);
                        if (c + 64 < g.bn) fetch_residual(c + 64);
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            float r[8];
                            unpack8<T>(ld_shared16(staged(area, lane, i)), r);
#pragma unroll
                            for (int j = 0; j < 8; j += 2) {
                                const float2 s = add2(make_float2(v[8 * i + j], v[8 * i + j + 1]), make_float2(r[j], r[j + 1]));
                                v[8 * i + j] = s.x;
                                v[8 * i + j + 1] = s.y;
                            }
                        }
                    }
                    leave(g.e.out, g.e.ldo, g.e.vec_out);
                }
                if constexpr (EPI == EPI_STORE) {
                    // 32-bit sums: rows and columns of this strip, the padding of the rows included
                    const long long at = (long long)row0 * g.e.ldacc + col;
                    const int wide = min(32, (int)g.e.ldacc - col);
                    if (g.e.acc_out) {
                        leave_sums(area, v, g.e.acc_out + (long long)sp * g.e.acc_split_stride + at, g.e.acc_in ? g.e.acc_in + at : nullptr,
                                   g.e.ldacc, wide, g.m - row0, lane);
                    } else {
                        if (g.e.acc_in && row_ok) {
                            const float* p = g.e.acc_in + (long long)row * g.e.ldacc + col;
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                if (i < wide) {
                                    const float4 f = *reinterpret_cast<const float4*>(p + i);
                                    v[i] += f.x;
                                    v[i + 1] += f.y;
                                    v[i + 2] += f.z;
                                    v[i + 3] += f.w;
                                }
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 s = mul2(make_float2(v[i], v[i + 1]), make_float2(scale, scale));
                            v[i] = s.x;
                            v[i + 1] = s.y;
                        }
                        leave(g.e.out, g.e.ldo, g.e.vec_out);
                    }
                }
                if constexpr (EPI == EPI_CE_STATS) {
                    const int l = label - col;
                    if (l >= 0 && l < 32) {   // element l of the strip, by its bits
                        float a[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) a[i] = l & 16 ? v[i + 16] : v[i];
#pragma unroll
                        for (int w = 8; w; w >>= 1)
#pragma unroll
                            for (int i = 0; i < w; i++) a[i] = l & w ? a[i + w] : a[i];
                        if (label < g.n) g.e.zlabel[row] = a[0];
                    }
                    // four sums, not one chain of 32; of z / classes: two classes that the type's lowest value masks add up to more than
                    // fp32 holds, their mean does not
                    if (g.e.want_zsum) {
                        const float2 inv = make_float2(g.e.inv_classes, g.e.inv_classes);
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
                    const float strip = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), now = fmaxf(run.m, strip), base = finite_max(now);
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
                if constexpr (EPI == EPI_CE_GRAD) {
                    const float2 off = make_float2(-top, -top), unit = make_float2(kLog2e, kLog2e);
                    const float2 mul_v = make_float2(mul, mul), add_v = make_float2(add, add);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 d = mul2(add2(make_float2(v[i], v[i + 1]), off), unit);
                        const float2 p = fma2(make_float2(exp2_fast(d.x), exp2_fast(d.y)), mul_v, add_v);
                        v[i] = p.x;
                        v[i + 1] = p.y;
                    }
                    const int l = label - col;
                    if (l >= 0 && l < 32) {
#pragma unroll
                        for (int i = 0; i < 32; i++) v[i] = i == l ? at_label : v[i];
                    }
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = counted ? v[i] : 0.0f;   // whatever the row held
                    // rounded to the element type, as an operand of two products has to be; column sums are made of what it was before
#pragma unroll
                    for (int i = 0; i < 4; i++) st_shared16(staged(area, lane, i), pack8<T>(v + 8 * i));
                    if (g.e.col_part) {
                        // Column sums over the warp's rows: at every step a lane keeps the half of its columns that its own
                        // number's next bit names and hands the other half to its partner. Lane l ends with column l.
#pragma unroll
                        for (int w = 16; w; w >>= 1) {
                            const bool upper = lane & w;
#pragma unroll
                            for (int i = 0; i < w; i++) {
                                const float keep = upper ? v[i + w] : v[i], send = upper ? v[i] : v[i + w];
                                v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, send, w);
                            }
                        }
                        if (lane < count) g.e.col_part[(long long)(row0 >> 5) * g.e.ldcol + col + lane] = v[0];
                    }
                    __syncwarp();
                    // the rows are padded to whole pieces, which nothing reads
                    copy_strip(area, reinterpret_cast<T*>(g.e.out), g.e.ldo, true, col, min(32, (count + 7) & ~7), row0, g.m - row0, lane);
                }
            }
            if (g.bn <= share * 32) release();   // a tile of one strip: the other warps have nothing to read
            if constexpr (EPI == EPI_CE_STATS) {
                if (row_ok) {
                    const long long plane = (long long)g.e.parts * g.m, at = (long long)(2 * nb + share) * g.m + row;
                    g.e.part[at] = run.m;
                    g.e.part[plane + at] = run.s;
                    if (g.e.want_zsum) g.e.part[2 * plane + at] = zsum;
                }
            }
        }
        __syncwarp();
    }
    tc::fence_before();
    if constexpr (CG == 2)
        tc::cluster_sync();
    else
        __syncthreads();
    tc::fence_after();
    if (warp == 2) tc::tmem_free<CG>(tmem);
    // the last arrival that the other CTA's products bring here (what it needs is read anew: kept, it costs the epilogues spills)
    if (CG == 2 && threadIdx.x == 32 && tc::cta_rank() == 1) tc::bar_drain(tc::smem_u32(&bars[36]), 0, g.wait_cycles);
}

// ---- host side -----------------------------------------------------------------------------------------
// One operand: `rows` x `cols` elements, row r at data + r * ld, columns contiguous. transposed = false: rows are the
// product's m or n, columns its contracted axis; true: the other way round.
struct Operand {
    const void* data;
    long long ld;
    int rows, cols;
    bool transposed;
    int outer() const { return transposed ? cols : rows; }
    int inner() const { return transposed ? rows : cols; }
};

struct DeviceInfo {
    int sms, index;
    int* status;              // the library-wide status word
};
int device_info(DeviceInfo* out);   // of the current device; 0 or an error code
// A map of an operand's 64 x box_rows boxes in the 128-byte swizzle.
int make_map(CUtensorMap* map, const Operand& o, bool bf16, int box_rows, const char* what);
// Rows on 16-byte boundaries, as a tensor-map copy needs them.
static inline bool map_ready(const Operand& o) {
    return ((uintptr_t)o.data & 15) == 0 && (o.rows <= 1 || (o.ld & 7) == 0);
}

// How a product is cut: columns per tile, CTAs per tile, pieces of the contracted axis.
struct GemmPlan {
    int bn, cg, splits, tiles_m, tiles_n, kblocks, kblocks_per_split;
};
GemmPlan gemm_plan(const DeviceInfo& dev, int m, int n, int k, bool b_transposed, bool may_split, int bn_most = kTileNMax);

template <typename T, bool A_MN, bool B_MN, int EPI, int CG>
int gemm_launch_as(const GemmArgs& g, const DeviceInfo& dev, cudaStream_t stream, const char* what) {
    auto* kernel = gemm_kernel<T, A_MN, B_MN, EPI, CG>;
    constexpr size_t smem = kRingBytes + kEpiWarps * kStageBytes + 1024;
    static unsigned long long ready;   // a bit for each device whose kernel has its shared-memory limit
    int rc;
    if (!(__atomic_load_n(&ready, __ATOMIC_RELAXED) >> dev.index & 1)) {
        rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), what);
        if (rc) return rc;
        __atomic_fetch_or(&ready, 1ull << dev.index, __ATOMIC_RELAXED);
    }
    const long long tiles = (long long)g.tiles_m * g.tiles_n * g.splits, slots = dev.sms / CG;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((tiles < slots ? tiles : slots) * CG));
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CG;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CG == 2 ? 2 : 1;
    rc = check_cuda(cudaLaunchKernelEx(&cfg, kernel, g), what);
    if (rc) return rc;
    count_launch();
    return RB200_OK;
}

// Waits of a product: default limit, no self-test.
struct GemmWait {
    int* status;
    unsigned long long cycles;
    int skip_block;
};

// Fills the launch block. Both operands are map_ready.
int gemm_args(GemmArgs* g, const DeviceInfo& dev, int epi, bool bf16, const Operand& a, const Operand& b, const Operand* b_alt, const int* b_select, const GemmPlan& plan,
              const EpiArgs& e, const GemmWait& wait, const char* what);

template <int EPI, bool A_MN, bool B_MN>
int gemm_launch(bool bf16, const Operand& a, const Operand& b, const Operand* b_alt, const int* b_select, const GemmPlan& plan, const EpiArgs& e,
                const GemmWait& wait, cudaStream_t stream, const char* what) {
    GemmArgs g;
    DeviceInfo dev;
    int rc = device_info(&dev);
    if (rc) return rc;
    rc = gemm_args(&g, dev, EPI, bf16, a, b, b_alt, b_select, plan, e, wait, what);
    if (rc) return rc;
    if (plan.cg == 2)
        return bf16 ? gemm_launch_as<__nv_bfloat16, A_MN, B_MN, EPI, 2>(g, dev, stream, what)
                    : gemm_launch_as<__half, A_MN, B_MN, EPI, 2>(g, dev, stream, what);
    return bf16 ? gemm_launch_as<__nv_bfloat16, A_MN, B_MN, EPI, 1>(g, dev, stream, what)
                : gemm_launch_as<__half, A_MN, B_MN, EPI, 1>(g, dev, stream, what);
}

// The products with a plain epilogue (gemm.cu): x w^T (KK), dz w (KN), dz^T x (NN: both operands transposed).
enum { GEMM_KK = 0, GEMM_KN = 1, GEMM_NN = 2 };
int gemm_store(int kind, bool bf16, const Operand& a, const Operand& b, const Operand* b_alt, const int* b_select, const GemmPlan& plan,
               const EpiArgs& e, const GemmWait& wait, cudaStream_t stream, const char* what);
// The same including the second launch that joins the pieces of a split product. `partials`: gemm_partial_bytes of the plan.
size_t gemm_partial_bytes(const GemmPlan& plan, int m, int n);
int gemm_store_joined(int kind, bool bf16, const Operand& a, const Operand& b, const Operand* b_alt, const int* b_select, const GemmPlan& plan,
                      EpiArgs e, void* partials, const GemmWait& wait, cudaStream_t stream, const char* what);
// Joins the pieces: sum over splits (and acc_in), to acc_out, or scaled with bias, activation and residual to out.
int gemm_join(bool bf16, const float* partials, int splits, int m, int n, const EpiArgs& e, cudaStream_t stream, const char* what);
// An operand as a product reads it: in place, or from a copy in the workspace (operands whose rows no tensor map can
// describe). pack_operands makes the copies of up to two operands in one launch.
struct Packed {
    Operand src, use;
    bool copy;
};
int pack_operands(const Packed* a, const Packed* b, cudaStream_t stream, const char* what);

// out[c] = scale * sum over planes of part[plane * ldpart + c] (linear.cu). Many planes are first summed in groups, which take
// the place of the first planes.
int sum_planes(bool bf16, float* part, long long ldpart, int planes, int cols, void* out, const Scale& scale, cudaStream_t stream, const char* what);

static inline long long round_up(long long v, long long to) { return (v + to - 1) / to * to; }

// Carves 256-byte aligned pieces out of a workspace; with base == nullptr it only counts.
struct Carver {
    uint8_t* base;
    size_t used = 0;
    explicit Carver(void* b) : base((uint8_t*)b) {}
    void* take(size_t bytes) {
        void* p = base ? base + used : nullptr;
        used += (size_t)round_up((long long)bytes, 256);
        return p;
    }
};

}  // namespace rb200
