// rb200k_linear: out = act(x W^T + b) + r, and its gradients. The products run on the tensor cores (gemm.cuh), those of a few
// rows on the ordinary ones (few_rows_kernel). The passes over the gradient of the output that the products do not make
// (activation slope, column sums, sums over rows that share a residual row) are memory-bound and made by rows_kernel in one sweep.
#include "matrix_args.cuh"

namespace rb200 {

// ---- sweeps over a gradient matrix ------------------------------------------------------------------------
// Rows j, j + period, j + 2 period, ... of `src` are summed into partial sums [chunk][j][column] in 32 bits; with
// `preact` the elements are first multiplied by the activation's slope, and with `dst` what was read (multiplied) is
// written, in the element type: dz is an operand of two products on the tensor cores, which take 16 bits, and splitting it into two
// such numbers would double both (dx and dW are 1.4 times as far from 64 bits as with dz in 32 bits). A block takes up to 256 columns (8 a thread, as many threads side by side as the columns
// need, the others on further rows) and a chunk of the repeats; a thread has two or four rows in flight. The row sums meet in
// shared memory, chunks meet in sum_chunks_kernel, always in the same order. Bound by memory.
struct RowsArgs {
    const void* src;
    long long lds;
    const void* preact;
    long long ldp;
    void* dst;
    long long ldd;
    float* part;              // [chunks][period][ldpart] or null
    long long ldpart;
    void* out;                // one chunk only: the sums in the element type, [period][ldo], or null
    long long ldo;
    int rows, cols, period, chunks, per_chunk;   // per_chunk: repeats of a chunk
    int across;               // threads side by side: a power of two up to 32
    int act, vec_src, vec_pre;
};

template <typename T, bool SLOPE>
__global__ void __launch_bounds__(256, 4) rows_kernel(RowsArgs a) {
    constexpr int U = SLOPE ? 2 : 4;   // rows in flight
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float sums[256 * 8];
    __shared__ float half[256];
    const int lane = threadIdx.x & (a.across - 1), sub = threadIdx.x / a.across, subs = 256 / a.across, wide = a.across * 8;
    const int col = blockIdx.x * wide + lane * 8, count = a.cols - col;
    const int repeats = a.rows / a.period;
    const long long units = (long long)a.period * a.chunks;
    for (long long u = blockIdx.y; u < units; u += gridDim.y) {
        const int chunk = (int)(u / a.period), j = (int)(u - (long long)chunk * a.period);
        const int t_end = min(repeats, (chunk + 1) * a.per_chunk);
        float acc[8] = {};
        auto fetch = [&](int t, uint4& w, uint4& z) {
            const long long row = (long long)t * a.period + j;
            w = load8(reinterpret_cast<const T*>(a.src) + row * a.lds + col, count, a.vec_src);
            if (SLOPE) z = load8(reinterpret_cast<const T*>(a.preact) + row * a.ldp + col, count, a.vec_pre);
        };
        auto take = [&](int t, const uint4& w, const uint4& z) {
            float v[8];
            unpack8<T>(w, v);
            if (SLOPE) {
                float s[8];
                unpack8<T>(z, s);
                act_slopes<8>(s, a.act);
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] *= s[k];
            }
            if (a.dst) {   // the destination's rows are padded to whole vectors
                const long long row = (long long)t * a.period + j;
                *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.dst) + row * a.ldd + col) =
                    make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]), Elem<T>::pack(v[6], v[7]));
            }
#pragma unroll
            for (int k = 0; k < 8; k++) acc[k] += v[k];
        };
        if (count > 0) {
            int t = chunk * a.per_chunk + sub;
            uint4 w[U], z[U];
            for (; t + (U - 1) * subs < t_end; t += U * subs) {
#pragma unroll
                for (int i = 0; i < U; i++) fetch(t + i * subs, w[i], z[i]);
#pragma unroll
                for (int i = 0; i < U; i++) take(t + i * subs, w[i], z[i]);
            }
            for (; t < t_end; t += subs) {
                fetch(t, w[0], z[0]);
                take(t, w[0], z[0]);
            }
        }
        if (a.part || a.out) {
            // 256 / wide threads a column, 8 row sums each, then the first `wide` threads
#pragma unroll
            for (int k = 0; k < 8; k++) sums[sub * wide + lane * 8 + k] = acc[k];
            __syncthreads();
            const int c = threadIdx.x & (wide - 1), piece = threadIdx.x / wide;
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k++) s += sums[(piece * 8 + k) * wide + c];
            half[threadIdx.x] = s;
            __syncthreads();
            const int out_col = blockIdx.x * wide + c;
            if (piece == 0 && out_col < a.cols) {
                for (int k = 1; k < 256 / wide; k++) s += half[k * wide + c];
                if (a.part) a.part[u * a.ldpart + out_col] = s;
                if (a.out) reinterpret_cast<T*>(a.out)[j * a.ldo + out_col] = Elem<T>::from_float(s);
            }
            __syncthreads();
        }
    }
}

// out[j][c] = scale * sum over planes of part[plane][j][c]: 8 columns a block, planes spread over 32 threads a column.
template <typename T>
__global__ void __launch_bounds__(256) sum_chunks_kernel(const float* __restrict__ part, long long ldpart, int planes, int rows, int cols, T* out,
                                                         long long ldo, Scale scale) {
    __shared__ float sums[32][9];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 7, sub = threadIdx.x >> 3, col = blockIdx.x * 8 + lane;
    const float factor = scale.value();
    for (int j = blockIdx.y; j < rows; j += gridDim.y) {
        float s = 0.0f;
        if (col < cols) {
#pragma unroll 4
            for (int p = sub; p < planes; p += 32) s += part[((long long)p * rows + j) * ldpart + col];
        }
        sums[sub][lane] = s;
        __syncthreads();
        if (sub == 0 && col < cols) {
#pragma unroll
            for (int i = 1; i < 32; i++) s += sums[i][lane];
            out[j * ldo + col] = Elem<T>::from_float(s * factor);
        }
        __syncthreads();
    }
}

// The same for few planes: a thread takes one sum.
template <typename T>
__global__ void __launch_bounds__(256) sum_few_kernel(const float* __restrict__ part, long long ldpart, int planes, int rows, int cols, T* out,
                                                      long long ldo, Scale scale) {
    pdl_launch_dependents();
    pdl_wait();
    const float factor = scale.value();
    const long long total = (long long)rows * cols;
    for (long long t = blockIdx.x * 256ll + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
        const long long j = t / cols;
        const int col = (int)(t - j * cols);
        float s = 0.0f;
#pragma unroll 4
        for (int p = 0; p < planes; p++) s += part[((long long)p * rows + j) * ldpart + col];
        out[j * ldo + col] = Elem<T>::from_float(s * factor);
    }
}

// How the block's threads lie and how many pieces the repeats are cut into: four blocks an SM (as many as fit), at least eight
// repeats a thread.
static void cut_rows(RowsArgs* a, int sms) {
    a->across = 1;
    while (a->across < 32 && a->across * 8 < a->cols) a->across *= 2;
    const int repeats = a->rows / a->period, wide = a->across * 8, least = 256 / a->across * 8;
    const long long blocks = (long long)((a->cols + wide - 1) / wide) * a->period;
    long long chunks = 4ll * sms / blocks;
    if (chunks > (repeats + least - 1) / least) chunks = (repeats + least - 1) / least;
    if (chunks < 1) chunks = 1;
    a->per_chunk = (int)((repeats + chunks - 1) / chunks);
    a->chunks = (repeats + a->per_chunk - 1) / a->per_chunk;
}

static int rows_launch(bool bf16, const RowsArgs& a, cudaStream_t stream, const char* what) {
    const long long units = (long long)a.period * a.chunks;
    const int wide = a.across * 8;
    const dim3 grid((unsigned)((a.cols + wide - 1) / wide), (unsigned)(units < 32768 ? units : 32768));
    auto* kernel = bf16 ? (a.preact ? rows_kernel<__nv_bfloat16, true> : rows_kernel<__nv_bfloat16, false>)
                        : (a.preact ? rows_kernel<__half, true> : rows_kernel<__half, false>);
    int rc = check_cuda(launch_overlapped(kernel, grid, dim3(256), 0, stream, a), what);
    if (rc) return rc;
    count_launch();
    return RB200_OK;
}

template <typename T>
static cudaError_t sum_launch(const float* part, long long ldpart, int planes, int rows, int cols, T* out, long long ldo, const Scale& scale,
                              cudaStream_t stream) {
    const long long blocks = ((long long)rows * cols + 255) / 256;
    const dim3 grid = planes < 32 ? dim3((unsigned)(blocks < 148 * 16 ? blocks : 148 * 16))
                                  : dim3((unsigned)((cols + 7) / 8), (unsigned)(rows < 32768 ? rows : 32768));
    return launch_overlapped(planes < 32 ? sum_few_kernel<T> : sum_chunks_kernel<T>, grid, dim3(256), 0, stream, part, ldpart, planes, rows, cols,
                             out, ldo, scale);
}
static int sum_chunks(bool bf16, const float* part, long long ldpart, int planes, int rows, int cols, void* out, long long ldo, const Scale& scale,
               cudaStream_t stream, const char* what) {
    int rc = check_cuda(bf16 ? sum_launch(part, ldpart, planes, rows, cols, (__nv_bfloat16*)out, ldo, scale, stream)
                             : sum_launch(part, ldpart, planes, rows, cols, (__half*)out, ldo, scale, stream),
                        what);
    if (rc) return rc;
    count_launch();
    return RB200_OK;
}

// part[g] = sum of the planes g, g + groups, g + 2 groups, ...: a thread takes one column of one group, in place (the planes
// of a group are read by the one thread that writes the group's).
__global__ void __launch_bounds__(256) group_planes_kernel(float* part, long long ldpart, int planes, int cols, int groups) {
    pdl_launch_dependents();
    pdl_wait();
    const int col = blockIdx.x * 32 + (threadIdx.x & 31);
    const int g = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (col >= cols || g >= groups) return;
    float s = 0.0f;
#pragma unroll 8
    for (int p = g; p < planes; p += groups) s += part[p * ldpart + col];
    part[g * ldpart + col] = s;
}

int sum_planes(bool bf16, float* part, long long ldpart, int planes, int cols, void* out, const Scale& scale, cudaStream_t stream, const char* what) {
    constexpr int kGroups = 256;
    if (planes > 2 * kGroups) {
        const dim3 grid((unsigned)((cols + 31) / 32), kGroups / 8);
        int rc = check_cuda(launch_overlapped(group_planes_kernel, grid, dim3(256), 0, stream, part, ldpart, planes, cols, kGroups), what);
        if (rc) return rc;
        count_launch();
        planes = kGroups;
    }
    return sum_chunks(bf16, part, ldpart, planes, 1, cols, out, 0, scale, stream, what);
}

static int check_shape(const char* what, int dtype, int act, long long rows, long long in, long long out) {
    int rc = check_dtype(what, dtype);
    if (rc) return rc;
    if (act < RB200_ACT_NONE || act > RB200_ACT_SILU) {
        set_error("%s: activation %d is not one of RB200_ACT_*", what, act);
        return RB200_E_INVALID;
    }
    return check_extents(what, rows, "in_features", in, "out_features", out);
}

// ---- a few rows ------------------------------------------------------------------------------------------------
// Up to kFewRows rows: every element of W is used so few times that the product is a read of W, which bounds it, and a tile of
// the tensor cores would be nearly empty. A warp takes C columns and a slice of the contracted axis; a lane holds 8 elements
// of each column (16 bytes) against the same 8 of every row, whose few KB come from L1, while its next reads of W are in flight. Sums
// in 32 bits, in pairs of elements (fma.f32x2), joined across lanes and then across the block's slices in a fixed order. Rows that
// are not on 16-byte boundaries are read by elements, without packing. Several rows share what a row costs in L1 reads and
// conversions between two columns. 1 x 2048 -> 1000: 4.0 us (tensor cores 8.9), the call 6.6 us of host time (8.2: two tensor maps).
struct FewArgs {
    const void *x, *w;
    long long ldx, ldw;
    int rows, cols, k;
    int slices, per_slice;    // a power of two up to 8; elements of a slice, a multiple of 256
    EpiArgs e;
};
constexpr int kFewRows = 4;

__device__ __forceinline__ unsigned long long pair_bits(float2 f) {
    return (unsigned long long)__float_as_uint(f.y) << 32 | __float_as_uint(f.x);
}
__device__ __forceinline__ unsigned long long fma_pairs(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

template <typename T, int R, int C, bool VEC>
__global__ void __launch_bounds__(256) few_rows_kernel(const FewArgs a) {
    constexpr int N = R * C, LOG = N == 1 ? 0 : N == 4 ? 2 : 3;
    static_assert(N == 1 << LOG, "sums of a warp");
    __shared__ float part[8][N];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slice = warp & (a.slices - 1);
    const long long col0 = ((long long)blockIdx.x * (8 / a.slices) + warp / a.slices) * C;
    const int k0 = slice * a.per_slice, k1 = min(a.k, k0 + a.per_slice);
    const T *x[R], *w[C];
#pragma unroll
    for (int r = 0; r < R; r++) x[r] = reinterpret_cast<const T*>(a.x) + min(r, a.rows - 1) * a.ldx;   // what is not there is read, not kept
#pragma unroll
    for (int c = 0; c < C; c++) w[c] = reinterpret_cast<const T*>(a.w) + min(col0 + c, (long long)a.cols - 1) * a.ldw;
    float v[N];
    if constexpr (VEC) {
        unsigned long long acc[R][C] = {};
        auto add = [&](const uint4* wv, const uint4* xv) {
            unsigned long long p[C][4];
#pragma unroll
            for (int c = 0; c < C; c++) {
                p[c][0] = pair_bits(Elem<T>::unpack(wv[c].x));
                p[c][1] = pair_bits(Elem<T>::unpack(wv[c].y));
                p[c][2] = pair_bits(Elem<T>::unpack(wv[c].z));
                p[c][3] = pair_bits(Elem<T>::unpack(wv[c].w));
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                const unsigned long long q[4] = {pair_bits(Elem<T>::unpack(xv[r].x)), pair_bits(Elem<T>::unpack(xv[r].y)),
                                                 pair_bits(Elem<T>::unpack(xv[r].z)), pair_bits(Elem<T>::unpack(xv[r].w))};
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int c = 0; c < C; c++) acc[r][c] = fma_pairs(p[c][i], q[i], acc[r][c]);
            }
        };
        int k = k0 + lane * 8;
        constexpr int U = C == 1 ? 4 : 2;   // steps whose reads of W are in flight while the ones before are summed
        uint4 next[U][C];
        auto fetch = [&](int at) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int c = 0; c < C; c++) next[u][c] = __ldg(reinterpret_cast<const uint4*>(w[c] + at + 256 * u));
        };
        auto whole = [&](int at) { return at + 256 * (U - 1) + 8 <= k1; };
        if (whole(k)) fetch(k);
#pragma unroll 1
        for (; whole(k); k += 256 * U) {
            uint4 wv[U][C];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int c = 0; c < C; c++) wv[u][c] = next[u][c];
            if (whole(k + 256 * U)) fetch(k + 256 * U);
#pragma unroll
            for (int u = 0; u < U; u++) {
                uint4 xv[R];
#pragma unroll
                for (int r = 0; r < R; r++) xv[r] = __ldg(reinterpret_cast<const uint4*>(x[r] + k + 256 * u));
                add(wv[u], xv);
            }
        }
#pragma unroll 1
        for (; k < k1; k += 256) {
            uint4 wv[C], xv[R];
#pragma unroll
            for (int c = 0; c < C; c++) wv[c] = load8(w[c] + k, k1 - k, true);
#pragma unroll
            for (int r = 0; r < R; r++) xv[r] = load8(x[r] + k, k1 - k, true);
            add(wv, xv);
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < C; c++) v[r * C + c] = __uint_as_float((uint32_t)acc[r][c]) + __uint_as_float((uint32_t)(acc[r][c] >> 32));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = 0.0f;
#pragma unroll 4
        for (int k = k0 + lane; k < k1; k += 32) {
            float p[C];
#pragma unroll
            for (int c = 0; c < C; c++) p[c] = Elem<T>::to_float(w[c][k]);
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float q = Elem<T>::to_float(x[r][k]);
#pragma unroll
                for (int c = 0; c < C; c++) v[r * C + c] = fmaf(p[c], q, v[r * C + c]);
            }
        }
    }
    // Halves of the lanes exchange halves of the sums, until each sum is in 32 >> LOG neighbouring lanes, then those lanes join theirs.
#pragma unroll
    for (int s = 0; s < 5; s++) {
        const int d = 16 >> s;
        if (s < LOG) {
            const int h = N >> (s + 1);
            const bool upper = lane & d;
#pragma unroll
            for (int i = 0; i < h; i++) {
                const float give = upper ? v[i] : v[i + h], keep = upper ? v[i + h] : v[i];
                v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, d);
            }
        } else {
            v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], d);
        }
    }
    const int at = lane >> (5 - LOG);   // the sum that the lane holds
    const bool owner = (lane & ((32 >> LOG) - 1)) == 0;
    float z = v[0];
    if (a.slices > 1) {
        if (owner) part[warp][at] = z;
        __syncthreads();
        if (slice) return;
        for (int s = 1; s < a.slices; s++) z += part[warp + s][at];
    }
    const int row = at / C;
    const long long col = col0 + at % C;
    if (!owner || row >= a.rows || col >= a.cols) return;
    if (a.e.bias) z += Elem<T>::to_float(reinterpret_cast<const T*>(a.e.bias)[col]);
    if (a.e.preact) reinterpret_cast<T*>(a.e.preact)[row * a.e.ldp + col] = Elem<T>::from_float(z);
    act_values<1>(&z, a.e.act);
    if (a.e.residual) z += Elem<T>::to_float(reinterpret_cast<const T*>(a.e.residual)[row % a.e.residual_rows * a.e.ldr + col]);
    reinterpret_cast<T*>(a.e.out)[row * a.e.ldo + col] = Elem<T>::from_float(z);
}

// Rows on 16-byte boundaries: one or two rows read W at up to 4.8 TB/s whatever its size (1 x 4096 -> 4096: 9.6 us, tensor cores and
// their joining launch 13.9; 8192 -> 8192: 28 against 31); three and four are as long as the tensor cores at 2^24 elements (12.0
// against 13.9 us) and slower beyond (39 against 31). Other rows would have to be packed first: 4 x 8191 -> 8192 takes 58 us against
// 121. A long contracted axis needs more slices than a block's eight (1 x 100000 -> 1024: 65 against 41 us).
static bool few_vec(const rb200_linear_params& p) {
    return map_ready(operand(p.x, p.ldx, p.rows, p.in_features, false)) && map_ready(operand(p.weight, p.ldw, p.out_features, p.in_features, false));
}
static bool few_rows(const rb200_linear_params& p) {
    return p.rows <= kFewRows && p.in_features <= 16384 && (p.rows <= 2 || p.in_features * p.out_features <= (1 << 24) || !few_vec(p));
}
template <typename T>
static int few_launch(FewArgs& a, bool vec, int sms, cudaStream_t stream, const char* what) {
    const int columns = a.rows == 1 ? 1 : 2;
    const long long warps = (a.cols + columns - 1) / columns;
    a.slices = 1;
    // eight warps an SM; single elements, of which a warp has less in flight, want more of them (2 x 8191 -> 8192: 64 us, then 45; whole
    // vectors lose by it: 1 x 4096 -> 4096 9.6 us, then 11.8)
    while (a.slices < 8 && a.k > 256 * a.slices && (warps * a.slices < 8ll * sms || (!vec && a.k >= 2048 * a.slices && warps * a.slices < 192ll * sms)))
        a.slices *= 2;
    a.per_slice = (int)round_up((a.k + a.slices - 1) / a.slices, 256);
    const dim3 grid((unsigned)((warps * a.slices + 7) / 8));
    void (*kernel)(FewArgs) = a.rows == 1   ? (vec ? few_rows_kernel<T, 1, 1, true> : few_rows_kernel<T, 1, 1, false>)
                              : a.rows == 2 ? (vec ? few_rows_kernel<T, 2, 2, true> : few_rows_kernel<T, 2, 2, false>)
                                            : (vec ? few_rows_kernel<T, 4, 2, true> : few_rows_kernel<T, 4, 2, false>);
    const int rc = check_cuda(launch_overlapped(kernel, grid, dim3(256), 0, stream, a), what);
    if (rc) return rc;
    count_launch();
    return RB200_OK;
}

// ---- forward ------------------------------------------------------------------------------------------------
struct LinearPlan {
    bool few;
    Packed x, w;
    GemmPlan gemm;
    void* partials;
    size_t bytes;
};
static LinearPlan plan_linear(const rb200_linear_params& p, const DeviceInfo& dev, void* ws) {
    LinearPlan l;
    Carver c(ws);
    l.few = few_rows(p);
    l.bytes = 0;
    if (l.few) return l;
    l.x = plan_pack(operand(p.x, p.ldx, p.rows, p.in_features, false), &c);
    l.w = plan_pack(operand(p.weight, p.ldw, p.out_features, p.in_features, false), &c);
    l.gemm = gemm_plan(dev, (int)p.rows, (int)p.out_features, (int)p.in_features, false, true);
    l.partials = c.take(gemm_partial_bytes(l.gemm, (int)p.rows, (int)p.out_features));
    l.bytes = c.used;
    return l;
}

static int linear_run(const rb200_linear_params* p, void* stream_v, GemmWait wait) {
    const char* what = "rb200k_linear";
    if (!p) {
        set_error("%s: params is null", what);
        return RB200_E_INVALID;
    }
    int rc = check_shape(what, p->dtype, p->activation, p->rows, p->in_features, p->out_features);
    if (rc) return rc;
    if (p->rows == 0) return RB200_OK;
    if ((rc = check_matrix(what, "x", p->x, p->ldx, p->rows, p->in_features))) return rc;
    if ((rc = check_matrix(what, "weight", p->weight, p->ldw, p->out_features, p->in_features))) return rc;
    if ((rc = check_matrix(what, "out", p->out, p->ldo, p->rows, p->out_features))) return rc;
    if (p->bias && (rc = check_matrix(what, "bias", p->bias, 0, 1, p->out_features))) return rc;
    if (p->preact && (rc = check_matrix(what, "preact", p->preact, p->ldp, p->rows, p->out_features))) return rc;
    if (p->residual) {
        if (p->residual_rows < 1 || p->rows % p->residual_rows) {
            set_error("%s: residual_rows %lld does not divide rows %lld", what, (long long)p->residual_rows, (long long)p->rows);
            return RB200_E_INVALID;
        }
        if ((rc = check_matrix(what, "residual", p->residual, p->ldr, p->residual_rows, p->out_features))) return rc;
    }
    DeviceInfo dev;
    if ((rc = device_info(&dev))) return rc;
    const LinearPlan l = plan_linear(*p, dev, p->workspace);
    if ((rc = check_workspace(what, p->workspace, p->workspace_bytes, l.bytes))) return rc;
    cudaStream_t stream = (cudaStream_t)stream_v;
    const bool bf16 = p->dtype == RB200_BF16;
    EpiArgs e = {};
    e.out = p->out;
    e.ldo = p->ldo;
    e.bias = p->bias;
    e.residual = p->residual;
    e.ldr = p->ldr;
    e.residual_rows = (int)p->residual_rows;
    e.preact = p->preact;
    e.ldp = p->ldp;
    e.act = p->activation;
    if (l.few) {
        FewArgs a = {p->x, p->weight, p->ldx, p->ldw, (int)p->rows, (int)p->out_features, (int)p->in_features, 1, 0, e};
        const bool vec = few_vec(*p);
        return bf16 ? few_launch<__nv_bfloat16>(a, vec, dev.sms, stream, what) : few_launch<__half>(a, vec, dev.sms, stream, what);
    }
    if ((rc = pack_operands(&l.x, &l.w, stream, what))) return rc;
    wait.status = p->status;
    if (l.gemm.splits > 1) {
        EpiArgs part = {};
        part.acc_out = (float*)l.partials;
        part.ldacc = round_up(p->out_features, 4);
        part.acc_split_stride = part.ldacc * p->rows;
        if ((rc = gemm_store(GEMM_KK, bf16, l.x.use, l.w.use, nullptr, nullptr, l.gemm, part, wait, stream, what))) return rc;
        return gemm_join(bf16, (const float*)l.partials, l.gemm.splits, (int)p->rows, (int)p->out_features, e, stream, what);
    }
    if (e.residual) return gemm_launch<EPI_LINEAR_ADD, false, false>(bf16, l.x.use, l.w.use, nullptr, nullptr, l.gemm, e, wait, stream, what);
    return gemm_launch<EPI_LINEAR, false, false>(bf16, l.x.use, l.w.use, nullptr, nullptr, l.gemm, e, wait, stream, what);
}

// ---- backward -----------------------------------------------------------------------------------------------
struct LinearBackwardPlan {
    Packed x, w;
    Operand dz;               // [rows][out]: dout itself, or the copy that rows_kernel writes
    bool own_dz, sums, reuse; // sums: rows_kernel makes the column sums; reuse: they come from the residual's
    RowsArgs bias_rows, res_rows;
    GemmPlan gx, gw;
    void *px, *pw;
    size_t bytes;
};
static LinearBackwardPlan plan_backward(const rb200_linear_backward_params& p, const DeviceInfo& dev, void* ws) {
    LinearBackwardPlan l = {};
    Carver c(ws);
    const int n = (int)p.rows, k = (int)p.in_features, m = (int)p.out_features;
    const Operand dout = operand(p.dout, p.lddo, p.rows, p.out_features, false);
    const bool products = p.dx || p.dweight;
    l.own_dz = products && (p.activation != RB200_ACT_NONE || !map_ready(dout));
    l.dz = dout;
    if (l.own_dz) {
        l.dz.ld = round_up(m, 8);
        l.dz.data = c.take((size_t)l.dz.ld * n * 2);
    }
    if (p.dx) {
        l.w = plan_pack(operand(p.weight, p.ldw, m, k, true), &c);
        l.gx = gemm_plan(dev, n, k, m, true, true);
        l.px = c.take(gemm_partial_bytes(l.gx, n, k));
    }
    if (p.dweight) {
        l.x = plan_pack(operand(p.x, p.ldx, n, k, true), &c);
        l.gw = gemm_plan(dev, m, k, n, true, true);
        l.pw = c.take(gemm_partial_bytes(l.gw, m, k));
    }
    RowsArgs a = {};
    a.src = p.dout;
    a.lds = p.lddo;
    a.rows = n;
    a.cols = m;
    a.vec_src = map_ready(dout);
    a.ldpart = round_up(m, 4);
    if (p.dresidual) {
        l.res_rows = a;
        l.res_rows.period = (int)p.residual_rows;
        cut_rows(&l.res_rows, dev.sms);
        // whole sums leave in the element type at once; 32-bit ones are kept for further sums
        if (l.res_rows.chunks == 1) {
            l.res_rows.out = p.dresidual;
            l.res_rows.ldo = p.lddr;
        }
        // without an activation the column sums are the sums of the residual's sums, if those are few: no second sweep
        l.reuse = p.dbias && p.activation == RB200_ACT_NONE && (long long)l.res_rows.chunks * l.res_rows.period <= 1024;
        if (l.res_rows.chunks > 1 || l.reuse)
            l.res_rows.part = (float*)c.take((size_t)l.res_rows.chunks * l.res_rows.period * a.ldpart * sizeof(float));
    }
    l.sums = p.dbias && !l.reuse;
    l.bias_rows = a;
    l.bias_rows.period = 1;
    cut_rows(&l.bias_rows, dev.sms);
    if (p.activation != RB200_ACT_NONE) {
        l.bias_rows.preact = p.preact;
        l.bias_rows.ldp = p.ldp;
        l.bias_rows.act = p.activation;
        l.bias_rows.vec_pre = map_ready(operand(p.preact, p.ldp, p.rows, p.out_features, false));
    }
    if (l.own_dz) {
        l.bias_rows.dst = const_cast<void*>(l.dz.data);
        l.bias_rows.ldd = l.dz.ld;
    }
    if (l.sums) l.bias_rows.part = (float*)c.take((size_t)l.bias_rows.chunks * a.ldpart * sizeof(float));
    l.bytes = c.used;
    return l;
}

static int backward_run(const rb200_linear_backward_params* p, void* stream_v) {
    const char* what = "rb200k_linear_backward";
    if (!p) {
        set_error("%s: params is null", what);
        return RB200_E_INVALID;
    }
    int rc = check_shape(what, p->dtype, p->activation, p->rows, p->in_features, p->out_features);
    if (rc) return rc;
    cudaStream_t stream = (cudaStream_t)stream_v;
    const long long n = p->rows, k = p->in_features, m = p->out_features;
    if (p->dweight && (rc = check_matrix(what, "dweight", p->dweight, p->lddw, m, k))) return rc;
    if (p->dbias && (rc = check_matrix(what, "dbias", p->dbias, 0, 1, m))) return rc;
    if (p->dresidual) {
        if (p->residual_rows < 1 || n % p->residual_rows) {
            set_error("%s: residual_rows %lld does not divide rows %lld", what, (long long)p->residual_rows, n);
            return RB200_E_INVALID;
        }
        if ((rc = check_matrix(what, "dresidual", p->dresidual, p->lddr, p->residual_rows, m))) return rc;
    }
    if (n == 0) {   // nothing flows back: the sums over no rows are zero
        if (p->dweight && (rc = clear_matrix(p->dweight, p->lddw, m, k, stream, what))) return rc;
        if (p->dbias && (rc = clear_matrix(p->dbias, 0, 1, m, stream, what))) return rc;
        if (p->dresidual && (rc = clear_matrix(p->dresidual, p->lddr, p->residual_rows, m, stream, what))) return rc;
        return RB200_OK;
    }
    if ((rc = check_matrix(what, "dout", p->dout, p->lddo, n, m))) return rc;
    if (p->dx && ((rc = check_matrix(what, "weight", p->weight, p->ldw, m, k)) || (rc = check_matrix(what, "dx", p->dx, p->lddx, n, k)))) return rc;
    if (p->dweight && (rc = check_matrix(what, "x", p->x, p->ldx, n, k))) return rc;
    if (p->activation != RB200_ACT_NONE && (p->dx || p->dweight || p->dbias) && (rc = check_matrix(what, "preact", p->preact, p->ldp, n, m)))
        return rc;
    DeviceInfo dev;
    if ((rc = device_info(&dev))) return rc;
    const LinearBackwardPlan l = plan_backward(*p, dev, p->workspace);
    if ((rc = check_workspace(what, p->workspace, p->workspace_bytes, l.bytes))) return rc;
    const bool bf16 = p->dtype == RB200_BF16;
    if (p->dresidual) {
        const RowsArgs& r = l.res_rows;
        if ((rc = rows_launch(bf16, r, stream, what))) return rc;
        if (!r.out && (rc = sum_chunks(bf16, r.part, r.ldpart, r.chunks, r.period, (int)m, p->dresidual, p->lddr, Scale(), stream, what))) return rc;
        if (l.reuse &&
            (rc = sum_chunks(bf16, r.part, r.ldpart, r.chunks * r.period, 1, (int)m, p->dbias, 0, Scale(), stream, what)))
            return rc;
    }
    if (l.sums || l.own_dz) {
        const RowsArgs& r = l.bias_rows;
        if ((rc = rows_launch(bf16, r, stream, what))) return rc;
        if (l.sums && (rc = sum_chunks(bf16, r.part, r.ldpart, r.chunks, 1, (int)m, p->dbias, 0, Scale(), stream, what))) return rc;
    }
    const GemmWait wait = {p->status, 0, -1};
    if ((rc = pack_operands(p->dx ? &l.w : nullptr, p->dweight ? &l.x : nullptr, stream, what))) return rc;
    EpiArgs e = {};
    if (p->dx) {
        e.out = p->dx;
        e.ldo = p->lddx;
        if ((rc = gemm_store_joined(GEMM_KN, bf16, l.dz, l.w.use, nullptr, nullptr, l.gx, e, l.px, wait, stream, what))) return rc;
    }
    if (p->dweight) {
        e.out = p->dweight;
        e.ldo = p->lddw;
        Operand dzt = l.dz;
        dzt.transposed = true;
        if ((rc = gemm_store_joined(GEMM_NN, bf16, dzt, l.x.use, nullptr, nullptr, l.gw, e, l.pw, wait, stream, what))) return rc;
    }
    return RB200_OK;
}

}  // namespace rb200

using namespace rb200;

extern "C" uint64_t rb200k_linear_workspace_bytes(const rb200_linear_params* p) {
    DeviceInfo dev;
    if (!p || check_shape("rb200k_linear_workspace_bytes", p->dtype, p->activation, p->rows, p->in_features, p->out_features) || p->rows == 0 ||
        device_info(&dev))
        return 0;
    return plan_linear(*p, dev, nullptr).bytes;
}
extern "C" int rb200k_linear(const rb200_linear_params* p, void* stream) { return linear_run(p, stream, GemmWait{nullptr, 0, -1}); }
extern "C" int rb200k_linear_probe(const rb200_linear_params* p, void* stream, uint64_t wait_cycles, int skip_block) {
    return linear_run(p, stream, GemmWait{nullptr, wait_cycles, skip_block});
}
extern "C" uint64_t rb200k_linear_backward_workspace_bytes(const rb200_linear_backward_params* p) {
    DeviceInfo dev;
    if (!p || check_shape("rb200k_linear_backward_workspace_bytes", p->dtype, p->activation, p->rows, p->in_features, p->out_features) ||
        p->rows == 0 || (p->dresidual && (p->residual_rows < 1 || p->rows % p->residual_rows)) || device_info(&dev))
        return 0;
    return plan_backward(*p, dev, nullptr).bytes;
}
extern "C" int rb200k_linear_backward(const rb200_linear_backward_params* p, void* stream) { return backward_run(p, stream); }
