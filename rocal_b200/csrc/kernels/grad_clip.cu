// rb200k_grad_clip: norm over many tensors and clipping. Two sweeps, both bound by memory: the first adds the squares,
// the second multiplies. The tensors' table travels in the launch's own parameters (no copy, nothing to keep alive, and
// a captured graph holds it). Tensors are cut into chunks of one size, which blocks take in turn; the second sweep walks
// the chunks backwards, so that what the first one read last is still in L2. Few elements take one launch.
#include <algorithm>
#include <new>
#include <vector>

#include "gemm.cuh"

namespace rb200 {

constexpr int kClipThreads = 256, kClipBlocksPerSm = 8;
constexpr int kClipMaxBlocks = 148 * kClipBlocksPerSm;   // partial sums a launch leaves at most

struct ClipEntry {
    const void* grad;
    void* out;
    long long count;
    int chunk0;         // of this tensor, counted over the launch's table
    short grad_dtype, out_dtype;
};
template <int CAP>
struct ClipTable {
    ClipEntry e[CAP];
    int n, chunks;
    int chunk;          // elements
};

template <int CAP>
__device__ __forceinline__ int find_tensor(const ClipTable<CAP>& t, int c) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].chunk0 <= c)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

template <typename T>
struct Values;   // of one 16-byte vector
template <>
struct Values<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const uint4& w, float* v) {
        v[0] = __uint_as_float(w.x);
        v[1] = __uint_as_float(w.y);
        v[2] = __uint_as_float(w.z);
        v[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ uint4 put(const float* v) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    static __device__ __forceinline__ float to_float(float v) { return v; }
    static __device__ __forceinline__ float from_float(float v) { return v; }
};
template <typename T>
struct Values16 {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& w, float* v) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = Elem<T>::unpack(u[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 put(const float* v) {
        return make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]), Elem<T>::pack(v[6], v[7]));
    }
    static __device__ __forceinline__ float to_float(T v) { return Elem<T>::to_float(v); }
    static __device__ __forceinline__ T from_float(float v) { return Elem<T>::from_float(v); }
};
template <>
struct Values<__half> : Values16<__half> {};
template <>
struct Values<__nv_bfloat16> : Values16<__nv_bfloat16> {};

// ---- sum of squares ---------------------------------------------------------------------------------------
// STAYS: nothing writes the gradients while the kernel runs, so that they may be read past the coherent path.
template <bool STAYS>
__device__ __forceinline__ uint4 load_vector(const uint4* p) {
    if constexpr (STAYS)
        return __ldg(p);
    else
        return *p;
}
template <bool STAYS, typename T>
__device__ __forceinline__ double square_sum(const T* p, int count) {
    constexpr int N = Values<T>::N;
    double s = 0.0;
    const int head = min(count, (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T)));   // up to the 16-byte boundary
    if ((int)threadIdx.x < head) {
        const double v = Values<T>::to_float(p[threadIdx.x]);
        s = v * v;
    }
    p += head;
    count -= head;
    const uint4* q = reinterpret_cast<const uint4*>(p);
    const int vectors = count / N;
    auto add = [&](const uint4& w) {
        float v[N];
        Values<T>::get(w, v);
#pragma unroll
        for (int j = 0; j < N; j++) s += (double)v[j] * (double)v[j];
    };
    int i = threadIdx.x;
    for (; i + 3 * kClipThreads < vectors; i += 4 * kClipThreads) {   // four vectors in flight
        uint4 w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = load_vector<STAYS>(q + i + k * kClipThreads);
#pragma unroll
        for (int k = 0; k < 4; k++) add(w[k]);
    }
    for (; i < vectors; i += kClipThreads) add(load_vector<STAYS>(q + i));
    const int tail = vectors * N + threadIdx.x;
    if (tail < count) {
        const double v = Values<T>::to_float(p[tail]);
        s += v * v;
    }
    return s;
}

template <bool STAYS>
__device__ __forceinline__ double square_piece(const ClipEntry& e, long long begin, int count) {
    if (e.grad_dtype == RB200_FP32) return square_sum<STAYS>(reinterpret_cast<const float*>(e.grad) + begin, count);
    if (e.grad_dtype == RB200_FP16) return square_sum<STAYS>(reinterpret_cast<const __half*>(e.grad) + begin, count);
    return square_sum<STAYS>(reinterpret_cast<const __nv_bfloat16*>(e.grad) + begin, count);
}

// The block's sum, in thread 0.
__device__ __forceinline__ double block_sum(double s, double* shared) {
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int i = 1; i < kClipThreads / 32; i++) s += shared[i];
    return s;
}

template <int CAP>
__global__ void __launch_bounds__(kClipThreads) clip_norm_kernel(const __grid_constant__ ClipTable<CAP> t, double* partial) {
    __shared__ double shared[kClipThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    double s = 0.0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const ClipEntry& e = t.e[find_tensor(t, c)];
        const long long begin = (long long)(c - e.chunk0) * t.chunk;
        const int count = (int)min((long long)t.chunk, e.count - begin);
        s += square_piece<true>(e, begin, count);
    }
    s = block_sum(s, shared);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// ---- multiplication -----------------------------------------------------------------------------------------
template <int W>
__device__ __forceinline__ void load_words(const uint32_t* p, uint32_t* w) {
    if constexpr (W == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x;
        w[1] = v.y;
    }
}
// One output vector: as many gradients as sixteen bytes of the output hold, so that a warp's stores are whole lines.
template <typename T, typename O>
__device__ __forceinline__ uint4 scale_words(const uint32_t* w, float factor) {
    constexpr int N = Values<O>::N;
    float v[N];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = __uint_as_float(w[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float2 f = Elem<T>::unpack(w[j / 2]);
            v[j] = f.x;
            v[j + 1] = f.y;
        }
    }
#pragma unroll
    for (int j = 0; j < N; j++) v[j] *= factor;
    return Values<O>::put(v);
}
// SHIFT < 0: the gradients have boundaries of their own words where the output has its 16-byte ones. Outputs are written
// past L2, where gradients still wait for their second read.
template <typename T, typename O, int SHIFT>
__device__ __forceinline__ void scale_vectors(const T* g, O* o, int vectors, float factor) {
    constexpr int W = Values<O>::N * (int)sizeof(T) / 4, U = 16 / W;   // U vectors in flight
    const uint32_t* q = reinterpret_cast<const uint32_t*>((uintptr_t)g & ~(uintptr_t)(4 * W - 1));
    const int bits = (int)((uintptr_t)g & 3) * 8;
    uint4* out = reinterpret_cast<uint4*>(o);
    auto fetch = [&](int i, uint32_t (&w)[W]) {   // the second vector is one that the window reaches into
        if constexpr (SHIFT < 0) {
            load_words<W>(q + i * W, w);
        } else {
            uint32_t both[2 * W];
            load_words<W>(q + i * W, both);
            load_words<W>(q + (i + 1) * W, both + W);
            window<W, SHIFT>(both, w, bits);
        }
    };
    int i = threadIdx.x;
    for (; i + (U - 1) * kClipThreads < vectors; i += U * kClipThreads) {
        uint32_t w[U][W];
#pragma unroll
        for (int k = 0; k < U; k++) fetch(i + k * kClipThreads, w[k]);
#pragma unroll
        for (int k = 0; k < U; k++) __stcs(out + i + k * kClipThreads, scale_words<T, O>(w[k], factor));
    }
    for (; i < vectors; i += kClipThreads) {
        uint32_t w[W];
        fetch(i, w);
        __stcs(out + i, scale_words<T, O>(w, factor));
    }
}
// Whole vectors are written where the output has its 16-byte boundaries; the gradients that belong there are cut out of
// the aligned vectors that hold them.
template <typename T, typename O>
__device__ __forceinline__ void scale_chunk(const T* g, O* o, int count, float factor) {
    constexpr int N = Values<O>::N, W = N * (int)sizeof(T) / 4;
    const int head = min(count, (int)(((16 - ((uintptr_t)o & 15)) & 15) / sizeof(O)));
    if ((int)threadIdx.x < head) o[threadIdx.x] = Values<O>::from_float(Values<T>::to_float(g[threadIdx.x]) * factor);
    g += head;
    o += head;
    count -= head;
    const int vectors = count / N, offset = (int)((uintptr_t)g & (4 * W - 1));
    if (offset == 0) {
        scale_vectors<T, O, -1>(g, o, vectors, factor);
    } else if (W == 2) {
        if (offset < 4)
            scale_vectors<T, O, 0>(g, o, vectors, factor);
        else
            scale_vectors<T, O, 1>(g, o, vectors, factor);
    } else {
        switch (offset >> 2) {
            case 0: scale_vectors<T, O, 0>(g, o, vectors, factor); break;
            case 1: scale_vectors<T, O, 1>(g, o, vectors, factor); break;
            case 2: scale_vectors<T, O, W == 2 ? 0 : 2>(g, o, vectors, factor); break;
            default: scale_vectors<T, O, W == 2 ? 1 : 3>(g, o, vectors, factor); break;
        }
    }
    const int tail = vectors * N + threadIdx.x;
    if (tail < count) o[tail] = Values<O>::from_float(Values<T>::to_float(g[tail]) * factor);
}
__device__ __forceinline__ void scale_piece(const ClipEntry& e, long long begin, int count, float factor) {
    if (factor == 1.0f && e.out == e.grad) return;
    if (e.grad_dtype == RB200_FP32) {
        scale_chunk(reinterpret_cast<const float*>(e.grad) + begin, reinterpret_cast<float*>(e.out) + begin, count, factor);
    } else if (e.grad_dtype == RB200_FP16) {
        const __half* g = reinterpret_cast<const __half*>(e.grad) + begin;
        if (e.out_dtype == RB200_FP32)
            scale_chunk(g, reinterpret_cast<float*>(e.out) + begin, count, factor);
        else
            scale_chunk(g, reinterpret_cast<__half*>(e.out) + begin, count, factor);
    } else {
        const __nv_bfloat16* g = reinterpret_cast<const __nv_bfloat16*>(e.grad) + begin;
        if (e.out_dtype == RB200_FP32)
            scale_chunk(g, reinterpret_cast<float*>(e.out) + begin, count, factor);
        else
            scale_chunk(g, reinterpret_cast<__nv_bfloat16*>(e.out) + begin, count, factor);
    }
}
// The norm and the factor of a sum of squares.
__device__ __forceinline__ float clip_factor(double sum, float max_norm, float inv_scale, float* norm) {
    const float n = (float)(sqrt(sum) * (double)inv_scale);
    const float c = max_norm / (n + 1e-6f);
    if (norm) *norm = n;
    return (c > 1.0f ? 1.0f : c) * inv_scale;   // NaN stays
}

template <int CAP>
__global__ void __launch_bounds__(kClipThreads) clip_scale_kernel(const __grid_constant__ ClipTable<CAP> t, const double* __restrict__ partial,
                                                                  int partials, float max_norm, float inv_scale, float* norm) {
    __shared__ double shared[kClipThreads / 32];
    __shared__ float factor_s;
    pdl_launch_dependents();
    pdl_wait();
    double s = 0.0;
    for (int i = threadIdx.x; i < partials; i += kClipThreads) s += partial[i];
    s = block_sum(s, shared);
    if (threadIdx.x == 0) factor_s = clip_factor(s, max_norm, inv_scale, blockIdx.x == 0 ? norm : nullptr);
    __syncthreads();
    const float factor = factor_s;
    for (int i = blockIdx.x; i < t.chunks; i += gridDim.x) {
        const int c = t.chunks - 1 - i;
        const ClipEntry& e = t.e[find_tensor(t, c)];
        const long long begin = (long long)(c - e.chunk0) * t.chunk;
        scale_piece(e, begin, (int)min((long long)t.chunk, e.count - begin), factor);
    }
}

// ---- both sweeps in one launch ----------------------------------------------------------------------------------
// Few elements: one cluster of eight blocks, which exchange their sums through distributed shared memory. Sums are added in
// rank order by every block, so all of them have the same factor.
constexpr int kClipCluster = 8;
constexpr long long kClipFew = 131072;
// Eight blocks take the tensors one after another, 0.2 us each: 60 of them 12 us. Two launches over as many blocks as there are tensors
// take the device 6 us, but the host 18.
constexpr size_t kClipFewTensors = 96;
template <int CAP>
__global__ void __launch_bounds__(kClipThreads) __cluster_dims__(kClipCluster, 1, 1)
    clip_few_kernel(const __grid_constant__ ClipTable<CAP> t, float max_norm, float inv_scale, float* norm) {
    __shared__ double shared[kClipThreads / 32];
    __shared__ double sums[kClipCluster];
    __shared__ float factor_s;
    tc::cluster_arrive();
    pdl_launch_dependents();
    pdl_wait();
    double s = 0.0;
    for (int c = blockIdx.x; c < t.chunks; c += kClipCluster) {
        const ClipEntry& e = t.e[find_tensor(t, c)];
        const long long begin = (long long)(c - e.chunk0) * t.chunk;
        s += square_piece<false>(e, begin, (int)min((long long)t.chunk, e.count - begin));   // written below, in place
    }
    s = block_sum(s, shared);
    __syncwarp();
    tc::cluster_wait();   // all eight blocks have started: their shared memory may be written
    if (threadIdx.x == 0) {
        const uint32_t mine = tc::smem_u32(&sums[tc::cta_rank()]);
#pragma unroll
        for (int r = 0; r < kClipCluster; r++)
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(tc::map_to_rank(mine, r)), "d"(s) : "memory");
    }
    __syncwarp();
    tc::cluster_sync();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int r = 0; r < kClipCluster; r++) s += sums[r];
        factor_s = clip_factor(s, max_norm, inv_scale, blockIdx.x == 0 ? norm : nullptr);
    }
    __syncthreads();
    const float factor = factor_s;
    for (int c = blockIdx.x; c < t.chunks; c += kClipCluster) {
        const ClipEntry& e = t.e[find_tensor(t, c)];
        const long long begin = (long long)(c - e.chunk0) * t.chunk;
        scale_piece(e, begin, (int)min((long long)t.chunk, e.count - begin), factor);
    }
}

// ---- host ---------------------------------------------------------------------------------------------------
constexpr int kClipMedium = 192, kClipLarge = 960;   // 960 entries: 30 KB of launch parameters

enum { CLIP_NORM, CLIP_SCALE, CLIP_FEW };
template <int CAP>
static int clip_table_launch(const ClipEntry* entries, int n, int chunks, int chunk, int sweep, double* partial, int partials, float max_norm,
                             float inv_scale, float* norm, int blocks, cudaStream_t stream) {
    ClipTable<CAP> t;
    for (int i = 0; i < n; i++) t.e[i] = entries[i];
    t.n = n;
    t.chunks = chunks;
    t.chunk = chunk;
    const dim3 grid(blocks), block(kClipThreads);
    int rc = check_cuda(sweep == CLIP_NORM    ? launch_overlapped(clip_norm_kernel<CAP>, grid, block, 0, stream, t, partial)
                        : sweep == CLIP_SCALE ? launch_overlapped(clip_scale_kernel<CAP>, grid, block, 0, stream, t, (const double*)partial, partials,
                                                                  max_norm, inv_scale, norm)
                                              : launch_overlapped(clip_few_kernel<CAP>, grid, block, 0, stream, t, max_norm, inv_scale, norm),
                        "rb200k_grad_clip");
    if (rc) return rc;
    count_launch();
    return RB200_OK;
}

static size_t clip_bytes(int dtype) { return dtype == RB200_FP32 ? 4 : 2; }

// No output meets another output or another tensor's gradients. Outputs and gradients are put in order on their own, which they
// usually are already (allocated one after another, or pieces of one buffer): a walk through both then takes 2 us for the 600
// ranges of 300 tensors, where sorting them together took 7 to 30.
struct ClipRange {
    uintptr_t begin, end;
};
static void order_ranges(std::vector<ClipRange>& r) {
    for (size_t i = 1; i < r.size(); i++)
        if (r[i].begin < r[i - 1].begin) {
            std::sort(r.begin(), r.end(), [](const ClipRange& a, const ClipRange& b) { return a.begin < b.begin; });
            return;
        }
}
static bool outputs_disjoint(const std::vector<ClipEntry>& v) {
    std::vector<ClipRange> outs, grads;   // gradients that are not their own outputs
    outs.reserve(v.size());
    for (const ClipEntry& e : v) {
        const uintptr_t g = (uintptr_t)e.grad, o = (uintptr_t)e.out;
        outs.push_back({o, o + e.count * clip_bytes(e.out_dtype)});
        if (g != o) {
            if (grads.empty()) grads.reserve(v.size());
            grads.push_back({g, g + e.count * clip_bytes(e.grad_dtype)});
        }
    }
    order_ranges(outs);
    order_ranges(grads);
    for (size_t i = 1; i < outs.size(); i++)
        if (outs[i].begin < outs[i - 1].end) return false;
    size_t o = 0;   // outputs do not overlap, so their ends are in order, too
    for (const ClipRange& g : grads) {
        while (o < outs.size() && outs[o].end <= g.begin) o++;
        if (o < outs.size() && outs[o].begin < g.end) return false;
    }
    return true;
}

static int clip_run(const rb200_grad_tensor* tensors, int n, float max_norm, float inv_scale, float* norm, void* ws, uint64_t ws_bytes,
                    cudaStream_t stream) {
    const char* what = "rb200k_grad_clip";
    if (n < 0 || (n && !tensors) || !norm || ((uintptr_t)norm & 3)) {
        set_error("%s: null pointer, misaligned norm or negative count", what);
        return RB200_E_INVALID;
    }
    if (!(max_norm >= 0.0f) || !(inv_scale > 0.0f && inv_scale <= 3.4028235e38f)) {
        set_error("%s: max_norm %g, inv_scale %g", what, max_norm, inv_scale);
        return RB200_E_INVALID;
    }
    std::vector<ClipEntry> v;
    v.reserve(n);
    long long total = 0;
    for (int i = 0; i < n; i++) {
        const rb200_grad_tensor& t = tensors[i];
        if (t.count == 0) continue;
        if (t.count < 0 || t.count > (1ll << 40) || !t.grad || !t.out) {
            set_error("%s: tensor %d is null or has %lld elements", what, i, (long long)t.count);
            return RB200_E_INVALID;
        }
        if ((t.grad_dtype != RB200_FP32 && t.grad_dtype != RB200_FP16 && t.grad_dtype != RB200_BF16) ||
            (t.out_dtype != t.grad_dtype && t.out_dtype != RB200_FP32)) {
            set_error("%s: tensor %d: types %d -> %d", what, i, t.grad_dtype, t.out_dtype);
            return RB200_E_INVALID;
        }
        if ((uintptr_t)t.grad % clip_bytes(t.grad_dtype) || (uintptr_t)t.out % clip_bytes(t.out_dtype)) {
            set_error("%s: tensor %d is not aligned to its elements", what, i);
            return RB200_E_INVALID;
        }
        v.push_back({t.grad, t.out, t.count, 0, (short)t.grad_dtype, (short)t.out_dtype});
        total += t.count;
    }
    if (total == 0) return check_cuda(cudaMemsetAsync(norm, 0, sizeof(float), stream), what);
    for (const ClipEntry& e : v)
        if (e.out == e.grad && e.out_dtype != e.grad_dtype) {
            set_error("%s: an output in place of gradients of another type", what);
            return RB200_E_INVALID;
        }
    if (!outputs_disjoint(v)) {
        set_error("%s: an output overlaps another output or another tensor's gradients", what);
        return RB200_E_INVALID;
    }
    const uint64_t need = rb200k_grad_clip_workspace_bytes(n);
    if (!ws || ws_bytes < need || ((uintptr_t)ws & 15)) {
        set_error("%s: the workspace has %llu bytes, the call needs %llu, 16-byte aligned", what, (unsigned long long)(ws ? ws_bytes : 0),
                  (unsigned long long)need);
        return RB200_E_INVALID;
    }
    DeviceInfo dev;
    int rc = device_info(&dev);
    if (rc) return rc;
    const int most = std::min(dev.sms * kClipBlocksPerSm, kClipMaxBlocks);
    // chunks: about four for every block, so that the ends of tensors even out; between 2048 elements and 16384
    long long chunk = round_up((total + 4 * most - 1) / (4 * most), 2048);
    chunk = std::min(chunk, 16384ll);
    while (total / chunk > (1ll << 30)) chunk *= 2;
    const bool few = total <= kClipFew && v.size() <= kClipFewTensors;
    if (few) chunk = round_up((total + kClipCluster - 1) / kClipCluster, 2048);
    double* partial = (double*)ws;
    int partials = 0;
    for (int pass = 0; pass < (few ? 1 : 2); pass++) {
        const size_t tables = (v.size() + kClipLarge - 1) / kClipLarge;
        for (size_t k = 0; k < tables; k++) {
            const size_t b = pass ? tables - 1 - k : k;   // the second sweep starts with the last table
            ClipEntry* first = v.data() + b * kClipLarge;
            const int count = (int)std::min<size_t>(kClipLarge, v.size() - b * kClipLarge);
            int chunks = 0;
            for (int i = 0; i < count; i++) {
                first[i].chunk0 = chunks;
                chunks += (int)((first[i].count + chunk - 1) / chunk);
            }
            const int blocks = few ? kClipCluster : std::min(chunks, most);
            auto* launch = count <= 16            ? clip_table_launch<16>
                           : count <= 64          ? clip_table_launch<64>
                           : count <= kClipMedium ? clip_table_launch<kClipMedium>
                           : count <= 448         ? clip_table_launch<448>
                                                  : clip_table_launch<kClipLarge>;
            rc = launch(first, count, chunks, (int)chunk, few ? CLIP_FEW : pass ? CLIP_SCALE : CLIP_NORM, pass ? partial : partial + partials, partials, max_norm, inv_scale,
                        k == 0 ? norm : nullptr, blocks, stream);
            if (rc) return rc;
            if (pass == 0) partials += blocks;
        }
    }
    return RB200_OK;
}

}  // namespace rb200

using namespace rb200;

extern "C" uint64_t rb200k_grad_clip_workspace_bytes(int num_tensors) {
    if (num_tensors <= 0) return 0;
    return (uint64_t)((num_tensors + kClipLarge - 1) / kClipLarge) * kClipMaxBlocks * sizeof(double);
}
extern "C" int rb200k_grad_clip(const rb200_grad_tensor* tensors, int num_tensors, float max_norm, float inv_scale, float* norm, void* workspace,
                                uint64_t workspace_bytes, void* stream) {
    try {
        return clip_run(tensors, num_tensors, max_norm, inv_scale, norm, workspace, workspace_bytes, (cudaStream_t)stream);
    } catch (const std::bad_alloc&) {
        set_error("rb200k_grad_clip: out of host memory");
        return RB200_E_LIMIT;
    }
}
