// Host side of the matrix products (gemm.cuh): tensor maps, how a product is cut, the plain-epilogue instances, and the
// small kernels around them (joining split products, packing operands).
#include "gemm.cuh"

namespace rb200 {

int device_info(DeviceInfo* out) {
    int dev = 0, rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
    if (rc) return rc;
    if (dev < 0 || dev >= 64) {
        set_error("device %d: only devices 0..63 are supported", dev);
        return RB200_E_LIMIT;
    }
    // A thread that has not used CUDA yet (autograd's, for one) has a current device but no context, which the driver's
    // tensor-map call needs; setting the device makes its primary context current.
    static thread_local int bound = -1;
    if (bound != dev) {
        rc = check_cuda(cudaSetDevice(dev), "cudaSetDevice");
        if (rc) return rc;
        bound = dev;
    }
    // properties of the device; every writer writes the same values
    static int sms[64];
    static int* words[64];
    int v = __atomic_load_n(&sms[dev], __ATOMIC_ACQUIRE);
    if (!v) {
        rc = check_cuda(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
        if (rc) return rc;
        int* word = default_status_word();
        if (!word) {
            set_error("the library-wide status word could not be found");
            return RB200_E_CUDA;
        }
        __atomic_store_n(&words[dev], word, __ATOMIC_RELAXED);
        __atomic_store_n(&sms[dev], v, __ATOMIC_RELEASE);
    }
    out->sms = v;
    out->index = dev;
    out->status = __atomic_load_n(&words[dev], __ATOMIC_RELAXED);
    return RB200_OK;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

int make_map(CUtensorMap* map, const Operand& o, bool bf16, int box_rows, const char* what) {
    EncodeTiled fn = encode_tiled();
    if (!fn) {
        set_error("%s: the driver has no cuTensorMapEncodeTiled", what);
        return RB200_E_CUDA;
    }
    const cuuint64_t dims[2] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows};
    // the pitch of a single row is never used, but has to be a legal one
    const cuuint64_t pitch[1] = {(cuuint64_t)(o.rows > 1 ? o.ld : round_up(o.cols, 8)) * 2};
    const cuuint32_t box[2] = {(cuuint32_t)kTileK, (cuuint32_t)box_rows};
    const cuuint32_t one[2] = {1, 1};
    const CUresult rc = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(o.data), dims, pitch,
                           box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) {
        set_error("%s: cuTensorMapEncodeTiled refused a %d x %d operand of pitch %lld (%d)", what, o.rows, o.cols, o.ld, (int)rc);
        return RB200_E_CUDA;
    }
    return RB200_OK;
}

// A model of the kernel's time in clocks, good enough to order the ways of cutting a product:
//   a k-block of a tile takes the longer of the tensor cores' time (2 bn clocks: 128 rows per SM and 4096 products a
//   clock, but 290 at least: they read all 128 rows of A however few the columns are) and the copies' (about 48 bytes of
//   operands per SM and clock while most SMs copy, up to twice that while few do);
//   a tile also keeps its group of epilogue warps busy (about 16 clocks a column; two groups take turns);
//   the last tile's epilogue is not hidden, and pieces of the contracted axis have to be joined by another launch (about 8000,
//   half of it on the host). Clusters whose CTAs join their pieces through distributed shared memory were tried instead: 14 us against
//   9 us for one row of 2048 x 1000, because clusters of full-size CTAs do not fill the GPU.
// A sum of very many products is cut whatever the model says, so that what the tensor cores cut off stays small (gemm.cuh): 32768 products of
// one sign in one accumulator come off by 1e-4, a fifth of half an fp16 step. (524288 rows in one: 3e-3. Split, 524288 x 2048 x 2048 takes
// 3.6 -> 3.8 ms; 131072 x 4096 x 1024 and 65536 x 4096 x 4096 as long as before, within the 5% that runs differ by.)
constexpr int kLongestSum = 32768;
GemmPlan gemm_plan(const DeviceInfo& dev, int m, int n, int k, bool b_transposed, bool may_split, int bn_most) {
    GemmPlan best = {};
    double best_cost = 0;
    const int kblocks = (k + kTileK - 1) / kTileK, a_rows = m < kTileM ? m : kTileM;
    const long long least = may_split ? (k + (long long)kLongestSum - 1) / kLongestSum : 1;
    for (int cg = 2; cg >= 1; cg--) {
        if (cg == 2 && m <= kTileM) continue;
        const int unit = (b_transposed ? 64 : 32) * cg, slots = dev.sms / cg;
        const int tiles_m = (m + kTileM * cg - 1) / (kTileM * cg);
        for (int bn = bn_most; bn >= unit; bn -= unit) {
            const int tiles_n = (n + bn - 1) / bn;
            if (bn > unit && (n + bn - unit - 1) / (bn - unit) == tiles_n && bn - unit >= n) continue;   // wider than the matrix
            const long long tiles = (long long)tiles_m * tiles_n;
            const double products = 2.0 * bn > 290 ? 2.0 * bn : 290, epilogue = 16.0 * bn + 500;
            // one piece, or as many as the free SMs take in one or two rounds
            long long choices[3] = {least, least, least};
            if (may_split && kblocks >= 16) {
                for (int r = 1; r <= 2; r++) {
                    long long s = r * slots / tiles;
                    if (s > kblocks / 8) s = kblocks / 8;
                    choices[r] = s > least ? s : least;
                }
            }
            for (long long s : choices) {
                const int per = (int)((kblocks + s - 1) / s), splits = (kblocks + per - 1) / per;   // none of them empty
                const long long units = tiles * splits, waves = (units + slots - 1) / slots;
                const double rate = units * 2 >= slots ? 48.0 : 96.0 - 96.0 * units / slots;
                const double copies = (a_rows + bn / cg) * 128 / rate, block = copies > products ? copies : products, work = per * block + 300;
                double cost = waves * (work > epilogue / 2 ? work : epilogue / 2) + epilogue + 1000;
                if (splits > 1) cost += 8000 + 8.0 * splits * m * n / 2500;   // partial sums: about 2500 bytes a clock
                if (best_cost == 0 || cost < best_cost * 0.99) {
                    best_cost = cost;
                    best = {bn, cg, splits, tiles_m, tiles_n, kblocks, per};
                }
            }
        }
    }
    return best;
}

int gemm_args(GemmArgs* g, const DeviceInfo& dev, int epi, bool bf16, const Operand& a, const Operand& b, const Operand* b_alt, const int* b_select,
              const GemmPlan& plan, const EpiArgs& e, const GemmWait& wait, const char* what) {
    const int m = a.outer(), n = b.outer();
    if ((double)plan.tiles_m * plan.tiles_n * plan.splits > 2e9) {
        set_error("%s: a product of %d x %d has more than 2e9 tiles", what, m, n);
        return RB200_E_LIMIT;
    }
    g->a_box_rows = kTileM;
    if (!a.transposed && m < kTileM) g->a_box_rows = (int)round_up(m, 8);
    const int bn_cta = plan.bn / plan.cg, b_box = b.transposed ? kTileK : bn_cta;
    int rc = make_map(&g->a, a, bf16, a.transposed ? kTileK : g->a_box_rows, what);
    if (rc) return rc;
    rc = make_map(&g->b, b, bf16, b_box, what);
    if (rc) return rc;
    g->b_select = b_alt ? b_select : nullptr;
    if (b_alt && (rc = make_map(&g->b_alt, *b_alt, bf16, b_box, what))) return rc;
    g->e = e;
    auto vec = [](const void* p, long long ld, int rows) { return ((uintptr_t)p & 15) == 0 && (rows <= 1 || (ld & 7) == 0); };
    g->e.vec_out = vec(e.out, e.ldo, m);
    g->e.vec_pre = vec(e.preact, e.ldp, m);
    g->e.vec_res = vec(e.residual, e.ldr, e.residual_rows);
    g->m = m;
    g->n = n;
    g->k = a.inner();
    g->bn = plan.bn;
    g->tiles_m = plan.tiles_m;
    g->tiles_n = plan.tiles_n;
    g->splits = plan.splits;
    g->kblocks = plan.kblocks;
    g->kblocks_per_split = plan.kblocks_per_split;
    // several accumulators where the sums are kept in 32 bits and a tile's columns leave room (gemm.cuh)
    int sums = epi == EPI_CE_STATS ? kTileNMax / plan.bn : 1;
    if (sums > plan.kblocks_per_split / 8) sums = plan.kblocks_per_split / 8;
    if (sums < 1) sums = 1;
    g->kblocks_per_sum = (plan.kblocks_per_split + sums - 1) / sums;
    g->idesc = tc::instr_desc(bf16, a.transposed, b.transposed, kTileM * plan.cg, plan.bn);
    g->block_bytes = (uint32_t)(kTileM + bn_cta) * kTileK * 2;
    g->stage_blocks = 8 * g->block_bytes <= kRingBytes ? 2 : 1;   // two while four stages remain
    g->stages = kRingBytes / (g->stage_blocks * g->block_bytes);
    if (g->stages > 12) g->stages = 12;
    g->status = wait.status ? wait.status : dev.status;
    // The longest wait is for all products of a tile. A contracted block takes 290 clocks at least, some 2000 when every SM reads its operands
    // from memory; with 8192 for each, the ordinary limit holds for sums of any length.
    g->wait_cycles = wait.cycles ? wait.cycles : kDefaultWaitCycles + 8192ull * plan.kblocks_per_split;
    g->skip_block = wait.skip_block;
    return RB200_OK;
}

int gemm_store(int kind, bool bf16, const Operand& a, const Operand& b, const Operand* b_alt, const int* b_select, const GemmPlan& plan,
               const EpiArgs& e, const GemmWait& wait, cudaStream_t stream, const char* what) {
    if (kind == GEMM_KK) return gemm_launch<EPI_STORE, false, false>(bf16, a, b, b_alt, b_select, plan, e, wait, stream, what);
    if (kind == GEMM_KN) return gemm_launch<EPI_STORE, false, true>(bf16, a, b, b_alt, b_select, plan, e, wait, stream, what);
    return gemm_launch<EPI_STORE, true, true>(bf16, a, b, b_alt, b_select, plan, e, wait, stream, what);
}

// ---- joining split products -----------------------------------------------------------------------------
// Pieces are added in an order of their own, so the result does not depend on which CTA finished first. SUBS threads
// share the pieces of four columns: one where there are few pieces, eight where there are many (few outputs then).
template <typename T, int SUBS>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ part, int splits, long long stride, long long ldacc, int m, int n,
                                                   EpiArgs e) {
    constexpr int OUT = 256 / SUBS;
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float4 sums[SUBS][OUT];
    const long long groups = (n + 3) / 4, total = groups * m;
    const float alpha = e.scale.value();
    const int lane = threadIdx.x % OUT, sub = threadIdx.x / OUT;
    for (long long t0 = (long long)blockIdx.x * OUT; t0 < total; t0 += (long long)gridDim.x * OUT) {
        const long long t = t0 + lane;
        const int row = (int)(t / groups), col = (int)(t - row * groups) * 4;
        const long long at = row * ldacc + col;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (t < total) {
#pragma unroll 4
            for (int s = sub; s < splits; s += SUBS) {
                const float4 f = *reinterpret_cast<const float4*>(part + at + s * stride);
                v[0] += f.x;
                v[1] += f.y;
                v[2] += f.z;
                v[3] += f.w;
            }
        }
        if (SUBS > 1) {
            __syncthreads();
            sums[sub][lane] = make_float4(v[0], v[1], v[2], v[3]);
            __syncthreads();
            if (sub) continue;
#pragma unroll
            for (int s = 1; s < SUBS; s++) {
                const float4 f = sums[s][lane];
                v[0] += f.x;
                v[1] += f.y;
                v[2] += f.z;
                v[3] += f.w;
            }
        }
        if (t >= total) continue;
        if (e.acc_in) {
            const float4 f = *reinterpret_cast<const float4*>(e.acc_in + at);
            v[0] += f.x;
            v[1] += f.y;
            v[2] += f.z;
            v[3] += f.w;
        }
        if (e.acc_out) {
            *reinterpret_cast<float4*>(e.acc_out + at) = make_float4(v[0], v[1], v[2], v[3]);
            continue;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (col + i >= n) break;
            float z = v[i] * alpha;
            if (e.bias) z += Elem<T>::to_float(reinterpret_cast<const T*>(e.bias)[col + i]);
            if (e.preact) reinterpret_cast<T*>(e.preact)[row * e.ldp + col + i] = Elem<T>::from_float(z);
            v[i] = z;
        }
        act_values<4>(v, e.act);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (col + i >= n) break;
            float z = v[i];
            if (e.residual) z += Elem<T>::to_float(reinterpret_cast<const T*>(e.residual)[(long long)(row % e.residual_rows) * e.ldr + col + i]);
            reinterpret_cast<T*>(e.out)[row * e.ldo + col + i] = Elem<T>::from_float(z);
        }
    }
}

size_t gemm_partial_bytes(const GemmPlan& plan, int m, int n) {
    return plan.splits > 1 ? (size_t)plan.splits * m * round_up(n, 4) * sizeof(float) : 0;
}

template <typename T>
static cudaError_t join_launch(const float* partials, int splits, int m, int n, const EpiArgs& e, cudaStream_t stream) {
    const long long ldacc = round_up(n, 4), total = ldacc / 4 * m;
    const int out = splits >= 16 ? 32 : 256;
    const long long blocks = (total + out - 1) / out;
    const dim3 grid((unsigned)(blocks < 148 * 16 ? blocks : 148 * 16));
    return launch_overlapped(splits >= 16 ? join_kernel<T, 8> : join_kernel<T, 1>, grid, dim3(256), 0, stream, partials, splits, ldacc * m, ldacc, m,
                             n, e);
}
int gemm_join(bool bf16, const float* partials, int splits, int m, int n, const EpiArgs& e, cudaStream_t stream, const char* what) {
    int rc = check_cuda(bf16 ? join_launch<__nv_bfloat16>(partials, splits, m, n, e, stream) : join_launch<__half>(partials, splits, m, n, e, stream),
                        what);
    if (rc) return rc;
    count_launch();
    return RB200_OK;
}

int gemm_store_joined(int kind, bool bf16, const Operand& a, const Operand& b, const Operand* b_alt, const int* b_select, const GemmPlan& plan,
                      EpiArgs e, void* partials, const GemmWait& wait, cudaStream_t stream, const char* what) {
    if (plan.splits == 1) return gemm_store(kind, bf16, a, b, b_alt, b_select, plan, e, wait, stream, what);
    const int m = a.outer(), n = b.outer();
    EpiArgs part = {};
    part.acc_out = (float*)partials;
    part.ldacc = round_up(n, 4);
    part.acc_split_stride = part.ldacc * m;
    int rc = gemm_store(kind, bf16, a, b, b_alt, b_select, plan, part, wait, stream, what);
    if (rc) return rc;
    return gemm_join(bf16, (const float*)partials, plan.splits, m, n, e, stream, what);
}

// ---- packing --------------------------------------------------------------------------------------------
struct PackArgs {
    const uint16_t* src[2];
    uint16_t* dst[2];
    long long lds[2], ldd[2], total[2];   // total: pieces of 8 elements
    int cols[2];
};
// Eight elements at any address: cut out of the two aligned vectors that hold them (the second only if they reach into it;
// neither leaves the 16-byte granules of the row's elements).
__device__ __forceinline__ uint4 load8_anywhere(const uint16_t* p, int count) {
    const int offset = (int)((uintptr_t)p & 15);
    const uint4* q = reinterpret_cast<const uint4*>((uintptr_t)p - offset);
    const uint4 a = __ldg(q);
    const uint4 b = offset + 2 * min(count, 8) > 16 ? __ldg(q + 1) : make_uint4(0, 0, 0, 0);
    const uint32_t both[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t w[4];
    const int bits = (offset & 3) * 8;
    switch (offset >> 2) {
        case 0: window<4, 0>(both, w, bits); break;
        case 1: window<4, 1>(both, w, bits); break;
        case 2: window<4, 2>(both, w, bits); break;
        default: window<4, 3>(both, w, bits); break;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Rows are padded to whole pieces; what the padding holds does not matter, the tensor map ends before it.
__global__ void __launch_bounds__(256) pack_kernel(PackArgs a) {
    constexpr int U = 4;   // pieces in flight
    pdl_launch_dependents();
    pdl_wait();
    const int w = blockIdx.y, cols = a.cols[w];
    const long long groups = (cols + 7) / 8, stride = (long long)gridDim.x * 256;
    for (long long t0 = blockIdx.x * 256ll + threadIdx.x; t0 < a.total[w]; t0 += U * stride) {
        uint4 v[U];
        long long at[U];
#pragma unroll
        for (int i = 0; i < U; i++) {
            const long long t = t0 + i * stride;
            at[i] = -1;
            if (t >= a.total[w]) continue;
            const long long row = a.total[w] < (1ll << 31) ? (long long)((uint32_t)t / (uint32_t)groups) : t / groups;
            const int col = (int)(t - row * groups) * 8;
            v[i] = load8_anywhere(a.src[w] + row * a.lds[w] + col, cols - col);
            at[i] = row * a.ldd[w] + col;
        }
#pragma unroll
        for (int i = 0; i < U; i++)
            if (at[i] >= 0) *reinterpret_cast<uint4*>(a.dst[w] + at[i]) = v[i];
    }
}

int pack_operands(const Packed* a, const Packed* b, cudaStream_t stream, const char* what) {
    PackArgs p = {};
    int n = 0;
    long long most = 0;
    for (const Packed* o : {a, b}) {
        if (!o || !o->copy) continue;
        p.src[n] = (const uint16_t*)o->src.data;
        p.lds[n] = o->src.ld;
        p.cols[n] = o->src.cols;
        p.dst[n] = (uint16_t*)const_cast<void*>(o->use.data);
        p.ldd[n] = o->use.ld;
        p.total[n] = (long long)((o->src.cols + 7) / 8) * o->src.rows;
        if (p.total[n] > most) most = p.total[n];
        n++;
    }
    if (n == 0) return RB200_OK;
    const long long blocks = (most + 255) / 256;
    int rc = check_cuda(launch_overlapped(pack_kernel, dim3((unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), n), dim3(256), 0, stream, p), what);
    if (rc) return rc;
    count_launch();
    return RB200_OK;
}

}  // namespace rb200
