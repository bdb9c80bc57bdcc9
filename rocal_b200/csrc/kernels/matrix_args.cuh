// Argument checks and operand preparation shared by the head operators (host side).
#pragma once

#include "gemm.cuh"

namespace rb200 {

// ---- argument checks ------------------------------------------------------------------------------------
constexpr long long kMaxExtent = 1ll << 30;

static inline int check_dtype(const char* what, int dtype) {
    if (dtype != RB200_FP16 && dtype != RB200_BF16) {
        set_error("%s: dtype %d is neither RB200_FP16 nor RB200_BF16", what, dtype);
        return RB200_E_INVALID;
    }
    return RB200_OK;
}

static inline int check_extents(const char* what, long long rows, const char* name_in, long long in, const char* name_out, long long out) {
    if (rows < 0 || in < 1 || out < 1) {
        set_error("%s: rows %lld, %s %lld, %s %lld", what, rows, name_in, in, name_out, out);
        return RB200_E_INVALID;
    }
    if (rows > kMaxExtent || in > kMaxExtent || out > kMaxExtent) {
        set_error("%s: %lld x %lld x %lld exceeds 2^30 in one extent", what, rows, in, out);
        return RB200_E_LIMIT;
    }
    return RB200_OK;
}

// A matrix argument: present, its rows not overlapping, its elements on their own boundaries.
static inline int check_matrix(const char* what, const char* name, const void* data, long long ld, long long rows, long long cols) {
    if (!data) {
        set_error("%s: %s is null", what, name);
        return RB200_E_INVALID;
    }
    if ((uintptr_t)data & 1) {
        set_error("%s: %s is not aligned to its elements", what, name);
        return RB200_E_INVALID;
    }
    if (rows > 1 && (ld < cols || ld > (1ll << 38))) {
        set_error("%s: leading dimension %lld of %s, %lld columns", what, ld, name, cols);
        return RB200_E_INVALID;
    }
    return RB200_OK;
}

static inline int check_workspace(const char* what, const void* ws, uint64_t have, uint64_t need) {
    if (need == 0) return RB200_OK;
    if (!ws || have < need) {
        set_error("%s: the workspace has %llu bytes, the call needs %llu", what, (unsigned long long)(ws ? have : 0), (unsigned long long)need);
        return RB200_E_INVALID;
    }
    if ((uintptr_t)ws & 255) {
        set_error("%s: the workspace must be 256-byte aligned", what);
        return RB200_E_INVALID;
    }
    return RB200_OK;
}

static inline Operand operand(const void* data, long long ld, long long rows, long long cols, bool transposed) {
    Operand o = {data, ld, (int)rows, (int)cols, transposed};
    return o;
}

static inline Packed plan_pack(const Operand& o, Carver* c) {
    Packed p = {o, o, !map_ready(o)};
    if (p.copy) {
        p.use.ld = round_up(o.cols, 8);
        p.use.data = c->take((size_t)p.use.ld * o.rows * 2);
    }
    return p;
}
// Zeroes a matrix of 16-bit elements.
static inline int clear_matrix(void* data, long long ld, long long rows, long long cols, cudaStream_t stream, const char* what) {
    return check_cuda(cudaMemset2DAsync(data, (size_t)(rows > 1 ? ld : cols) * 2, 0, (size_t)cols * 2, (size_t)rows, stream), what);
}

}  // namespace rb200
