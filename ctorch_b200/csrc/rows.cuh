// rows.cuh — operators over the rows of [..., cols] matrices (the norm, the projection with its cross entropy, the
// balance loss): where each operand of a row lies, for any leading dims and strides, and the host's checks of them.
//
// A "row" is one position of the leading dims of the first matrix. Further matrices have its leading shape;
// numbers a row broadcast (right-aligned) to it, results a row have exactly it. The plan drops leading dims of
// extent 1 and merges neighbours that chain in every operand, so that contiguous operands are addressed by row * stride.
#pragma once

#include <cuda_bf16.h>

#include <exception>
#include <string>

#include "common.cuh"
#include "plan.cuh"

namespace ctb {

template <int N> struct RowViews {
    void* ptr[N];
    int32_t dtype[N];
    int64_t stride[N][kMaxDims];  // over the merged leading dims
    int64_t inner[N];             // along the row
    int rank;                     // of the merged leading dims, >= 1
    FastDiv div[kMaxDims];        // divisors = their extents
    int64_t ext[kMaxDims];
    int64_t rows, cols;
};

template <int N> __device__ __forceinline__ int64_t row_offset(const RowViews<N>& v, int slot, int64_t row) {
    if (v.rank == 1) return row * v.stride[slot][0];
    int64_t off = 0;
    uint64_t r = static_cast<uint64_t>(row);
    for (int d = v.rank - 1; d > 0; --d) {
        uint64_t q, c;
        v.div[d].divmod(r, q, c);
        off += static_cast<int64_t>(c) * v.stride[slot][d];
        r = q;
    }
    return off + static_cast<int64_t>(r) * v.stride[slot][0];
}

// A number of the row as float64: float32, float64, bfloat16 or bool.
__device__ __forceinline__ double real_at(const void* p, int dt, int64_t off) {
    switch (dt) {
    case CTB_FLOAT32: return static_cast<const float*>(p)[off];
    case CTB_FLOAT64: return static_cast<const double*>(p)[off];
    case CTB_BFLOAT16: return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[off]);
    default: return static_cast<const uint8_t*>(p)[off] ? 1.0 : 0.0;
    }
}

__device__ __forceinline__ int64_t index_at(const void* p, int dt, int64_t off) {
    return dt == CTB_INT32 ? static_cast<int64_t>(static_cast<const int32_t*>(p)[off])
                           : static_cast<const int64_t*>(p)[off];
}

template <class T> __device__ __forceinline__ float to_float(T x) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(x);
    else return static_cast<float>(x);
}
template <class T> __device__ __forceinline__ T from_float(float x) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(x);
    else return static_cast<T>(x);
}

// Records a bad index for the host (the 16-byte status of include/ctb/ctb.h). The first one wins.
__device__ __forceinline__ void record_bad_index(int32_t* status, int64_t index) {
    if (status && atomicCAS(status, 0, 1) == 0) *reinterpret_cast<int64_t*>(status + 2) = index;
}

// ------------------------------------------------------------------------------------------------
// host side

inline int check_row_view(const ctb_view* v, const char* what) {
    const std::string name(what);
    if (!v) return fail(CTB_ERR_ARGUMENT, name + ": null view");
    if (v->ndim < 0 || v->ndim > kMaxDims)
        return fail(CTB_ERR_SHAPE, "CUDA backend does not support tensor rank > 16 (got " + std::to_string(v->ndim) + ")");
    if (v->dtype < 0 || v->dtype > CTB_FLOAT8_E4M3) return fail(CTB_ERR_ARGUMENT, name + ": malformed view");
    int64_t n = 1;
    for (int d = 0; d < v->ndim; ++d) {
        if (v->shape[d] < 0) return fail(CTB_ERR_ARGUMENT, name + ": malformed view");
        n *= v->shape[d];
    }
    if (!v->data && n != 0) return fail(CTB_ERR_ARGUMENT, name + ": null data pointer");
    return CTB_OK;
}

// An element that several positions of an output share would be written by several threads.
inline int check_written(const ctb_view* v, const char* what) {
    for (int d = 0; d < v->ndim; ++d)
        if (v->shape[d] > 1 && v->strides[d] == 0)
            return fail(CTB_ERR_ARGUMENT, std::string(what) + " must not be a broadcast view");
    return CTB_OK;
}

constexpr unsigned kDtypeReal = 1u << CTB_FLOAT32 | 1u << CTB_FLOAT64;
constexpr unsigned kDtypeIndex = 1u << CTB_INT32 | 1u << CTB_INT64;
constexpr unsigned kDtypeWeight = kDtypeReal | 1u << CTB_BOOL;
constexpr unsigned kDtypeMatrix = 1u << CTB_FLOAT32 | 1u << CTB_BFLOAT16;

inline int check_row_dtype(const ctb_view* v, unsigned allowed, const char* what) {
    if (allowed >> v->dtype & 1u) return CTB_OK;
    std::string names;
    for (int t = 0; t <= CTB_FLOAT8_E4M3; ++t)
        if (allowed >> t & 1u) names += (names.empty() ? "" : " or ") + std::string(dtype_name(t));
    return fail(CTB_ERR_DTYPE, std::string(what) + " must be " + names + " (got " + dtype_name(v->dtype) + ")");
}

template <int N> struct RowBuilder {
    RowViews<N> v{};
    const ctb_view* first = nullptr;
    std::string name;
    int lead = 0;

    // The matrix that gives the rows.
    int begin(int slot, const ctb_view* x, unsigned allowed, const char* what) {
        if (int rc = check_row_view(x, what)) return rc;
        if (int rc = check_row_dtype(x, allowed, what)) return rc;
        if (x->ndim < 1) return fail(CTB_ERR_SHAPE, std::string(what) + " must have at least one dim");
        first = x;
        name = what;
        lead = x->ndim - 1;
        v.cols = x->shape[lead];
        if (v.cols < 1) return fail(CTB_ERR_SHAPE, std::string(what) + ": rows are empty");
        if (v.cols >= (int64_t(1) << 31)) return fail(CTB_ERR_SHAPE, std::string(what) + ": rows of 2^31 or more elements are not supported");
        v.rows = 1;
        for (int d = 0; d < lead; ++d) v.rows *= x->shape[d];
        if (v.rows >= (int64_t(1) << 31)) return fail(CTB_ERR_SHAPE, std::string(what) + ": 2^31 or more rows are not supported");
        v.ptr[slot] = x->data;
        v.dtype[slot] = x->dtype;
        v.inner[slot] = x->strides[lead];
        for (int d = 0; d < lead; ++d) v.stride[slot][d] = x->shape[d] == 1 ? 0 : x->strides[d];
        return CTB_OK;
    }

    // A number a row, broadcast.
    int operand(int slot, const ctb_view* x, unsigned allowed, const char* what) {
        if (int rc = check_row_view(x, what)) return rc;
        if (int rc = check_row_dtype(x, allowed, what)) return rc;
        return leading(slot, x, x->ndim, what, true);
    }

    // [..., cols]: the leading shape exactly and `cols` columns; `written` for outputs.
    int matrix(int slot, const ctb_view* x, unsigned allowed, int64_t cols, bool written, const char* what) {
        if (int rc = check_row_view(x, what)) return rc;
        if (int rc = check_row_dtype(x, allowed, what)) return rc;
        if (x->ndim != lead + 1 || x->shape[x->ndim - 1] != cols)
            return fail(CTB_ERR_SHAPE, std::string(what) + " does not have " + name + "'s leading dims and " +
                                           std::to_string(cols) + " columns");
        v.inner[slot] = x->strides[lead];
        if (int rc = leading(slot, x, lead, what, false)) return rc;
        return written ? check_written(x, what) : CTB_OK;
    }

    // A result a row: exactly the leading shape.
    int result(int slot, const ctb_view* x, unsigned allowed, const char* what) {
        if (!x) return CTB_OK;
        if (int rc = check_row_view(x, what)) return rc;
        if (int rc = check_row_dtype(x, allowed, what)) return rc;
        if (int rc = leading(slot, x, x->ndim, what, false)) return rc;
        return check_written(x, what);
    }

    int leading(int slot, const ctb_view* x, int ndim, const char* what, bool broadcast) {
        ctb_view head = *x;
        head.ndim = ndim;
        bool same = ndim == lead;
        for (int d = 0; same && d < lead; ++d) same = x->shape[d] == first->shape[d];
        if ((!broadcast && !same) || !broadcast_strides(head, lead, first->shape, v.stride[slot]))
            return fail(CTB_ERR_SHAPE, std::string(what) + " does not match " + name + "'s leading dims");
        v.ptr[slot] = x->data;
        v.dtype[slot] = x->dtype;
        return CTB_OK;
    }

    void finish() {
        int r = 0;
        for (int d = 0; d < lead; ++d) {
            if (first->shape[d] == 1) continue;
            bool chain = r > 0;
            for (int s = 0; chain && s < N; ++s)
                if (v.ptr[s] && v.stride[s][r - 1] != v.stride[s][d] * first->shape[d]) chain = false;
            const int at = chain ? r - 1 : r;
            for (int s = 0; s < N; ++s) v.stride[s][at] = v.stride[s][d];
            v.ext[at] = chain ? v.ext[at] * first->shape[d] : first->shape[d];
            r = at + 1;
        }
        if (r == 0) {
            v.ext[0] = v.rows;
            for (int s = 0; s < N; ++s) v.stride[s][0] = 0;
            r = 1;
        }
        v.rank = r;
        for (int d = 0; d < r; ++d) v.div[d] = FastDiv(static_cast<uint64_t>(v.ext[d] > 0 ? v.ext[d] : 1));
    }
};

inline int check_row_status(const int32_t* status) {
    return reinterpret_cast<uintptr_t>(status) % 8 ? fail(CTB_ERR_ARGUMENT, "the status must start on an 8-byte boundary")
                                                   : CTB_OK;
}

inline int check_row_scratch(const void* scratch, size_t have, size_t need, size_t align) {
    if (need && (!scratch || have < need))
        return fail(CTB_ERR_SCRATCH, "scratch buffer too small: need " + std::to_string(need) + " bytes");
    if (reinterpret_cast<uintptr_t>(scratch) % align)
        return fail(CTB_ERR_ARGUMENT, "scratch must start on a " + std::to_string(align) + "-byte boundary");
    return CTB_OK;
}

// No exception crosses the C ABI.
template <class F> int c_entry(F&& f) {
    try {
        fail(CTB_OK, "");
        return f();
    } catch (const std::exception& e) {
        return fail(CTB_ERR_CUDA, std::string("internal error: ") + e.what());
    } catch (...) {
        return fail(CTB_ERR_CUDA, "internal error");
    }
}

#define CTB_CHECK(call)                   \
    do {                                  \
        if (int rc_ = (call)) return rc_; \
    } while (0)

}  // namespace ctb
