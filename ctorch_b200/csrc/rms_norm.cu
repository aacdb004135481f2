// rms_norm.cu — the root-mean-square norm of rows with the residual's addition, to the rows' type or to 8 bits with
// scales, and its backward pass (include/ctb/ctb.h).
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "rows.cuh"

namespace ctb {

namespace {

enum NormRow : int { kNmX = 0, kNmResidual, kNmSummed, kNmOut, kNmRstd, kNmScales, kNmViews };
enum NormGradRow : int { kNgUp = 0, kNgSummed, kNgPassed, kNgGradX, kNgRstd, kNgViews };

constexpr int kScaleBlock = 128;  // columns that share a scale
constexpr float kE4M3Max = 448.0f;

struct NormArgs {
    RowViews<kNmViews> v;
    const void* weight;
    int32_t weight_dtype;
    int64_t weight_stride;
    float eps;
    int quant;  // 0: none, 1: a scale a row, 2: a scale for every 128 columns
};

struct NormGradArgs {
    RowViews<kNgViews> v;
    const void* weight;
    int32_t weight_dtype;
    int64_t weight_stride;
    void* grad_weight;
    int64_t grad_weight_stride;
    float* partial;  // [CTAs][cols] sums of grad_weight
    int ctas;
};

__device__ __forceinline__ float weight_at(const void* p, int dt, int64_t off) {
    return dt == CTB_FLOAT32 ? static_cast<const float*>(p)[off] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[off]);
}

// The larger of two, or NaN if one is.
__device__ __forceinline__ float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}

// scale = amax / 448, the value that 1 stands for; 1 where all is 0. Its reciprocal stays finite.
__device__ __forceinline__ float scale_of(float amax) { return amax == 0.0f ? 1.0f : max_nan(amax / kE4M3Max, 1.17549435e-38f); }

__device__ __forceinline__ uint8_t to_e4m3(float x) { return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }

template <int THREADS> __device__ __forceinline__ float block_sum(float x) {
    __shared__ float sm[THREADS / 32];
    for (int d = 16; d >= 1; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0.0f;
    for (int w = 0; w < THREADS / 32; ++w) x += sm[w];
    return x;
}

template <int THREADS> __device__ __forceinline__ float block_max(float x) {
    __shared__ float sm[THREADS / 32];
    for (int d = 16; d >= 1; d >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, d));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = x;
    __syncthreads();
    x = sm[0];
    for (int w = 1; w < THREADS / 32; ++w) x = max_nan(x, sm[w]);
    return x;
}

constexpr int kAnyThreads = 256;

// Any layout: a CTA a row, element by element; the sum is read back by the thread that wrote it.
template <class T> __global__ void __launch_bounds__(kAnyThreads) norm_rows_any(NormArgs a) {
    dependent_wait();
    const RowViews<kNmViews>& v = a.v;
    const int64_t cols = v.cols;
    for (int64_t r = blockIdx.x; r < v.rows; r += gridDim.x) {
        const T* const x = static_cast<const T*>(v.ptr[kNmX]) + row_offset(v, kNmX, r);
        const T* const res = v.ptr[kNmResidual] ? static_cast<const T*>(v.ptr[kNmResidual]) + row_offset(v, kNmResidual, r) : nullptr;
        T* const kept = v.ptr[kNmSummed] ? static_cast<T*>(v.ptr[kNmSummed]) + row_offset(v, kNmSummed, r) : nullptr;
        auto element = [&](int64_t j) {
            float s = to_float(x[j * v.inner[kNmX]]);
            return res ? to_float(from_float<T>(s + to_float(res[j * v.inner[kNmResidual]]))) : s;
        };
        // `kept` may be x's or the residual's own view, so once it is written the sum is read from there
        float ss = 0.0f;
        for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) {
            const float s = element(j);
            if (kept) kept[j * v.inner[kNmSummed]] = from_float<T>(s);
            ss += s * s;
        }
        ss = block_sum<kAnyThreads>(ss);
        const float rstd = 1.0f / sqrtf(ss / static_cast<float>(cols) + a.eps);
        if (threadIdx.x == 0 && v.ptr[kNmRstd]) static_cast<float*>(v.ptr[kNmRstd])[row_offset(v, kNmRstd, r)] = rstd;
        __syncthreads();
        auto normed = [&](int64_t j) {
            const float s = kept ? to_float(kept[j * v.inner[kNmSummed]]) : element(j);
            return s * rstd * weight_at(a.weight, a.weight_dtype, j * a.weight_stride);
        };
        if (a.quant == 0) {
            T* const out = static_cast<T*>(v.ptr[kNmOut]) + row_offset(v, kNmOut, r);
            for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) out[j * v.inner[kNmOut]] = from_float<T>(normed(j));
            continue;
        }
        uint8_t* const out = static_cast<uint8_t*>(v.ptr[kNmOut]) + row_offset(v, kNmOut, r);
        float* const scales = static_cast<float*>(v.ptr[kNmScales]) + row_offset(v, kNmScales, r);
        if (a.quant == 1) {
            float top = 0.0f;
            for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) top = max_nan(top, fabsf(normed(j)));
            const float scale = scale_of(block_max<kAnyThreads>(top)), inv = 1.0f / scale;
            if (threadIdx.x == 0) *scales = scale;
            for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) out[j * v.inner[kNmOut]] = to_e4m3(normed(j) * inv);
        } else {
            for (int64_t at = threadIdx.x >> 5; at * kScaleBlock < cols; at += kAnyThreads / 32) {
                const int64_t j0 = at * kScaleBlock + (threadIdx.x & 31);
                float top = 0.0f;
                for (int64_t j = j0; j < min(cols, (at + 1) * kScaleBlock); j += 32) top = max_nan(top, fabsf(normed(j)));
                for (int d = 16; d >= 1; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float scale = scale_of(top), inv = 1.0f / scale;
                if ((threadIdx.x & 31) == 0) scales[at * v.inner[kNmScales]] = scale;
                for (int64_t j = j0; j < min(cols, (at + 1) * kScaleBlock); j += 32) out[j * v.inner[kNmOut]] = to_e4m3(normed(j) * inv);
            }
        }
    }
    allow_dependents();
}

// Any layout: a CTA takes every gridDim-th row; a thread's columns of grad_weight are summed where only it writes.
template <class T> __global__ void __launch_bounds__(kAnyThreads) norm_grad_any(NormGradArgs a) {
    dependent_wait();
    const RowViews<kNgViews>& v = a.v;
    const int64_t cols = v.cols;
    float* const part = a.grad_weight ? a.partial + blockIdx.x * cols : nullptr;
    if (part)
        for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) part[j] = 0.0f;
    for (int64_t r = blockIdx.x; r < v.rows; r += gridDim.x) {
        const T* const up = static_cast<const T*>(v.ptr[kNgUp]) + row_offset(v, kNgUp, r);
        const T* const x = static_cast<const T*>(v.ptr[kNgSummed]) + row_offset(v, kNgSummed, r);
        const T* const passed = v.ptr[kNgPassed] ? static_cast<const T*>(v.ptr[kNgPassed]) + row_offset(v, kNgPassed, r) : nullptr;
        T* const grad = static_cast<T*>(v.ptr[kNgGradX]) + row_offset(v, kNgGradX, r);
        const float rstd = static_cast<const float*>(v.ptr[kNgRstd])[row_offset(v, kNgRstd, r)];
        float dot = 0.0f;
        for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) {
            const float g = to_float(up[j * v.inner[kNgUp]]), hat = to_float(x[j * v.inner[kNgSummed]]) * rstd;
            if (part) part[j] += g * hat;
            dot += g * weight_at(a.weight, a.weight_dtype, j * a.weight_stride) * hat;
        }
        dot = block_sum<kAnyThreads>(dot) / static_cast<float>(cols);
        for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) {
            const float hat = to_float(x[j * v.inner[kNgSummed]]) * rstd;
            float y = rstd * (to_float(up[j * v.inner[kNgUp]]) * weight_at(a.weight, a.weight_dtype, j * a.weight_stride) - hat * dot);
            if (passed) y += to_float(passed[j * v.inner[kNgPassed]]);
            grad[j * v.inner[kNgGradX]] = from_float<T>(y);
        }
    }
    allow_dependents();
}

// grad_weight: the CTAs' sums added in their order, in float64.
__global__ void __launch_bounds__(256) norm_grad_weight(NormGradArgs a) {
    dependent_wait();
    allow_dependents();
    for (int64_t j = blockIdx.x * 256 + threadIdx.x; j < a.v.cols; j += gridDim.x * 256) {
        double s = 0.0;
        for (int c = 0; c < a.ctas; ++c) s += a.partial[c * a.v.cols + j];
        const float y = static_cast<float>(s);
        if (a.weight_dtype == CTB_FLOAT32) static_cast<float*>(a.grad_weight)[j * a.grad_weight_stride] = y;
        else static_cast<__nv_bfloat16*>(a.grad_weight)[j * a.grad_weight_stride] = __float2bfloat16_rn(y);
    }
}

// ------------------------------------------------------------------------------------------------
// host side

int weight_of(const ctb_view* w, int64_t cols, const char* what) {
    CTB_CHECK(check_row_view(w, what));
    CTB_CHECK(check_row_dtype(w, kDtypeMatrix, what));
    if (w->ndim != 1 || w->shape[0] != cols) return fail(CTB_ERR_SHAPE, std::string(what) + " must be [" + std::to_string(cols) + "]");
    return CTB_OK;
}

int grad_ctas(int64_t rows) { return static_cast<int>(std::min<int64_t>(rows, sm_count() * 4)); }

}  // namespace
}  // namespace ctb

using namespace ctb;

extern "C" {

int ctb_rms_norm(const ctb_view* x, const ctb_view* weight, const ctb_view* residual, double eps, int quant,
                 const ctb_view* out, const ctb_view* summed, const ctb_view* rstd, const ctb_view* scales, ctb_stream stream) {
    return c_entry([&]() -> int {
        NormArgs a{};
        RowBuilder<kNmViews> b;
        CTB_CHECK(b.begin(kNmX, x, kDtypeMatrix, "x"));
        const int64_t cols = b.v.cols;
        CTB_CHECK(weight_of(weight, cols, "weight"));
        if (residual) CTB_CHECK(b.matrix(kNmResidual, residual, 1u << x->dtype, cols, false, "residual"));
        if (!residual != !summed) return fail(CTB_ERR_ARGUMENT, "summed goes with residual");
        if (summed) CTB_CHECK(b.matrix(kNmSummed, summed, 1u << x->dtype, cols, true, "summed"));
        if (quant < 0 || quant > 2) return fail(CTB_ERR_ARGUMENT, "quant must be 0, 1 or 2");
        CTB_CHECK(b.matrix(kNmOut, out, quant ? 1u << CTB_FLOAT8_E4M3 : 1u << x->dtype, cols, true, "out"));
        CTB_CHECK(b.result(kNmRstd, rstd, 1u << CTB_FLOAT32, "rstd"));
        if (!quant != !scales) return fail(CTB_ERR_ARGUMENT, "scales go with an output in 8 bits");
        if (quant == 1) CTB_CHECK(b.result(kNmScales, scales, 1u << CTB_FLOAT32, "scales"));
        if (quant == 2) CTB_CHECK(b.matrix(kNmScales, scales, 1u << CTB_FLOAT32, (cols + kScaleBlock - 1) / kScaleBlock, true, "scales"));
        if (!(eps >= 0.0 && eps <= 1e30)) return fail(CTB_ERR_ARGUMENT, "eps must be finite and not negative");
        b.finish();
        a.v = b.v;
        a.weight = weight->data;
        a.weight_dtype = weight->dtype;
        a.weight_stride = weight->strides[0];
        a.eps = static_cast<float>(eps);
        a.quant = quant;
        if (a.v.rows == 0) return CTB_OK;
        auto kernel = x->dtype == CTB_FLOAT32 ? norm_rows_any<float> : norm_rows_any<__nv_bfloat16>;
        launch_dependent(kernel, grid_for(a.v.rows, 8), kAnyThreads, 0, static_cast<cudaStream_t>(stream), a);
        count_launch();
        return check_launch("rms norm");
    });
}

size_t ctb_rms_norm_backward_scratch_bytes(const ctb_view* summed) {
    if (!summed || summed->ndim < 1 || summed->ndim > kMaxDims) return 0;
    int64_t rows = 1;
    for (int d = 0; d < summed->ndim - 1; ++d) rows *= summed->shape[d];
    return static_cast<size_t>(grad_ctas(rows)) * static_cast<size_t>(summed->shape[summed->ndim - 1]) * sizeof(float);
}

int ctb_rms_norm_backward(const ctb_view* grad_out, const ctb_view* summed, const ctb_view* weight, const ctb_view* rstd,
                          const ctb_view* grad_summed, const ctb_view* grad_x, const ctb_view* grad_weight, void* scratch,
                          size_t scratch_bytes, ctb_stream stream) {
    return c_entry([&]() -> int {
        NormGradArgs a{};
        RowBuilder<kNgViews> b;
        CTB_CHECK(b.begin(kNgUp, grad_out, kDtypeMatrix, "grad_out"));
        const int64_t cols = b.v.cols;
        const unsigned type = 1u << grad_out->dtype;
        CTB_CHECK(b.matrix(kNgSummed, summed, type, cols, false, "summed"));
        CTB_CHECK(weight_of(weight, cols, "weight"));
        CTB_CHECK(check_row_view(rstd, "rstd"));
        CTB_CHECK(b.operand(kNgRstd, rstd, 1u << CTB_FLOAT32, "rstd"));
        if (grad_summed) CTB_CHECK(b.matrix(kNgPassed, grad_summed, type, cols, false, "grad_summed"));
        CTB_CHECK(b.matrix(kNgGradX, grad_x, type, cols, true, "grad_x"));
        if (grad_weight) {
            CTB_CHECK(weight_of(grad_weight, cols, "grad_weight"));
            CTB_CHECK(check_written(grad_weight, "grad_weight"));
            if (grad_weight->dtype != weight->dtype) return fail(CTB_ERR_DTYPE, "grad_weight's dtype must equal weight's");
            a.grad_weight = grad_weight->data;
            a.grad_weight_stride = grad_weight->strides[0];
        }
        a.ctas = grad_ctas(b.v.rows);
        if (grad_weight)
            CTB_CHECK(check_row_scratch(scratch, scratch_bytes, static_cast<size_t>(a.ctas) * static_cast<size_t>(cols) * sizeof(float), 16));
        b.finish();
        a.v = b.v;
        a.weight = weight->data;
        a.weight_dtype = weight->dtype;
        a.weight_stride = weight->strides[0];
        a.partial = static_cast<float*>(scratch);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (a.ctas) {
            auto kernel = grad_out->dtype == CTB_FLOAT32 ? norm_grad_any<float> : norm_grad_any<__nv_bfloat16>;
            launch_dependent(kernel, static_cast<unsigned>(a.ctas), kAnyThreads, 0, st, a);
            count_launch();
            CTB_CHECK(check_launch("rms norm backward"));
        }
        if (grad_weight) {
            launch_dependent(norm_grad_weight, grid_for((cols + 255) / 256, 4), 256, 0, st, a);
            count_launch();
            CTB_CHECK(check_launch("rms norm backward"));
        }
        return CTB_OK;
    });
}

}  // extern "C"
