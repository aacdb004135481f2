// rms_norm.cu — the root-mean-square norm of rows with the residual's addition, to the rows' type or to 8 bits with
// scales, and its backward pass (include/ctb/ctb.h).
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "ctb/ctb_debug.h"
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
    bool weight_whole;  // contiguous, on 16 bytes
    float eps;
    int quant;  // 0: none, 1: a scale a row, 2: a scale for every 128 columns
};

struct NormGradArgs {
    RowViews<kNgViews> v;
    const void* weight;
    int32_t weight_dtype;
    int64_t weight_stride;
    bool weight_whole;
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

// scale = amax / 448, the value that 1 stands for; 1 where all is 0. A normal number, so that its reciprocal is finite.
__device__ __forceinline__ float scale_of(float amax) { return amax == 0.0f ? 1.0f : max_nan(amax / kE4M3Max, 1.17549435e-38f); }

// Quotients by a scale, rounded to nearest: what is left of y after the quotient by the rounded reciprocal, which a fused
// multiply-add gives exactly, corrects it (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990). By the reciprocal alone quotients next to a tie of e4m3 fell to its other side. B200, 8192 x 8192
// bfloat16, a scale for 128 columns: 83.2 us by the reciprocal, 85.9 so in pairs, 114 with a division.
struct Divisor {
    float minus, inverse;  // of the scale; by an infinite one quotients are 0, by NaN and of an infinite y NaN
    __device__ __forceinline__ explicit Divisor(float scale) : minus(scale < INFINITY ? -scale : 0.0f), inverse(1.0f / scale) {}
    __device__ __forceinline__ float operator()(float y) const {
        const float q = y * inverse;
        return fmaf(fmaf(q, minus, y), inverse, q);
    }
};

// Two quotients in packed operations.
__device__ __forceinline__ float2 quotients(float2 y, const Divisor& d) {
    const float2 minus = make_float2(d.minus, d.minus), inverse = make_float2(d.inverse, d.inverse);
    float2 q;
    asm("{\n\t.reg .b64 q, r;\n\tmul.rn.f32x2 q, %1, %3;\n\tfma.rn.f32x2 r, q, %2, %1;\n\tfma.rn.f32x2 %0, r, %3, q;\n\t}"
        : "=l"(reinterpret_cast<unsigned long long&>(q))
        : "l"(reinterpret_cast<const unsigned long long&>(y)), "l"(reinterpret_cast<const unsigned long long&>(minus)),
          "l"(reinterpret_cast<const unsigned long long&>(inverse)));
    return q;
}

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
            const float scale = scale_of(block_max<kAnyThreads>(top));
            const Divisor quotient(scale);
            if (threadIdx.x == 0) *scales = scale;
            for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) out[j * v.inner[kNmOut]] = to_e4m3(quotient(normed(j)));
        } else {
            for (int64_t at = threadIdx.x >> 5; at * kScaleBlock < cols; at += kAnyThreads / 32) {
                const int64_t j0 = at * kScaleBlock + (threadIdx.x & 31);
                float top = 0.0f;
                for (int64_t j = j0; j < min(cols, (at + 1) * kScaleBlock); j += 32) top = max_nan(top, fabsf(normed(j)));
                for (int d = 16; d >= 1; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float scale = scale_of(top);
                const Divisor quotient(scale);
                if ((threadIdx.x & 31) == 0) scales[at * v.inner[kNmScales]] = scale;
                for (int64_t j = j0; j < min(cols, (at + 1) * kScaleBlock); j += 32) out[j * v.inner[kNmOut]] = to_e4m3(quotient(normed(j)));
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

// grad_weight: the CTAs' sums added in float64, in an order that their number alone gives: 32 warps of a CTA take every
// 32nd sum of 32 columns each.
__global__ void __launch_bounds__(1024) norm_grad_weight(NormGradArgs a) {
    dependent_wait();
    allow_dependents();
    __shared__ double sm[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    double s = 0.0;
    if (j < a.v.cols) {
#pragma unroll 4
        for (int c = warp; c < a.ctas; c += 32) s += a.partial[c * a.v.cols + j];
    }
    sm[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || j >= a.v.cols) return;
    s = 0.0;
    for (int w = 0; w < 32; ++w) s += sm[w][lane];
    const float y = static_cast<float>(s);
    if (a.weight_dtype == CTB_FLOAT32) static_cast<float*>(a.grad_weight)[j * a.grad_weight_stride] = y;
    else static_cast<__nv_bfloat16*>(a.grad_weight)[j * a.grad_weight_stride] = __float2bfloat16_rn(y);
}

// ------------------------------------------------------------------------------------------------
// rows held in registers

// A group of G threads has a row, NP packs of VEC elements a thread: pack q of thread t is columns (q G + t) VEC and
// on. Groups of one warp share a CTA of 128 threads, larger ones are a CTA. A row is read once and written once; what
// keeps reads on their way while other rows are reduced is the number of groups an SM holds.
constexpr int kRingPacks = 2048;  // of a row that passes through shared memory: longer ones do not fit it

template <int G> constexpr int group_threads() { return G == 32 ? 128 : G; }
// CTAs an SM that the registers have to leave room for: 768 threads (80 registers each), 1024 in two groups of 512; 512
// (128) in backward passes whose rows start anywhere.
template <int G> constexpr int group_ctas(int threads) { return threads / group_threads<G>() > 1 ? threads / group_threads<G>() : 1; }
template <int G> constexpr int forward_ctas() { return G == 512 ? 2 : group_ctas<G>(768); }
template <int G, bool ODD> constexpr int backward_ctas() { return group_ctas<G>(ODD ? 512 : 768); }

// The sum (or maximum) over the group; `turn` alternates between calls, so one barrier a call is enough.
template <int G, bool MAX> __device__ __forceinline__ float group_join(float x, float (&sm)[2][32], int& turn) {
    for (int d = 16; d >= 1; d >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, x, d);
        x = MAX ? max_nan(x, o) : x + o;
    }
    if constexpr (G > 32) {
        if ((threadIdx.x & 31) == 0) sm[turn][threadIdx.x >> 5] = x;
        __syncthreads();
        x = sm[turn][0];
#pragma unroll
        for (int w = 1; w < G / 32; ++w) x = MAX ? max_nan(x, sm[turn][w]) : x + sm[turn][w];
        turn ^= 1;
    }
    return x;
}

template <class T, int VEC> __device__ __forceinline__ Pack<T, VEC> read_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, VEC>*>(p);
}

// VEC weights from column j on, as they lie (float32 or the rows' type) when they are contiguous.
template <class T, int VEC>
__device__ __forceinline__ void read_weights(float (&w)[VEC], const void* p, int dt, int64_t stride, bool whole, int64_t j) {
    if (whole && dt == CTB_FLOAT32) {
        constexpr int kPart = VEC < 4 ? VEC : 4;
#pragma unroll
        for (int h = 0; h < VEC; h += kPart) {
            const Pack<float, kPart> v = read_pack<float, kPart>(static_cast<const float*>(p) + j + h);
#pragma unroll
            for (int q = 0; q < kPart; ++q) w[h + q] = v.v[q];
        }
    } else if (whole) {
        const Pack<__nv_bfloat16, VEC> v = read_pack<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16*>(p) + j);
#pragma unroll
        for (int q = 0; q < VEC; ++q) w[q] = __bfloat162float(v.v[q]);
    } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) w[q] = weight_at(p, dt, (j + q) * stride);
    }
}

template <class T, int VEC, int G, int NP, bool RES, int QUANT>
__global__ void __launch_bounds__(group_threads<G>(), group_ctas<G>(1024)) norm_rows_held(NormArgs a) {
    dependent_wait();
    __shared__ float sm[2][32];
    int turn = 0;
    const RowViews<kNmViews>& v = a.v;
    constexpr int kGroups = group_threads<G>() / G;
    const int t = threadIdx.x % G, cols = static_cast<int>(v.cols);
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / G; r < v.rows; r += static_cast<int64_t>(gridDim.x) * kGroups) {
        const T* const x = static_cast<const T*>(v.ptr[kNmX]) + row_offset(v, kNmX, r);
        Pack<T, VEC> s[NP], res[RES ? NP : 1];
#pragma unroll
        for (int q = 0; q < NP; ++q)
            if ((q * G + t) * VEC < cols) s[q] = read_pack<T, VEC>(x + (q * G + t) * VEC);
        if (RES) {
            const T* const from = static_cast<const T*>(v.ptr[kNmResidual]) + row_offset(v, kNmResidual, r);
            T* const kept = static_cast<T*>(v.ptr[kNmSummed]) + row_offset(v, kNmSummed, r);
#pragma unroll
            for (int q = 0; q < NP; ++q)
                if ((q * G + t) * VEC < cols) res[q] = read_pack<T, VEC>(from + (q * G + t) * VEC);
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                if ((q * G + t) * VEC >= cols) continue;
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[q].v[e] = from_float<T>(to_float(s[q].v[e]) + to_float(res[q].v[e]));
                store_pack_split<T, VEC>(kept + (q * G + t) * VEC, s[q]);
            }
        }
        float ss = 0.0f;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            if ((q * G + t) * VEC >= cols) continue;
#pragma unroll
            for (int e = 0; e < VEC; ++e) ss = fmaf(to_float(s[q].v[e]), to_float(s[q].v[e]), ss);
        }
        ss = group_join<G, false>(ss, sm, turn);
        const float rstd = 1.0f / sqrtf(ss / static_cast<float>(cols) + a.eps);
        if (t == 0 && v.ptr[kNmRstd]) static_cast<float*>(v.ptr[kNmRstd])[row_offset(v, kNmRstd, r)] = rstd;
        if constexpr (QUANT == 0) {
            T* const out = static_cast<T*>(v.ptr[kNmOut]) + row_offset(v, kNmOut, r);
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const int j = (q * G + t) * VEC;
                if (j >= cols) continue;
                float w[VEC];
                read_weights<T, VEC>(w, a.weight, a.weight_dtype, a.weight_stride, a.weight_whole, j);
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[q].v[e] = from_float<T>(to_float(s[q].v[e]) * rstd * w[e]);
                store_pack_split<T, VEC>(out + j, s[q]);
            }
        } else {
            uint8_t* const out = static_cast<uint8_t*>(v.ptr[kNmOut]) + row_offset(v, kNmOut, r);
            float* const scales = static_cast<float*>(v.ptr[kNmScales]) + row_offset(v, kNmScales, r);
            float y[NP][VEC], top = 0.0f;
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const int j = (q * G + t) * VEC;
                if (j < cols) read_weights<T, VEC>(y[q], a.weight, a.weight_dtype, a.weight_stride, a.weight_whole, j);
                float mine = 0.0f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    y[q][e] = j < cols ? to_float(s[q].v[e]) * rstd * y[q][e] : 0.0f;
                    mine = max_nan(mine, fabsf(y[q][e]));
                }
                if (QUANT == 1) {
                    top = max_nan(top, mine);
                    continue;
                }
                // the threads that have 128 columns are neighbours in a warp
                constexpr int kShare = kScaleBlock / VEC;
#pragma unroll
                for (int d = kShare / 2; d >= 1; d >>= 1) mine = max_nan(mine, __shfl_xor_sync(0xffffffffu, mine, d));
                const float scale = scale_of(mine);
                const Divisor quotient(scale);
                if (j < cols && t % kShare == 0) scales[(j / kScaleBlock) * v.inner[kNmScales]] = scale;
#pragma unroll
                for (int e = 0; e < VEC; ++e) y[q][e] = quotient(y[q][e]);
            }
            if (QUANT == 1) {
                const float scale = scale_of(group_join<G, true>(top, sm, turn));
                const Divisor quotient(scale);
                if (t == 0) *scales = scale;
#pragma unroll
                for (int q = 0; q < NP; ++q)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) y[q][e] = quotient(y[q][e]);
            }
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const int j = (q * G + t) * VEC;
                if (j >= cols) continue;
                Pack<uint8_t, VEC> b;
                if constexpr (VEC >= 2) {
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) {
                        const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(make_float2(y[q][e], y[q][e + 1]), __NV_SATFINITE, __NV_E4M3);
                        b.v[e] = static_cast<uint8_t>(two);
                        b.v[e + 1] = static_cast<uint8_t>(two >> 8);
                    }
                } else {
                    b.v[0] = to_e4m3(y[q][0]);
                }
                *reinterpret_cast<Pack<uint8_t, VEC>*>(out + j) = b;
            }
        }
    }
    allow_dependents();
}

// The same for 16-byte packs, the rows on their way through shared memory: a thread copies its own packs of the next
// kRing - 1 rows ahead (cp.async) and is the only one to read them, so nothing but the row's sum waits for other threads,
// and the bytes on their way do not take registers. B200, 16384 x 4096 bfloat16 with a residual: 106 us with the rows in
// registers, 87 so (537 MB: 96% of the copy rate).
// Stages of the ring for `arrays` matrices: what the CTAs that an SM holds have room for, two at least and eight at most.
// What is on its way has to cover the memory's latency whatever the group (B200, 16384 x 4095 bfloat16, one
// CTA an SM: 279 us with three stages).
template <int G, int NP> constexpr int ring_stages(int arrays, int ctas) {
    const int fit = 222 * 1024 / ctas / (arrays * NP * 16 * group_threads<G>());
    return fit < 2 ? 2 : fit > 8 ? 8 : fit;
}
template <int G, int NP> constexpr int ring_bytes(int arrays, int ctas) { return ring_stages<G, NP>(arrays, ctas) * arrays * NP * 16 * group_threads<G>(); }

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int STAGES> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory"); }

template <class T, int VEC> __device__ __forceinline__ Pack<T, VEC> ring_pack(uint32_t at) {
    Pack<T, VEC> v;
    uint32_t* const u = reinterpret_cast<uint32_t*>(&v);
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]) : "r"(at));
    return v;
}

// The rows and columns of a group of threads. ODD: rows start anywhere, all matrices' alike; packs are those of memory, so
// the first and the last one of a row may be in part its neighbours': they are read whole where they lie inside the
// matrix (pack_inside), else, and when they are written, element by element. How far a row starts behind a pack repeats
// every `period` rows (a power of two), and a group takes rows of one kind: its columns, and with them its weights and
// sums of grad_weight, stay the same.
template <int VEC, bool ODD> struct Share {
    int64_t lo, hi, first, period;  // rows first + period * [lo, hi)
    int behind;                     // elements from a pack's start to the row's

    __host__ __device__ __forceinline__ Share(int64_t rows, int64_t group, int64_t groups, int base, int64_t stride) {
        first = 0;
        period = 1;
        behind = 0;
        if (ODD) {
            const int off = static_cast<int>(stride & (VEC - 1));
            while ((off * static_cast<int>(period)) & (VEC - 1)) period *= 2;
            first = group & (period - 1);
            group /= period;
            groups /= period;
            rows = (rows - first + period - 1) / period;  // at most period - 1 groups may have none
            if (rows < 0) rows = 0;
            behind = (base + off * static_cast<int>(first)) & (VEC - 1);
        }
        lo = rows * group / groups;
        hi = rows * (group + 1) / groups;
    }
    __host__ __device__ __forceinline__ int64_t row(int64_t i) const { return ODD ? first + period * i : i; }
    __host__ __device__ __forceinline__ int column(int pack) const { return pack * VEC - behind; }
    // 2: all of the pack is the row's, 1: a part, 0: nothing
    __host__ __device__ __forceinline__ int kind(int j, int cols) const {
        if (!ODD) return j < cols ? 2 : 0;
        return j >= 0 && j + VEC <= cols ? 2 : j + VEC > 0 && j < cols ? 1 : 0;
    }
};

// Whether a pack that has columns j to j + VEC - 1 in or next to row r lies inside the matrix, gaps between rows counted in: all
// but the first row's first and the last row's last one, as rows have VEC - 1 elements at least (alike()).
template <int VEC> __host__ __device__ __forceinline__ bool pack_inside(int j, int cols, int64_t r, int64_t rows) {
    return (j >= 0 || r > 0) && (j + VEC <= cols || r + 1 < rows);
}

// A thread's pack of a row on its way into its place in the ring. What is in part the row's and reaches out of the matrix is
// read element by element at once.
template <class T, int VEC, bool ODD>
__device__ __forceinline__ void fetch_pack(uint32_t to, const T* row, int kind, int j, int cols, int64_t r, int64_t rows) {
    if (!kind) return;
    if (!ODD || kind == 2 || pack_inside<VEC>(j, cols, r, rows)) {
        copy16(to, row + j);
        return;
    }
#pragma unroll 1
    for (int e = 0; e < VEC; ++e)
        if (j + e >= 0 && j + e < cols) {
            if constexpr (sizeof(T) == 4) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + e * 4), "f"(row[j + e]) : "memory");
            else asm volatile("st.shared.b16 [%0], %1;" ::"r"(to + e * 2), "h"(*reinterpret_cast<const uint16_t*>(row + j + e)) : "memory");
        }
}

// The pack; what is not the row's is 0.
template <class T, int VEC, bool ODD> __device__ __forceinline__ Pack<T, VEC> take_pack(uint32_t at, int kind, int j, int cols) {
    Pack<T, VEC> v = ring_pack<T, VEC>(at);
    if (ODD && kind == 1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v.v[e] = j + e >= 0 && j + e < cols ? v.v[e] : from_float<T>(0.0f);
    }
    return v;
}

// Writes a pack; one that is in part the row's element by element, by way of the thread's place `at` in the ring (a loop, not
// VEC copies of it: rows pass faster when their code fits the instruction cache).
template <class T, int VEC, bool ODD>
__device__ __forceinline__ void put_pack(int kind, T* row, int j, int cols, const Pack<T, VEC>& v, uint32_t at) {
    if (!ODD || kind == 2) {
        if constexpr (sizeof(T) * VEC >= 16) store_pack_split<T, VEC>(row + j, v);
        else *reinterpret_cast<Pack<T, VEC>*>(row + j) = v;
        return;
    }
    const uint32_t* const u = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(v)) / 4; ++k) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + k * 4), "r"(u[k]) : "memory");
#pragma unroll 1
    for (int e = max(0, -j); e < min(VEC, cols - j); ++e) {
        uint32_t x;
        if constexpr (sizeof(T) == 4) {
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(at + e * 4) : "memory");
            *reinterpret_cast<uint32_t*>(row + j + e) = x;
        } else if constexpr (sizeof(T) == 2) {
            uint16_t y;
            asm volatile("ld.shared.b16 %0, [%1];" : "=h"(y) : "r"(at + e * 2) : "memory");
            *reinterpret_cast<uint16_t*>(row + j + e) = y;
        } else {
            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(x) : "r"(at + e) : "memory");
            *reinterpret_cast<uint8_t*>(row + j + e) = static_cast<uint8_t>(x);
        }
    }
}
template <class T, int VEC, bool ODD>
__device__ __forceinline__ void weights_of_pack(float (&w)[VEC], const void* p, int dt, int64_t stride, bool whole, int j, int cols) {
    if constexpr (ODD) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] = j + e >= 0 && j + e < cols ? weight_at(p, dt, (j + e) * stride) : 0.0f;
    } else {
        read_weights<T, VEC>(w, p, dt, stride, whole, j);
    }
}
template <class T, int VEC> __device__ __forceinline__ int elements_behind(const void* p) {
    return static_cast<int>(reinterpret_cast<uintptr_t>(p) / sizeof(T) & (VEC - 1));
}

template <class T, int VEC, int G, int NP, bool RES, int QUANT, bool ODD>
__global__ void __launch_bounds__(group_threads<G>(), forward_ctas<G>()) norm_rows_ring(NormArgs a) {
    extern __shared__ __align__(16) unsigned char ring[];
    dependent_wait();
    __shared__ float sm[2][32];
    int turn = 0;
    const RowViews<kNmViews>& v = a.v;
    __shared__ uint32_t block_tops[2][group_threads<G>() / G][ODD && QUANT == 2 ? kRingPacks * VEC / kScaleBlock + 1 : 1];
    int turns = 0;
    if (ODD && QUANT == 2) {
        for (int k = threadIdx.x % G; k <= v.cols / kScaleBlock; k += G) block_tops[0][threadIdx.x / G][k] = 0u;
        __syncwarp();  // a group of one warp meets nowhere else before its first row's maxima
    }
    constexpr int kGroups = group_threads<G>() / G, kArrays = RES ? 2 : 1, kRing = ring_stages<G, NP>(kArrays, forward_ctas<G>());
    const int t = threadIdx.x % G, cols = static_cast<int>(v.cols);
    const int64_t groups = static_cast<int64_t>(gridDim.x) * kGroups, group = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / G;
    const Share<VEC, ODD> share(v.rows, group, groups, elements_behind<T, VEC>(v.ptr[kNmX]), v.stride[kNmX][0]);
    const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + threadIdx.x * 16;
    constexpr uint32_t kStep = group_threads<G>() * 16;  // from one pack of a thread to its next
    auto fetch = [&](int64_t i, int stage) {
        if (i < share.hi) {
            const int64_t r = share.row(i);
            auto matrix = [&](int slot, int array) {
                const T* const row = static_cast<const T*>(v.ptr[slot]) + row_offset(v, slot, r);
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    const int j = share.column(q * G + t);
                    fetch_pack<T, VEC, ODD>(mine + ((stage * kArrays + array) * NP + q) * kStep, row, share.kind(j, cols), j, cols, r, v.rows);
                }
            };
            matrix(kNmX, 0);
            if (RES) matrix(kNmResidual, 1);
        }
        copies_commit();
    };
#pragma unroll 1
    for (int s = 0; s < kRing - 1; ++s) fetch(share.lo + s, s);
    float w[NP][VEC];
#pragma unroll
    for (int q = 0; q < NP; ++q)
        if (share.kind(share.column(q * G + t), cols))
            weights_of_pack<T, VEC, ODD>(w[q], a.weight, a.weight_dtype, a.weight_stride, a.weight_whole, share.column(q * G + t), cols);
    int stage = 0, ahead = kRing - 1;
    for (int64_t i = share.lo; i < share.hi; ++i) {
        const int64_t r = share.row(i);
        copies_wait<kRing>();
        Pack<T, VEC> s[NP];
        T* const kept = RES ? static_cast<T*>(v.ptr[kNmSummed]) + row_offset(v, kNmSummed, r) : nullptr;
        float ss = 0.0f;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int j = share.column(q * G + t), kind = share.kind(j, cols);
            if (!kind) continue;
            s[q] = take_pack<T, VEC, ODD>(mine + (stage * kArrays * NP + q) * kStep, kind, j, cols);
            if (RES) {
                const Pack<T, VEC> o = take_pack<T, VEC, ODD>(mine + (stage * kArrays * NP + NP + q) * kStep, kind, j, cols);
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[q].v[e] = from_float<T>(to_float(s[q].v[e]) + to_float(o.v[e]));
                put_pack<T, VEC, ODD>(kind, kept, j, cols, s[q], mine + (stage * kArrays * NP + q) * kStep);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) ss = fmaf(to_float(s[q].v[e]), to_float(s[q].v[e]), ss);
        }
        fetch(i + kRing - 1, ahead);
        const int taken = stage;
        stage = stage + 1 == kRing ? 0 : stage + 1;
        ahead = ahead + 1 == kRing ? 0 : ahead + 1;
        ss = group_join<G, false>(ss, sm, turn);
        const float rstd = 1.0f / sqrtf(ss / static_cast<float>(cols) + a.eps);
        if (t == 0 && v.ptr[kNmRstd]) static_cast<float*>(v.ptr[kNmRstd])[row_offset(v, kNmRstd, r)] = rstd;
        if constexpr (QUANT == 0) {
            T* const out = static_cast<T*>(v.ptr[kNmOut]) + row_offset(v, kNmOut, r);
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const int j = share.column(q * G + t), kind = share.kind(j, cols);
                if (!kind) continue;
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[q].v[e] = from_float<T>(to_float(s[q].v[e]) * rstd * w[q][e]);
                put_pack<T, VEC, ODD>(kind, out, j, cols, s[q], mine + (taken * kArrays * NP + q) * kStep);
            }
        } else {
            uint8_t* const out = static_cast<uint8_t*>(v.ptr[kNmOut]) + row_offset(v, kNmOut, r);
            float* const scales = static_cast<float*>(v.ptr[kNmScales]) + row_offset(v, kNmScales, r);
            Divisor quotient(1.0f);
            // packs that reach over 128 columns' borders: the blocks' maxima meet in shared memory (as the bits of numbers that
            // are not negative, which order like them, NaN above all)
            constexpr bool kMeet = ODD && QUANT == 2;
            uint32_t* const tops = kMeet ? block_tops[turns][threadIdx.x / G] : nullptr;
            if constexpr (kMeet) {
                for (int k = t; k <= cols / kScaleBlock; k += G) block_tops[turns ^ 1][threadIdx.x / G][k] = 0u;
                turns ^= 1;
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    const int j = share.column(q * G + t);
                    if (!share.kind(j, cols)) continue;
                    const int left = max(j, 0) / kScaleBlock, border = (left + 1) * kScaleBlock - j;
                    uint32_t low = 0u, high = 0u;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const uint32_t bits = __float_as_uint(fabsf(to_float(s[q].v[e]) * rstd * w[q][e]));
                        if (j + e < 0 || j + e >= cols) continue;
                        if (e < border) low = max(low, bits);
                        else high = max(high, bits);
                    }
                    atomicMax(tops + left, low);
                    if (border < VEC && j + border < cols) atomicMax(tops + left + 1, high);
                }
                if (G > 32) __syncthreads();
                else __syncwarp();
                for (int k = t; k * kScaleBlock < cols; k += G) scales[k * v.inner[kNmScales]] = scale_of(__uint_as_float(tops[k]));
            }
            if (QUANT == 1) {
                float top = 0.0f;
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    if (share.kind(share.column(q * G + t), cols))
#pragma unroll
                        for (int e = 0; e < VEC; ++e) top = max_nan(top, fabsf(to_float(s[q].v[e]) * rstd * w[q][e]));
                const float scale = scale_of(group_join<G, true>(top, sm, turn));
                quotient = Divisor(scale);
                if (t == 0) *scales = scale;
            }
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const int j = share.column(q * G + t), kind = share.kind(j, cols);
                const bool live = kind != 0;
                float y[VEC], top = 0.0f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    y[e] = live ? to_float(s[q].v[e]) * rstd * w[q][e] : 0.0f;
                    top = max_nan(top, fabsf(y[e]));
                }
                Divisor high = quotient;
                int border = VEC;
                if (kMeet) {
                    if (live) {
                        const int left = max(j, 0) / kScaleBlock;
                        border = (left + 1) * kScaleBlock - j;
                        quotient = Divisor(scale_of(__uint_as_float(tops[left])));
                        high = border < VEC && j + border < cols ? Divisor(scale_of(__uint_as_float(tops[left + 1]))) : quotient;
                    }
                } else if (QUANT == 2) {
                    // the threads that have 128 columns are neighbours in a warp
                    constexpr int kShare = kScaleBlock / VEC;
#pragma unroll
                    for (int d = kShare / 2; d >= 1; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const float scale = scale_of(top);
                    quotient = Divisor(scale);
                    if (live && t % kShare == 0) scales[(j / kScaleBlock) * v.inner[kNmScales]] = scale;
                }
                if (!live) continue;
                Pack<uint8_t, VEC> b;
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    float2 q;
                    if constexpr (kMeet) {  // (selects in place of the branches: 232 us against 168, 8192 x 4099 bfloat16)
                        if (e >= border) quotient = high;
                        q.x = quotient(y[e]);
                        if (e + 1 >= border) quotient = high;
                        q.y = quotient(y[e + 1]);
                    } else {
                        q = quotients(make_float2(y[e], y[e + 1]), quotient);
                    }
                    const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, __NV_E4M3);
                    b.v[e] = static_cast<uint8_t>(two);
                    b.v[e + 1] = static_cast<uint8_t>(two >> 8);
                }
                put_pack<uint8_t, VEC, ODD>(kind, out, j, cols, b, mine + (taken * kArrays * NP + q) * kStep);
            }
        }
    }
    allow_dependents();
}

// The groups' sums of a CTA's rows, joined in their order, as the CTA's row of partial sums.
template <int VEC, int G, int NP>
__device__ __forceinline__ void put_partial(const NormGradArgs& a, const float (&sums)[NP][VEC], int t, int cols, int behind) {
    float* const part = a.partial + static_cast<int64_t>(blockIdx.x) * cols;
    constexpr int kGroups = group_threads<G>() / G;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
        if (k > 0) __syncthreads();
        if (static_cast<int>(threadIdx.x) / G != k) continue;
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int j = (q * G + t) * VEC + e - behind;
                if (j >= 0 && j < cols) part[j] = k > 0 ? part[j] + sums[q][e] : sums[q][e];
            }
    }
}

// A thread keeps its columns' sums of grad_weight in registers over all rows of its group; the groups of a CTA are joined
// in their order at the end.
template <class T, int VEC, int G, int NP, bool PASSED>
__global__ void __launch_bounds__(group_threads<G>(), group_ctas<G>(768)) norm_grad_held(NormGradArgs a) {
    dependent_wait();
    __shared__ float sm[2][32];
    int turn = 0;
    const RowViews<kNgViews>& v = a.v;
    constexpr int kGroups = group_threads<G>() / G;
    const int t = threadIdx.x % G, cols = static_cast<int>(v.cols);
    float sums[NP][VEC];
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sums[q][e] = 0.0f;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / G; r < v.rows; r += static_cast<int64_t>(gridDim.x) * kGroups) {
        const T* const up = static_cast<const T*>(v.ptr[kNgUp]) + row_offset(v, kNgUp, r);
        const T* const x = static_cast<const T*>(v.ptr[kNgSummed]) + row_offset(v, kNgSummed, r);
        Pack<T, VEC> g[NP], s[NP], p[PASSED ? NP : 1];
        float rstd = 0.0f;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int j = (q * G + t) * VEC;
            if (j >= cols) continue;
            g[q] = read_pack<T, VEC>(up + j);
            s[q] = read_pack<T, VEC>(x + j);
        }
        if (PASSED) {
            const T* const from = static_cast<const T*>(v.ptr[kNgPassed]) + row_offset(v, kNgPassed, r);
#pragma unroll
            for (int q = 0; q < NP; ++q)
                if ((q * G + t) * VEC < cols) p[q] = read_pack<T, VEC>(from + (q * G + t) * VEC);
        }
        rstd = static_cast<const float*>(v.ptr[kNgRstd])[row_offset(v, kNgRstd, r)];
        float dot = 0.0f;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int j = (q * G + t) * VEC;
            if (j >= cols) continue;
            float w[VEC];
            read_weights<T, VEC>(w, a.weight, a.weight_dtype, a.weight_stride, a.weight_whole, j);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float up_e = to_float(g[q].v[e]), hat = to_float(s[q].v[e]) * rstd;
                sums[q][e] = fmaf(up_e, hat, sums[q][e]);
                dot = fmaf(up_e * w[e], hat, dot);
            }
        }
        dot = group_join<G, false>(dot, sm, turn) / static_cast<float>(cols);
        T* const grad = static_cast<T*>(v.ptr[kNgGradX]) + row_offset(v, kNgGradX, r);
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int j = (q * G + t) * VEC;
            if (j >= cols) continue;
            float w[VEC];
            read_weights<T, VEC>(w, a.weight, a.weight_dtype, a.weight_stride, a.weight_whole, j);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float hat = to_float(s[q].v[e]) * rstd;
                float y = rstd * (to_float(g[q].v[e]) * w[e] - hat * dot);
                if (PASSED) y += to_float(p[q].v[e]);
                s[q].v[e] = from_float<T>(y);
            }
            store_pack_split<T, VEC>(grad + j, s[q]);
        }
    }
    if (a.grad_weight) put_partial<VEC, G, NP>(a, sums, t, cols, 0);
    allow_dependents();
}

// The same with 16-byte packs on their way through shared memory, as norm_rows_ring (B200, 16384 x 4096 bfloat16 with a
// gradient passed on: 173 us with the rows in registers, 97 so, 537 MB).
template <class T, int VEC, int G, int NP, bool PASSED, bool ODD>
__global__ void __launch_bounds__(group_threads<G>(), backward_ctas<G, ODD>()) norm_grad_ring(NormGradArgs a) {
    extern __shared__ __align__(16) unsigned char ring[];
    dependent_wait();
    __shared__ float sm[2][32];
    int turn = 0;
    const RowViews<kNgViews>& v = a.v;
    constexpr int kGroups = group_threads<G>() / G, kArrays = PASSED ? 3 : 2, kRing = ring_stages<G, NP>(kArrays, backward_ctas<G, ODD>());
    const int t = threadIdx.x % G, cols = static_cast<int>(v.cols);
    const int64_t groups = static_cast<int64_t>(gridDim.x) * kGroups, group = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / G;
    const Share<VEC, ODD> share(v.rows, group, groups, elements_behind<T, VEC>(v.ptr[kNgUp]), v.stride[kNgUp][0]);
    const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + threadIdx.x * 16;
    constexpr uint32_t kStep = group_threads<G>() * 16;
    auto fetch = [&](int64_t i, int stage) {
        if (i < share.hi) {
            const int64_t r = share.row(i);
            auto matrix = [&](int slot, int array) {
                const T* const row = static_cast<const T*>(v.ptr[slot]) + row_offset(v, slot, r);
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    const int j = share.column(q * G + t);
                    fetch_pack<T, VEC, ODD>(mine + ((stage * kArrays + array) * NP + q) * kStep, row, share.kind(j, cols), j, cols, r, v.rows);
                }
            };
            matrix(kNgUp, 0);
            matrix(kNgSummed, 1);
            if (PASSED) matrix(kNgPassed, 2);
        }
        copies_commit();
    };
#pragma unroll 1
    for (int s = 0; s < kRing - 1; ++s) fetch(share.lo + s, s);
    float w[NP][VEC], sums[NP][VEC];
#pragma unroll
    for (int q = 0; q < NP; ++q) {
        if (share.kind(share.column(q * G + t), cols))
            weights_of_pack<T, VEC, ODD>(w[q], a.weight, a.weight_dtype, a.weight_stride, a.weight_whole, share.column(q * G + t), cols);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sums[q][e] = 0.0f;
    }
    const float* const rstds = static_cast<const float*>(v.ptr[kNgRstd]);
    float rstd = share.lo < share.hi ? rstds[row_offset(v, kNgRstd, share.row(share.lo))] : 0.0f;
    int stage = 0, ahead = kRing - 1;
    for (int64_t i = share.lo; i < share.hi; ++i) {
        const int64_t r = share.row(i);
        copies_wait<kRing>();
        Pack<T, VEC> g[NP], s[NP];
        float dot = 0.0f;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int j = share.column(q * G + t), kind = share.kind(j, cols);
            if (!kind) continue;
            g[q] = take_pack<T, VEC, ODD>(mine + (stage * kArrays * NP + q) * kStep, kind, j, cols);
            s[q] = take_pack<T, VEC, ODD>(mine + (stage * kArrays * NP + NP + q) * kStep, kind, j, cols);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float up = to_float(g[q].v[e]), hat = to_float(s[q].v[e]) * rstd;
                sums[q][e] = fmaf(up, hat, sums[q][e]);
                dot = fmaf(up * w[q][e], hat, dot);
            }
        }
        const float next = i + 1 < share.hi ? rstds[row_offset(v, kNgRstd, share.row(i + 1))] : 0.0f;
        fetch(i + kRing - 1, ahead);
        ahead = ahead + 1 == kRing ? 0 : ahead + 1;
        dot = group_join<G, false>(dot, sm, turn) / static_cast<float>(cols);
        T* const grad = static_cast<T*>(v.ptr[kNgGradX]) + row_offset(v, kNgGradX, r);
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int j = share.column(q * G + t), kind = share.kind(j, cols);
            if (!kind) continue;
            Pack<T, VEC> p;
            if (PASSED)
                p = take_pack<T, VEC, ODD>(mine + (stage * kArrays * NP + 2 * NP + q) * kStep, kind, j, cols);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float hat = to_float(s[q].v[e]) * rstd;
                float y = rstd * (to_float(g[q].v[e]) * w[q][e] - hat * dot);
                if (PASSED) y += to_float(p.v[e]);
                s[q].v[e] = from_float<T>(y);
            }
            put_pack<T, VEC, ODD>(kind, grad, j, cols, s[q], mine + (stage * kArrays * NP + q) * kStep);
        }
        stage = stage + 1 == kRing ? 0 : stage + 1;
        rstd = next;
    }
    if (a.grad_weight) put_partial<VEC, G, NP>(a, sums, t, cols, share.behind);
    allow_dependents();
}

// ------------------------------------------------------------------------------------------------
// host side

int weight_of(const ctb_view* w, int64_t cols, const char* what) {
    CTB_CHECK(check_row_view(w, what));
    CTB_CHECK(check_row_dtype(w, kDtypeMatrix, what));
    if (w->ndim != 1 || w->shape[0] != cols) return fail(CTB_ERR_SHAPE, std::string(what) + " must be [" + std::to_string(cols) + "]");
    return CTB_OK;
}

bool weight_whole(const ctb_view* w) { return (w->strides[0] == 1 || w->shape[0] == 1) && aligned16(w->data); }

// Elements a pack: 16 bytes where every row of every given matrix starts on that and is whole packs, else 1; 0 where the
// columns of one are not contiguous.
template <int N> int pack_of(const RowViews<N>& v, std::initializer_list<int> slots) {
    int vec = 16 / static_cast<int>(dtype_size(v.dtype[0]));
    if (v.cols % vec) vec = 1;
    for (int s : slots) {
        if (!v.ptr[s]) continue;
        if (v.inner[s] != 1 && v.cols > 1) return 0;
        const int64_t size = static_cast<int64_t>(dtype_size(v.dtype[s])), align = size == 1 ? 16 / static_cast<int64_t>(dtype_size(v.dtype[0])) : 16;
        if (reinterpret_cast<uintptr_t>(v.ptr[s]) % align) vec = 1;
        for (int d = 0; d < v.rank; ++d)
            if (v.stride[s][d] * size % align) vec = 1;
    }
    return vec;
}

// Whether rows fill a pack but for one element, so that a pack of memory touches two of them at most.
constexpr bool wide_rows(int64_t cols, int vec) { return cols >= vec - 1; }

// Whether all rows of the given matrices start equally far behind a pack (16 bytes of the rows' type), with unit strides along
// and one stride across, and are wide enough: packs of memory then serve all of them.
template <int N> bool alike(const RowViews<N>& v, std::initializer_list<int> slots) {
    const int64_t size = static_cast<int64_t>(dtype_size(v.dtype[0])), vec = 16 / size;
    if (v.rank != 1 || !wide_rows(v.cols, static_cast<int>(vec))) return false;
    const int64_t base = reinterpret_cast<uintptr_t>(v.ptr[0]) / size % vec;
    for (int s : slots) {
        if (!v.ptr[s]) continue;
        const int64_t own = static_cast<int64_t>(dtype_size(v.dtype[s]));
        if (reinterpret_cast<uintptr_t>(v.ptr[s]) % own || static_cast<int64_t>(reinterpret_cast<uintptr_t>(v.ptr[s]) / own % vec) != base ||
            ((v.stride[s][0] - v.stride[0][0]) & (vec - 1)) || (v.rows > 1 && v.stride[s][0] < v.cols))
            return false;
    }
    return true;
}

// Calls f(group, packs a thread) for the smallest group that holds `packs`, as compile-time numbers; false where none does. A
// thread has 16 elements at most, so that a backward pass has room for their weights and sums; longer rows are held by 1024
// threads of up to 8 packs.
template <int VEC, class F> bool with_group(int64_t packs, F&& f) {
    auto take = [&](auto g, auto np) {
        if (packs > static_cast<int64_t>(g) * np) return false;
        f(g, np);
        return true;
    };
#define CTB_TAKE(G, NP) take(std::integral_constant<int, G>{}, std::integral_constant<int, NP>{})
    if constexpr (VEC == 4) {
        return CTB_TAKE(32, 1) || CTB_TAKE(32, 2) || CTB_TAKE(32, 4) || CTB_TAKE(64, 4) || CTB_TAKE(128, 3) || CTB_TAKE(128, 4) ||
               CTB_TAKE(256, 3) || CTB_TAKE(256, 4) || CTB_TAKE(512, 3) || CTB_TAKE(512, 4) || CTB_TAKE(1024, 4);
    } else if constexpr (VEC == 8) {
        return CTB_TAKE(32, 1) || CTB_TAKE(32, 2) || CTB_TAKE(64, 2) || CTB_TAKE(128, 2) || CTB_TAKE(256, 2) || CTB_TAKE(512, 2) ||
               CTB_TAKE(1024, 2) || CTB_TAKE(1024, 4);
    } else {
        return CTB_TAKE(32, 2) || CTB_TAKE(128, 2) || CTB_TAKE(256, 2) || CTB_TAKE(512, 2) || CTB_TAKE(1024, 2) || CTB_TAKE(1024, 4) ||
               CTB_TAKE(1024, 8);
    }
#undef CTB_TAKE
}

// CTAs an SM in a grid: what is resident, or eight times that where several groups share an SM and no row waits for a
// second sum and there are enough of them: the SMs do not all stream alike (B200, 16384 x 4096 with a residual: 89 us, 96 without; to 8 bits with a
// scale for every 128 columns, 8192 x 8192, the other way round: 123 against 109).
int norm_grid(int resident, int quant, int64_t rows) {
    return resident > 2 && !quant && rows >= static_cast<int64_t>(sm_count()) * resident * 16 ? 8 * resident : resident;
}

// Starts a kernel whose rows pass through shared memory, `per_sm` CTAs an SM at most.
template <class A, class K> void launch_ring(K kernel, const A& a, unsigned grid, int threads, int bytes, cudaStream_t st) {
    if (bytes > 47 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    launch_dependent(kernel, grid, threads, bytes, st, a);
}

template <class T, int VEC, bool ODD> bool run_norm_held(const NormArgs& a, cudaStream_t st) {
    const int64_t packs = ODD ? (a.v.cols + 2 * VEC - 2) / VEC : (a.v.cols + VEC - 1) / VEC;
    if (ODD && packs > kRingPacks) return false;
    return with_group<VEC>(packs, [&](auto g, auto np) {
        constexpr int G = decltype(g)::value, NP = decltype(np)::value, threads = group_threads<G>(), groups = threads / G;
        const bool res = a.v.ptr[kNmResidual] != nullptr;
        unsigned grid = grid_for((a.v.rows + groups - 1) / groups, VEC > 1 && G * NP <= kRingPacks ? norm_grid(forward_ctas<G>(), a.quant, a.v.rows) : 64);
        if (ODD) grid = grid < VEC ? VEC : grid / VEC * VEC;  // whole periods of kinds of rows
        if constexpr (VEC > 1 && G * NP <= kRingPacks) {
            auto launch = [&](auto kernel, int arrays) { launch_ring(kernel, a, grid, threads, ring_bytes<G, NP>(arrays, forward_ctas<G>()), st); };
            if (a.quant == 0) res ? launch(norm_rows_ring<T, VEC, G, NP, true, 0, ODD>, 2) : launch(norm_rows_ring<T, VEC, G, NP, false, 0, ODD>, 1);
            else if (a.quant == 1) res ? launch(norm_rows_ring<T, VEC, G, NP, true, 1, ODD>, 2) : launch(norm_rows_ring<T, VEC, G, NP, false, 1, ODD>, 1);
            else res ? launch(norm_rows_ring<T, VEC, G, NP, true, 2, ODD>, 2) : launch(norm_rows_ring<T, VEC, G, NP, false, 2, ODD>, 1);
        } else if constexpr (!ODD) {
            auto plain = [&](auto kernel) { launch_dependent(kernel, grid, threads, 0, st, a); };
            if (a.quant == 0) res ? plain(norm_rows_held<T, VEC, G, NP, true, 0>) : plain(norm_rows_held<T, VEC, G, NP, false, 0>);
            else if (a.quant == 1) res ? plain(norm_rows_held<T, VEC, G, NP, true, 1>) : plain(norm_rows_held<T, VEC, G, NP, false, 1>);
            else if constexpr (VEC > 1) res ? plain(norm_rows_held<T, VEC, G, NP, true, 2>) : plain(norm_rows_held<T, VEC, G, NP, false, 2>);
        }
    });
}

template <class T> void run_norm(const NormArgs& a, cudaStream_t st) {
    constexpr int kVec = 16 / sizeof(T);
    const int vec = pack_of(a.v, {kNmX, kNmResidual, kNmSummed, kNmOut});
    const bool held = vec == kVec ? run_norm_held<T, kVec, false>(a, st)
                                  : vec == 1 && ((alike(a.v, {kNmX, kNmResidual, kNmSummed, kNmOut}) && run_norm_held<T, kVec, true>(a, st)) ||
                                                 (a.quant != 2 && run_norm_held<T, 1, false>(a, st)));
    if (!held) launch_dependent(norm_rows_any<T>, grid_for(a.v.rows, 8), kAnyThreads, 0, st, a);
    count_launch();
}

// CTAs of the backward pass at most, each with a row of partial sums: as many as are resident, fewer on longer rows.
int64_t grad_ctas(int64_t rows, int64_t row_bytes) {
    return std::min<int64_t>(rows, static_cast<int64_t>(sm_count()) * (row_bytes <= 4096 ? 6 : row_bytes <= 8192 ? 3 : 2));
}

template <class T, int VEC, bool ODD> bool run_grad_held(NormGradArgs& a, cudaStream_t st) {
    const int64_t packs = ODD ? (a.v.cols + 2 * VEC - 2) / VEC : (a.v.cols + VEC - 1) / VEC;
    if (ODD && (packs > kRingPacks || a.ctas < VEC)) return false;
    return with_group<VEC>(packs, [&](auto g, auto np) {
        constexpr int G = decltype(g)::value, NP = decltype(np)::value;
        const bool passed = a.v.ptr[kNgPassed] != nullptr;
        constexpr int groups = group_threads<G>() / G, per_sm = backward_ctas<G, ODD>();
        a.ctas = static_cast<int>(std::min<int64_t>({a.ctas, (a.v.rows + groups - 1) / groups, static_cast<int64_t>(sm_count()) * per_sm}));
        if (ODD) a.ctas = a.ctas / VEC * VEC > 0 ? a.ctas / VEC * VEC : VEC;  // whole periods of kinds of rows
        const unsigned grid = static_cast<unsigned>(a.ctas);
        if constexpr (VEC > 1 && G * NP <= kRingPacks) {
            auto launch = [&](auto kernel, int arrays) { launch_ring(kernel, a, grid, group_threads<G>(), ring_bytes<G, NP>(arrays, backward_ctas<G, ODD>()), st); };
            passed ? launch(norm_grad_ring<T, VEC, G, NP, true, ODD>, 3) : launch(norm_grad_ring<T, VEC, G, NP, false, ODD>, 2);
        } else if constexpr (!ODD) {
            auto plain = [&](auto kernel) { launch_dependent(kernel, grid, group_threads<G>(), 0, st, a); };
            passed ? plain(norm_grad_held<T, VEC, G, NP, true>) : plain(norm_grad_held<T, VEC, G, NP, false>);
        }
    });
}

template <class T> void run_grad(NormGradArgs& a, cudaStream_t st) {
    constexpr int kVec = 16 / sizeof(T);
    const int vec = pack_of(a.v, {kNgUp, kNgSummed, kNgPassed, kNgGradX});
    const bool held = vec == kVec ? run_grad_held<T, kVec, false>(a, st)
                                  : vec == 1 && ((alike(a.v, {kNgUp, kNgSummed, kNgPassed, kNgGradX}) && run_grad_held<T, kVec, true>(a, st)) ||
                                                 run_grad_held<T, 1, false>(a, st));
    if (!held) launch_dependent(norm_grad_any<T>, static_cast<unsigned>(a.ctas), kAnyThreads, 0, st, a);
    count_launch();
}

// The elements that the ring's packs read of a matrix, by the kernels' own arithmetic: the first and the last one that is part of
// a pack read whole.
template <int VEC> void packs_read(int64_t rows, int cols, int64_t stride, int base, int64_t& lowest, int64_t& highest) {
    lowest = highest = 0;
    if (!wide_rows(cols, VEC)) return;  // such rows are read element by element
    for (int64_t group = 0; group < VEC; ++group) {
        const Share<VEC, true> share(rows, group, VEC, base, stride);
        for (int64_t i = share.lo; i < share.hi; ++i) {
            const int64_t r = share.row(i);
            for (int pack = 0; pack <= (cols + 2 * VEC - 2) / VEC; ++pack) {
                const int j = share.column(pack), kind = share.kind(j, cols);
                if (kind == 2 || (kind == 1 && pack_inside<VEC>(j, cols, r, rows))) {
                    lowest = std::min(lowest, r * stride + j);
                    highest = std::max(highest, r * stride + j + VEC - 1);
                }
            }
        }
    }
}

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
        a.weight_whole = weight_whole(weight);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (x->dtype == CTB_FLOAT32) run_norm<float>(a, st);
        else run_norm<__nv_bfloat16>(a, st);
        return check_launch("rms norm");
    });
}

size_t ctb_rms_norm_backward_scratch_bytes(const ctb_view* summed) {
    if (!summed || summed->ndim < 1 || summed->ndim > kMaxDims) return 0;
    int64_t rows = 1;
    for (int d = 0; d < summed->ndim - 1; ++d) rows *= summed->shape[d];
    const int64_t cols = summed->shape[summed->ndim - 1];
    return static_cast<size_t>(grad_ctas(rows, cols * static_cast<int64_t>(dtype_size(summed->dtype))) * cols) * sizeof(float);
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
        a.ctas = static_cast<int>(grad_ctas(b.v.rows, cols * static_cast<int64_t>(dtype_size(grad_out->dtype))));
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
            a.weight_whole = weight_whole(weight);
            if (grad_out->dtype == CTB_FLOAT32) run_grad<float>(a, st);
            else run_grad<__nv_bfloat16>(a, st);
            CTB_CHECK(check_launch("rms norm backward"));
        }
        if (grad_weight) {
            launch_dependent(norm_grad_weight, static_cast<unsigned>((cols + 31) / 32), 1024, 0, st, a);
            count_launch();
            CTB_CHECK(check_launch("rms norm backward"));
        }
        return CTB_OK;
    });
}

int ctb_debug_norm_reads(int64_t rows, int cols, int64_t stride, int base, int elem_bytes, int64_t* lowest, int64_t* highest) {
    if (rows < 1 || cols < 1 || (rows > 1 && stride < cols) || base < 0 || !lowest || !highest) return CTB_ERR_ARGUMENT;
    if (elem_bytes == 4) packs_read<4>(rows, cols, stride, base, *lowest, *highest);
    else if (elem_bytes == 2) packs_read<8>(rows, cols, stride, base, *lowest, *highest);
    else return CTB_ERR_ARGUMENT;
    return CTB_OK;
}

}  // extern "C"
