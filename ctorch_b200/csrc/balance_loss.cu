// balance_loss.cu — the balance loss of routed experts, with the experts' counts and the router's gradient
// (include/ctb/ctb.h).
//
// For a group of rows of which n count, with p = softmax(x) of a row, its k chosen experts and lse = log sum exp x:
//     f_e = (times e was chosen) / (n k),  P_e = mean p_e,  loss = coef E sum_e f_e P_e + z_coef mean lse^2
//     dloss/dx_j = p_j / n (a_j - sum_e a_e p_e + 2 z_coef lse),  a_e = coef E f_e
// A row's gradient needs the whole group's counts. They are taken in the same pass as the sums of p, so the logits are read
// twice: balance_rows sums a run of rows of one group per CTA, balance_join adds the runs in their order, balance_grad writes
// the gradient. (The counts need experts and mask alone: counted first, one read of the logits would do.)
#include <algorithm>
#include <cmath>

#include "rows.cuh"

namespace ctb {

namespace {

enum BalanceRow : int { kBlX = 0, kBlExperts, kBlMask, kBlGrad, kBlViews };

constexpr int kMaxExperts = 4096;
constexpr int kMaxGroups = 1 << 20;
constexpr int kThreads = 256, kWarps = kThreads / 32;

struct BalanceRun {  // of one CTA's rows
    double lse2;
    int32_t rows, bad;
};

struct BalanceGroup {
    double lse2, rows;  // mean of lse^2; rows that count, 1 at least
    int32_t bad, pad;
};

struct BalanceArgs {
    RowViews<kBlViews> v;
    int64_t chosen, groups, length;  // experts a row; rows a group
    int64_t runs, run_rows;          // CTAs a group, rows of each
    double coef, z_coef;
    float* run_probs;    // [groups * runs][E]
    int32_t* run_counts; // the same
    BalanceRun* run;     // [groups * runs]
    float* slope;        // [groups][E] a_e
    BalanceGroup* group; // [groups]
    double* inner;       // [groups][chunks] sums of a_e P_e over 32 experts each
    float2* row_stats;   // [rows] (maximum, sum of exponentials)
    int64_t chunks;
    float* loss;
    int64_t* counts;
    int64_t counts_stride[2];
    float* probs;
    int64_t probs_stride[2];
    int32_t* status;
};

__device__ __forceinline__ float warp_max(float x) {
    for (int d = 16; d >= 1; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}
__device__ __forceinline__ float warp_sum(float x) {
    for (int d = 16; d >= 1; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

__device__ __forceinline__ bool row_counts(const BalanceArgs& a, int64_t r) {
    return !a.v.ptr[kBlMask] || real_at(a.v.ptr[kBlMask], a.v.dtype[kBlMask], row_offset(a.v, kBlMask, r)) != 0.0;
}

struct RowStats {
    float m, s;  // maximum, sum of exp(x - m); s is NaN where the row has no softmax
};

template <class T> __device__ __forceinline__ RowStats row_stats(const T* x, int64_t inner, int experts) {
    RowStats o{-INFINITY, 0.0f};
    for (int e = threadIdx.x & 31; e < experts; e += 32) o.m = fmaxf(o.m, to_float(x[e * inner]));
    o.m = warp_max(o.m);
    for (int e = threadIdx.x & 31; e < experts; e += 32) o.s += expf(to_float(x[e * inner]) - o.m);
    o.s = warp_sum(o.s);
    return o;
}

// A run's results out of shared memory: the warps' sums in their order.
__device__ __forceinline__ void put_run(const BalanceArgs& a, const int32_t* counts, const float* sums, const double* lse2,
                                        const int32_t* live, int32_t bad) {
    const int experts = static_cast<int>(a.v.cols);
    float* const out = a.run_probs + blockIdx.x * a.v.cols;
    int32_t* const out_counts = a.run_counts + blockIdx.x * a.v.cols;
    for (int e = threadIdx.x; e < experts; e += kThreads) {
        float s = 0.0f;
        for (int w = 0; w < kWarps; ++w) s += sums[w * experts + e];
        out[e] = s;
        out_counts[e] = counts[e];
    }
    if (threadIdx.x == 0) {
        BalanceRun b{0.0, 0, bad};
        for (int w = 0; w < kWarps; ++w) {
            b.lse2 += lse2[w];
            b.rows += live[w];
        }
        a.run[blockIdx.x] = b;
    }
}

// Any layout and number of experts: a warp a row; every lane keeps its columns' sums of p in its warp's part of shared memory.
template <class T> __global__ void __launch_bounds__(kThreads) balance_rows(BalanceArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    dependent_wait();
    const int experts = static_cast<int>(a.v.cols), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int32_t* const counts = reinterpret_cast<int32_t*>(smem);
    float* const sums = reinterpret_cast<float*>(counts + experts);  // [kWarps][experts]
    __shared__ double lse2[kWarps];
    __shared__ int32_t live[kWarps];
    __shared__ int32_t bad;
    for (int e = threadIdx.x; e < experts; e += kThreads) counts[e] = 0;
    for (int e = threadIdx.x; e < experts * kWarps; e += kThreads) sums[e] = 0.0f;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    const int64_t group = blockIdx.x / a.runs, run = blockIdx.x % a.runs;
    const int64_t lo = group * a.length + run * a.run_rows, hi = min(lo + a.run_rows, (group + 1) * a.length);
    double l2 = 0.0;
    int n = 0;
    for (int64_t r = lo + warp; r < hi; r += kWarps) {
        if (!row_counts(a, r)) continue;
        ++n;
        const T* const x = static_cast<const T*>(a.v.ptr[kBlX]) + row_offset(a.v, kBlX, r);
        const RowStats o = row_stats(x, a.v.inner[kBlX], experts);
        const float inv = 1.0f / o.s;
        for (int e = lane; e < experts; e += 32) sums[warp * experts + e] += expf(to_float(x[e * a.v.inner[kBlX]]) - o.m) * inv;
        const double lse = static_cast<double>(o.m) + log(static_cast<double>(o.s));
        l2 += lse * lse;
        const int64_t at = row_offset(a.v, kBlExperts, r);
        for (int64_t k = lane; k < a.chosen; k += 32) {
            const int64_t e = index_at(a.v.ptr[kBlExperts], a.v.dtype[kBlExperts], at + k * a.v.inner[kBlExperts]);
            if (e >= 0 && e < experts) {
                atomicAdd(counts + e, 1);  // integers: any order gives the same
            } else {
                bad = 1;
                record_bad_index(a.status, e);
            }
        }
    }
    if (lane == 0) {
        lse2[warp] = l2;
        live[warp] = n;
    }
    __syncthreads();
    put_run(a, counts, sums, lse2, live, bad);
    allow_dependents();
}

// 32 experts of a group: its runs added in float64, in an order that their number alone gives (32 warps take every 32nd).
constexpr int kJoinThreads = 1024;
__global__ void __launch_bounds__(kJoinThreads) balance_join(BalanceArgs a) {
    dependent_wait();
    allow_dependents();
    __shared__ double sums[32][33], lse2[32], rows[32];
    __shared__ int64_t counts[32][33];
    __shared__ int32_t bads[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t g = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, e = chunk * 32 + lane, experts = a.v.cols;
    double p = 0.0;
    int64_t c = 0;
    if (e < experts) {
#pragma unroll 4
        for (int64_t i = warp; i < a.runs; i += 32) {
            p += a.run_probs[(g * a.runs + i) * experts + e];
            c += a.run_counts[(g * a.runs + i) * experts + e];
        }
    }
    sums[warp][lane] = p;
    counts[warp][lane] = c;
    double l2 = 0.0, n = 0.0;
    int32_t bad = 0;
    for (int64_t i = threadIdx.x; i < a.runs; i += kJoinThreads) {
        const BalanceRun b = a.run[g * a.runs + i];
        l2 += b.lse2;
        n += b.rows;
        bad |= b.bad;
    }
    for (int d = 16; d >= 1; d >>= 1) {
        l2 += __shfl_xor_sync(0xffffffffu, l2, d);
        n += __shfl_xor_sync(0xffffffffu, n, d);
        bad |= __shfl_xor_sync(0xffffffffu, bad, d);
    }
    if (lane == 0) {
        lse2[warp] = l2;
        rows[warp] = n;
        bads[warp] = bad;
    }
    __syncthreads();
    if (warp != 0) return;
    l2 = n = 0.0;
    bad = 0;
    p = 0.0;
    c = 0;
    for (int w = 0; w < 32; ++w) {
        l2 += lse2[w];
        n += rows[w];
        bad |= bads[w];
        p += sums[w][lane];
        c += counts[w][lane];
    }
    n = fmax(n, 1.0);
    double inner = 0.0;
    if (e < experts) {
        p /= n;
        const double slope = a.coef * static_cast<double>(experts) * static_cast<double>(c) / (n * static_cast<double>(a.chosen));
        inner = slope * p;
        a.slope[g * experts + e] = bad ? NAN : static_cast<float>(slope);
        if (a.counts) a.counts[g * a.counts_stride[0] + e * a.counts_stride[1]] = c;
        if (a.probs) a.probs[g * a.probs_stride[0] + e * a.probs_stride[1]] = static_cast<float>(p);
    }
    for (int d = 16; d >= 1; d >>= 1) inner += __shfl_xor_sync(0xffffffffu, inner, d);
    if (lane == 0) {
        a.inner[g * a.chunks + chunk] = bad ? nan("") : inner;
        if (chunk == 0) a.group[g] = BalanceGroup{l2 / n, n, bad, 0};
    }
}

// The scalar, by one warp of the last kernel: the groups' losses in their order.
__device__ __forceinline__ void put_loss(const BalanceArgs& a) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < a.groups * a.chunks; i += 32) s += a.inner[i];
    if (a.z_coef != 0.0)
        for (int64_t g = threadIdx.x; g < a.groups; g += 32) s += a.z_coef * a.group[g].lse2;
    for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (threadIdx.x == 0) *a.loss = static_cast<float>(s / static_cast<double>(a.groups));
}

// ------------------------------------------------------------------------------------------------
// rows held in registers: L lanes of a warp have a row, NP packs of VEC experts each; a warp has kRows rows of its run
// under way at a time for each of its 32 / L groups of lanes. VEC is 4 where every row starts on 4 elements. Bound by the
// reads and, in the first pass, by what a row's maximum, sum and log wait for (B200, 131072 x 256 float32: 56 and 52 us,
// element by element 170 and 190).

__device__ __forceinline__ float exp_approx(float x) {  // of x <= 0: 2^-22 and its argument's rounding
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.44269504f));
    return y;
}

template <int L> __device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
    for (int d = L / 2; d >= 1; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
template <int L> __device__ __forceinline__ float lanes_max(float x) {
#pragma unroll
    for (int d = L / 2; d >= 1; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}

template <class T, int VEC, int L, int NP> struct HeldRow {
    static constexpr int kOf = VEC * NP;
    float x[kOf];
    // Experts that there are none of are -inf.
    __device__ __forceinline__ void load(const T* p, int lane, int experts) {
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int e = (q * L + lane) * VEC;
            if (e < experts) {
                const Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC>*>(p + e);
#pragma unroll
                for (int k = 0; k < VEC; ++k) x[q * VEC + k] = to_float(v.v[k]);
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k) x[q * VEC + k] = -INFINITY;
            }
        }
    }
};

template <class T, int VEC, int L, int NP, int ROWS>
__global__ void __launch_bounds__(kThreads) balance_rows_held(BalanceArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    dependent_wait();
    constexpr int kOf = VEC * NP, kSub = 32 / L;  // experts a lane; rows of a warp side by side
    const int experts = static_cast<int>(a.v.cols), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, in = lane % L, sub = lane / L;
    int32_t* const counts = reinterpret_cast<int32_t*>(smem);
    float* const sums = reinterpret_cast<float*>(counts + experts);  // [kWarps][experts]
    __shared__ double lse2[kWarps];
    __shared__ int32_t live[kWarps];
    __shared__ int32_t bad;
    for (int e = threadIdx.x; e < experts; e += kThreads) counts[e] = 0;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    const int64_t group = blockIdx.x / a.runs, run = blockIdx.x % a.runs;
    const int64_t lo = group * a.length + run * a.run_rows, hi = min(lo + a.run_rows, (group + 1) * a.length);
    const T* const logits = static_cast<const T*>(a.v.ptr[kBlX]);
    float acc[kOf];
#pragma unroll
    for (int k = 0; k < kOf; ++k) acc[k] = 0.0f;
    double l2 = 0.0;
    int n = 0;
    for (int64_t first = lo + warp * (kSub * ROWS); first < hi; first += kWarps * kSub * ROWS) {
        HeldRow<T, VEC, L, NP> h[ROWS];
        bool on[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int64_t r = first + i * kSub + sub;
            on[i] = r < hi && row_counts(a, r);
            h[i].load(logits + (on[i] ? row_offset(a.v, kBlX, r) : 0), in, on[i] ? experts : 0);
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int64_t r = first + i * kSub + sub;
            float m = h[i].x[0];
#pragma unroll
            for (int k = 1; k < kOf; ++k) m = fmaxf(m, h[i].x[k]);
            m = lanes_max<L>(m);
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < kOf; ++k) {
                // an expert that there is none of must stay out of a row without a softmax too
                const bool there = ((k / VEC) * L + in) * VEC + k % VEC < experts;
                h[i].x[k] = there ? exp_approx(h[i].x[k] - m) : 0.0f;
                s += h[i].x[k];
            }
            s = lanes_sum<L>(s);
            if (!on[i]) continue;
            const float inv = 1.0f / s;
#pragma unroll
            for (int k = 0; k < kOf; ++k) acc[k] = fmaf(h[i].x[k], inv, acc[k]);
            if (in == 0) {
                a.row_stats[r] = make_float2(m, s);
                const double lse = static_cast<double>(m + logf(s));
                l2 += lse * lse;
                ++n;
            }
            const int64_t at = row_offset(a.v, kBlExperts, r);
            for (int64_t k = in; k < a.chosen; k += L) {
                const int64_t e = index_at(a.v.ptr[kBlExperts], a.v.dtype[kBlExperts], at + k * a.v.inner[kBlExperts]);
                if (e >= 0 && e < experts) {
                    atomicAdd(counts + e, 1);  // integers: any order gives the same
                } else {
                    bad = 1;
                    record_bad_index(a.status, e);
                }
            }
        }
    }
    __syncwarp();
    // the warp's groups of lanes, then its warps
#pragma unroll
    for (int k = 0; k < kOf; ++k)
#pragma unroll
        for (int d = L; d < 32; d <<= 1) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], d);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
        l2 += __shfl_xor_sync(0xffffffffu, l2, d);
        n += __shfl_xor_sync(0xffffffffu, n, d);
    }
    if (sub == 0) {
#pragma unroll
        for (int k = 0; k < kOf; ++k) {
            const int e = ((k / VEC) * L + in) * VEC + k % VEC;
            if (e < experts) sums[warp * experts + e] = acc[k];
        }
    }
    if (lane == 0) {
        lse2[warp] = l2;
        live[warp] = n;
    }
    __syncthreads();
    put_run(a, counts, sums, lse2, live, bad);
    allow_dependents();
}

template <class T, int VEC, int L, int NP, int ROWS>
__global__ void __launch_bounds__(kThreads) balance_grad_held(BalanceArgs a) {
    dependent_wait();
    if (a.loss && blockIdx.x == 0 && threadIdx.x < 32) put_loss(a);
    constexpr int kOf = VEC * NP, kSub = 32 / L;
    const int experts = static_cast<int>(a.v.cols), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, in = lane % L, sub = lane / L;
    const int64_t group = blockIdx.x / a.runs, run = blockIdx.x % a.runs;
    const int64_t lo = group * a.length + run * a.run_rows, hi = min(lo + a.run_rows, (group + 1) * a.length);
    const T* const logits = static_cast<const T*>(a.v.ptr[kBlX]);
    T* const grads = static_cast<T*>(a.v.ptr[kBlGrad]);
    float slope[kOf];
#pragma unroll
    for (int k = 0; k < kOf; ++k) {
        const int e = ((k / VEC) * L + in) * VEC + k % VEC;
        slope[k] = e < experts ? a.slope[group * experts + e] : 0.0f;
    }
    const float f = static_cast<float>(1.0 / (a.group[group].rows * static_cast<double>(a.groups)));
    const float z2 = static_cast<float>(2.0 * a.z_coef);
    for (int64_t first = lo + warp * (kSub * ROWS); first < hi; first += kWarps * kSub * ROWS) {
        HeldRow<T, VEC, L, NP> h[ROWS];
        float2 stats[ROWS];
        bool on[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int64_t r = first + i * kSub + sub;
            on[i] = r < hi && row_counts(a, r);
            h[i].load(logits + (on[i] ? row_offset(a.v, kBlX, r) : 0), in, on[i] ? experts : 0);
            stats[i] = on[i] ? a.row_stats[r] : make_float2(0.0f, 1.0f);
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int64_t r = first + i * kSub + sub;
            const float inv = 1.0f / stats[i].y;
            float dot = 0.0f;
#pragma unroll
            for (int k = 0; k < kOf; ++k) {
                h[i].x[k] = exp_approx(h[i].x[k] - stats[i].x) * inv;
                const bool there = ((k / VEC) * L + in) * VEC + k % VEC < experts;
                dot = there ? fmaf(slope[k], h[i].x[k], dot) : dot;
            }
            dot = lanes_sum<L>(dot);
            if (r >= hi) continue;
            const float up = z2 != 0.0f ? z2 * (stats[i].x + logf(stats[i].y)) : 0.0f;
            T* const out = grads + row_offset(a.v, kBlGrad, r);
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const int e = (q * L + in) * VEC;
                if (e >= experts) continue;
                Pack<T, VEC> v;
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    v.v[k] = from_float<T>(on[i] ? h[i].x[q * VEC + k] * (slope[q * VEC + k] - dot + up) * f : 0.0f);
                *reinterpret_cast<Pack<T, VEC>*>(out + e) = v;
            }
        }
    }
    allow_dependents();
}

template <class T> __global__ void __launch_bounds__(kThreads) balance_grad(BalanceArgs a) {
    dependent_wait();
    const int experts = static_cast<int>(a.v.cols), lane = threadIdx.x & 31;
    if (a.loss && blockIdx.x == 0 && threadIdx.x < 32) put_loss(a);
    if (!a.v.ptr[kBlGrad]) return;
    for (int64_t r = blockIdx.x * kWarps + (threadIdx.x >> 5); r < a.v.rows; r += gridDim.x * kWarps) {
        T* const grad = static_cast<T*>(a.v.ptr[kBlGrad]) + row_offset(a.v, kBlGrad, r);
        if (!row_counts(a, r)) {
            for (int e = lane; e < experts; e += 32) grad[e * a.v.inner[kBlGrad]] = from_float<T>(0.0f);
            continue;
        }
        const T* const x = static_cast<const T*>(a.v.ptr[kBlX]) + row_offset(a.v, kBlX, r);
        const int64_t g = r / a.length;
        const float* const slope = a.slope + g * experts;
        const RowStats o = row_stats(x, a.v.inner[kBlX], experts);
        const float inv = 1.0f / o.s;
        float dot = 0.0f;
        for (int e = lane; e < experts; e += 32) dot += slope[e] * expf(to_float(x[e * a.v.inner[kBlX]]) - o.m) * inv;
        dot = warp_sum(dot);
        const double lse = static_cast<double>(o.m) + log(static_cast<double>(o.s));
        const float up = a.z_coef != 0.0 ? static_cast<float>(2.0 * a.z_coef * lse) : 0.0f;
        const float f = static_cast<float>(1.0 / (a.group[g].rows * static_cast<double>(a.groups)));
        for (int e = lane; e < experts; e += 32) {
            const float p = expf(to_float(x[e * a.v.inner[kBlX]]) - o.m) * inv;
            grad[e * a.v.inner[kBlGrad]] = from_float<T>(p * (slope[e] - dot + up) * f);
        }
    }
    allow_dependents();
}

// ------------------------------------------------------------------------------------------------
// host side

struct Layout {
    int64_t runs, run_rows;
    size_t probs, counts, run, slope, group, inner, stats, bytes;
};

// Runs: enough CTAs for the GPU, of at least 32 rows each.
Layout lay_out(int64_t rows, int64_t experts, int64_t groups) {
    Layout l;
    const int64_t length = rows / groups;
    const int64_t want = std::max<int64_t>(1, sm_count() * 4 / groups);
    l.run_rows = std::max<int64_t>(32, (length + want - 1) / want);
    l.runs = std::max<int64_t>(1, (length + l.run_rows - 1) / l.run_rows);
    size_t at = 0;
    auto add = [&](int64_t n, size_t size) {
        const size_t here = at;
        at += (static_cast<size_t>(n) * size + 15) / 16 * 16;
        return here;
    };
    l.probs = add(groups * l.runs * experts, 4);
    l.counts = add(groups * l.runs * experts, 4);
    l.run = add(groups * l.runs, sizeof(BalanceRun));
    l.slope = add(groups * experts, 4);
    l.group = add(groups, sizeof(BalanceGroup));
    l.inner = add(groups * ((experts + 31) / 32), 8);
    l.stats = add(rows, 8);
    l.bytes = at;
    return l;
}

int check_groups(int64_t rows, int64_t groups) {
    if (groups < 1 || groups > kMaxGroups)
        return fail(CTB_ERR_ARGUMENT, "groups must be 1 to " + std::to_string(kMaxGroups));
    if (rows % groups) return fail(CTB_ERR_SHAPE, "the rows do not divide into " + std::to_string(groups) + " groups");
    return CTB_OK;
}

// 4 where rows of logits and gradient start on 4 elements and are whole packs, 1 where their experts are contiguous, else 0.
int pack_of(const BalanceArgs& a) {
    int vec = a.v.cols % 4 ? 1 : 4;
    for (int s : {static_cast<int>(kBlX), static_cast<int>(kBlGrad)}) {
        if (!a.v.ptr[s]) continue;
        if (a.v.inner[s] != 1 && a.v.cols > 1) return 0;
        const uintptr_t bytes = 4 * dtype_size(a.v.dtype[s]);
        if (reinterpret_cast<uintptr_t>(a.v.ptr[s]) % bytes) vec = 1;
        for (int d = 0; d < a.v.rank; ++d)
            if (a.v.stride[s][d] % 4) vec = 1;
    }
    return vec;
}

int wide_shared(const void* kernel, size_t bytes) {
    if (bytes <= 47 * 1024) return CTB_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxExperts * 4 * (kWarps + 1));
    if (e == cudaSuccess) return CTB_OK;
    cudaGetLastError();
    return fail(CTB_ERR_CUDA, std::string("balance loss: ") + cudaGetErrorString(e));
}

template <class T, class R, class G> int run(const BalanceArgs& a, R rows, G grad, unsigned grad_grid, cudaStream_t st) {
    const size_t smem = static_cast<size_t>(a.v.cols) * 4 * (kWarps + 1);
    CTB_CHECK(wide_shared(reinterpret_cast<const void*>(rows), smem));
    launch_dependent(rows, static_cast<unsigned>(a.groups * a.runs), kThreads, smem, st, a);
    count_launch();
    CTB_CHECK(check_launch("balance loss"));
    launch_dependent(balance_join, static_cast<unsigned>(a.groups * a.chunks), kJoinThreads, 0, st, a);
    count_launch();
    CTB_CHECK(check_launch("balance loss"));
    launch_dependent(grad, grad_grid, kThreads, 0, st, a);
    count_launch();
    return check_launch("balance loss");
}

template <class T, int VEC, int L, int NP> int run_held(const BalanceArgs& a, cudaStream_t st) {
    // rows under way: B200, 131072 x 256 float32 64 us with one, 56 with two, 92 with four; 16368 x 60 bfloat16 6.4 with two,
    // 8.8 with four (registers: fewer warps an SM)
    constexpr int kRows = VEC * NP >= 16 ? 1 : 2;
    auto grad = balance_grad_held<T, VEC, L, NP, kRows>;
    // without a gradient the kernel is there for the scalar alone
    if (!a.v.ptr[kBlGrad]) return run<T>(a, balance_rows_held<T, VEC, L, NP, kRows>, balance_grad<T>, 1u, st);
    return run<T>(a, balance_rows_held<T, VEC, L, NP, kRows>, grad, static_cast<unsigned>(a.groups * a.runs), st);
}

template <class T, int VEC> int run_packs(const BalanceArgs& a, cudaStream_t st) {
    const int64_t packs = (a.v.cols + VEC - 1) / VEC;
    if (packs <= 2) return run_held<T, VEC, 2, 1>(a, st);
    if (packs <= 4) return run_held<T, VEC, 4, 1>(a, st);
    if (packs <= 8) return run_held<T, VEC, 8, 1>(a, st);
    if (packs <= 16) return run_held<T, VEC, 16, 1>(a, st);
    if (packs <= 32) return run_held<T, VEC, 32, 1>(a, st);
    if (packs <= 64) return run_held<T, VEC, 32, 2>(a, st);
    if (packs <= 128) return run_held<T, VEC, 32, 4>(a, st);
    if (packs <= 256) return run_held<T, VEC, 32, 8>(a, st);
    return run<T>(a, balance_rows<T>, balance_grad<T>, a.v.ptr[kBlGrad] ? grid_for((a.v.rows + kWarps - 1) / kWarps, 8) : 1u, st);
}

template <class T> int run_any(const BalanceArgs& a, cudaStream_t st) {
    const int vec = pack_of(a);
    if (vec == 4) return run_packs<T, 4>(a, st);
    if (vec == 1) return run_packs<T, 1>(a, st);
    return run<T>(a, balance_rows<T>, balance_grad<T>, a.v.ptr[kBlGrad] ? grid_for((a.v.rows + kWarps - 1) / kWarps, 8) : 1u, st);
}

}  // namespace
}  // namespace ctb

using namespace ctb;

extern "C" {

size_t ctb_balance_loss_scratch_bytes(const ctb_view* logits, int64_t groups) {
    if (!logits || logits->ndim < 1 || logits->ndim > kMaxDims || groups < 1 || groups > kMaxGroups) return 0;
    int64_t rows = 1;
    for (int d = 0; d < logits->ndim - 1; ++d) rows *= logits->shape[d];
    return lay_out(rows, logits->shape[logits->ndim - 1], groups).bytes;
}

int ctb_balance_loss(const ctb_view* logits, const ctb_view* experts, const ctb_view* mask, int64_t groups, double coef,
                     double z_coef, const ctb_view* loss, const ctb_view* counts, const ctb_view* probs,
                     const ctb_view* grad, int32_t* d_status, void* scratch, size_t scratch_bytes, ctb_stream stream) {
    return c_entry([&]() -> int {
        BalanceArgs a{};
        RowBuilder<kBlViews> b;
        CTB_CHECK(b.begin(kBlX, logits, kDtypeMatrix, "logits"));
        if (b.v.cols > kMaxExperts) return fail(CTB_ERR_SHAPE, "more than " + std::to_string(kMaxExperts) + " experts are not supported");
        CTB_CHECK(check_groups(b.v.rows, groups));
        CTB_CHECK(check_row_view(experts, "experts"));
        if (experts->ndim < 1) return fail(CTB_ERR_SHAPE, "experts must be [..., chosen]");
        a.chosen = experts->shape[experts->ndim - 1];
        if (a.chosen < 1) return fail(CTB_ERR_SHAPE, "experts must name at least one expert a row");
        CTB_CHECK(b.matrix(kBlExperts, experts, kDtypeIndex, a.chosen, false, "experts"));
        if (mask) CTB_CHECK(b.operand(kBlMask, mask, kDtypeWeight, "mask"));
        if (!(std::fabs(coef) <= 1e30)) return fail(CTB_ERR_ARGUMENT, "coef must be finite");
        if (!(std::fabs(z_coef) <= 1e30)) return fail(CTB_ERR_ARGUMENT, "z_coef must be finite");
        if (loss) {
            CTB_CHECK(check_row_view(loss, "loss"));
            CTB_CHECK(check_row_dtype(loss, 1u << CTB_FLOAT32, "loss"));
            for (int d = 0; d < loss->ndim; ++d)
                if (loss->shape[d] != 1) return fail(CTB_ERR_SHAPE, "loss must hold one element");
            a.loss = static_cast<float*>(loss->data);
        }
        auto table = [&](const ctb_view* t, int dtype, const char* what, int64_t (&strides)[2]) -> int {
            CTB_CHECK(check_row_view(t, what));
            CTB_CHECK(check_row_dtype(t, 1u << dtype, what));
            if (t->ndim != 2 || t->shape[0] != groups || t->shape[1] != b.v.cols)
                return fail(CTB_ERR_SHAPE, std::string(what) + " must be [groups, experts]");
            strides[0] = t->strides[0];
            strides[1] = t->strides[1];
            return check_written(t, what);
        };
        if (counts) {
            CTB_CHECK(table(counts, CTB_INT64, "counts", a.counts_stride));
            a.counts = static_cast<int64_t*>(counts->data);
        }
        if (probs) {
            CTB_CHECK(table(probs, CTB_FLOAT32, "probs", a.probs_stride));
            a.probs = static_cast<float*>(probs->data);
        }
        if (grad) CTB_CHECK(b.matrix(kBlGrad, grad, 1u << logits->dtype, b.v.cols, true, "grad"));
        CTB_CHECK(check_row_status(d_status));
        const Layout l = lay_out(b.v.rows, b.v.cols, groups);
        CTB_CHECK(check_row_scratch(scratch, scratch_bytes, l.bytes, 16));
        b.finish();
        a.v = b.v;
        a.groups = groups;
        a.length = b.v.rows / groups;
        a.runs = l.runs;
        a.run_rows = l.run_rows;
        a.coef = coef;
        a.z_coef = z_coef;
        a.status = d_status;
        unsigned char* const s = static_cast<unsigned char*>(scratch);
        a.run_probs = reinterpret_cast<float*>(s + l.probs);
        a.run_counts = reinterpret_cast<int32_t*>(s + l.counts);
        a.run = reinterpret_cast<BalanceRun*>(s + l.run);
        a.slope = reinterpret_cast<float*>(s + l.slope);
        a.group = reinterpret_cast<BalanceGroup*>(s + l.group);
        a.inner = reinterpret_cast<double*>(s + l.inner);
        a.row_stats = reinterpret_cast<float2*>(s + l.stats);
        a.chunks = (a.v.cols + 31) / 32;
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        return logits->dtype == CTB_FLOAT32 ? run_any<float>(a, st) : run_any<__nv_bfloat16>(a, st);
    });
}

}  // extern "C"
