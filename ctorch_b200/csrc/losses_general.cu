// losses_general.cu — the losses over logits rows for any layout and type: one CTA a row, element by
// element through the strides, the row read twice (statistics, then gradient; the second read comes
// from L2 unless the row is huge). Rows of unit stride in float32 or bfloat16 have kernels of their
// own (losses_stream.cu, losses_held.cu); this one takes float64, rows that are strided along the
// vocabulary, and losses over rows that those cannot hold: policy loss and distillation of more than 262144 bf16 or
// 131072 float32 logits (8 slices of 64 KiB), distillation with more entries than fit beside three of the slices
// (from 187 a row on, where slices are 64 KiB; losses_held.cu). It is 4 to 8 times slower. B200: policy loss on
// [8192, 131072] bf16 6.3 ms against 0.78 ms; on [2048, 131072] float32 361 us by the other kernel, on [2048, 131080] 1508 us
// by this one; float64 [1024, 131072] 1377 us, 24% of the copy rate.
#include "losses.cuh"

namespace ctb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Sum (or maximum) over the CTA, the same in every thread; the order depends on the thread count alone.
__device__ __forceinline__ double cta_sum(double v, double* sm) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < kWarps; ++w) t += sm[w];
    return t;
}

__device__ __forceinline__ double cta_max(double v, double* sm) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, d));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = sm[0];
    for (int w = 1; w < kWarps; ++w) t = fmax(t, sm[w]);
    return t;
}

template <class Acc> __device__ __forceinline__ void cta_join(const LossArgs& a, RowSum<Acc>& r, Acc* sm) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
        const Acc om = __shfl_xor_sync(0xffffffffu, r.m, d), os = __shfl_xor_sync(0xffffffffu, r.s, d);
        r.join(a, om, os);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
        sm[2 * (threadIdx.x >> 5)] = r.m;
        sm[2 * (threadIdx.x >> 5) + 1] = r.s;
    }
    __syncthreads();
    r.m = sm[0];
    r.s = sm[1];
    for (int w = 1; w < kWarps; ++w) r.join(a, sm[2 * w], sm[2 * w + 1]);
}

template <class T, int OP> __global__ void __launch_bounds__(kThreads) loss_rows_any(LossArgs a) {
    dependent_wait();
    using E = LossElem<T>;
    using Acc = typename E::Acc;
    __shared__ double sm_d[kWarps];
    __shared__ Acc sm_a[2 * kWarps];
    __shared__ double sh[4];
    __shared__ int bad;
    // distill: which columns the teacher names (one bit each), and the gradient on them
    extern __shared__ __align__(16) unsigned char any_smem[];
    Acc* fix = reinterpret_cast<Acc*>(any_smem);
    uint32_t* bits = reinterpret_cast<uint32_t*>(any_smem + (OP == kLossDistill ? sizeof(Acc) * a.top : 0));
    if (OP == kLossDistill) {
        for (int64_t i = threadIdx.x; i < (a.cols + 31) / 32; i += kThreads) bits[i] = 0u;
        __syncthreads();
    }
    const T* X = static_cast<const T*>(a.ptr[kLrX]);
    T* G = static_cast<T*>(a.ptr[kLrGrad]);
    double total = 0.0;  // thread 0
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = X + loss_offset(a, kLrX, row);
        T* g = G ? G + loss_offset(a, kLrGrad, row) : nullptr;
        const double w = row_weight(a, row);
        bool counts = w != 0.0;
        double tm = 0.0, tl = 0.0;  // teacher: maximum of the scaled logits, log-sum-exp
        int64_t t_off = 0, ti_off = 0;
        int entries = 0;
        if (OP == kLossDistill && counts) {
            t_off = loss_offset(a, kLrTeacher, row);
            ti_off = loss_offset(a, kLrTeacherIdx, row);
            double mx = -INFINITY, n = 0.0;
            for (int k = threadIdx.x; k < a.top; k += kThreads) {
                const double z = load_real(a.ptr[kLrTeacher], a.dtype[kLrTeacher], t_off + k * a.t_in) * a.inv_temp;
                mx = fmax(mx, z);
                n += z != -INFINITY;
            }
            tm = cta_max(mx, sm_d);
            entries = static_cast<int>(cta_sum(n, sm_d));
            counts = entries > 0;
            if (a.tail) {
                tl = counts ? row_real(a, kLrTeacherLse, row) : 0.0;
            } else if (counts) {
                double s = 0.0;
                for (int k = threadIdx.x; k < a.top; k += kThreads)
                    s += exp(load_real(a.ptr[kLrTeacher], a.dtype[kLrTeacher], t_off + k * a.t_in) * a.inv_temp - tm);
                tl = tm + log(cta_sum(s, sm_d));
            }
        }
        if (!counts) {
            if (threadIdx.x == 0) put_empty_row(a, row);
            if (g)
                for (int64_t j = threadIdx.x; j < a.cols; j += kThreads) g[j * a.g_in] = E::down(Acc(0));
            __syncthreads();
            continue;
        }
        RowSum<Acc> named;
        named.init();
        if (OP == kLossDistill) {
            if (threadIdx.x == 0) bad = 0;
            __syncthreads();
            for (int k = threadIdx.x; k < a.top; k += kThreads) {
                if (load_real(a.ptr[kLrTeacher], a.dtype[kLrTeacher], t_off + k * a.t_in) == -INFINITY) continue;
                const int64_t j = load_index(a.ptr[kLrTeacherIdx], a.dtype[kLrTeacherIdx], ti_off + k * a.ti_in);
                if (j < 0 || j >= a.cols || (atomicOr(&bits[j >> 5], 1u << (j & 31)) >> (j & 31) & 1u)) {
                    bad = 1;
                    note_bad_index(a, j);
                } else if (a.tail) {
                    named.add(a, E::up(x[j * a.x_in]));
                }
            }
            __syncthreads();
        }
        // pass 1: the row's maximum and sum (tail: of the columns that the teacher does not name)
        RowSum<Acc> r;
        r.init();
        for (int64_t j = threadIdx.x; j < a.cols; j += kThreads) {
            if (OP == kLossDistill && a.tail && (bits[j >> 5] >> (j & 31) & 1u)) continue;
            r.add(a, E::up(x[j * a.x_in]));
        }
        cta_join(a, r, sm_a);
        double s_rest = 0.0, lift = 1.0, below = 0.0;
        Acc at = r.m;  // what the gradient's exponentials are relative to
        if (OP == kLossDistill && a.tail) {
            cta_join(a, named, sm_a);
            s_rest = r.s;
            r.join(a, named.m, named.s);
            lift = at == r.m ? Acc(1) : row_exp(a, at, r.m);
            below = (static_cast<double>(at) - r.m) * a.inv_temp;
            if (at == static_cast<Acc>(-INFINITY)) at = 0;
        }
        r.finish();
        const double m = r.m, s = r.s;
        int64_t target = -1;
        if (OP != kLossDistill) {
            if (threadIdx.x == 0) {
                target = load_index(a.ptr[kLrTarget], a.dtype[kLrTarget], loss_offset(a, kLrTarget, row));
                const bool ok = target >= 0 && target < a.cols;
                if (!ok) note_bad_index(a, target);
                const double logp = ok ? target_logp(a, E::up(x[target * a.x_in]), m, s) : quiet_nan();
                if (OP == kLossToken) {
                    put_row(a, kLrLogp, row, logp);
                    put_row(a, kLrLse, row, m * a.inv_temp + log(s));
                } else {
                    const double d = a.ptr[kLrRef] ? row_real(a, kLrRef, row) - logp : 0.0;
                    const PolicyTerms o = policy_terms(a, w, row_real(a, kLrAdv, row),
                                                       exp(logp - row_real(a, kLrOld, row)), d, expm1(d));
                    put_row(a, kLrLogp, row, logp);
                    put_row(a, kLrRowLoss, row, o.loss);
                    put_row(a, kLrKl, row, o.kl);
                    total += w * o.loss;
                    sh[0] = -o.g / s;
                    sh[1] = -o.g * expm1(logp);  // g (1 - p_t)
                    if (!ok) target = -1;
                }
            }
        } else {
            double cross = 0.0, mass = 0.0;
            for (int k = threadIdx.x; k < a.top; k += kThreads) {
                const double z = load_real(a.ptr[kLrTeacher], a.dtype[kLrTeacher], t_off + k * a.t_in) * a.inv_temp;
                if (z == -INFINITY) continue;
                const double q = exp(z - tl);
                mass += q;
                if (!bad && q != 0.0) {
                    const int64_t j = load_index(a.ptr[kLrTeacherIdx], a.dtype[kLrTeacherIdx], ti_off + k * a.ti_in);
                    cross += q * ((z - tl) - target_logp(a, E::up(x[j * a.x_in]), m, s));
                }
            }
            cross = cta_sum(cross, sm_d);
            mass = cta_sum(mass, sm_d);
            double big_q;
            double slope = distill_slope(a, w, s, s_rest, lift, mass, entries == a.cols, big_q);
            double loss = distill_loss_of(a, s, s_rest, below, cross, mass, entries == a.cols);
            if (bad || !(s > 0.0)) slope = loss = quiet_nan();
            for (int k = threadIdx.x; k < a.top; k += kThreads) {
                const double z = load_real(a.ptr[kLrTeacher], a.dtype[kLrTeacher], t_off + k * a.t_in) * a.inv_temp;
                if (z == -INFINITY || bad) continue;
                const int64_t j = load_index(a.ptr[kLrTeacherIdx], a.dtype[kLrTeacherIdx], ti_off + k * a.ti_in);
                fix[k] = static_cast<Acc>(w * a.inv_temp * (big_q * exp(target_logp(a, E::up(x[j * a.x_in]), m, s)) - exp(z - tl)));
            }
            if (threadIdx.x == 0) {
                put_row(a, kLrRowLoss, row, loss);
                total += w * loss;
                sh[0] = slope;
            }
        }
        if (!g && OP != kLossDistill) {
            __syncthreads();
            continue;
        }
        __syncthreads();
        // pass 2: the gradient, then the named positions
        if (g) {
            const Acc ga = static_cast<Acc>(sh[0]);
            for (int64_t j = threadIdx.x; j < a.cols; j += kThreads)
                g[j * a.g_in] = E::down(ga * row_exp(a, E::up(x[j * a.x_in]), at));
            __syncthreads();
        }
        if (OP == kLossDistill) {
            for (int k = threadIdx.x; k < a.top; k += kThreads) {
                if (load_real(a.ptr[kLrTeacher], a.dtype[kLrTeacher], t_off + k * a.t_in) == -INFINITY) continue;
                const int64_t j = load_index(a.ptr[kLrTeacherIdx], a.dtype[kLrTeacherIdx], ti_off + k * a.ti_in);
                if (j < 0 || j >= a.cols) continue;
                if (g && !bad) g[j * a.g_in] = E::down(fix[k]);
                bits[j >> 5] = 0u;
            }
        } else if (threadIdx.x == 0 && target >= 0) {
            g[target * a.g_in] = E::down(static_cast<Acc>(sh[1]));
        }
        __syncthreads();
    }
    allow_dependents();
    if (a.partials && threadIdx.x == 0) a.partials[blockIdx.x] = total;
}

// The gradient of sum up * logp from what the forward pass kept: with the row's anchor (backward_row)
//     p_j = exp((x_j - at) / T + shift),   g_j = -(up / T) p_j, and (up / T)(1 - p_t) at the target.
template <class T> __global__ void __launch_bounds__(kThreads) loss_backward_any(LossArgs a) {
    dependent_wait();
    using E = LossElem<T>;
    using Acc = typename E::Acc;
    __shared__ BackwardRow<Acc> b;
    const T* X = static_cast<const T*>(a.ptr[kLrX]);
    T* G = static_cast<T*>(a.ptr[kLrGrad]);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = X + loss_offset(a, kLrX, row);
        T* g = G + loss_offset(a, kLrGrad, row);
        if (threadIdx.x == 0) b = backward_row<T>(a, row, x, row_upstream(a, row));
        __syncthreads();
        const BackwardRow<Acc> c = b;
        for (int64_t j = threadIdx.x; j < a.cols; j += kThreads)
            g[j * a.g_in] = E::down(c.zero ? Acc(0) : c.a * row_exp_shifted(a, E::up(x[j * a.x_in]), c.at, c.shift));
        __syncthreads();
        if (threadIdx.x == 0 && c.target >= 0) g[c.target * a.g_in] = E::down(c.at_target);
        __syncthreads();
    }
    allow_dependents();
}

template <class T> int rows_typed(const LossPlan& p, int* ctas, cudaStream_t st) {
    const LossArgs& a = p.args;
    size_t smem = 0;
    if (p.op == kLossDistill) smem = sizeof(typename LossElem<T>::Acc) * a.top + static_cast<size_t>((a.cols + 31) / 32) * 4;
    void (*fn)(LossArgs) = p.op == kLossToken    ? loss_rows_any<T, kLossToken>
                           : p.op == kLossPolicy ? loss_rows_any<T, kLossPolicy>
                                                 : loss_rows_any<T, kLossDistill>;
    // the most that any call may ask for, so that no later call lowers it under a concurrent launch
    constexpr int kMost = kLossMaxTop * sizeof(double) + kLossMaxDistillCols / 8;
    static_assert(kMost <= 227 * 1024, "the bitmap and the entries fit an SM's shared memory");
    if (smem > 48 * 1024 && cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kMost) != cudaSuccess)
        return check_launch("loss rows smem attribute");
    const int per_sm = resident_ctas(reinterpret_cast<const void*>(fn), kThreads, smem);
    int64_t grid = static_cast<int64_t>(sm_count()) * per_sm;
    if (grid > a.rows) grid = a.rows;
    if (grid > kLossMaxCtas) grid = kLossMaxCtas;
    *ctas = static_cast<int>(grid);
    launch_dependent(fn, static_cast<unsigned>(grid), kThreads, smem, st, a);
    count_launch();
    return check_launch("loss rows");
}

template <class T> int backward_typed(const LossArgs& a, cudaStream_t st) {
    void (*fn)(LossArgs) = loss_backward_any<T>;
    const int per_sm = resident_ctas(reinterpret_cast<const void*>(fn), kThreads, 0);
    launch_dependent(fn, grid_for(a.rows, per_sm), kThreads, 0, st, a);
    count_launch();
    return check_launch("loss backward");
}

}  // namespace

int loss_rows_general(const LossPlan& p, int* ctas, cudaStream_t st) {
    switch (p.args.dtype[kLrX]) {
    case CTB_FLOAT32: return rows_typed<float>(p, ctas, st);
    case CTB_BFLOAT16: return rows_typed<__nv_bfloat16>(p, ctas, st);
    default: return rows_typed<double>(p, ctas, st);
    }
}

int loss_backward_general(const LossArgs& a, cudaStream_t st) {
    switch (a.dtype[kLrX]) {
    case CTB_FLOAT32: return backward_typed<float>(a, st);
    case CTB_BFLOAT16: return backward_typed<__nv_bfloat16>(a, st);
    default: return backward_typed<double>(a, st);
    }
}

}  // namespace ctb
