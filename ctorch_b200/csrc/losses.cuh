// losses.cuh — what the loss kernels share: the description of a call (LossArgs), the row's own
// arithmetic, and the reads and writes of the small per-row operands.
//
// Every loss here is a function of one row x[0..V) of logits through z = x / T, the row's maximum m
// and the sum s = sum_j exp(z_j - m / T), so that log-sum-exp is m / T + log s and
// p_j = exp((x_j - m) / T) / s. Its gradient on that row has one form,
//     g_j = A * exp((x_j - m) / T)      for every j but a few named positions,
// with one number A a row; the named positions (the target, the teacher's entries) get their own
// value. The kernels differ in how they get a row past the two passes (statistics, then gradient);
// the functions below turn the statistics into the outputs, A and the named values.
//
// Precision. Elements and their sums are float32 for bfloat16 and float32 logits (float64 for
// float64 ones); differences are taken before scaling, (x_j - m) * (log2(e) / T), so that a row of
// the type's lowest values still gives a uniform p instead of an overflow, and a common offset of
// the logits costs nothing. What happens once a row (logarithms, ratios, the loss) is float64: it
// is a few hundred instructions a row, and the losses subtract numbers that nearly cancel. (Float32 are:
// the joining of a row's partial sums in losses_held.cu and losses_short.cu, and the teacher's probabilities in the former.)
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace ctb {

enum LossOp : int { kLossToken = 0, kLossPolicy = 1, kLossDistill = 2 };

// Per-row operands and results, each addressed by the row's coordinates over the leading dims.
enum LossRow : int {
    kLrX = 0,        // logits (offset of the row's first element)
    kLrGrad,         // gradient row, optional
    kLrTarget,       // int32/int64
    kLrWeight,       // bool/float32/float64, optional; 0 = the row does not count
    kLrOld,          // policy: old log-probability
    kLrAdv,          // policy: advantage
    kLrRef,          // policy: reference log-probability, optional
    kLrTeacher,      // distill: teacher logits (offset of the row's first entry)
    kLrTeacherIdx,   // distill: their vocabulary indices
    kLrTeacherLse,   // distill: the teacher's log-sum-exp, optional
    kLrLogp,         // out (backward: in)
    kLrRowLoss,      // out, optional
    kLrKl,           // out, optional
    kLrLse,          // out, optional (backward: in)
    kLrUp,           // backward: gradient of the log-probability
    kLossRowViews
};

struct LossArgs {
    void* ptr[kLossRowViews];
    int32_t dtype[kLossRowViews];
    int64_t stride[kLossRowViews][kMaxDims];  // over the collapsed leading dims
    int rank;                                 // of the collapsed leading dims, >= 1
    int64_t ext[kMaxDims];                    // their extents
    FastDiv div[kMaxDims];                    // divisors = the extents
    int64_t rows, cols;
    int64_t x_in, g_in;   // strides along the vocabulary
    int64_t t_in, ti_in;  // strides along the teacher's entries
    int top;              // the teacher's entries a row
    void* lists;          // distill: scratch for the teacher's prepared entries (losses_held.cu)
    int tail;             // distill: the mass outside the top entries is one more event
    double temp, inv_temp;
    float c2;             // log2(e) / T
    float c2_down, c2_rest;  // the same rounded down, and what that leaves (positive)
    double scale;         // multiplies every weight
    double clip_lo, clip_hi, kl_coef;
    const void* offsets;  // preference, packed rows: rows before the first offset or from the last one on
    int32_t offsets_dtype;  // belong to no sequence and do not count
    int64_t offsets_end;    // element offset of the last one
    bool up_final;        // preference: kLrUp is 0 in rows that do not count, and says by NaN that no row is valid
    double* partials;     // one weighted loss sum a CTA, optional
    int32_t* status;      // optional: int32 flag, int64 offending index at byte 8; written on error only
    unsigned long long* timeouts;  // device counter of timed-out waits (async_copy.cuh)
};

__device__ __forceinline__ int64_t loss_offset(const LossArgs& a, int view, int64_t row) {
    if (a.rank == 1) return row * a.stride[view][0];
    int64_t off = 0;
    uint64_t r = static_cast<uint64_t>(row);
    for (int d = a.rank - 1; d > 0; --d) {
        uint64_t q, c;
        a.div[d].divmod(r, q, c);
        off += static_cast<int64_t>(c) * a.stride[view][d];
        r = q;
    }
    return off + static_cast<int64_t>(r) * a.stride[view][0];
}

__device__ __forceinline__ double load_real(const void* p, int dt, int64_t off) {
    switch (dt) {
    case CTB_FLOAT32: return static_cast<const float*>(p)[off];
    case CTB_FLOAT64: return static_cast<const double*>(p)[off];
    case CTB_BFLOAT16: return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[off]);
    default: return static_cast<const uint8_t*>(p)[off] ? 1.0 : 0.0;  // bool
    }
}

__device__ __forceinline__ int64_t load_index(const void* p, int dt, int64_t off) {
    return dt == CTB_INT32 ? static_cast<int64_t>(static_cast<const int32_t*>(p)[off])
                           : static_cast<const int64_t*>(p)[off];
}

__device__ __forceinline__ double row_real(const LossArgs& a, int view, int64_t row) {
    return load_real(a.ptr[view], a.dtype[view], loss_offset(a, view, row));
}

// A result of the row, rounded once to its own type (a no-op where the caller did not ask for it).
__device__ __forceinline__ void put_row(const LossArgs& a, int view, int64_t row, double v) {
    if (!a.ptr[view]) return;
    const int64_t off = loss_offset(a, view, row);
    if (a.dtype[view] == CTB_FLOAT32) static_cast<float*>(a.ptr[view])[off] = static_cast<float>(v);
    else static_cast<double*>(a.ptr[view])[off] = v;
}

__device__ __forceinline__ double quiet_nan() { return __longlong_as_double(0x7ff8000000000000ll); }

// The weight of a row, 0 for a row that does not count (its logits and operands are not looked at).
__device__ __forceinline__ double row_weight(const LossArgs& a, int64_t row) {
    if (a.offsets && (row < load_index(a.offsets, a.offsets_dtype, 0) ||
                      row >= load_index(a.offsets, a.offsets_dtype, a.offsets_end)))
        return 0.0;
    return a.ptr[kLrWeight] ? a.scale * row_real(a, kLrWeight, row) : a.scale;
}

// Records an index that points outside the row, or a teacher index that occurs twice. The first one wins.
__device__ __forceinline__ void note_bad_index(const LossArgs& a, int64_t index) {
    if (a.status && atomicCAS(a.status, 0, 1) == 0) *reinterpret_cast<int64_t*>(a.status + 2) = index;
}

// ------------------------------------------------------------------------------------------------
// element types

template <class T> struct LossElem;
template <> struct LossElem<float> {
    using Acc = float;
    __device__ static __forceinline__ float up(float x) { return x; }
    __device__ static __forceinline__ float down(float x) { return x; }
};
template <> struct LossElem<__nv_bfloat16> {
    using Acc = float;
    __device__ static __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
    __device__ static __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};
template <> struct LossElem<double> {
    using Acc = double;
    __device__ static __forceinline__ double up(double x) { return x; }
    __device__ static __forceinline__ double down(double x) { return x; }
};

// 2^t. The float form is the hardware's approximation (relative error below 2^-22), which the
// float32 sums and products around it do not outdo.
__device__ __forceinline__ float exp2_fast(float t) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
    return y;
}

// exp((x - at) / T) for a row's element
__device__ __forceinline__ float row_exp(const LossArgs& a, float x, float at) { return exp2_fast((x - at) * a.c2); }
__device__ __forceinline__ double row_exp(const LossArgs& a, double x, double at) { return exp((x - at) * a.inv_temp); }

// The running maximum and sum of one thread's share of a row: s is relative to m.
template <class Acc> struct RowSum {
    Acc m, s;
    __device__ __forceinline__ void init() {
        m = static_cast<Acc>(-INFINITY);
        s = 0;
    }
    __device__ __forceinline__ void add(const LossArgs& a, Acc x) {
        if (x > m) {
            s = s * row_exp(a, m, x) + 1;  // m = -inf: s is 0 and the factor 0
            m = x;
        } else if (x != static_cast<Acc>(-INFINITY)) {  // NaN comes here too, and stays
            s += row_exp(a, x, m);
        }
    }
    __device__ __forceinline__ void join(const LossArgs& a, Acc om, Acc os) {
        if (om > m) {
            s = s * row_exp(a, m, om) + os;
            m = om;
        } else {
            s += om == m ? os : os * row_exp(a, om, m);
        }
    }
    // Of the whole row: a maximum of +inf has no softmax (x - m is NaN there, 0 elsewhere).
    __device__ __forceinline__ void finish() {
        if (m == static_cast<Acc>(INFINITY)) s = static_cast<Acc>(NAN);
    }
};

// ------------------------------------------------------------------------------------------------
// one row's arithmetic

// Log-probability of a target from the row's statistics: (x_t - m) / T - log s.
__device__ __forceinline__ double target_logp(const LossArgs& a, double xt, double m, double s) {
    return (xt - m) * a.inv_temp - log(s);
}

// The clipped policy loss of one row; with r = exp(logp - old), d = ref - logp and ed = exp(d) - 1,
//     loss = -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl_coef (ed - d)
//     dloss/dlogp = (r A <= clip(r) A ? -r A : 0) - kl_coef ed
// and dlogp/dx_j = (1[j = t] - p_j) / T. Comparisons are written so that a NaN stays one.
struct PolicyTerms {
    double loss, kl;
    double g;  // w / T dloss/dlogp
};

__device__ __forceinline__ PolicyTerms policy_terms(const LossArgs& a, double w, double adv, double r, double d, double ed) {
    const double lo = 1.0 - a.clip_lo, hi = 1.0 + a.clip_hi;
    const double u = r * adv, c = (r < lo ? lo : r > hi ? hi : r) * adv;
    const bool free = !(u > c);
    PolicyTerms t;
    t.loss = free ? -u : -c;
    t.kl = a.ptr[kLrRef] ? ed - d : 0.0;
    double slope = free ? -u : 0.0;
    if (a.kl_coef != 0.0) {
        t.loss += a.kl_coef * t.kl;
        slope -= a.kl_coef * ed;
    }
    t.g = w * slope * a.inv_temp;
    return t;
}

// Outputs of a row that does not count.
__device__ __forceinline__ void put_empty_row(const LossArgs& a, int64_t row) {
    put_row(a, kLrLogp, row, 0.0);
    put_row(a, kLrRowLoss, row, 0.0);
    put_row(a, kLrKl, row, 0.0);
    put_row(a, kLrLse, row, 0.0);
}

// The loss and A of a distilled row, from sums over the teacher's entries: cross = sum q (log q - log p),
// mass = sum q. The columns outside the entries keep a maximum m' and a sum s' of their own, because all of them
// may lie so far below the entries that nothing of them is left in s (masked with a large finite value, or a low
// temperature): lift = exp((m' - m) / T) may be 0 where s' is not. With q' = 1 - mass the rest's share under the
// teacher, log p' = log s' + (m' - m) / T - log s under the student (tail only, else q' = 0) and Q = mass + q',
//     loss    = cross + q' (log q' - log p')
//     dl/dx_j = (Q p_j - q_j) / T on an entry, p_j (Q - q' / p') / T elsewhere,
// the latter as A exp((x_j - m') / T) with A = (Q lift / s - q' / s') / T; renormalised entries have Q = 1.
__device__ __forceinline__ double rest_of_teacher(const LossArgs& a, double mass, bool every_column) {
    if (!a.tail || every_column) return 0.0;
    return mass < 1.0 ? 1.0 - mass : mass == mass ? 0.0 : mass;
}

__device__ __forceinline__ double distill_slope(const LossArgs& a, double w, double s, double s_rest, double lift, double mass,
                                                bool every_column, double& big_q) {
    const double q_rest = rest_of_teacher(a, mass, every_column);
    big_q = a.tail ? mass + q_rest : 1.0;
    if (!a.tail) return w * a.inv_temp * lift / s;
    // with no mass outside the entries every other p_j is 0 and so is its gradient
    return s_rest > 0.0 ? w * a.inv_temp * (big_q * lift / s - q_rest / s_rest) : s_rest == 0.0 ? 0.0 : s_rest;
}

// below = (m' - m) / T
__device__ __forceinline__ double distill_loss_of(const LossArgs& a, double s, double s_rest, double below, double cross, double mass,
                                                  bool every_column) {
    const double q_rest = rest_of_teacher(a, mass, every_column);
    return q_rest == 0.0 ? cross : cross + q_rest * (log(q_rest) - (log(s_rest) + below - log(s)));
}

// What the backward pass needs of a row: p_j = exp((x_j - at) / T) 2^shift, g_j = a p_j.
//
// The forward pass keeps log-sum-exp and the target's log-probability, each rounded to the row type.
// log-sum-exp alone would lose p: at a common offset of the logits of 1000 its float32 rounding is
// 3e-5, an error of every p_j, and at the type's lowest value nothing of p is left in it. The target
// gives a second anchor, x_t - T logp, whose error is the rounding of logp alone, so the row takes the
// anchor with the smaller magnitude. The anchor's own rounding to the element type goes into `a`.
template <class Acc> struct BackwardRow {
    Acc at, shift, a, at_target;
    int64_t target;  // -1: no value of its own
    int zero;        // nothing comes back to this row: its logits are not read
};

__device__ __forceinline__ double row_upstream(const LossArgs& a, int64_t row) {
    return a.up_final || row_weight(a, row) != 0.0 ? row_real(a, kLrUp, row) : 0.0;
}

template <class T>
__device__ __forceinline__ BackwardRow<typename LossElem<T>::Acc> backward_row(const LossArgs& a, int64_t row, const T* x,
                                                                               double up) {
    using Acc = typename LossElem<T>::Acc;
    BackwardRow<Acc> b;
    b.at = b.shift = b.a = b.at_target = 0;
    b.target = -1;
    b.zero = up == 0.0;
    if (b.zero) return b;
    const double g = up * a.inv_temp;
    const int64_t t = load_index(a.ptr[kLrTarget], a.dtype[kLrTarget], loss_offset(a, kLrTarget, row));
    if (t < 0 || t >= a.cols) {
        note_bad_index(a, t);
        b.a = static_cast<Acc>(quiet_nan());
        return b;
    }
    const double xt = LossElem<T>::up(x[t * a.x_in]);
    const double lse = row_real(a, kLrLse, row);
    const double kept = row_real(a, kLrLogp, row);
    const bool by_target = fabs(kept) <= fabs(lse) && kept != -INFINITY;
    const double logp = by_target ? kept : xt * a.inv_temp - lse;
    double rest;  // log2 of what the anchor in the element type leaves over
    if (by_target) {
        b.at = static_cast<Acc>(xt);
        b.shift = static_cast<Acc>(logp * 1.4426950408889634);
        rest = logp * 1.4426950408889634 - static_cast<double>(b.shift);
    } else {
        b.at = static_cast<Acc>(lse * a.temp);
        b.shift = 0;
        rest = (static_cast<double>(b.at) * a.inv_temp - lse) * 1.4426950408889634;
    }
    b.a = static_cast<Acc>(-g * exp2(rest));
    b.at_target = static_cast<Acc>(-g * expm1(logp));
    b.target = t;
    return b;
}

// One multiply-add with log2(e)/T as a float32 and the hardware's 2^t as it is: a p_j of the backward pass is off by up to
// 6e-8 |t| to one side, t the exponent, and 5e-8 more. The forward kernels correct for both (losses_ring.cuh) because
// sequences add their results up; a gradient's elements are rounded one by one.
__device__ __forceinline__ float row_exp_shifted(const LossArgs& a, float x, float at, float shift) {
    return exp2_fast(fmaf(x - at, a.c2, shift));
}
__device__ __forceinline__ double row_exp_shifted(const LossArgs& a, double x, double at, double shift) {
    return exp2((x - at) * a.inv_temp * 1.4426950408889634 + shift);
}

// ------------------------------------------------------------------------------------------------
// host side

struct LossPlan {
    LossArgs args;
    int op = 0;
    bool empty = false;  // no rows
};

constexpr int kLossMaxTop = 2048;                      // the teacher's entries a row
constexpr int64_t kLossMaxDistillCols = int64_t(1) << 20;  // columns of a distilled row (its bitmap)

// CTAs (partial sums) of the forward-and-gradient kernels, whatever the shape: an upper bound, for
// the scratch query.
constexpr int kLossMaxCtas = 148 * 16;

bool loss_stream_fit(const LossArgs& a);                                      // losses_stream.cu
int loss_token_stream(const LossArgs& a, cudaStream_t st);                    // losses_stream.cu
int loss_backward_stream(const LossArgs& a, cudaStream_t st);                 // losses_stream.cu
bool loss_short_fit(const LossPlan& p);                                       // losses_short.cu
bool loss_backward_short_fit(const LossArgs& a);                              // losses_short.cu
int loss_short(const LossPlan& p, int* parts, cudaStream_t st);               // losses_short.cu
int loss_backward_short(const LossArgs& a, cudaStream_t st);                  // losses_short.cu
// *parts: how many partial sums were written; negative when the rows are too long (nothing was launched).
int loss_held(const LossPlan& p, int* parts, cudaStream_t st);                // losses_held.cu
size_t loss_lists_bytes(int64_t rows, int64_t top);                           // losses_held.cu
int loss_rows_general(const LossPlan& p, int* ctas, cudaStream_t st);      // losses_general.cu
int loss_backward_general(const LossArgs& a, cudaStream_t st);              // losses_general.cu

}  // namespace ctb
