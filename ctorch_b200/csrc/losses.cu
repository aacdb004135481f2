// losses.cu — the entry points of the losses over logits rows (include/ctb/ctb.h): checks, the plan of a
// call (its rows and where each operand of a row lies), the choice of kernel, and the two small
// kernels around the row kernels: the sum of the weighted losses, and the preference loss's pairs.
#include <cmath>
#include <exception>
#include <initializer_list>
#include <string>

#include "losses.cuh"
#include "plan.cuh"

namespace ctb {

unsigned long long* wait_timeout_counter();  // async.cu

namespace {

// ------------------------------------------------------------------------------------------------
// kernels

// out = the partial sums added in a fixed order, rounded once (0 when there are none).
__global__ void __launch_bounds__(256) loss_total(const double* partials, int n, void* out, int out_dtype) {
    dependent_wait();
    allow_dependents();
    __shared__ double sm[8];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += partials[i];
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < 8; ++w) t += sm[w];
        if (out_dtype == CTB_FLOAT32) *static_cast<float*>(out) = static_cast<float>(t);
        else *static_cast<double*>(out) = t;
    }
}

constexpr int kPairThreads = 512;

struct PairArgs {
    const double* logp;  // [rows], by row number
    double* up;          // [rows] gradient of each log-probability, optional
    double* weighted;    // [pairs]
    int64_t pairs, length;  // rows a sequence when there are no offsets
    const void* offsets;
    int32_t offsets_dtype;
    int64_t offsets_stride;
    const void* weights;  // [pairs], optional
    int32_t weights_dtype;
    int64_t weights_stride;
    void *pair_loss, *rewards;
    int32_t out_dtype;
    int64_t pair_loss_stride, rewards_stride;
    double scale, beta, smoothing;
    int average;
};

__device__ __forceinline__ void put_real(void* p, int dt, int64_t off, double v) {
    if (!p) return;
    if (dt == CTB_FLOAT32) static_cast<float*>(p)[off] = static_cast<float>(v);
    else static_cast<double*>(p)[off] = v;
}

// CTA p: pair p, sequences p (chosen) and pairs + p (rejected). With R_s = beta times the sum (or mean)
// of logp - ref over the sequence's counted rows and h = R_p - R_{pairs + p},
//     loss = (1 - e) log(1 + exp(-h)) + e log(1 + exp(h))
//     dloss/dR_p = e sigma(h) - (1 - e) sigma(-h) = -dloss/dR_{pairs + p}.
// With offsets, one more CTA clears the rows of no sequence. Reads a few numbers a row, so it is bound by its latency (B200,
// 8 pairs of 2 x 255 rows: about 10 us with the kernel for the total, between the two passes over the logits).
__global__ void __launch_bounds__(kPairThreads) loss_pairs(LossArgs a, PairArgs p) {
    dependent_wait();
    allow_dependents();
    __shared__ double sm[kPairThreads / 32][4];
    __shared__ int bad;
    const int64_t n = 2 * p.pairs;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    auto offset = [&](int64_t s) -> int64_t {
        return p.offsets ? load_index(p.offsets, p.offsets_dtype, s * p.offsets_stride) : s * p.length;
    };
    // offsets that fall, or point outside the rows, would give one row to two sequences: then no pair is valid
    if (p.offsets) {
        for (int64_t s = threadIdx.x; s <= n; s += kPairThreads) {
            const int64_t o = offset(s);
            if (o < 0 || o > a.rows || (s > 0 && o < offset(s - 1))) {
                bad = 1;
                if (blockIdx.x == 0) note_bad_index(a, o);
            }
        }
        __syncthreads();
    }
    if (static_cast<int64_t>(blockIdx.x) == p.pairs) {
        const int64_t first = bad ? a.rows : offset(0), last = bad ? a.rows : offset(n);
        for (int64_t r = threadIdx.x; r < a.rows; r += kPairThreads)
            if (r < first || r >= last) {
                put_row(a, kLrLogp, r, bad ? quiet_nan() : 0.0);
                if (p.up) p.up[r] = bad ? quiet_nan() : 0.0;
            }
        return;
    }
    const int64_t pair = blockIdx.x;
    double w = p.scale;
    if (p.weights) w *= load_real(p.weights, p.weights_dtype, pair * p.weights_stride);
    double reward[2] = {0.0, 0.0}, share[2] = {1.0, 1.0};
    if (bad) {
        if (threadIdx.x == 0) {
            p.weighted[pair] = quiet_nan();
            put_real(p.pair_loss, p.out_dtype, pair * p.pair_loss_stride, quiet_nan());
            put_real(p.rewards, p.out_dtype, pair * p.rewards_stride, quiet_nan());
            put_real(p.rewards, p.out_dtype, (p.pairs + pair) * p.rewards_stride, quiet_nan());
        }
        return;
    }
    auto counts = [&](int64_t r) { return !a.ptr[kLrWeight] || row_real(a, kLrWeight, r) != 0.0; };
    uint32_t seen[2] = {0u, 0u};  // which of this thread's first 32 rows of a side count
    // both sequences' sums and counts, joined together
    double sums[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const int64_t s = side * p.pairs + pair, first = offset(s), last = offset(s + 1);
        int i = 0;
        for (int64_t r = first + threadIdx.x; r < last; r += kPairThreads, ++i) {
            // all loads at once; what a row that does not count holds is not used
            const double lp = p.logp[r], ref = a.ptr[kLrRef] ? row_real(a, kLrRef, r) : 0.0;
            const bool on = counts(r);
            put_row(a, kLrLogp, r, on ? lp : 0.0);
            if (on) {
                sums[2 * side] += lp - ref;
                sums[2 * side + 1] += 1.0;
                if (i < 32) seen[side] |= 1u << i;
            }
        }
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1)
#pragma unroll
        for (int v = 0; v < 4; ++v) sums[v] += __shfl_xor_sync(0xffffffffu, sums[v], d);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int v = 0; v < 4; ++v) sm[threadIdx.x >> 5][v] = sums[v];
    __syncthreads();
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        double sum = 0.0, count = 0.0;
#pragma unroll
        for (int w = 0; w < kPairThreads / 32; ++w) {
            sum += sm[w][2 * side];
            count += sm[w][2 * side + 1];
        }
        if (p.average) share[side] = 1.0 / fmax(count, 1.0);
        reward[side] = p.beta * sum * share[side];
    }
    const double h = reward[0] - reward[1], e = p.smoothing;
    // from t = exp(-|h|): sigma(|h|) = 1 / (1 + t), sigma(-|h|) = t / (1 + t), log(1 + e^h) = max(h, 0) + log(1 + t)
    const double t = exp(-fabs(h)), high = 1.0 / (1.0 + t), low = t * high;
    const double dh = w * p.beta * (h >= 0.0 ? e * high - (1.0 - e) * low : e * low - (1.0 - e) * high);
    if (threadIdx.x == 0) {
        const double rest = log1p(t), loss = (1.0 - e) * (fmax(-h, 0.0) + rest) + e * (fmax(h, 0.0) + rest);
        p.weighted[pair] = w == 0.0 ? 0.0 : w * loss;
        put_real(p.pair_loss, p.out_dtype, pair * p.pair_loss_stride, loss);
        put_real(p.rewards, p.out_dtype, pair * p.rewards_stride, reward[0]);
        put_real(p.rewards, p.out_dtype, (p.pairs + pair) * p.rewards_stride, reward[1]);
    }
    if (!p.up) return;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const int64_t s = side * p.pairs + pair, first = offset(s), last = offset(s + 1);
        const double g = w == 0.0 ? 0.0 : (side ? -dh : dh) * share[side];
        int i = 0;
        for (int64_t r = first + threadIdx.x; r < last; r += kPairThreads, ++i)
            p.up[r] = (i < 32 ? (seen[side] >> i & 1u) != 0u : counts(r)) ? g : 0.0;
    }
}

// ------------------------------------------------------------------------------------------------
// checks and planning

int check_view(const ctb_view* v, const char* what) {
    const std::string name(what);
    if (!v) return fail(CTB_ERR_ARGUMENT, name + ": null view");
    if (v->ndim < 0 || v->ndim > kMaxDims)
        return fail(CTB_ERR_SHAPE, "CUDA backend does not support tensor rank > 16 (got " + std::to_string(v->ndim) + ")");
    if (v->dtype < 0 || v->dtype > CTB_BFLOAT16) return fail(CTB_ERR_ARGUMENT, name + ": malformed view");
    int64_t n = 1;
    for (int d = 0; d < v->ndim; ++d) {
        if (v->shape[d] < 0) return fail(CTB_ERR_ARGUMENT, name + ": malformed view");
        n *= v->shape[d];
    }
    if (!v->data && n != 0) return fail(CTB_ERR_ARGUMENT, name + ": null data pointer");
    return CTB_OK;
}

bool is_index(int dt) { return dt == CTB_INT32 || dt == CTB_INT64; }
bool is_real(int dt) { return dt == CTB_FLOAT32 || dt == CTB_FLOAT64; }

// The type of a row's results: float32, or float64 for float64 logits.
int result_dtype(const ctb_view* logits) { return logits->dtype == CTB_FLOAT64 ? CTB_FLOAT64 : CTB_FLOAT32; }

struct Builder {
    LossPlan plan;
    const ctb_view* logits;
    int lead;  // leading dims

    LossArgs& a() { return plan.args; }

    int begin(const ctb_view* x, double temperature, int32_t* status) {
        plan.args = LossArgs{};
        logits = x;
        if (int rc = check_view(x, "logits")) return rc;
        if (x->dtype != CTB_FLOAT32 && x->dtype != CTB_FLOAT64 && x->dtype != CTB_BFLOAT16)
            return fail(CTB_ERR_DTYPE, std::string("logits must be float32, float64 or bfloat16 (got ") + dtype_name(x->dtype) + ")");
        if (x->ndim < 1) return fail(CTB_ERR_SHAPE, "logits must have at least one dim (the vocabulary, last)");
        lead = x->ndim - 1;
        LossArgs& p = a();
        p.cols = x->shape[lead];
        if (p.cols < 1) return fail(CTB_ERR_SHAPE, "logits rows are empty (a softmax over no entries has no value)");
        if (p.cols >= (int64_t(1) << 31)) return fail(CTB_ERR_SHAPE, "rows of 2^31 or more logits are not supported");
        if (!(temperature > 0.0) || temperature > 1e30 || temperature < 1e-30)
            return fail(CTB_ERR_ARGUMENT, "temperature must be positive (1e-30 to 1e30)");
        p.rows = 1;
        for (int d = 0; d < lead; ++d) p.rows *= x->shape[d];
        plan.empty = p.rows == 0;
        p.temp = temperature;
        p.inv_temp = 1.0 / temperature;
        p.c2 = static_cast<float>(1.4426950408889634 * p.inv_temp);
        const double c2 = 1.4426950408889634 * p.inv_temp;
        float down = static_cast<float>(c2);
        if (static_cast<double>(down) > c2) down = std::nextafterf(down, 0.0f);
        p.c2_down = down;
        p.c2_rest = std::fmax(static_cast<float>(c2 - down), 1.2e-38f);
        p.scale = 1.0;
        p.status = status;
        p.ptr[kLrX] = x->data;
        p.dtype[kLrX] = x->dtype;
        p.x_in = x->strides[lead];
        for (int d = 0; d < lead; ++d) p.stride[kLrX][d] = x->shape[d] == 1 ? 0 : x->strides[d];
        return CTB_OK;
    }

    // An operand of one number a row, right-aligned broadcast over the leading dims.
    int operand(int slot, const ctb_view* v, const char* what) { return strides_of(slot, v, v->ndim, what, true); }

    // A result of one number a row: exactly the leading shape.
    int result(int slot, const ctb_view* v, const char* what) {
        if (!v) return CTB_OK;
        if (int rc = check_view(v, what)) return rc;
        if (v->dtype != result_dtype(logits))
            return fail(CTB_ERR_DTYPE, std::string(what) + " must be " + dtype_name(result_dtype(logits)));
        return strides_of(slot, v, v->ndim, what, false);
    }

    // The gradient: the logits' shape and type; it may be the logits' own view.
    int gradient(const ctb_view* v) {
        if (!v) return CTB_OK;
        if (int rc = check_view(v, "grad")) return rc;
        if (v->dtype != logits->dtype) return fail(CTB_ERR_DTYPE, "the gradient's dtype must equal the logits'");
        if (v->ndim != logits->ndim || v->shape[lead] != a().cols)
            return fail(CTB_ERR_SHAPE, "the gradient's shape must equal the logits'");
        if (int rc = strides_of(kLrGrad, v, lead, "grad", false)) return rc;
        a().g_in = v->strides[lead];
        if (a().cols > 1 && a().g_in == 0) return fail(CTB_ERR_ARGUMENT, "grad must not be a broadcast view");
        return CTB_OK;
    }

    // The teacher's entries: the leading shape (broadcast) and one more dim.
    int entries(int slot, const ctb_view* v, const char* what, int64_t& inner) {
        if (v->ndim < 1) return fail(CTB_ERR_SHAPE, std::string(what) + " must have at least one dim (the entries, last)");
        if (int rc = strides_of(slot, v, v->ndim - 1, what, true)) return rc;
        inner = v->strides[v->ndim - 1];
        return CTB_OK;
    }

    int strides_of(int slot, const ctb_view* v, int ndim, const char* what, bool broadcast) {
        ctb_view head = *v;
        head.ndim = ndim;
        bool same = ndim == lead;
        for (int d = 0; same && d < lead; ++d) same = v->shape[d] == logits->shape[d];
        if ((!broadcast && !same) || !broadcast_strides(head, lead, logits->shape, a().stride[slot]))
            return fail(CTB_ERR_SHAPE, std::string(what) + " does not match the logits' leading dims");
        if (!broadcast)
            for (int d = 0; d < lead; ++d)
                if (v->shape[d] > 1 && v->strides[d] == 0)
                    return fail(CTB_ERR_ARGUMENT, std::string(what) + " must not be a broadcast view");
        a().ptr[slot] = v->data;
        a().dtype[slot] = v->dtype;
        return CTB_OK;
    }

    // Drops leading dims of extent 1 and merges neighbours that chain in every operand.
    void finish() {
        LossArgs& p = a();
        int64_t ext[kMaxDims];
        int r = 0;
        for (int d = 0; d < lead; ++d) {
            if (logits->shape[d] == 1) continue;
            bool chain = r > 0;
            for (int s = 0; chain && s < kLossRowViews; ++s)
                if (p.ptr[s] && p.stride[s][r - 1] != p.stride[s][d] * logits->shape[d]) chain = false;
            const int at = chain ? r - 1 : r;
            for (int s = 0; s < kLossRowViews; ++s) p.stride[s][at] = p.stride[s][d];
            ext[at] = chain ? ext[at] * logits->shape[d] : logits->shape[d];
            r = at + 1;
        }
        if (r == 0) {
            ext[0] = p.rows;
            for (int s = 0; s < kLossRowViews; ++s) p.stride[s][0] = 0;
            r = 1;
        }
        p.rank = r;
        for (int d = 0; d < r; ++d) {
            p.ext[d] = ext[d];
            p.div[d] = FastDiv(static_cast<uint64_t>(ext[d] > 0 ? ext[d] : 1));
        }
        p.timeouts = wait_timeout_counter();
    }
};

int weights_of(Builder& b, const ctb_view* v, double scale, const char* what) {
    b.a().scale = scale;
    if (!v) return CTB_OK;
    if (int rc = check_view(v, what)) return rc;
    if (v->dtype != CTB_BOOL && !is_real(v->dtype))
        return fail(CTB_ERR_DTYPE, std::string(what) + " must be bool, float32 or float64");
    return b.operand(kLrWeight, v, what);
}

int indices_of(Builder& b, int slot, const ctb_view* v, const char* what) {
    if (int rc = check_view(v, what)) return rc;
    if (!is_index(v->dtype)) return fail(CTB_ERR_DTYPE, std::string(what) + " must be int32 or int64");
    return slot == kLrTeacherIdx ? CTB_OK : b.operand(slot, v, what);
}

int reals_of(Builder& b, int slot, const ctb_view* v, const char* what) {
    if (int rc = check_view(v, what)) return rc;
    if (!is_real(v->dtype)) return fail(CTB_ERR_DTYPE, std::string(what) + " must be float32 or float64");
    return b.operand(slot, v, what);
}

int total_of(const Builder& b, const ctb_view* v) {
    if (!v) return CTB_OK;
    if (int rc = check_view(v, "loss")) return rc;
    if (v->dtype != result_dtype(b.logits))
        return fail(CTB_ERR_DTYPE, std::string("loss must be ") + dtype_name(result_dtype(b.logits)));
    for (int d = 0; d < v->ndim; ++d)
        if (v->shape[d] != 1) return fail(CTB_ERR_SHAPE, "loss must hold one element");
    return CTB_OK;
}

size_t partial_bytes(int64_t rows) {
    return static_cast<size_t>(rows < kLossMaxCtas ? rows : kLossMaxCtas) * sizeof(double);
}

size_t distill_bytes(int64_t rows, int64_t top) { return partial_bytes(rows) + loss_lists_bytes(rows, top); }

size_t preference_bytes(int64_t rows, int64_t pairs) {
    return static_cast<size_t>(3 * rows + pairs) * sizeof(double);
}

int check_scratch(const void* scratch, size_t have, size_t need) {
    if (need && (!scratch || have < need))
        return fail(CTB_ERR_SCRATCH, "scratch buffer too small: need " + std::to_string(need) + " bytes");
    if (reinterpret_cast<uintptr_t>(scratch) % sizeof(double))
        return fail(CTB_ERR_ARGUMENT, "scratch must start on an 8-byte boundary");
    return CTB_OK;
}

int check_status(const int32_t* status) {
    return reinterpret_cast<uintptr_t>(status) % 8 ? fail(CTB_ERR_ARGUMENT, "the status must start on an 8-byte boundary")
                                                   : CTB_OK;
}

int run_rows(const LossPlan& p, int* parts, cudaStream_t st) {
    if (loss_short_fit(p)) return loss_short(p, parts, st);
    if (loss_stream_fit(p.args)) {
        if (p.op == kLossToken) return loss_token_stream(p.args, st);
        if (int rc = loss_held(p, parts, st)) return rc;
        if (*parts >= 0) return CTB_OK;
    }
    return loss_rows_general(p, parts, st);
}

int run_backward(const LossArgs& a, cudaStream_t st) {
    if (loss_backward_short_fit(a)) return loss_backward_short(a, st);
    return loss_stream_fit(a) ? loss_backward_stream(a, st) : loss_backward_general(a, st);
}

int run_total(const double* partials, int n, const ctb_view* out, cudaStream_t st) {
    launch_dependent(loss_total, 1, 256, 0, st, partials, n, out->data, out->dtype);
    count_launch();
    return check_launch("loss total");
}

// Rows with their weighted sum: the forward-and-gradient kernels.
int run_loss(Builder& b, const ctb_view* loss, void* scratch, size_t scratch_bytes, cudaStream_t st) {
    const bool lists = b.plan.op == kLossDistill;
    const size_t need = lists ? distill_bytes(b.a().rows, b.a().top) : loss ? partial_bytes(b.a().rows) : 0;
    if (int rc = check_scratch(scratch, scratch_bytes, need)) return rc;
    b.finish();
    if (lists) b.a().lists = static_cast<unsigned char*>(scratch) + partial_bytes(b.a().rows);
    b.a().partials = loss ? static_cast<double*>(scratch) : nullptr;
    int ctas = 0;
    if (!b.plan.empty)
        if (int rc = run_rows(b.plan, &ctas, st)) return rc;
    return loss ? run_total(static_cast<const double*>(scratch), ctas, loss, st) : CTB_OK;
}

template <class F> int guarded(F&& f) {
    try {
        fail(CTB_OK, "");
        return f();
    } catch (const std::exception& e) {
        return fail(CTB_ERR_CUDA, std::string("internal error: ") + e.what());
    } catch (...) {
        return fail(CTB_ERR_CUDA, "internal error");
    }
}

#define CTB_TRY(call)                    \
    do {                                 \
        if (int rc_ = (call)) return rc_; \
    } while (0)

}  // namespace
}  // namespace ctb

using namespace ctb;

extern "C" {

int ctb_token_logprobs(const ctb_view* logits, const ctb_view* targets, const ctb_view* mask, double temperature,
                       const ctb_view* logprobs, const ctb_view* lse, int32_t* d_status, ctb_stream stream) {
    return guarded([&]() -> int {
        Builder b;
        CTB_TRY(b.begin(logits, temperature, d_status));
        CTB_TRY(indices_of(b, kLrTarget, targets, "targets"));
        CTB_TRY(weights_of(b, mask, 1.0, "mask"));
        CTB_TRY(check_view(logprobs, "logprobs"));
        CTB_TRY(b.result(kLrLogp, logprobs, "logprobs"));
        CTB_TRY(b.result(kLrLse, lse, "lse"));
        CTB_TRY(check_status(d_status));
        b.finish();
        b.plan.op = kLossToken;
        int ctas = 0;
        return b.plan.empty ? CTB_OK : run_rows(b.plan, &ctas, static_cast<cudaStream_t>(stream));
    });
}

int ctb_token_logprobs_backward(const ctb_view* grad_logprobs, const ctb_view* logits, const ctb_view* targets,
                                const ctb_view* logprobs, const ctb_view* lse, const ctb_view* mask,
                                double temperature, const ctb_view* grad, int32_t* d_status, ctb_stream stream) {
    return guarded([&]() -> int {
        Builder b;
        CTB_TRY(b.begin(logits, temperature, d_status));
        CTB_TRY(reals_of(b, kLrUp, grad_logprobs, "grad_logprobs"));
        CTB_TRY(indices_of(b, kLrTarget, targets, "targets"));
        CTB_TRY(check_view(logprobs, "logprobs"));
        CTB_TRY(check_view(lse, "lse"));
        CTB_TRY(b.result(kLrLogp, logprobs, "logprobs"));
        CTB_TRY(b.result(kLrLse, lse, "lse"));
        CTB_TRY(weights_of(b, mask, 1.0, "mask"));
        CTB_TRY(check_view(grad, "grad"));
        CTB_TRY(b.gradient(grad));
        CTB_TRY(check_status(d_status));
        b.finish();
        return b.plan.empty ? CTB_OK : run_backward(b.a(), static_cast<cudaStream_t>(stream));
    });
}

size_t ctb_loss_scratch_bytes(const ctb_view* logits, int64_t pairs, int64_t top) {
    if (!logits || logits->ndim < 1 || logits->ndim > kMaxDims || pairs < 0 || top < 0 || top > kLossMaxTop) return 0;
    int64_t rows = 1;
    for (int d = 0; d < logits->ndim - 1; ++d) rows *= logits->shape[d];
    return pairs ? preference_bytes(rows, pairs) : top ? distill_bytes(rows, top) : partial_bytes(rows);
}

int ctb_distill_loss(const ctb_view* logits, const ctb_view* teacher_logits, const ctb_view* teacher_indices,
                     const ctb_view* teacher_lse, const ctb_view* weights, double weight_scale, double temperature,
                     const ctb_view* loss, const ctb_view* row_loss, const ctb_view* grad, int32_t* d_status,
                     void* scratch, size_t scratch_bytes, ctb_stream stream) {
    return guarded([&]() -> int {
        Builder b;
        CTB_TRY(b.begin(logits, temperature, d_status));
        LossArgs& a = b.a();
        CTB_TRY(check_view(teacher_logits, "teacher_logits"));
        if (!is_real(teacher_logits->dtype) && teacher_logits->dtype != CTB_BFLOAT16)
            return fail(CTB_ERR_DTYPE, "teacher_logits must be float32, float64 or bfloat16");
        CTB_TRY(b.entries(kLrTeacher, teacher_logits, "teacher_logits", a.t_in));
        CTB_TRY(indices_of(b, kLrTeacherIdx, teacher_indices, "teacher_indices"));
        CTB_TRY(b.entries(kLrTeacherIdx, teacher_indices, "teacher_indices", a.ti_in));
        const int64_t top = teacher_logits->shape[teacher_logits->ndim - 1];
        if (teacher_indices->shape[teacher_indices->ndim - 1] != top)
            return fail(CTB_ERR_SHAPE, "teacher_logits and teacher_indices must have the same number of entries");
        if (top < 1 || top > kLossMaxTop)
            return fail(CTB_ERR_SHAPE, "1 to " + std::to_string(kLossMaxTop) + " teacher entries a row are supported (got " +
                                           std::to_string(top) + ")");
        if (a.cols > kLossMaxDistillCols)
            return fail(CTB_ERR_SHAPE, "distilled rows of more than " + std::to_string(kLossMaxDistillCols) +
                                           " logits are not supported");
        a.top = static_cast<int>(top);
        if (teacher_lse) CTB_TRY(reals_of(b, kLrTeacherLse, teacher_lse, "teacher_lse"));
        a.tail = teacher_lse != nullptr;
        CTB_TRY(weights_of(b, weights, weight_scale, "weights"));
        CTB_TRY(total_of(b, loss));
        CTB_TRY(b.result(kLrRowLoss, row_loss, "row_loss"));
        CTB_TRY(b.gradient(grad));
        CTB_TRY(check_status(d_status));
        b.plan.op = kLossDistill;
        return run_loss(b, loss, scratch, scratch_bytes, static_cast<cudaStream_t>(stream));
    });
}

int ctb_policy_loss(const ctb_view* logits, const ctb_view* targets, const ctb_view* old_logprobs,
                    const ctb_view* advantages, const ctb_view* ref_logprobs, const ctb_view* weights,
                    double weight_scale, double clip_low, double clip_high, double kl_coef, double temperature,
                    const ctb_view* loss, const ctb_view* row_loss, const ctb_view* logprobs, const ctb_view* kl,
                    const ctb_view* grad, int32_t* d_status, void* scratch, size_t scratch_bytes, ctb_stream stream) {
    return guarded([&]() -> int {
        Builder b;
        CTB_TRY(b.begin(logits, temperature, d_status));
        LossArgs& a = b.a();
        CTB_TRY(indices_of(b, kLrTarget, targets, "targets"));
        CTB_TRY(reals_of(b, kLrOld, old_logprobs, "old_logprobs"));
        CTB_TRY(reals_of(b, kLrAdv, advantages, "advantages"));
        if (ref_logprobs) CTB_TRY(reals_of(b, kLrRef, ref_logprobs, "ref_logprobs"));
        if (!(clip_low >= 0.0 && clip_low <= 1.0)) return fail(CTB_ERR_ARGUMENT, "clip_low must be in [0, 1]");
        if (!(clip_high >= 0.0)) return fail(CTB_ERR_ARGUMENT, "clip_high must not be negative");
        if (!(kl_coef >= 0.0) || kl_coef > 1e300) return fail(CTB_ERR_ARGUMENT, "kl_coef must be finite and not negative");
        if (kl_coef != 0.0 && !ref_logprobs) return fail(CTB_ERR_ARGUMENT, "kl_coef needs ref_logprobs");
        a.clip_lo = clip_low;
        a.clip_hi = clip_high;
        a.kl_coef = kl_coef;
        CTB_TRY(weights_of(b, weights, weight_scale, "weights"));
        CTB_TRY(total_of(b, loss));
        CTB_TRY(b.result(kLrRowLoss, row_loss, "row_loss"));
        CTB_TRY(b.result(kLrLogp, logprobs, "logprobs"));
        CTB_TRY(b.result(kLrKl, kl, "kl"));
        CTB_TRY(b.gradient(grad));
        CTB_TRY(check_status(d_status));
        b.plan.op = kLossPolicy;
        return run_loss(b, loss, scratch, scratch_bytes, static_cast<cudaStream_t>(stream));
    });
}

int ctb_preference_loss(const ctb_view* logits, const ctb_view* targets, int64_t pairs, const ctb_view* offsets,
                        const ctb_view* ref_logprobs, const ctb_view* mask, const ctb_view* weights,
                        double weight_scale, double beta, double label_smoothing, int average, const ctb_view* loss,
                        const ctb_view* pair_loss, const ctb_view* rewards, const ctb_view* logprobs,
                        const ctb_view* grad, int32_t* d_status, void* scratch, size_t scratch_bytes,
                        ctb_stream stream) {
    return guarded([&]() -> int {
        Builder b;
        CTB_TRY(b.begin(logits, 1.0, d_status));
        LossArgs& a = b.a();
        CTB_TRY(indices_of(b, kLrTarget, targets, "targets"));
        if (pairs < 1 || pairs > (int64_t(1) << 30)) return fail(CTB_ERR_ARGUMENT, "pairs must be at least 1");
        if (offsets) {
            CTB_TRY(check_view(offsets, "offsets"));
            if (!is_index(offsets->dtype)) return fail(CTB_ERR_DTYPE, "offsets must be int32 or int64");
            if (offsets->ndim != 1 || offsets->shape[0] != 2 * pairs + 1)
                return fail(CTB_ERR_SHAPE, "offsets must be [2 * pairs + 1]");
            if (logits->ndim != 2) return fail(CTB_ERR_SHAPE, "packed sequences need [rows, vocabulary] logits");
        } else if (a.rows % (2 * pairs)) {
            return fail(CTB_ERR_SHAPE, "the logits' rows do not divide into " + std::to_string(2 * pairs) + " sequences");
        }
        if (ref_logprobs) CTB_TRY(reals_of(b, kLrRef, ref_logprobs, "ref_logprobs"));
        CTB_TRY(weights_of(b, mask, 1.0, "mask"));
        if (!(beta > 0.0) || beta > 1e300) return fail(CTB_ERR_ARGUMENT, "beta must be positive and finite");
        if (!(label_smoothing >= 0.0 && label_smoothing < 0.5))
            return fail(CTB_ERR_ARGUMENT, "label_smoothing must be in [0, 0.5)");
        CTB_TRY(total_of(b, loss));
        PairArgs p{};
        const int rt = result_dtype(logits);
        auto vector_of = [&](const ctb_view* v, int64_t n, const char* what) -> int {
            CTB_TRY(check_view(v, what));
            if (v->ndim != 1 || v->shape[0] != n)
                return fail(CTB_ERR_SHAPE, std::string(what) + " must be [" + std::to_string(n) + "]");
            return CTB_OK;
        };
        if (weights) {
            CTB_TRY(vector_of(weights, pairs, "weights"));
            if (weights->dtype != CTB_BOOL && !is_real(weights->dtype))
                return fail(CTB_ERR_DTYPE, "weights must be bool, float32 or float64");
            p.weights = weights->data;
            p.weights_dtype = weights->dtype;
            p.weights_stride = weights->strides[0];
        }
        for (const ctb_view* v : {pair_loss, rewards}) {
            if (!v) continue;
            const char* what = v == rewards ? "rewards" : "pair_loss";
            CTB_TRY(vector_of(v, v == rewards ? 2 * pairs : pairs, what));
            if (v->dtype != rt) return fail(CTB_ERR_DTYPE, std::string(what) + " must be " + dtype_name(rt));
            if (v->shape[0] > 1 && v->strides[0] == 0)
                return fail(CTB_ERR_ARGUMENT, std::string(what) + " must not be a broadcast view");
        }
        CTB_TRY(b.result(kLrLogp, logprobs, "logprobs"));
        CTB_TRY(b.gradient(grad));
        CTB_TRY(check_status(d_status));
        CTB_TRY(check_scratch(scratch, scratch_bytes, preference_bytes(a.rows, pairs)));
        b.finish();
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (offsets) {
            a.offsets = p.offsets = offsets->data;
            a.offsets_dtype = p.offsets_dtype = offsets->dtype;
            p.offsets_stride = offsets->strides[0];
            a.offsets_end = 2 * pairs * offsets->strides[0];
        }
        double* const logp = static_cast<double*>(scratch);
        double* const lse = logp + a.rows;
        double* const up = lse + a.rows;
        // 1: log-probabilities, in float64 and by row number. A sequence's sum is the difference of long sums
        // of them, so they are not rounded on the way.
        LossPlan forward = b.plan;
        forward.op = kLossToken;
        forward.args.ptr[kLrGrad] = nullptr;
        auto by_row = [&](LossArgs& f, int slot, double* to) {
            f.ptr[slot] = to;
            f.dtype[slot] = CTB_FLOAT64;
            int64_t step = 1;
            for (int d = f.rank - 1; d >= 0; --d) {
                f.stride[slot][d] = step;
                step *= f.ext[d];
            }
        };
        by_row(forward.args, kLrLogp, logp);
        by_row(forward.args, kLrLse, lse);
        int ctas = 0;
        if (!b.plan.empty) CTB_TRY(run_rows(forward, &ctas, st));
        // 2: the pairs
        p.logp = logp;
        p.up = grad ? up : nullptr;
        p.weighted = up + a.rows;
        p.pairs = pairs;
        p.length = a.rows / (2 * pairs);
        p.pair_loss = pair_loss ? pair_loss->data : nullptr;
        p.pair_loss_stride = pair_loss ? pair_loss->strides[0] : 0;
        p.rewards = rewards ? rewards->data : nullptr;
        p.rewards_stride = rewards ? rewards->strides[0] : 0;
        p.out_dtype = rt;
        p.scale = weight_scale;
        p.beta = beta;
        p.smoothing = label_smoothing;
        p.average = average;
        launch_dependent(loss_pairs, static_cast<unsigned>(pairs + (offsets ? 1 : 0)), kPairThreads, 0, st, a, p);
        count_launch();
        CTB_TRY(check_launch("loss pairs"));
        // 3: the gradient
        if (grad && !b.plan.empty) {
            LossArgs back = a;
            by_row(back, kLrLogp, logp);
            by_row(back, kLrLse, lse);
            by_row(back, kLrUp, up);
            back.up_final = true;
            CTB_TRY(run_backward(back, st));
        }
        return loss ? run_total(p.weighted, static_cast<int>(pairs), loss, st) : CTB_OK;
    });
}

}  // extern "C"
