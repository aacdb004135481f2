// losses_held.cu — the policy and distillation losses over rows of unit stride (float32, bfloat16): each logit is
// read from memory once, and its gradient is written from the same pass.
//
// A row belongs to a thread-block cluster of C CTAs (C = 1 for rows that one CTA can hold), a CTA to a
// contiguous slice of the row's 16-byte packs. Clusters are persistent: cluster c takes rows c, c + n,
// c + 2n, ... In a CTA
//   * the producer warp copies the slices of the coming rows into a ring of shared-memory stages, one stage a
//     row (bulk asynchronous copies), and reads the rows' small operands, 32 rows at a time;
//   * the consumer warps fold a slice into each warp's (m_w, sum of exp((x - m_w) / T)) and send it to every CTA
//     of the cluster (st.async into its mailbox, completion counted on its mbarrier: no cluster-wide barrier);
//   * the row warp joins the C * W partial sums and publishes the row's coefficient A;
//   * the consumers write g = A exp((x - m) / T) from the stage to memory and give the stage back.
// The consumers fold up to three rows ahead of the row that they write, so that the exchange of a row (0.2 us) and the
// row warp's arithmetic (0.7 us) pass while they work. What a row's losses need is kept by the row warp and worked
// out for 32 rows at once, a lane a row.
//
// Each logit takes two exponentials, one for the sum and one for the gradient, both from the stage. Keeping the first
// in registers instead halves the use of the exponential unit, but that code is unrolled through and through (the
// warps wait for instructions) and slices are half as wide. Policy loss on [8192, 131072] bf16, B200: 962 us with
// exponentials kept (two CTAs of eight warps an SM), 1018 us kept for two rows, 780 us this way. Writing the gradient
// into the stage and from there by bulk copies took 790 us (distillation 715 us against 627 us: the stage is given
// back later). Measured: policy loss [8192, 131072] bf16 780 us (90% of the rows count; 5.2 TB/s), [3001, 50021] bf16 with
// rows padded to 50048 (85%) 136 us; distillation [4096, 131072] bf16 with 128 entries a row and a tail 530 us. On
// wide slices nothing is used up (80% of the copy rate; the exponential pipe and instruction issue a little over half busy),
// but of 64 KiB stages there are three: one is folded, one written, one loads. Narrow ones are bound by what every row
// costs whatever its length (about 2 us a cluster).
//
// Distillation. The teacher's entries are prepared by a kernel of their own (loss_lists), a warp a row: q and the
// sums that need no logit. Two list warps, in turns, join them with the rows: read the named logits, and put -inf in
// their place in the landed stage, so that the consumers' sum is that of the others (1 - sum p would lose it to
// cancellation) and their gradient there 0; when the consumers have written the row, the list warp writes the named
// elements' own gradient over that. With a 64 KiB slice three stages fit, and beside them the entries only up to 186 a
// row: more go to losses_general.cu ([4096, 131072] bf16 with 186 entries 617 us, with 187 3.9 ms; [4096, 32768] 182 and
// 790 us). On narrower slices many entries leave an SM one CTA of few warps ([8192, 6144] with 64 entries 104 us, with 256
// 572 us; the sizes below were chosen for the policy loss).
#include <string>

#include "losses_ring.cuh"

namespace ctb {

namespace {

// ------------------------------------------------------------------------------------------------
// the teacher's entries

// Of one row's entries, by loss_lists.
struct ListSums {
    double q_logq, mass;  // sum q log q, sum q
    int count, bad;       // entries that are not padding; an index outside the row
};

// Scratch of a distillation: [rows] ListSums, then q and columns [rows, top].
__host__ __device__ inline size_t list_sums_bytes(int64_t rows) { return static_cast<size_t>(rows) * sizeof(ListSums); }

// q_k = exp(z_k - base) * weight with z = teacher / T: renormalised over the entries (base their maximum, weight
// 1 / sum), or with the teacher's own log-sum-exp. Sums are float64; q itself is kept in float32, half the bytes a list
// warp fetches, and so sum q x and with it the loss carry up to 2^-24 sum q |x - max| / T (a KL of nearly 0 is not exact
// below that; the row's float32 sum leaves it no better). A warp a row; a few numbers a row, bound by latency
// (a few microseconds, the first of them beside the kernel before it).
__global__ void __launch_bounds__(256) loss_lists(const __grid_constant__ LossArgs a) {
    dependent_wait();
    allow_dependents();
    const int lane = threadIdx.x & 31;
    ListSums* sums = static_cast<ListSums*>(a.lists);
    float* qs = reinterpret_cast<float*>(static_cast<unsigned char*>(a.lists) + list_sums_bytes(a.rows));
    int* columns = reinterpret_cast<int*>(qs + a.rows * a.top);
    for (int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; row < a.rows;
         row += (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5) {
        ListSums out;
        out.q_logq = out.mass = 0.0;
        out.count = out.bad = 0;
        if (row_weight(a, row) != 0.0) {
            const int64_t t_off = loss_offset(a, kLrTeacher, row), ti_off = loss_offset(a, kLrTeacherIdx, row);
            auto scaled = [&](int k) {
                return load_real(a.ptr[kLrTeacher], a.dtype[kLrTeacher], t_off + k * a.t_in) * a.inv_temp;
            };
            double base = -INFINITY;
            int count = 0;
            for (int k = lane; k < a.top; k += 32) {
                const double z = scaled(k);
                base = fmax(base, z);
                count += z != -INFINITY;
            }
            out.count = __reduce_add_sync(0xffffffffu, count);
            if (out.count) {
                double log_sum = 0.0, weight = 1.0;
                if (a.tail) {
                    base = row_real(a, kLrTeacherLse, row);
                } else {
#pragma unroll
                    for (int d = 16; d >= 1; d >>= 1) base = fmax(base, __shfl_xor_sync(0xffffffffu, base, d));
                    double sum = 0.0;
                    for (int k = lane; k < a.top; k += 32) sum += exp(scaled(k) - base);
                    sum = warp_sum(sum);
                    weight = 1.0 / sum;
                    log_sum = log(sum);
                }
                int bad = 0;
                for (int k = lane; k < a.top; k += 32) {
                    const double z = scaled(k), q = z == -INFINITY ? 0.0 : weight * exp(z - base);
                    int j = -1;
                    if (z != -INFINITY) {
                        const int64_t at = load_index(a.ptr[kLrTeacherIdx], a.dtype[kLrTeacherIdx], ti_off + k * a.ti_in);
                        if (at >= 0 && at < a.cols) {
                            j = static_cast<int>(at);
                        } else {
                            bad = 1;
                            note_bad_index(a, at);
                        }
                    }
                    if (q != 0.0) {  // NaN too
                        out.mass += q;
                        out.q_logq += q * (z - base - log_sum);
                    }
                    qs[row * a.top + k] = static_cast<float>(q);
                    columns[row * a.top + k] = j;
                }
                out.mass = warp_sum(out.mass);
                out.q_logq = warp_sum(out.q_logq);
                out.bad = __any_sync(0xffffffffu, bad);
            }
        }
        if (lane == 0) sums[row] = out;
    }
}

// ------------------------------------------------------------------------------------------------
// shared memory

// A row's operands, read before its logits.
struct RowMeta {
    double w;                 // 0: the row does not count
    double xt, adv;           // policy: the target's logit
    double old, ref;
    double exp_old, exp_ref;  // exp(-old), exp(ref)
    ListSums list;            // distill
    long long row;
    const void* src;          // this CTA's slice of the logits
    void* out;                // of the gradient, where its rows are aligned like the logits' (else null)
    void* grad;               // the gradient's row, null without one
    int count;                // packs of the slice
    int body;                 // column of the slice's first element
    int target;               // column of the target, -1: bad
    uint32_t edges;           // which of the 16 elements around the whole packs there are (CTA 0 of the cluster)
    int behind;               // column of the first element behind the whole packs
    int pad_;
};

// What joining a list with the row's logits gives the row warp.
struct ListInfo {
    double q_x, ref;  // sum of q (x - ref)
    double named;     // sum of exp((x - x_max) / T)
    float x_max;
    uint32_t edge_named;  // the list warp's own
};

struct Coef {
    float a, m;       // of every element but the named ones: a exp((x - m) / T)
    float named;      // policy: the target's gradient; distill: the row's maximum, for the entries' own
    float p_scale;    // distill: Q / s
};

constexpr int kMaxDepth = 3;               // rows folded before the oldest of them is written
constexpr int kSides = 2 * kMaxDepth + 2;  // rows whose sums and lists may be in use at once
constexpr int kMaxRing = 8;
static_assert(kMaxRing <= kSides, "a row waits for the row before in its stage by its side");
constexpr int kAhead = 4;      // entries a lane of a list warp fetches a row ahead
constexpr int kListWarps = 2;  // they take turns

// What lies behind the ring's stages.
template <int W> struct Shared {
    uint64_t mail[kSides][kMaxCluster * W];
    RowMeta meta[2][kBatch];
    float edge[2][kBatch][16];
    ListInfo list[kSides];
    Coef coef[kMaxDepth + 1];
    uint64_t full[kMaxRing], empty[kMaxRing];
    uint64_t meta_full[2], meta_empty[2];
    uint64_t list_full[kSides], done[kSides];
    uint64_t mail_full[kSides], coef_full[kMaxDepth + 1];
};

// Bytes behind the stages: Shared, then for distillation, for each list warp, a bit a column of the slice (a byte a
// pack) and the named logits of the rows in use.
template <int W> __host__ __device__ constexpr size_t bits_at() { return (sizeof(Shared<W>) + 15) / 16 * 16; }
__host__ __device__ inline size_t bits_bytes(int slice_packs) { return (slice_packs + 15) / 16 * 16; }
template <int W> __host__ __device__ inline size_t behind_bytes(int op, int top, int slice_packs) {
    return op == kLossDistill ? bits_at<W>() + kListWarps * bits_bytes(slice_packs) + static_cast<size_t>(kSides) * top * 4
                              : sizeof(Shared<W>);
}
template <int OP, int W> __host__ __device__ constexpr int held_threads() { return (W + 2 + (OP == kLossDistill ? kListWarps : 0)) * 32; }

// A position in the ring, advanced a row at a time.
struct Ring {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next(int stages) {
        if (++slot == stages) {
            slot = 0;
            phase ^= 1u;
        }
    }
};

// ------------------------------------------------------------------------------------------------

// W consumer warps; `stages` stages of `stage_bytes`.
template <class T, int OP, int W, int PER_SM>
__global__ void __launch_bounds__(held_threads<OP, W>(), PER_SM)
    loss_held_kernel(const __grid_constant__ LossArgs a, int stages, int stage_bytes, int slice_packs, int depth) {
    using P = PackOf<T>;
    using S = Shared<W>;
    constexpr int VE = P::VE, kCons = W * 32;
    extern __shared__ __align__(128) unsigned char sm[];
    S& sh = *reinterpret_cast<S*>(sm + static_cast<size_t>(stages) * stage_bytes);
    unsigned char* const behind = reinterpret_cast<unsigned char*>(&sh);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank()), size = static_cast<int>(cluster_size());
    const uint32_t mail_bytes = static_cast<uint32_t>(size) * W * 8;
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], W);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.meta_full[i], 1);
            mbar_init(&sh.meta_empty[i], W + 1 + (OP == kLossDistill ? kListWarps : 0));
        }
        for (int i = 0; i <= kMaxDepth; ++i) mbar_init(&sh.coef_full[i], 1);
        for (int i = 0; i < kSides; ++i) {
            mbar_init(&sh.list_full[i], 1);
            mbar_init(&sh.done[i], W);
            mbar_init(&sh.mail_full[i], 1);
        }
        mbar_fence_init();
        for (int i = 0; i < kSides; ++i) mbar_arrive_expect_tx(&sh.mail_full[i], mail_bytes);
    }
    __syncthreads();
    cluster_sync();
    dependent_wait();  // the previous kernel in the stream has completed and its writes are visible

    const int64_t cluster = blockIdx.x / size, clusters = gridDim.x / size;
    const int rows = static_cast<int>(cluster < a.rows ? (a.rows - cluster + clusters - 1) / clusters : 0);
    const float* list_q = nullptr;
    const int* list_col = nullptr;
    if (OP == kLossDistill) {
        list_q = reinterpret_cast<const float*>(static_cast<const unsigned char*>(a.lists) + list_sums_bytes(a.rows));
        list_col = reinterpret_cast<const int*>(list_q + a.rows * a.top);
    }
    bool ok = true;

    if (warp == W) {
        // ---- producer
        int prepared = 0;    // batches whose operands have been read
        uint32_t live = 0;   // rows that count, issued
        Ring ring;
        const T* X = static_cast<const T*>(a.ptr[kLrX]);
        T* G = static_cast<T*>(a.ptr[kLrGrad]);
        auto prepare = [&]() {
            const int b = prepared++, side = b & 1, n = min(kBatch, rows - b * kBatch);
            ok = __all_sync(0xffffffffu, wait_phase(&sh.meta_empty[side], ((b >> 1) & 1) ^ 1));
            if (!ok) return;
            RowMeta r{};
            int64_t x_off = 0;
            if (lane < n) {
                r.row = cluster + static_cast<int64_t>(b * kBatch + lane) * clusters;
                r.w = row_weight(a, r.row);
                if (OP == kLossDistill) {
                    r.list = static_cast<const ListSums*>(a.lists)[r.row];
                    if (r.list.count == 0) r.w = 0.0;  // nothing but padding
                }
                x_off = loss_offset(a, kLrX, r.row);
                const int64_t head64 = ((16 - (reinterpret_cast<uintptr_t>(X + x_off) & 15)) & 15) / sizeof(T);
                const int head = static_cast<int>(head64 < a.cols ? head64 : a.cols);
                const int packs = static_cast<int>((a.cols - head) / VE);
                int first;
                slice_of(packs, rank, size, first, r.count);
                r.body = head + first * VE;
                r.behind = head + packs * VE;
                r.src = X + x_off + r.body;
                if (G) {
                    T* g = G + loss_offset(a, kLrGrad, r.row);
                    r.grad = g;
                    if (a.g_in == 1 && (reinterpret_cast<uintptr_t>(g + r.body) & 15) == 0) r.out = g + r.body;
                }
                if (rank == 0) r.edges = edges_of(a, head, r.behind);
                r.target = -1;
                if (OP == kLossPolicy && r.w != 0.0) {
                    const int64_t t = load_index(a.ptr[kLrTarget], a.dtype[kLrTarget], loss_offset(a, kLrTarget, r.row));
                    r.old = row_real(a, kLrOld, r.row);
                    r.adv = row_real(a, kLrAdv, r.row);
                    if (a.ptr[kLrRef]) r.ref = row_real(a, kLrRef, r.row);
                    if (t >= 0 && t < a.cols) {
                        r.target = static_cast<int>(t);
                        r.xt = LossElem<T>::up(X[x_off + t]);
                    } else {
                        note_bad_index(a, t);
                    }
                    r.exp_old = exp(-r.old);
                    if (a.ptr[kLrRef]) r.exp_ref = exp(r.ref);
                }
                sh.meta[side][lane] = r;
            }
            if (rank == 0) read_edges(X, x_off, r.w != 0.0 ? r.edges : 0u, r.behind, n, lane, &sh.edge[side][0][0]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.meta_full[side]);
        };
        // Starts the copy of row i into the next stage.
        auto issue = [&](int i) {
            const RowMeta& r = sh.meta[i / kBatch & 1][i % kBatch];
            if (r.w == 0.0) return;
            ok = __all_sync(0xffffffffu, wait_phase(&sh.empty[ring.slot], ring.phase ^ 1u));
            if (!ok) return;
            if (lane == 0) {
                unsigned char* st = sm + static_cast<size_t>(ring.slot) * stage_bytes;
                const uint32_t bytes = static_cast<uint32_t>(r.count) * 16u;
                mbar_arrive_expect_tx(&sh.full[ring.slot], bytes);
                if (bytes) bulk_load(st, r.src, bytes, &sh.full[ring.slot]);
            }
            __syncwarp();
            ring.next(stages);
            ++live;
        };
        for (int i = 0; i < rows && ok; ++i) {
            if (i % kBatch == 0) prepare();
            if (ok) issue(i);
        }
        if (!ok) {
            if (lane == 0) note_timeout(a.timeouts);
            // the copies in flight land before the CTA's memory goes away
            for (int i = 0; i < stages; ++i)
                if (static_cast<uint32_t>(i) < live) mbar_wait(&sh.full[i], i < ring.slot ? ring.phase : ring.phase ^ 1u, 100000000ull);
        }
    } else if (warp == W + 1) {
        // ---- row warp: joins the sums, publishes the coefficient, and keeps what the losses are made of
        uint32_t live = 0;
        double total = 0.0, kept_s = 0.0, kept_rest = 0.0, kept_x = 0.0, kept_ref = 0.0;  // kept_x: ratio, or sum q (x - ref)
        float kept_m = 0.f, kept_mr = 0.f;
        for (int i = 0; i < rows && ok; ++i) {
            const int ms = i / kBatch & 1, mi = i % kBatch;
            if (mi == 0) ok = __all_sync(0xffffffffu, wait_phase(&sh.meta_full[ms], (i / kBatch >> 1) & 1));
            if (!ok) break;
            const RowMeta& r = sh.meta[ms][mi];
            if (r.w != 0.0) {
                const int cs = static_cast<int>(live % (kMaxDepth + 1)), side = static_cast<int>(live % kSides);
                const uint32_t phase = (live / kSides) & 1u;
                ok = wait_phase<true>(&sh.mail_full[side], phase);
                if (OP == kLossDistill) ok = ok && wait_phase(&sh.list_full[side], phase);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const int parts = size * W;
                constexpr int kJoin = kMaxCluster * W / 32;
                float pm[kJoin], ps[kJoin], mf = -INFINITY;
#pragma unroll
                for (int k = 0; k < kJoin; ++k) {
                    const uint64_t v = lane + 32 * k < parts ? sh.mail[side][lane + 32 * k] : 0xff800000ull;
                    pm[k] = __uint_as_float(static_cast<uint32_t>(v));
                    ps[k] = __uint_as_float(static_cast<uint32_t>(v >> 32));
                    mf = fmaxf(mf, pm[k]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(&sh.mail_full[side], mail_bytes);  // for the row kSides later
                const ListInfo& li = sh.list[side];
                const float mr = warp_max(mf);  // distill: of the columns that the teacher does not name
                mf = OP == kLossDistill ? fmaxf(mr, li.x_max) : mr;
                const double m = mf;
                // Every consumer of the cluster waits for the coefficient, so only what it needs is computed first:
                // no logarithm.
                double lift = 1.0;
                if (OP == kLossPolicy) lift = exp((m - r.xt) * a.inv_temp);
                float part = 0.f;
#pragma unroll
                for (int k = 0; k < kJoin; ++k)
                    if (32 * k < parts) part += pm[k] == -INFINITY ? ps[k] : ps[k] * (pm[k] == mr ? 1.f : exp_one(a, pm[k], mr));
                double s = warp_sum(part), s_rest = s;
                if (mf == INFINITY) s = s_rest = quiet_nan();
                Coef c;
                c.m = OP == kLossDistill && mr == -INFINITY ? 0.f : mr;
                c.named = c.p_scale = 0.f;
                double ratio = 0.0, big_q = 1.0;
                if (OP == kLossPolicy) {
                    // s relative to the target's logit instead of the maximum: r = exp(-old) / s', p_t = 1 / s'
                    const double st = s * lift, pt = 1.0 / st;
                    ratio = r.exp_old * pt;
                    double ed = r.exp_ref * st - 1.0, rest = 1.0 - pt;
                    if (!(st < 1e300 && r.exp_old < 1e300 && r.exp_old > 1e-300 && r.exp_ref < 1e300) || r.target < 0) {
                        // numbers outside these forms' range: through the logarithm
                        const double logp = r.target >= 0 ? (r.xt - m) * a.inv_temp - log(s) : quiet_nan();
                        ratio = exp(logp - r.old);
                        ed = expm1(r.ref - logp);
                        rest = -expm1(logp);
                    }
                    const double g = policy_terms(a, r.w, r.adv, ratio, 0.0, ed).g;
                    c.a = -static_cast<float>(g) / static_cast<float>(s);
                    c.named = static_cast<float>(g * rest);
                } else {
                    const float rise = mr == -INFINITY ? 0.f : exp_one(a, mr, mf);
                    s = s_rest * rise + li.named * (li.x_max == -INFINITY ? 0.f : exp_one(a, li.x_max, mf));
                    if (r.list.bad || !(s > 0.0)) s = quiet_nan();
                    c.a = static_cast<float>(distill_slope(a, r.w, s, s_rest, rise, r.list.mass, r.list.count == a.cols, big_q));
                    if (s != s) c.a = NAN;
                    c.p_scale = static_cast<float>(big_q) / static_cast<float>(s);
                    c.named = mf;
                }
                if (lane == 0) {
                    sh.coef[cs] = c;
                    mbar_arrive(&sh.coef_full[cs]);
                }
                if (lane == mi) {
                    kept_s = s;
                    kept_rest = s_rest;
                    kept_m = mf;
                    kept_mr = mr;
                    kept_x = OP == kLossPolicy ? ratio : li.q_x;
                    kept_ref = OP == kLossPolicy ? 0.0 : li.ref;
                }
                ++live;
            }
            __syncwarp();
            if (mi == kBatch - 1 || i + 1 == rows) {
                if (rank == 0 && lane <= mi) {
                    const RowMeta& mine = sh.meta[ms][lane];
                    const double m = kept_m;
                    if (mine.w == 0.0) {
                        put_empty_row(a, mine.row);
                    } else if (OP == kLossDistill) {
                        const double cross = mine.list.q_logq - a.inv_temp * (kept_x + (kept_ref - m) * mine.list.mass) +
                                             mine.list.mass * log(kept_s);
                        const double loss = distill_loss_of(a, kept_s, kept_rest, (kept_mr - m) * a.inv_temp, cross, mine.list.mass,
                                                            mine.list.count == a.cols);
                        put_row(a, kLrRowLoss, mine.row, loss);
                        total += mine.w * loss;
                    } else {
                        const double logp = mine.target >= 0 ? (mine.xt - m) * a.inv_temp - log(kept_s) : quiet_nan();
                        const double d = mine.ref - logp;
                        const PolicyTerms t = policy_terms(a, mine.w, mine.adv, kept_x, d, a.ptr[kLrRef] ? expm1(d) : 0.0);
                        put_row(a, kLrLogp, mine.row, logp);
                        put_row(a, kLrKl, mine.row, t.kl);
                        put_row(a, kLrRowLoss, mine.row, t.loss);
                        total += mine.w * t.loss;
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.meta_empty[ms]);
            }
        }
        if (!ok && lane == 0) note_timeout(a.timeouts);
        total = warp_sum(total);
        if (a.partials && rank == 0 && lane == 0) a.partials[cluster] = total;
    } else if (OP == kLossDistill && warp > W + 1) {
        // ---- list warps: every other row that counts
        const uint32_t mine = static_cast<uint32_t>(warp - W - 2);
        const T* X = static_cast<const T*>(a.ptr[kLrX]);
        unsigned char* bits = behind + bits_at<W>() + mine * bits_bytes(slice_packs);
        float* const e_xs = reinterpret_cast<float*>(behind + bits_at<W>() + kListWarps * bits_bytes(slice_packs));
        int col_ahead[kAhead];
        float q_ahead[kAhead];
        // Entries lane, lane + 32, ... of the first kAhead * 32 of a row, fetched a row ahead.
        auto fetch = [&](int64_t row) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int k = lane + 32 * u;
                col_ahead[u] = k < a.top ? list_col[row * a.top + k] : -1;
                q_ahead[u] = k < a.top ? list_q[row * a.top + k] : 0.f;
            }
        };
        // Waits until the consumers have written row l, the l-th that counts. The barrier is one of kSides, not the
        // stage's: with three stages the next row of a stage is the other list warp's, and its phase could come and go
        // before this warp looks. Row l + kSides is written only after this warp has given the list of row l + 4, which it
        // does after its last look at row l; and before it takes row l it has put row l - 4, so no earlier phase is open.
        auto written = [&](uint32_t l) { return wait_phase(&sh.done[l % kSides], (l / kSides) & 1u); };
        // Joins row i's entries with its logits, and takes those out of the slice.
        auto take = [&](int i, uint32_t l, const Ring& ring) {
            const int side = static_cast<int>(l % kSides), ms = i / kBatch & 1, mi = i % kBatch;
            const RowMeta& r = sh.meta[ms][mi];
            const T* x = X + loss_offset(a, kLrX, r.row);
            float* e_x = e_xs + side * a.top;
            T* st = reinterpret_cast<T*>(sm + static_cast<size_t>(ring.slot) * stage_bytes);
            ListInfo& li = sh.list[side];
            int col[kAhead];
            float q[kAhead];
            T raw[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                col[u] = col_ahead[u];
                q[u] = q_ahead[u];
                if (col[u] >= 0) raw[u] = x[col[u]];
            }
            for (int k = lane; k < (slice_packs + 15) / 16; k += 32) reinterpret_cast<uint4*>(bits)[k] = make_uint4(0u, 0u, 0u, 0u);
            if (lane == 0) li.edge_named = 0u;
            __syncwarp();  // other lanes set bits there (votes and shuffles order no memory)
            float x_max = -INFINITY;
            float xs[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                xs[u] = col[u] >= 0 ? LossElem<T>::up(raw[u]) : -INFINITY;
                x_max = fmaxf(x_max, xs[u]);
                if (lane + 32 * u < a.top) e_x[lane + 32 * u] = xs[u];
            }
            for (int k = lane + 32 * kAhead; k < a.top; k += 32) {
                const int j = list_col[r.row * a.top + k];
                const float xk = j >= 0 ? LossElem<T>::up(x[j]) : -INFINITY;
                x_max = fmaxf(x_max, xk);
                e_x[k] = xk;
            }
            x_max = warp_max(x_max);
            const float ref = x_max == -INFINITY ? 0.f : x_max;
            float named = 0.f;
            double q_x = 0.0;
            auto add = [&](float qk, int j, float xk) {
                if (j >= 0) named += exp_one(a, xk, ref);
                if (qk != 0.f) q_x += static_cast<double>(qk) * (static_cast<double>(xk) - ref);
            };
#pragma unroll
            for (int u = 0; u < kAhead; ++u) add(q[u], col[u], xs[u]);
            for (int k = lane + 32 * kAhead; k < a.top; k += 32)
                add(list_q[r.row * a.top + k], list_col[r.row * a.top + k], e_x[k]);
            named = warp_sum(named);
            q_x = warp_sum(q_x);
            // The row before in this stage may be the other list warp's: until that has landed, `full` still shows the
            // phase before, whose parity is this row's.
            ok = true;
            if (l >= static_cast<uint32_t>(stages)) ok = written(l - stages);
            ok = __all_sync(0xffffffffu, ok && wait_phase(&sh.full[ring.slot], ring.phase));
            if (!ok) return;
            // -inf in the place of each; a column named twice makes the whole row NaN
            T* twice_at = nullptr;
            float* twice_edge = nullptr;
            const int body = r.body, inside_end = r.count * VE, tail = r.behind;
            const uint32_t edges = r.edges;
            auto remove = [&](int j) {
                const int at = j - body;
                if (j < 0) return;
                if (at >= 0 && at < inside_end) {
                    const uint32_t bit = 1u << ((at / VE & 3) * 8 + at % VE);
                    const bool twice = atomicOr(reinterpret_cast<uint32_t*>(bits) + (at / VE >> 2), bit) & bit;
                    st[at] = LossElem<T>::down(-INFINITY);
                    if (twice) twice_at = st + at;
                } else if (rank == 0) {
                    const int l16 = j < 8 && (edges >> j & 1u) ? j : j >= tail ? 8 + j - tail : -1;
                    if (l16 < 0) return;
                    const bool twice = atomicOr(&li.edge_named, 1u << l16) >> l16 & 1u;
                    sh.edge[ms][mi][l16] = -INFINITY;
                    if (twice) twice_edge = &sh.edge[ms][mi][l16];
                } else {
                    return;
                }
                if (twice_at || twice_edge) note_bad_index(a, j);
            };
#pragma unroll
            for (int u = 0; u < kAhead; ++u) remove(col[u]);
            for (int k = lane + 32 * kAhead; k < a.top; k += 32) remove(list_col[r.row * a.top + k]);
            __syncwarp();
            if (twice_at) *twice_at = LossElem<T>::down(NAN);
            if (twice_edge) *twice_edge = NAN;
            release_fence();
            if (lane == 0) {
                li.q_x = q_x;
                li.ref = ref;
                li.named = named;
                li.x_max = x_max;
                mbar_arrive(&sh.list_full[side]);
            }
            __syncwarp();
        };
        // The named elements of this CTA's slice of row i, over what the consumers have left there.
        auto put = [&](int i, uint32_t l) {
            const RowMeta& r = sh.meta[i / kBatch & 1][i % kBatch];
            const float* e_x = e_xs + static_cast<int>(l % kSides) * a.top;
            int col[kAhead];
            float q[kAhead];
            auto entries = [&](int k0) {
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int k = k0 + lane + 32 * u;
                    col[u] = r.grad && k < a.top ? list_col[r.row * a.top + k] : -1;
                    q[u] = r.grad && k < a.top ? list_q[r.row * a.top + k] : 0.f;
                }
            };
            entries(0);
            ok = __all_sync(0xffffffffu, written(l));
            if (!ok) return;
            if (r.grad) {
                const Coef c = sh.coef[l % (kMaxDepth + 1)];
                T* gr = static_cast<T*>(r.grad);
                const float scale = static_cast<float>(r.w * a.inv_temp);
                // a bad row is NaN throughout: its named columns too, whoever found it
                const float poison = c.a == c.a ? 0.f : c.a;
                const int body = r.body, inside_end = r.count * VE, tail = r.behind;
                const uint32_t edges = r.edges;
                for (int k0 = 0; k0 < a.top; k0 += 32 * kAhead) {
                    if (k0) entries(k0);
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) {
                        const int j = col[u], at = j - body;
                        if (j < 0) continue;
                        const bool inside = at >= 0 && at < inside_end;
                        if (!inside && !((j < 8 && (edges >> j & 1u)) || (rank == 0 && j >= tail))) continue;
                        const T v = LossElem<T>::down(scale * (exp_one(a, e_x[k0 + lane + 32 * u], c.named) * c.p_scale - q[u]) + poison);
                        gr[j * a.g_in] = v;
                    }
                }
            }
            __syncwarp();
        };
        uint32_t live = 0, held_l = 0;
        int held = -1, freed = 0;  // the row that waits for its named elements; batches given back
        int64_t fetched = -1;
        Ring ring;
        for (int i = 0; i < rows && ok; ++i) {
            if (i % kBatch == 0) ok = __all_sync(0xffffffffu, wait_phase(&sh.meta_full[i / kBatch & 1], (i / kBatch >> 1) & 1));
            if (!ok) break;
            const RowMeta& r = sh.meta[i / kBatch & 1][i % kBatch];
            if (r.w != 0.0) {
                if (live % kListWarps == mine) {
                    if (fetched != r.row) fetch(r.row);
                    take(i, live, ring);
                    // this warp's next row, as far as it is known
                    const int end = min(rows, (i / kBatch + 1) * kBatch);
                    int k = i + 1, others = 0;
                    for (; k < end; ++k)
                        if (sh.meta[k / kBatch & 1][k % kBatch].w != 0.0 && ++others == kListWarps) break;
                    fetched = k < end ? sh.meta[k / kBatch & 1][k % kBatch].row : -1;
                    if (ok && fetched >= 0) fetch(fetched);
                    if (ok && held >= 0) put(held, held_l);
                    held = i;
                    held_l = live;
                }
                ring.next(stages);
                ++live;
            }
            // The operands of a batch are read again only when those of the one before the last are given back, so a
            // row does not wait past the end of the next batch, however few rows of that count.
            if (ok && i % kBatch == kBatch - 1 && held >= 0 && held < i / kBatch * kBatch) {
                put(held, held_l);
                held = -1;
            }
            for (; ok && (freed + 1) * kBatch <= (held >= 0 ? held : i + 1); ++freed)
                if (lane == 0) mbar_arrive(&sh.meta_empty[freed & 1]);
        }
        if (ok && held >= 0) put(held, held_l);
        if (!ok && lane == 0) note_timeout(a.timeouts);
    } else {
        // ---- consumers
        const int t = threadIdx.x;
        const ExpConst kc = exp_const(a);
        uint32_t live = 0, written = 0;  // rows that count: folded, written
        Ring ring, write_ring;
        int held[kMaxDepth] = {};  // the rows between, the latest first
        int freed = 0;             // batches given back
        auto stage_of = [&](const Ring& g) { return reinterpret_cast<uint4*>(sm + static_cast<size_t>(g.slot) * stage_bytes); };
        // Folds row i: its sum goes to the cluster.
        auto fold = [&](int i, const RowMeta& r) {
            const int side = static_cast<int>(live % kSides);
            if (OP == kLossDistill) ok = wait_phase(&sh.list_full[side], (live / kSides) & 1u);
            ok = __all_sync(0xffffffffu, ok && wait_phase(&sh.full[ring.slot], ring.phase));
            if (!ok) return;
            const uint4* st = stage_of(ring) + t;
            const float xe = t < 16 && (r.edges >> t & 1u) ? sh.edge[i / kBatch & 1][i % kBatch][t] : -INFINITY;
            const int count = r.count - t;  // packs t, t + kCons, ... of the slice
            float m, s0, s1;
            // a maximum a warp; the sum is brought down when it grows (a few times a row)
            constexpr int CP = 4;
            m = warp_max(xe);
            F2 sum = f2(exp_one(a, xe, m == -INFINITY ? 0.f : m), 0.f);
            for (int p0 = 0; p0 < r.count; p0 += CP * kCons) {
                uint4 raw[CP];
                float mx = -INFINITY;
#pragma unroll
                for (int u = 0; u < CP; ++u) {
                    raw[u] = p0 + u * kCons < count ? st[p0 + u * kCons] : P::lowest();
                    mx = fmaxf(mx, P::max(raw[u]));
                }
                mx = warp_max(mx);
                if (mx > m) {
                    const float down = exp_one(a, m, mx);
                    sum = mul2(sum, f2(down, down));
                    m = mx;
                }
                const float at = m == -INFINITY ? 0.f : m;
                const F2 minus = f2(-at, -at);
                F2 acc0 = f2(0.f, 0.f), acc1 = f2(0.f, 0.f);
#pragma unroll
                for (int u = 0; u < CP; ++u) {
                    F2 e[VE / 2];
                    P::up(raw[u], e);
#pragma unroll
                    for (int h = 0; h < VE / 2; h += 2) {
                        acc0 = add2(acc0, exp_pair(e[h], minus, kc));
                        acc1 = add2(acc1, exp_pair(e[h + 1], minus, kc));
                    }
                }
                sum = add2(sum, add2(acc0, acc1));
            }
            un(sum, s0, s1);
            const float s = warp_sum(s0 + s1);
            // A side of the mailbox is written again kSides = 2 depth + 2 rows later. This warp has by then waited for
            // the coefficient of depth + 1 rows ago, to which every warp of the cluster sent its sum after it had
            // itself waited for the one of depth + 1 rows before that, published when its CTA had read that side.
            if (lane < size)
                send8(&sh.mail[side][rank * W + warp], &sh.mail_full[side], lane,
                      static_cast<uint64_t>(__float_as_uint(m)) | static_cast<uint64_t>(__float_as_uint(s)) << 32);
        };
        // Writes the gradient of row i, the next one.
        auto write = [&](int i) {
            const RowMeta& r = sh.meta[i / kBatch & 1][i % kBatch];
            const uint32_t cs = written % (kMaxDepth + 1);
            ok = __all_sync(0xffffffffu, wait_phase(&sh.coef_full[cs], (written / (kMaxDepth + 1)) & 1u));
            if (!ok) return;
            const Coef c = sh.coef[cs];
            const uint4* st = stage_of(write_ring) + t;
            const int count = r.count - t;
            const F2 ga = f2(c.a, c.a), minus = f2(-c.m, -c.m);
            auto pack = [&](int p) {
                F2 e[VE / 2];
                P::up(st[p * kCons], e);
#pragma unroll
                for (int h = 0; h < VE / 2; ++h) e[h] = mul2(exp_pair(e[h], minus, kc), ga);
                return P::down(e);
            };
            if (r.out) {
                uint4* const to = static_cast<uint4*>(r.out) + t;
#pragma unroll 4
                for (int p = 0; p * kCons < count; ++p) to[p * kCons] = pack(p);
                if (OP == kLossPolicy) {
                    const int at = r.target - r.body;  // the target's own value, by the thread that wrote its pack
                    if (r.target >= 0 && at >= 0 && at < r.count * VE && (at / VE) % kCons == t)
                        static_cast<T*>(r.out)[at] = LossElem<T>::down(c.named);
                }
            } else if (r.grad) {
                // where the gradient's rows are not aligned like the logits', or strided: element by element
                T* gr = static_cast<T*>(r.grad);
                auto scatter = [&](int p, const uint4& o) {
                    const T* v = reinterpret_cast<const T*>(&o);
                    const int j = r.body + (p * kCons + t) * VE;
#pragma unroll
                    for (int k = 0; k < VE; ++k)
                        gr[(j + k) * a.g_in] = OP == kLossPolicy && j + k == r.target ? LossElem<T>::down(c.named) : v[k];
                };
                for (int p = 0; p * kCons < count; ++p) scatter(p, pack(p));
            }
            if (r.grad && t < 16 && (r.edges >> t & 1u)) {
                const int j = edge_column(t, r.behind);
                const float v = c.a * exp_one(a, sh.edge[i / kBatch & 1][i % kBatch][t], c.m);
                static_cast<T*>(r.grad)[j * a.g_in] = LossElem<T>::down(OP == kLossPolicy && j == r.target ? c.named : v);
            }
            release_fence();
            if (lane == 0) {
                mbar_arrive(&sh.empty[write_ring.slot]);
                if (OP == kLossDistill) mbar_arrive(&sh.done[written % kSides]);
            }
            write_ring.next(stages);
            ++written;
        };
        for (int i = 0; i < rows && ok; ++i) {
            if (i % kBatch == 0) ok = __all_sync(0xffffffffu, wait_phase(&sh.meta_full[i / kBatch & 1], (i / kBatch >> 1) & 1));
            if (!ok) break;
            const RowMeta& r = sh.meta[i / kBatch & 1][i % kBatch];
            if (r.w != 0.0) {
                fold(i, r);
                const int oldest = depth == 1 ? held[0] : depth == 2 ? held[1] : held[2];
                ring.next(stages);
                if (ok && live - written == static_cast<uint32_t>(depth)) write(oldest);
                if (!ok) break;
                held[2] = held[1];
                held[1] = held[0];
                held[0] = i;
                ++live;
            } else if (r.grad) {
                T* gr = static_cast<T*>(r.grad);
                if (r.out)
                    for (int p = t; p < r.count; p += kCons) static_cast<uint4*>(r.out)[p] = make_uint4(0u, 0u, 0u, 0u);
                else
                    for (int k = t; k < r.count * VE; k += kCons) gr[(r.body + k) * a.g_in] = LossElem<T>::down(0.f);
                if (t < 16 && (r.edges >> t & 1u)) gr[edge_column(t, r.behind) * a.g_in] = LossElem<T>::down(0.f);
            }
            __syncwarp();
            // The operands of a batch are read again only when those of the one before the last are given back, so a
            // row does not wait past the end of the next batch, however few rows of that count.
            auto first_waiting = [&]() {
                const uint32_t n = live - written;
                return n == 0 ? i + 1 : n == 1 ? held[0] : n == 2 ? held[1] : held[2];
            };
            if (i % kBatch == kBatch - 1)
                while (ok && first_waiting() < i / kBatch * kBatch) write(first_waiting());
            for (; ok && (freed + 1) * kBatch <= first_waiting(); ++freed)
                if (lane == 0) mbar_arrive(&sh.meta_empty[freed & 1]);
        }
        while (ok && written < live) write(live - written == 1 ? held[0] : live - written == 2 ? held[1] : held[2]);
        if (!ok && lane == 0) note_timeout(a.timeouts);
    }
    allow_dependents();
    leave_cluster(ok);
}

// ------------------------------------------------------------------------------------------------
// host side

// Launches with clusters of `cluster` CTAs; *parts < 0 when three stages do not fit.
template <class T, int OP, int W, int PER_SM>
int held_typed(const LossArgs& a, int64_t cluster, int most_stages, int* parts, cudaStream_t st) {
    const int64_t packs = a.cols / PackOf<T>::VE;
    int slice = static_cast<int>((packs + cluster - 1) / cluster);
    int stage = (slice < 1 ? 1 : slice) * 16;
    stage = (stage + 127) / 128 * 128;
    const size_t rest = behind_bytes<W>(OP, a.top, slice);
    // an equal share of an SM's shared memory (228 KiB, of which a CTA takes 1 KiB more than it asks for)
    const size_t room = (PER_SM > 1 ? 228 * 1024 / PER_SM - 1024 : static_cast<size_t>(kMaxSmem));
    int64_t stages = rest < room ? static_cast<int64_t>((room - rest) / stage) : 0;
    if (stages < 3) stages = rest < kMaxSmem ? static_cast<int64_t>((kMaxSmem - rest) / stage) : 0;
    if (stages > most_stages) stages = most_stages;
    *parts = -1;
    if (stages < 3) return CTB_OK;
    const size_t smem = static_cast<size_t>(stages) * stage + rest;
    auto fn = loss_held_kernel<T, OP, W, PER_SM>;
    constexpr int threads = held_threads<OP, W>();
    int n = 0;
    if (int rc = resident_blocks(reinterpret_cast<const void*>(fn), threads, static_cast<int>(cluster), smem, &n)) return rc;
    int64_t clusters = n < a.rows ? n : a.rows;
    if (clusters > kLossMaxCtas) clusters = kLossMaxCtas;
    *parts = static_cast<int>(clusters);
    if (OP == kLossDistill) {
        launch_dependent(loss_lists, grid_for((a.rows + 7) / 8, 8), 256, 0, st, a);
        count_launch();
        if (int rc = check_launch("loss lists")) return rc;
    }
    LossArgs args = a;
    int ring = static_cast<int>(stages);
    // besides the rows that wait and the one that is folded, two stages load: with one, nothing is on its way while a
    // stage is written and given back
    int depth = stages >= 6 ? 3 : stages >= 5 ? 2 : 1;
    void* argv[5] = {&args, &ring, &stage, &slice, &depth};
    return launch_cluster(reinterpret_cast<const void*>(fn), static_cast<unsigned>(clusters * cluster), threads,
                          static_cast<int>(cluster), smem, st, argv);
}

template <class T, int OP> int held_sized(const LossArgs& a, int* parts, cudaStream_t st) {
    const int64_t v = a.cols;
    auto share = [&](int64_t most) { return (v + most - 1) / most; };
    *parts = -1;
    const int64_t most = 65536 / sizeof(T);  // logits of a slice that leaves room for three stages
    int64_t c = share(most);
    if (c > kMaxCluster) return CTB_OK;
    // few rows: more CTAs a row, down to 8 KiB each
    while (c * 2 <= kMaxCluster && a.rows * c * 2 <= sm_count() && v * static_cast<int64_t>(sizeof(T)) >= c * 2 * 8192) c *= 2;
    // A row costs a CTA about 2 us whatever its length (the exchange, the row's arithmetic, the copies' latency), so
    // short slices want several CTAs an SM. Policy loss on B200, us, by the slice's bytes (bf16 rows), CTAs an SM x
    // consumer warps:
    //     bytes     1 x 16   2 x 8   3 x 8   4 x 4
    //      8 KiB       701     411     409     266
    //     12 KiB       385     228     234     194
    //     16 KiB       391     249     234     411
    //     24 KiB       413     346     411     359
    //     32 KiB       435     484     432     793
    const int64_t bytes = (v + c - 1) / c * static_cast<int64_t>(sizeof(T));
    if (bytes <= 12 * 1024) return held_typed<T, OP, 4, 4>(a, c, kMaxRing, parts, st);
    if (bytes <= 18 * 1024) return held_typed<T, OP, 8, 3>(a, c, kMaxRing, parts, st);
    if (bytes <= 28 * 1024) return held_typed<T, OP, 8, 2>(a, c, kMaxRing, parts, st);
    return held_typed<T, OP, 16, 1>(a, c, kMaxRing, parts, st);
}

}  // namespace

size_t loss_lists_bytes(int64_t rows, int64_t top) { return list_sums_bytes(rows) + static_cast<size_t>(rows) * top * 8; }

int loss_held(const LossPlan& p, int* parts, cudaStream_t st) {
    const LossArgs& a = p.args;
    const bool bf = a.dtype[kLrX] == CTB_BFLOAT16;
    if (p.op == kLossPolicy)
        return bf ? held_sized<__nv_bfloat16, kLossPolicy>(a, parts, st) : held_sized<float, kLossPolicy>(a, parts, st);
    return bf ? held_sized<__nv_bfloat16, kLossDistill>(a, parts, st) : held_sized<float, kLossDistill>(a, parts, st);
}

}  // namespace ctb
