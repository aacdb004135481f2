// losses_rows.cu — the losses over rows of unit stride, float32 and bfloat16: each logit is read from
// memory once and each gradient element written once.
//
// A row belongs to a thread-block cluster of C CTAs (C = 1 for rows that one CTA can hold), a CTA to a
// contiguous slice of the row's 16-byte packs. Clusters are persistent: cluster c takes rows c, c + n,
// c + 2n, ... A CTA has eight consumer warps and two helpers:
//   * the producer warp streams the slices of the coming rows into a ring of shared-memory stages with
//     bulk asynchronous copies (async_copy.cuh) and reads the rows' small operands ahead, 32 rows a time;
//   * the consumers take a slice out of the ring into registers, find the warp's maximum, turn the
//     logits into e = exp((x - m_w) / T) and send each warp's (m_w, sum e) to every CTA of the cluster
//     (st.async into its mailbox, completion counted on its mbarrier: no cluster-wide barrier);
//   * the row warp joins the C * 8 partial sums, does the row's own arithmetic in float64 and publishes
//     the row's coefficient A; the consumers then write g = e * A exp((m_w - m) / T) from registers.
// So a logit costs one exponential, not two, and the exchange of one cluster hides behind the other
// clusters of the SM and behind the copies of the next rows.
//
// Accuracy of the sum. log2(e)/T as one float32 is off by up to 6e-8 relative, and so is every t = d log2(e)/T
// and with it, one-sidedly, the sum; a sequence's log-probabilities add that up. t is therefore corrected
// with the rest of log2(e)/T, one fused multiply-add (log-probabilities on B200, [8192, 32768] bfloat16: mean
// error -6e-9, of the order of the hardware's 2^t). Long sums are taken in two levels, a stage's share of a
// thread and then the stages, so that small terms are not lost against a grown sum ([2048, 131072] logits of
// standard deviation 4 in one level: 1.7e-7 low on average).
#include <map>
#include <mutex>
#include <string>
#include <tuple>

#include "async_copy.cuh"
#include "losses.cuh"

namespace ctb {

namespace {

constexpr int kConsWarps = 8;
constexpr int kCons = kConsWarps * 32;
constexpr int kProducer = kConsWarps;  // warp numbers
constexpr int kRowWarp = kConsWarps + 1;
constexpr int kThreads = kCons + 64;
constexpr int kMaxCluster = 8;
constexpr int kAhead = 4;   // teacher entries a lane of the producer fetches a row ahead
constexpr int kBatch = 32;  // rows whose operands the producer reads together, one a lane
constexpr int kMaxSmem = 227 * 1024;

// ------------------------------------------------------------------------------------------------
// pairs of floats (one instruction for two elements on sm_100)

struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void un(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// The largest of the warp's values (NaN loses against any number).
__device__ __forceinline__ float warp_max(float x) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// A 16-byte pack as pairs of floats, its maximum, and back (rounded to nearest even).
template <class T> struct PackOf;
template <> struct PackOf<float> {
    static constexpr int VE = 4;
    __device__ static __forceinline__ float max(const uint4& p) {
        return fmaxf(fmaxf(__uint_as_float(p.x), __uint_as_float(p.y)), fmaxf(__uint_as_float(p.z), __uint_as_float(p.w)));
    }
    __device__ static __forceinline__ void up(const uint4& p, F2* o) {
        o[0] = f2(__uint_as_float(p.x), __uint_as_float(p.y));
        o[1] = f2(__uint_as_float(p.z), __uint_as_float(p.w));
    }
    __device__ static __forceinline__ uint4 down(const F2* e) {
        float a, b, c, d;
        un(e[0], a, b);
        un(e[1], c, d);
        return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
    }
    __device__ static __forceinline__ uint4 lowest() {
        return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);  // -inf
    }
};
template <> struct PackOf<__nv_bfloat16> {
    static constexpr int VE = 8;
    __device__ static __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    __device__ static __forceinline__ float max(const uint4& p) {
        const uint32_t m = max2(max2(p.x, p.y), max2(p.z, p.w));
        return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
    __device__ static __forceinline__ F2 pair(uint32_t w) { return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    __device__ static __forceinline__ void up(const uint4& p, F2* o) {
        o[0] = pair(p.x);
        o[1] = pair(p.y);
        o[2] = pair(p.z);
        o[3] = pair(p.w);
    }
    __device__ static __forceinline__ uint32_t two(F2 e) {
        float a, b;
        un(e, a, b);
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));  // first operand in the upper half
        return r;
    }
    __device__ static __forceinline__ uint4 down(const F2* e) { return make_uint4(two(e[0]), two(e[1]), two(e[2]), two(e[3])); }
    __device__ static __forceinline__ uint4 lowest() {
        return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
    }
};

// exp of pairs: t = d c + d c rho with c = log2(e)/T rounded down and rho >= 1e-30 its rest, so that
// d = -inf stays -inf.
struct ExpConst {
    F2 c, rho;
};
__device__ __forceinline__ ExpConst exp_const(const LossArgs& a) {
    ExpConst k;
    k.c = f2(a.c2_down, a.c2_down);
    k.rho = f2(a.c2_rest, a.c2_rest);
    return k;
}
__device__ __forceinline__ F2 exp_pair(F2 x, F2 minus_m, const ExpConst& k) {
    const F2 d = mul2(add2(x, minus_m), k.c);
    const F2 t = fma2(d, k.rho, d);
    float a, b;
    un(t, a, b);
    return f2(exp2_fast(a), exp2_fast(b));
}
__device__ __forceinline__ float exp_one(const LossArgs& a, float x, float m) {
    const float d = (x - m) * a.c2_down;
    return exp2_fast(fmaf(d, a.c2_rest, d));
}

// Gives a stage back after the warp's reads of it. The reads may still be in flight when the next copy is
// allowed to start, and that copy belongs to another proxy: without the fence, a refill was seen to
// overtake them (a few packs at the start of a stage, once in some ten thousand stages).
__device__ __forceinline__ void release_fence() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}
__device__ __forceinline__ void release_stage(uint64_t* empty, int lane) {
    release_fence();
    if (lane == 0) mbar_arrive(empty);
}

// ------------------------------------------------------------------------------------------------
// clusters

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// Every thread of every CTA of the cluster. Used at the start (barriers are initialised before anyone
// sends to them) and at the end (no CTA leaves while another may still send to its memory).
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Stores 8 bytes to the same place in CTA `cta` of the cluster and counts them on its barrier.
__device__ __forceinline__ void send8(const void* local, uint64_t* local_bar, uint32_t cta, uint64_t v) {
    asm volatile(
        "{\n\t.reg .b32 ra, rb;\n\t"
        "mapa.shared::cluster.u32 ra, %0, %2;\n\t"
        "mapa.shared::cluster.u32 rb, %1, %2;\n\t"
        "st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [ra], %3, [rb];\n\t}" ::"r"(smem_addr(local)),
        "r"(smem_addr(local_bar)), "r"(cta), "l"(v)
        : "memory");
}

// The end of every warp's work. After a wait that ran out, another CTA may have sent what this one no longer
// waits for: it stays for a millisecond more, a thousand times what a store takes.
__device__ __forceinline__ void leave_cluster(bool ok) {
    __syncwarp();
    cluster_sync();
    if (!ok) {
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 1000000ull) {
        }
    }
}

// Waits for a phase that threads of other CTAs of the cluster contribute to.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity) {
    uint64_t t0 = 0;
    for (int i = 0;; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(smem_addr(bar)), "r"(parity)
            : "memory");
        if (done) return true;
        if (i % 32 == 0) {
            if (t0 == 0) t0 = global_ns();
            else if (global_ns() - t0 > kWaitLimitNs) return false;
        }
    }
}

// ------------------------------------------------------------------------------------------------
// shared memory

// What the producer knows of a row before its logits arrive.
struct RowMeta {
    double w;            // 0: the row does not count
    double xt;           // target's logit
    double old, adv, ref;
    double exp_old, exp_ref;  // exp(-old), exp(ref)
    long long row, g_off;
    int target;          // -1: bad
    int head, packs;     // elements before the first whole 16-byte pack, whole packs
    int first, count;    // this CTA's slice of the packs
    int pad_;
};

// What the producer knows of a teacher's list.
struct ListInfo {
    double q_logq, q_x, ref, mass;  // sums of q log q, q (x - ref) and q over the entries
    double named;                   // sum of exp((x - x_max) / T) over them
    float x_max;
    int count, bad;
    uint32_t edge_named;  // which of the 16 edge elements the teacher names (the producer's own)
};

struct Coef {
    float a, m, at_target, pad_;
};

template <class T, int E, int CP, int NS> struct Layout {
    static constexpr int VE = PackOf<T>::VE;
    static constexpr int RP = E / VE;        // packs a consumer thread holds
    static constexpr int NCH = RP / CP;      // stages a slice takes
    static constexpr int kChunkPacks = CP * kCons;
    static constexpr size_t kStage = static_cast<size_t>(kChunkPacks) * 16;
    static constexpr size_t kMail = NS * kStage;                       // uint64 [2][kMaxCluster * kConsWarps]
    static constexpr size_t kMeta = kMail + 2 * kMaxCluster * kConsWarps * 8;  // RowMeta [2][kBatch]
    static constexpr size_t kEdge = kMeta + 2 * kBatch * sizeof(RowMeta);      // float [2][kBatch][16]
    static constexpr size_t kCoef = kEdge + 2 * kBatch * 16 * sizeof(float);   // Coef [2]
    static constexpr size_t kBars = kCoef + 2 * sizeof(Coef);
    static constexpr int kNumBars = 2 * NS + 14;
    static constexpr size_t kList = kBars + kNumBars * 8;              // ListInfo [2]
    static constexpr size_t kBits = (kList + 2 * sizeof(ListInfo) + 15) / 16 * 16;  // bytes [kCons * RP]
    static constexpr size_t kEntries = kBits + kCons * RP;         // per side: int idx[K], float x[K], float q[K]
    static constexpr size_t bytes(int op, int top) {
        return op == kLossDistill ? kEntries + static_cast<size_t>(2) * 12 * top : kList;
    }
};

// The barriers of a CTA.
template <int NS> struct Bars {
    uint64_t full[NS], empty[NS];
    uint64_t meta_full[2], meta_empty[2];
    uint64_t list_full[2], list_empty[2];
    uint64_t mail[2], coef[2];
    uint64_t done[2];  // the consumers have written the row's slice
};

// Rank r's share of a row's packs.
__device__ __forceinline__ void slice_of(int packs, int rank, int size, int& first, int& count) {
    first = static_cast<int>(static_cast<int64_t>(packs) * rank / size);
    count = static_cast<int>(static_cast<int64_t>(packs) * (rank + 1) / size) - first;
}

// ------------------------------------------------------------------------------------------------
// the producer's reads

template <class T, int OP>
__device__ __forceinline__ RowMeta read_meta(const LossArgs& a, int64_t row, int rank, int size, int64_t& x_off) {
    RowMeta r;
    const T* X = static_cast<const T*>(a.ptr[kLrX]);
    r.row = row;
    r.w = row_weight(a, row);
    x_off = loss_offset(a, kLrX, row);
    r.g_off = a.ptr[kLrGrad] ? loss_offset(a, kLrGrad, row) : 0;
    const uintptr_t at = reinterpret_cast<uintptr_t>(X + x_off);
    const int64_t head = ((16 - (at & 15)) & 15) / sizeof(T);
    r.head = static_cast<int>(head < a.cols ? head : a.cols);
    r.packs = static_cast<int>((a.cols - r.head) / PackOf<T>::VE);
    slice_of(r.packs, rank, size, r.first, r.count);
    r.target = -1;
    r.xt = r.old = r.adv = r.ref = r.exp_old = r.exp_ref = 0.0;
    if (OP != kLossDistill && r.w != 0.0) {
        const int64_t t = load_index(a.ptr[kLrTarget], a.dtype[kLrTarget], loss_offset(a, kLrTarget, row));
        if (OP == kLossPolicy) {
            r.old = row_real(a, kLrOld, row);
            r.adv = row_real(a, kLrAdv, row);
            r.exp_old = exp(-r.old);
            if (a.ptr[kLrRef]) {
                r.ref = row_real(a, kLrRef, row);
                r.exp_ref = exp(r.ref);
            }
        }
        if (t >= 0 && t < a.cols) {
            r.target = static_cast<int>(t);
            r.xt = LossElem<T>::up(X[x_off + t]);
        } else {
            note_bad_index(a, t);
        }
    }
    return r;
}

// The elements around the whole packs: 0..7 before them, 8..15 behind them; -1 where there is none.
__device__ __forceinline__ int64_t edge_position(const LossArgs& a, int head, int packs, int ve, int l) {
    const int64_t behind = head + static_cast<int64_t>(packs) * ve;
    if (l < 8) return l < head ? l : -1;
    return behind + (l - 8) < a.cols ? behind + (l - 8) : -1;
}

// ------------------------------------------------------------------------------------------------
// forward passes: log-probabilities alone (token), losses with their gradient (policy, distill)

template <class T, int OP, int E, int CP, int NS, int PER_SM>
__global__ void __launch_bounds__(kThreads, PER_SM) loss_rows_kernel(const __grid_constant__ LossArgs a) {
    using L = Layout<T, E, CP, NS>;
    using P = PackOf<T>;
    constexpr int VE = L::VE, RP = L::RP;
    extern __shared__ __align__(128) unsigned char sm[];
    Bars<NS>& bars = *reinterpret_cast<Bars<NS>*>(sm + L::kBars);
    uint64_t* mail = reinterpret_cast<uint64_t*>(sm + L::kMail);
    RowMeta* metas = reinterpret_cast<RowMeta*>(sm + L::kMeta);
    float* edges = reinterpret_cast<float*>(sm + L::kEdge);
    Coef* coefs = reinterpret_cast<Coef*>(sm + L::kCoef);
    ListInfo* lists = reinterpret_cast<ListInfo*>(sm + L::kList);
    unsigned char* bits = sm + L::kBits;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank()), size = static_cast<int>(cluster_size());
    const uint32_t mail_bytes = static_cast<uint32_t>(size) * kConsWarps * 8;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.empty[i], kConsWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.meta_full[i], 1);
            mbar_init(&bars.meta_empty[i], kConsWarps + 1);
            mbar_init(&bars.list_full[i], 1);
            mbar_init(&bars.list_empty[i], kConsWarps + 1);
            mbar_init(&bars.mail[i], 1);
            mbar_init(&bars.coef[i], 1);
            mbar_init(&bars.done[i], kConsWarps);
        }
        mbar_fence_init();
        for (int i = 0; i < 2; ++i) mbar_arrive_expect_tx(&bars.mail[i], mail_bytes);
    }
    __syncthreads();
    cluster_sync();
    dependent_wait();  // the previous kernel in the stream has completed and its writes are visible

    const int64_t cluster = blockIdx.x / size, clusters = gridDim.x / size;
    const int64_t my_rows = cluster < a.rows ? (a.rows - cluster + clusters - 1) / clusters : 0;
    bool ok = true;

    if (warp == kProducer) {
        uint32_t g = 0;     // stages filled
        uint32_t live = 0;  // rows that count
        auto issue = [&](int64_t x_off, int head, int first, int count) {
            const T* src = static_cast<const T*>(a.ptr[kLrX]) + x_off + head + static_cast<int64_t>(first) * VE;
            for (int p = 0; p < count && ok; p += L::kChunkPacks, ++g) {
                const int slot = static_cast<int>(g % NS);
                ok = __all_sync(0xffffffffu, mbar_wait(&bars.empty[slot], ((g / NS) & 1u) ^ 1u));
                if (!ok) break;
                const int n = min(L::kChunkPacks, count - p);
                if (lane == 0) {
                    mbar_arrive_expect_tx(&bars.full[slot], static_cast<uint32_t>(n) * 16u);
                    bulk_load(sm + static_cast<size_t>(slot) * L::kStage, src + static_cast<int64_t>(p) * VE,
                              static_cast<uint32_t>(n) * 16u, &bars.full[slot]);
                }
                __syncwarp();
            }
        };
        // The teacher's list of one row. Entries lane, lane + 32, ... of the first kAhead * 32 are fetched a row
        // ahead into registers, as they lie in memory, so that nothing waits for them; longer lists are read in
        // place.
        uint64_t raw_t[kAhead], raw_at[kAhead];
        auto as_real = [&](uint64_t v) -> double {
            switch (a.dtype[kLrTeacher]) {
            case CTB_FLOAT32: return __uint_as_float(static_cast<uint32_t>(v));
            case CTB_FLOAT64: return __longlong_as_double(static_cast<long long>(v));
            default: return __uint_as_float(static_cast<uint32_t>(v) << 16);
            }
        };
        auto scaled = [&](int64_t t_off, int k) {
            return load_real(a.ptr[kLrTeacher], a.dtype[kLrTeacher], t_off + k * a.t_in) * a.inv_temp;
        };
        auto fetch_list = [&](int64_t row) {
            const int64_t t_off = loss_offset(a, kLrTeacher, row), ti_off = loss_offset(a, kLrTeacherIdx, row);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int k = lane + 32 * u;
                if (k < a.top) {
                    const int64_t o = t_off + k * a.t_in, io = ti_off + k * a.ti_in;
                    if (a.dtype[kLrTeacher] == CTB_FLOAT32) raw_t[u] = static_cast<const uint32_t*>(a.ptr[kLrTeacher])[o];
                    else if (a.dtype[kLrTeacher] == CTB_FLOAT64) raw_t[u] = static_cast<const uint64_t*>(a.ptr[kLrTeacher])[o];
                    else raw_t[u] = static_cast<const uint16_t*>(a.ptr[kLrTeacher])[o];
                    if (a.dtype[kLrTeacherIdx] == CTB_INT32) raw_at[u] = static_cast<const uint32_t*>(a.ptr[kLrTeacherIdx])[io];
                    else raw_at[u] = static_cast<const uint64_t*>(a.ptr[kLrTeacherIdx])[io];
                }
            }
        };
        // Joins the list of the row whose stages are g0 to g1 with the row's logits: sums for the row warp, and -inf
        // in place of the named logits, so that the consumers' sum is that of the others. `next`: the row to
        // fetch ahead, or -1.
        auto read_list = [&](int64_t row, int64_t next, int64_t x_off, int head, int packs, int first, int count, uint32_t g0,
                             uint32_t g1, float* edge) {
            const int side = static_cast<int>(live & 1u);
            int* e_idx = reinterpret_cast<int*>(sm + L::kEntries + static_cast<size_t>(side) * 12 * a.top);
            float* e_x = reinterpret_cast<float*>(e_idx + a.top);
            float* e_q = e_x + a.top;
            const T* x = static_cast<const T*>(a.ptr[kLrX]) + x_off;
            const int64_t t_off = loss_offset(a, kLrTeacher, row), ti_off = loss_offset(a, kLrTeacherIdx, row);
            double zr[kAhead];
            int jr[kAhead];
            T xraw[kAhead];
            int bad = 0;
            // all loads of logits first
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                zr[u] = lane + 32 * u < a.top ? as_real(raw_t[u]) * a.inv_temp : -INFINITY;
                const int64_t at = a.dtype[kLrTeacherIdx] == CTB_INT32 ? static_cast<int64_t>(static_cast<int32_t>(raw_at[u]))
                                                                       : static_cast<int64_t>(raw_at[u]);
                jr[u] = zr[u] == -INFINITY ? -1 : at >= 0 && at < a.cols ? static_cast<int>(at) : -2;
                if (jr[u] >= 0) xraw[u] = x[jr[u]];
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (jr[u] == -2) {
                    bad = 1;
                    if (rank == 0)
                        note_bad_index(a, a.dtype[kLrTeacherIdx] == CTB_INT32 ? static_cast<int64_t>(static_cast<int32_t>(raw_at[u]))
                                                                              : static_cast<int64_t>(raw_at[u]));
                    jr[u] = -1;
                }
            // a valid entry's column, -1 for padding and for an index outside the row
            auto column = [&](double zk, int64_t k) -> int {
                if (zk == -INFINITY) return -1;
                if (k >= 0 && k < a.cols) return static_cast<int>(k);
                bad = 1;
                if (rank == 0) note_bad_index(a, k);
                return -1;
            };
            if (next >= 0) fetch_list(next);
            // the teacher alone, while those are on their way: q = weight * exp(z - base), with weight 1 and the
            // teacher's own log-sum-exp, or 1 / sum and the maximum
            double base = -INFINITY, log_sum = 0.0, weight = 1.0;
            int entries = 0;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                base = fmax(base, zr[u]);
                entries += zr[u] != -INFINITY;
            }
            for (int k = lane + 32 * kAhead; k < a.top; k += 32) {
                const double zk = scaled(t_off, k);
                base = fmax(base, zk);
                entries += zk != -INFINITY;
            }
            entries = __reduce_add_sync(0xffffffffu, entries);
            if (a.tail) {
                base = entries ? row_real(a, kLrTeacherLse, row) : 0.0;
            } else {
#pragma unroll
                for (int d = 16; d >= 1; d >>= 1) base = fmax(base, __shfl_xor_sync(0xffffffffu, base, d));
            }
            double er[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) er[u] = zr[u] == -INFINITY ? 0.0 : exp(zr[u] - base);
            if (!a.tail) {
                double sum = 0.0;
#pragma unroll
                for (int u = 0; u < kAhead; ++u) sum += er[u];
                for (int k = lane + 32 * kAhead; k < a.top; k += 32) sum += exp(scaled(t_off, k) - base);
                sum = warp_sum(sum);
                weight = 1.0 / sum;
                log_sum = log(sum);
            }
            ok = __all_sync(0xffffffffu, mbar_wait(&bars.list_empty[side], ((live >> 1) & 1u) ^ 1u));
            if (!ok) return;
            float xr[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) xr[u] = jr[u] >= 0 ? LossElem<T>::up(xraw[u]) : -INFINITY;
            // which columns of this CTA's slice are named already
            uint4* b16 = reinterpret_cast<uint4*>(bits);
            for (int i = lane; i < kCons * RP / 16; i += 32) b16[i] = make_uint4(0u, 0u, 0u, 0u);
            if (lane == 0) lists[side].edge_named = 0u;
            float x_max = -INFINITY;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                x_max = fmaxf(x_max, xr[u]);
                if (lane + 32 * u < a.top) {
                    e_idx[lane + 32 * u] = jr[u];
                    e_x[lane + 32 * u] = xr[u];
                }
            }
            for (int k = lane + 32 * kAhead; k < a.top; k += 32) {
                const int j = column(scaled(t_off, k), load_index(a.ptr[kLrTeacherIdx], a.dtype[kLrTeacherIdx], ti_off + k * a.ti_in));
                const float xk = j >= 0 ? LossElem<T>::up(x[j]) : -INFINITY;
                x_max = fmaxf(x_max, xk);
                e_idx[k] = j;
                e_x[k] = xk;
            }
            x_max = warp_max(x_max);
            const double ref = x_max == -INFINITY ? 0.0 : static_cast<double>(x_max);
            double sums[4] = {0.0, 0.0, 0.0, 0.0};  // mass, q log q, q (x - ref), exp((x - x_max) / T)
            auto add = [&](int k, double zk, double ek, int j, float xk) {
                const double q = weight * ek;
                if (q != 0.0) {  // NaN too
                    sums[0] += q;
                    sums[1] += q * (zk - base - log_sum);
                    sums[2] += q * (static_cast<double>(xk) - ref);
                }
                if (j >= 0 && xk != -INFINITY) sums[3] += exp_one(a, xk, x_max);
                e_q[k] = static_cast<float>(q);
            };
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (lane + 32 * u < a.top) add(lane + 32 * u, zr[u], er[u], jr[u], xr[u]);
            for (int k = lane + 32 * kAhead; k < a.top; k += 32) {
                const double zk = scaled(t_off, k);
                add(k, zk, zk == -INFINITY ? 0.0 : exp(zk - base), e_idx[k], e_x[k]);
            }
#pragma unroll
            for (int d = 16; d >= 1; d >>= 1)
#pragma unroll
                for (int v = 0; v < 4; ++v) sums[v] += __shfl_xor_sync(0xffffffffu, sums[v], d);
            // the row's stages have landed: take the named logits out
            for (uint32_t k = g0; k != g1; ++k) ok = mbar_wait(&bars.full[k % NS], (k / NS) & 1u) && ok;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return;
            for (int k = lane; k < a.top; k += 32) {
                const int j = e_idx[k];
                if (j < 0) continue;
                const int b = j - head;
                uint32_t was = 0u, bit = 1u;
                if (b >= 0 && b < packs * VE) {
                    const int p = b / VE - first;
                    if (p >= 0 && p < count) {
                        bit = 1u << ((p & 3) * 8 + b % VE);
                        was = atomicOr(reinterpret_cast<uint32_t*>(bits) + (p >> 2), bit);
                        const uint32_t slot = (g0 + static_cast<uint32_t>(p / L::kChunkPacks)) % NS;
                        T* st = reinterpret_cast<T*>(sm + slot * L::kStage) + (p % L::kChunkPacks) * VE + b % VE;
                        *st = LossElem<T>::down(-INFINITY);
                    }
                } else if (rank == 0) {
                    const int l = b < 0 ? j : 8 + b - packs * VE;
                    bit = 1u << l;
                    was = atomicOr(&lists[side].edge_named, bit);
                    edge[l] = -INFINITY;
                }
                if (was & bit) {
                    bad = 1;
                    note_bad_index(a, j);
                }
            }
            bad = __any_sync(0xffffffffu, bad);
            release_fence();  // a later copy into these stages comes after these stores
            if (lane == 0) {
                ListInfo& li = lists[side];
                li.mass = sums[0];
                li.q_logq = sums[1];
                li.q_x = sums[2];
                li.named = sums[3];
                li.ref = ref;
                li.x_max = x_max;
                li.count = entries;
                li.bad = bad;
                mbar_arrive(&bars.list_full[side]);
            }
            __syncwarp();
        };
        for (int64_t b = 0; b * kBatch < my_rows && ok; ++b) {
            const int side = static_cast<int>(b & 1);
            const int n = static_cast<int>(min(static_cast<int64_t>(kBatch), my_rows - b * kBatch));
            ok = __all_sync(0xffffffffu, mbar_wait(&bars.meta_empty[side], ((b >> 1) & 1) ^ 1));
            if (!ok) break;
            int64_t x_off = 0;
            RowMeta r{};
            if (lane < n) {
                r = read_meta<T, OP>(a, cluster + (b * kBatch + lane) * clusters, rank, size, x_off);
                metas[side * kBatch + lane] = r;
            }
            if (rank == 0) {
                for (int i = 0; i < n; ++i) {
                    const int64_t off = __shfl_sync(0xffffffffu, x_off, i);
                    const int head = __shfl_sync(0xffffffffu, r.head, i), packs = __shfl_sync(0xffffffffu, r.packs, i);
                    const bool counts = __shfl_sync(0xffffffffu, r.w != 0.0, i);
                    if (lane < 16) {
                        const int64_t at = edge_position(a, head, packs, VE, lane);
                        edges[(side * kBatch + i) * 16 + lane] =
                            at >= 0 && counts ? LossElem<T>::up(static_cast<const T*>(a.ptr[kLrX])[off + at]) : -INFINITY;
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.meta_full[side]);
            const uint32_t counting = __ballot_sync(0xffffffffu, r.w != 0.0);
            // A list is joined with its row once that has landed, so the next row's copies are started first,
            // where the ring holds two rows.
            constexpr bool kTwo = OP == kLossDistill && NS >= 2 * L::NCH;
            uint32_t g_next = g;
            bool issued = false;
            for (uint32_t todo = counting; todo && ok; todo &= todo - 1) {
                const int i = __ffs(todo) - 1;
                const uint32_t later = todo & (todo - 1);
                const int i2 = later ? __ffs(later) - 1 : i;
                const int64_t off = __shfl_sync(0xffffffffu, x_off, i);
                const int head = __shfl_sync(0xffffffffu, r.head, i);
                const int first = __shfl_sync(0xffffffffu, r.first, i), count = __shfl_sync(0xffffffffu, r.count, i);
                uint32_t g0 = g_next, g1 = g;
                if (!issued) {
                    g0 = g;
                    issue(off, head, first, count);
                    g1 = g;
                }
                if (OP == kLossDistill && ok) {
                    const int64_t row = __shfl_sync(0xffffffffu, r.row, i), next = __shfl_sync(0xffffffffu, r.row, i2);
                    const int packs = __shfl_sync(0xffffffffu, r.packs, i);
                    if (todo == counting) fetch_list(row);  // the batch's first: nobody fetched it ahead
                    issued = kTwo && later;
                    if (issued) {
                        g_next = g;
                        issue(__shfl_sync(0xffffffffu, x_off, i2), __shfl_sync(0xffffffffu, r.head, i2),
                              __shfl_sync(0xffffffffu, r.first, i2), __shfl_sync(0xffffffffu, r.count, i2));
                    }
                    if (ok) read_list(row, later ? next : -1, off, head, packs, first, count, g0, g1, edges + (side * kBatch + i) * 16);
                }
                ++live;
            }
        }
        if (!ok) {
            if (lane == 0) note_timeout(a.timeouts);
            // the copies in flight land before the CTA's memory goes away
            for (uint32_t i = g > static_cast<uint32_t>(NS) ? g - NS : 0u; i < g; ++i)
                mbar_wait(&bars.full[i % NS], (i / NS) & 1u);
        }
    } else if (warp == kRowWarp) {
        uint32_t live = 0;
        double total = 0.0;
        for (int64_t i = 0; i < my_rows && ok; ++i) {
            const int64_t b = i / kBatch;
            const int side = static_cast<int>(b & 1);
            if (i % kBatch == 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars.meta_full[side], (b >> 1) & 1));
            if (!ok) break;
            const RowMeta& r = metas[side * kBatch + i % kBatch];
            const int64_t row = r.row;
            if (r.w == 0.0) {
                if (rank == 0 && lane == 0) put_empty_row(a, row);
            } else {
                const int par = static_cast<int>(live & 1u);
                const uint32_t phase = (live >> 1) & 1u;
                ok = mbar_wait_cluster(&bars.mail[par], phase);
                if (OP == kLossDistill) ok = ok && mbar_wait(&bars.list_full[par], phase);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                // the partial sums, joined in float64
                const int parts = size * kConsWarps;
                float pm[2], ps[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint64_t v = lane + 32 * k < parts ? mail[par * kMaxCluster * kConsWarps + lane + 32 * k] : 0xff800000ull;
                    pm[k] = __uint_as_float(static_cast<uint32_t>(v));
                    ps[k] = __uint_as_float(static_cast<uint32_t>(v >> 32));
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(&bars.mail[par], mail_bytes);  // for the row after the next
                float mf = warp_max(fmaxf(pm[0], pm[1]));
                const ListInfo* li = &lists[par];
                if (OP == kLossDistill) mf = fmaxf(mf, li->x_max);
                const double m = mf;
                if constexpr (OP == kLossToken) {
                    // nobody waits for these: joined in float64
                    double s = 0.0;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        s += pm[k] == -INFINITY ? static_cast<double>(ps[k])  // 0, or NaN
                                                : ps[k] * (pm[k] == mf ? 1.0 : exp((static_cast<double>(pm[k]) - mf) * a.inv_temp));
                    s = warp_sum(s);
                    if (mf == INFINITY) s = quiet_nan();
                    if (lane == 0) {
                        mbar_arrive(&bars.coef[par]);
                        if (rank == 0) {
                            const double log_s = log(s);
                            put_row(a, kLrLogp, row, r.target >= 0 ? (r.xt - m) * a.inv_temp - log_s : quiet_nan());
                            put_row(a, kLrLse, row, m * a.inv_temp + log_s);
                        }
                    }
                } else {
                    // Every consumer of the cluster waits from here to the coefficient, so only what it needs is
                    // computed first: no logarithm, and the row's losses after it is published.
                    float part = 0.f;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        part += pm[k] == -INFINITY ? ps[k] : ps[k] * (pm[k] == mf ? 1.f : exp_one(a, pm[k], mf));
                    Coef c;
                    c.m = mf;
                    c.at_target = c.pad_ = 0.f;
                    auto publish = [&]() {
                        if (lane == 0) {
                            coefs[par] = c;
                            mbar_arrive(&bars.coef[par]);
                        }
                    };
                    if constexpr (OP == kLossPolicy) {
                        // s relative to the target's logit instead of the maximum: r = exp(-old) / s', p_t = 1 / s'
                        const double lift = exp((m - r.xt) * a.inv_temp);
                        const double s = mf == INFINITY ? quiet_nan() : static_cast<double>(warp_sum(part));
                        const double st = s * lift;
                        const double pt = 1.0 / st;
                        double ratio = r.exp_old * pt, ed = r.exp_ref * st - 1.0, rest = 1.0 - pt, logp = 0.0;
                        const bool far = !(st < 1e300 && r.exp_old < 1e300 && r.exp_old > 1e-300 && r.exp_ref < 1e300) || r.target < 0;
                        if (far) {  // numbers outside these forms' range: through the logarithm
                            logp = r.target >= 0 ? (r.xt - m) * a.inv_temp - log(s) : quiet_nan();
                            ratio = exp(logp - r.old);
                            ed = expm1(r.ref - logp);
                            rest = -expm1(logp);
                        }
                        const double g = policy_terms(a, r.w, r.adv, ratio, 0.0, ed).g;
                        c.a = -static_cast<float>(g) / static_cast<float>(s);
                        c.at_target = static_cast<float>(g * rest);
                        publish();
                        if (rank == 0 && lane == 0) {
                            if (!far) logp = (r.xt - m) * a.inv_temp - log(s);
                            const double d = r.ref - logp;
                            const PolicyTerms t = policy_terms(a, r.w, r.adv, ratio, d, a.ptr[kLrRef] ? expm1(d) : 0.0);
                            put_row(a, kLrLogp, row, logp);
                            put_row(a, kLrKl, row, t.kl);
                            put_row(a, kLrRowLoss, row, t.loss);
                            total += r.w * t.loss;
                        }
                    } else {
                        const double s_rest = mf == INFINITY ? quiet_nan() : static_cast<double>(warp_sum(part));
                        const double s = s_rest + (li->count ? li->named * exp_one(a, li->x_max, mf) : 0.0);
                        const bool counts = li->count > 0;
                        double big_q;
                        c.a = static_cast<float>(distill_slope(a, r.w, s, s_rest, li->mass, li->count == a.cols, big_q));
                        if (!(s > 0.0)) c.a = NAN;
                        if (!counts) c.a = 0.f;
                        publish();
                        if (rank == 0 && lane == 0) {
                            const double log_s = log(s);
                            const double cross = li->q_logq - a.inv_temp * (li->q_x + (li->ref - m) * li->mass) + li->mass * log_s;
                            double loss = distill_loss_of(a, s, s_rest, cross, li->mass, li->count == a.cols);
                            if (!(s > 0.0)) loss = quiet_nan();
                            if (!counts) loss = 0.0;
                            put_row(a, kLrRowLoss, row, loss);
                            if (counts) total += r.w * loss;
                        }
                        __syncwarp();
                        // The named elements of this CTA's slice, over what the consumers have written there.
                        T* G = static_cast<T*>(a.ptr[kLrGrad]);
                        if (G && counts) {
                            ok = __all_sync(0xffffffffu, mbar_wait(&bars.done[par], phase));
                            if (!ok) break;
                            T* gr = G + r.g_off;
                            const int first = r.first, count = r.count;
                            const int* e_idx = reinterpret_cast<const int*>(sm + L::kEntries + static_cast<size_t>(par) * 12 * a.top);
                            const float* e_x = reinterpret_cast<const float*>(e_idx + a.top);
                            const float* e_q = e_x + a.top;
                            const float scale = static_cast<float>(r.w * a.inv_temp), p_scale = static_cast<float>(big_q / s);
                            // a bad row is NaN throughout: its named columns too, whoever found it
                            const float poison = c.a == c.a ? 0.f : c.a;
                            for (int k = lane; k < a.top; k += 32) {
                                const int j = e_idx[k];
                                if (j < 0) continue;
                                const int body = j - r.head;
                                const bool mine = body >= 0 && body < r.packs * VE ? body / VE >= first && body / VE < first + count
                                                                                   : rank == 0;
                                if (mine) gr[j * a.g_in] = LossElem<T>::down(scale * (exp_one(a, e_x[k], mf) * p_scale - e_q[k]) + poison);
                            }
                        }
                    }
                }
                __syncwarp();
                if (OP == kLossDistill && lane == 0) mbar_arrive(&bars.list_empty[par]);
                ++live;
            }
            __syncwarp();
            if (lane == 0 && (i % kBatch == kBatch - 1 || i + 1 == my_rows)) mbar_arrive(&bars.meta_empty[side]);
        }
        if (!ok && lane == 0) note_timeout(a.timeouts);
        if (a.partials && rank == 0 && lane == 0) a.partials[cluster] = total;
    } else {
        // ---- consumers
        const int t = threadIdx.x;
        const ExpConst kc = exp_const(a);
        uint32_t g = 0, live = 0;
        for (int64_t i = 0; i < my_rows && ok; ++i) {
            const int64_t b = i / kBatch;
            const int side = static_cast<int>(b & 1);
            if (i % kBatch == 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars.meta_full[side], (b >> 1) & 1));
            if (!ok) break;
            const RowMeta& r = metas[side * kBatch + i % kBatch];
            const int first = r.first, count = r.count;
            T* gr = a.ptr[kLrGrad] ? static_cast<T*>(a.ptr[kLrGrad]) + r.g_off : nullptr;
            // Packs are stored whole where the gradient's rows are aligned like the logits', element by element
            // elsewhere (which costs eight times the store instructions, and takes any stride).
            T* gs = gr + (r.head + static_cast<int64_t>(first) * VE) * a.g_in;
            const bool whole = a.g_in == 1 && (reinterpret_cast<uintptr_t>(gs) & 15) == 0;
            auto put_pack = [&](int p, const uint4& o) {
                if (whole) {
                    reinterpret_cast<uint4*>(gs)[p] = o;
                } else {
                    const T* ov = reinterpret_cast<const T*>(&o);
                    T* dst = gs + static_cast<int64_t>(p) * VE * a.g_in;
#pragma unroll
                    for (int k = 0; k < VE; ++k) dst[k * a.g_in] = ov[k];
                }
            };
            const bool edge = rank == 0 && t < 16;
            const int64_t edge_at = edge ? edge_position(a, r.head, r.packs, VE, t) : -1;
            auto zeros = [&]() {
                if (!gr) return;
                for (int p = t; p < count; p += kCons) put_pack(p, make_uint4(0u, 0u, 0u, 0u));
                if (edge_at >= 0) gr[edge_at * a.g_in] = LossElem<T>::down(0.f);
            };
            if (r.w == 0.0) {
                zeros();
            } else if constexpr (OP == kLossToken) {
                // Nothing is written back, so the slice is folded stage by stage, whatever its length: the warp
                // keeps one maximum, and its sum is brought down to a new one when that grows (a few times a row).
                float m = warp_max(edge_at >= 0 ? edges[(side * kBatch + i % kBatch) * 16 + t] : -INFINITY);
                F2 sum = f2(edge_at >= 0 ? exp_one(a, edges[(side * kBatch + i % kBatch) * 16 + t], m == -INFINITY ? 0.f : m) : 0.f, 0.f);
                for (int p0 = 0; p0 < count; p0 += L::kChunkPacks, ++g) {
                    const int slot = static_cast<int>(g % NS);
                    ok = __all_sync(0xffffffffu, mbar_wait(&bars.full[slot], (g / NS) & 1u));
                    if (!ok) break;
                    const uint4* st = reinterpret_cast<const uint4*>(sm + static_cast<size_t>(slot) * L::kStage);
                    uint4 raw[CP];
                    float mx = -INFINITY;
#pragma unroll
                    for (int u = 0; u < CP; ++u) {
                        raw[u] = p0 + u * kCons + t < count ? st[u * kCons + t] : P::lowest();
                        mx = fmaxf(mx, P::max(raw[u]));
                    }
                    release_stage(&bars.empty[slot], lane);
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
                float s0, s1;
                un(sum, s0, s1);
                const float s = warp_sum(s0 + s1);
                // the mailbox has two sides: the row before the last one must have been read, everywhere
                if (ok && live > 0)
                    ok = __all_sync(0xffffffffu, mbar_wait(&bars.coef[(live - 1) & 1u], ((live - 1) >> 1) & 1u));
                if (!ok) break;
                const int par = static_cast<int>(live & 1u);
                if (lane < size)
                    send8(&mail[par * kMaxCluster * kConsWarps + rank * kConsWarps + warp], &bars.mail[par], lane,
                          static_cast<uint64_t>(__float_as_uint(m)) | static_cast<uint64_t>(__float_as_uint(s)) << 32);
                ++live;
            } else {
                const int par = static_cast<int>(live & 1u);
                const uint32_t phase = (live >> 1) & 1u;
                if (OP == kLossDistill) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&bars.list_full[par], phase));
                    if (!ok) break;
                }
                // the slice, out of the ring
                uint4 raw[RP];
                float mx = -INFINITY;
#pragma unroll
                for (int ch = 0; ch < L::NCH; ++ch) {
                    if (ch * L::kChunkPacks < count) {
                        const int slot = static_cast<int>(g % NS);
                        ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars.full[slot], (g / NS) & 1u));
                        const uint4* st = reinterpret_cast<const uint4*>(sm + static_cast<size_t>(slot) * L::kStage);
#pragma unroll
                        for (int u = 0; u < CP; ++u) {
                            const int p = ch * L::kChunkPacks + u * kCons + t;
                            raw[ch * CP + u] = ok && p < count ? st[u * kCons + t] : P::lowest();
                        }
                        ++g;
                    } else {
#pragma unroll
                        for (int u = 0; u < CP; ++u) raw[ch * CP + u] = P::lowest();
                    }
                }
                if (!ok) break;
                float xe = -INFINITY;
                if (edge_at >= 0)
                    xe = edges[(side * kBatch + i % kBatch) * 16 + t];
#pragma unroll
                for (int p = 0; p < RP; ++p) mx = fmaxf(mx, P::max(raw[p]));
                const float mw = warp_max(fmaxf(mx, xe));
                const float at = mw == -INFINITY ? 0.f : mw;
                const F2 minus = f2(-at, -at);
                F2 e[RP][VE / 2];
                F2 acc0 = f2(0.f, 0.f), acc1 = f2(0.f, 0.f);
#pragma unroll
                for (int p = 0; p < RP; ++p) {
                    P::up(raw[p], e[p]);
#pragma unroll
                    for (int h = 0; h < VE / 2; ++h) {
                        e[p][h] = exp_pair(e[p][h], minus, kc);
                        if (h & 1) acc1 = add2(acc1, e[p][h]);
                        else acc0 = add2(acc0, e[p][h]);
                    }
                }
                const float ee = exp_one(a, xe, at);
                float s0, s1;
                un(add2(acc0, acc1), s0, s1);
                float s = warp_sum(s0 + s1 + ee);
                if (OP == kLossDistill && warp == 0 && lists[par].bad) s = NAN;
                if (lane < size)
                    send8(&mail[par * kMaxCluster * kConsWarps + rank * kConsWarps + warp], &bars.mail[par], lane,
                          static_cast<uint64_t>(__float_as_uint(mw)) | static_cast<uint64_t>(__float_as_uint(s)) << 32);
                // every lane's reads have arrived here: their values are in the sum
                release_fence();
                if (lane == 0)
                    for (uint32_t k = g - static_cast<uint32_t>((count + L::kChunkPacks - 1) / L::kChunkPacks); k != g; ++k)
                        mbar_arrive(&bars.empty[k % NS]);
                ok = __all_sync(0xffffffffu, mbar_wait(&bars.coef[par], phase));
                if (!ok) break;
                const Coef c = coefs[par];
                if (OP == kLossDistill && lists[par].count == 0) {
                    zeros();
                } else if (gr) {
                    const float f = c.a * exp_one(a, mw, c.m);
                    const F2 ff = f2(f, f);
                    const int tb = r.target - r.head;  // the target among the whole packs
                    const int tp = OP == kLossPolicy && tb >= 0 && r.target >= 0 ? tb / VE - first : -1;
#pragma unroll
                    for (int p = 0; p < RP; ++p) {
                        const int pk = p * kCons + t;
                        if (pk < count) {
#pragma unroll
                            for (int h = 0; h < VE / 2; ++h) e[p][h] = mul2(e[p][h], ff);
                            if (OP == kLossPolicy && pk == tp) {
#pragma unroll
                                for (int h = 0; h < VE / 2; ++h) {
                                    float x0, x1;
                                    un(e[p][h], x0, x1);
                                    if (tb % VE == 2 * h) x0 = c.at_target;
                                    if (tb % VE == 2 * h + 1) x1 = c.at_target;
                                    e[p][h] = f2(x0, x1);
                                }
                            }
                            put_pack(pk, P::down(e[p]));
                        }
                    }
                    if (edge_at >= 0)
                        gr[edge_at * a.g_in] = LossElem<T>::down(OP == kLossPolicy && r.target == edge_at ? c.at_target : ee * f);
                }
                if (OP == kLossDistill) {
                    __syncwarp();  // the warp's stores are ordered before the row warp's
                    if (lane == 0) {
                        mbar_arrive(&bars.list_empty[par]);
                        mbar_arrive(&bars.done[par]);
                    }
                }
                ++live;
            }
            __syncwarp();
            if (lane == 0 && (i % kBatch == kBatch - 1 || i + 1 == my_rows)) mbar_arrive(&bars.meta_empty[side]);
        }
        if (!ok && lane == 0) note_timeout(a.timeouts);
    }
    allow_dependents();
    leave_cluster(ok);
}

// ------------------------------------------------------------------------------------------------
// the backward pass of the log-probabilities

struct PullMeta {
    long long g_off;
    float at, shift, a, at_target;  // backward_row
    int target, zero;
    int head, packs;
};

template <class T, int CP, int NS> struct PullLayout {
    static constexpr int kChunkPacks = CP * kCons;
    static constexpr size_t kStage = static_cast<size_t>(kChunkPacks) * 16;
    static constexpr size_t kMeta = NS * kStage;  // PullMeta [2][kBatch]
    static constexpr size_t kEdge = kMeta + 2 * kBatch * sizeof(PullMeta);
    static constexpr size_t kBars = kEdge + 2 * kBatch * 16 * sizeof(float);
    static constexpr size_t kBytes = kBars + (2 * NS + 4) * 8;
};

// g_j = a exp((x_j - at) / T) 2^shift with numbers that are known when the row begins, so a row is a stream:
// out of the ring, through one exponential, to memory. CTA (row group, part): the parts of a row are
// independent. One producer warp, eight consumer warps; bound by the memory.
template <class T, int CP, int NS, int PER_SM>
__global__ void __launch_bounds__(kCons + 32, PER_SM) loss_pull_kernel(const __grid_constant__ LossArgs a, int parts) {
    using L = PullLayout<T, CP, NS>;
    using P = PackOf<T>;
    constexpr int VE = P::VE;
    extern __shared__ __align__(128) unsigned char sm[];
    PullMeta* metas = reinterpret_cast<PullMeta*>(sm + L::kMeta);
    float* edges = reinterpret_cast<float*>(sm + L::kEdge);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::kBars);
    uint64_t* empty = full + NS;
    uint64_t* meta_full = empty + NS;
    uint64_t* meta_empty = meta_full + 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kConsWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&meta_full[i], 1);
            mbar_init(&meta_empty[i], kConsWarps);
        }
        mbar_fence_init();
    }
    __syncthreads();
    dependent_wait();
    const int rank = static_cast<int>(blockIdx.x) % parts;
    const int64_t group = blockIdx.x / parts, groups = gridDim.x / parts;
    const int64_t my_rows = group < a.rows ? (a.rows - group + groups - 1) / groups : 0;
    const T* X = static_cast<const T*>(a.ptr[kLrX]);
    bool ok = true;
    uint32_t g = 0;
    if (warp == kProducer) {
        for (int64_t b = 0; b * kBatch < my_rows && ok; ++b) {
            const int side = static_cast<int>(b & 1);
            const int n = static_cast<int>(min(static_cast<int64_t>(kBatch), my_rows - b * kBatch));
            ok = __all_sync(0xffffffffu, mbar_wait(&meta_empty[side], ((b >> 1) & 1) ^ 1));
            if (!ok) break;
            int64_t x_off = 0;
            PullMeta r{};
            if (lane < n) {
                const int64_t row = group + (b * kBatch + lane) * groups;
                x_off = loss_offset(a, kLrX, row);
                r.g_off = loss_offset(a, kLrGrad, row);
                const int64_t head = ((16 - (reinterpret_cast<uintptr_t>(X + x_off) & 15)) & 15) / sizeof(T);
                r.head = static_cast<int>(head < a.cols ? head : a.cols);
                r.packs = static_cast<int>((a.cols - r.head) / VE);
                const BackwardRow<float> c = backward_row<T>(a, row, X + x_off);
                r.at = c.at;
                r.shift = c.shift;
                r.a = c.a;
                r.at_target = c.at_target;
                r.target = static_cast<int>(c.target);
                r.zero = c.zero;
                metas[side * kBatch + lane] = r;
            }
            if (rank == 0) {
                for (int i = 0; i < n; ++i) {
                    const int64_t off = __shfl_sync(0xffffffffu, x_off, i);
                    const int head = __shfl_sync(0xffffffffu, r.head, i), packs = __shfl_sync(0xffffffffu, r.packs, i);
                    const bool zero = __shfl_sync(0xffffffffu, r.zero, i);
                    if (lane < 16) {
                        const int64_t at = edge_position(a, head, packs, VE, lane);
                        if (at >= 0 && !zero) edges[(side * kBatch + i) * 16 + lane] = LossElem<T>::up(X[off + at]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&meta_full[side]);
            for (int i = 0; i < n && ok; ++i) {
                const int64_t off = __shfl_sync(0xffffffffu, x_off, i);
                const int head = __shfl_sync(0xffffffffu, r.head, i), packs = __shfl_sync(0xffffffffu, r.packs, i);
                if (__shfl_sync(0xffffffffu, r.zero, i)) continue;
                int first, count;
                slice_of(packs, rank, parts, first, count);
                const T* src = X + off + head + static_cast<int64_t>(first) * VE;
                for (int p = 0; p < count; p += L::kChunkPacks, ++g) {
                    const int slot = static_cast<int>(g % NS);
                    ok = __all_sync(0xffffffffu, mbar_wait(&empty[slot], ((g / NS) & 1u) ^ 1u));
                    if (!ok) break;
                    const uint32_t bytes = static_cast<uint32_t>(min(L::kChunkPacks, count - p)) * 16u;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&full[slot], bytes);
                        bulk_load(sm + static_cast<size_t>(slot) * L::kStage, src + static_cast<int64_t>(p) * VE, bytes, &full[slot]);
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok) {
            if (lane == 0) note_timeout(a.timeouts);
            for (uint32_t i = g > static_cast<uint32_t>(NS) ? g - NS : 0u; i < g; ++i)
                mbar_wait(&full[i % NS], (i / NS) & 1u);
        }
        return;
    }
    const int t = threadIdx.x;
    const F2 c2 = f2(a.c2, a.c2);
    for (int64_t i = 0; i < my_rows; ++i) {
        const int64_t b = i / kBatch;
        const int side = static_cast<int>(b & 1);
        if (i % kBatch == 0) ok = __all_sync(0xffffffffu, mbar_wait(&meta_full[side], (b >> 1) & 1));
        if (!ok) break;
        const PullMeta r = metas[side * kBatch + i % kBatch];
        int first, count;
        slice_of(r.packs, rank, parts, first, count);
        T* gr = static_cast<T*>(a.ptr[kLrGrad]) + r.g_off;
        T* gs = gr + (r.head + static_cast<int64_t>(first) * VE) * a.g_in;
        const bool whole = a.g_in == 1 && (reinterpret_cast<uintptr_t>(gs) & 15) == 0;
        auto put_pack = [&](int p, const uint4& o) {
            if (whole) {
                reinterpret_cast<uint4*>(gs)[p] = o;
            } else {
                const T* ov = reinterpret_cast<const T*>(&o);
                T* dst = gs + static_cast<int64_t>(p) * VE * a.g_in;
#pragma unroll
                for (int k = 0; k < VE; ++k) dst[k * a.g_in] = ov[k];
            }
        };
        const int64_t edge_at = rank == 0 && t < 16 ? edge_position(a, r.head, r.packs, VE, t) : -1;
        if (edge_at >= 0) {
            const float x = edges[(side * kBatch + i % kBatch) * 16 + t];
            const float v = r.zero ? 0.f : r.target == edge_at ? r.at_target : r.a * row_exp_shifted(a, x, r.at, r.shift);
            gr[edge_at * a.g_in] = LossElem<T>::down(v);
        }
        if (r.zero) {
            for (int p = t; p < count; p += kCons) put_pack(p, make_uint4(0u, 0u, 0u, 0u));
        } else {
            const F2 minus = f2(-r.at, -r.at), shift = f2(r.shift, r.shift), ga = f2(r.a, r.a);
            const int tb = r.target - r.head;
            const int tp = r.target >= 0 && tb >= 0 ? tb / VE - first : -1;
            for (int p0 = 0; p0 < count; p0 += L::kChunkPacks, ++g) {
                const int slot = static_cast<int>(g % NS);
                ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], (g / NS) & 1u));
                if (!ok) break;
                const uint4* st = reinterpret_cast<const uint4*>(sm + static_cast<size_t>(slot) * L::kStage);
                uint4 raw[CP];
#pragma unroll
                for (int u = 0; u < CP; ++u) raw[u] = p0 + u * kCons + t < count ? st[u * kCons + t] : P::lowest();
                release_stage(&empty[slot], lane);
#pragma unroll
                for (int u = 0; u < CP; ++u) {
                    const int pk = p0 + u * kCons + t;
                    if (pk >= count) continue;
                    F2 e[VE / 2];
                    P::up(raw[u], e);
#pragma unroll
                    for (int h = 0; h < VE / 2; ++h) {
                        float x0, x1;
                        un(fma2(add2(e[h], minus), c2, shift), x0, x1);
                        un(mul2(f2(exp2_fast(x0), exp2_fast(x1)), ga), x0, x1);
                        if (pk == tp) {
                            if (tb % VE == 2 * h) x0 = r.at_target;
                            if (tb % VE == 2 * h + 1) x1 = r.at_target;
                        }
                        e[h] = f2(x0, x1);
                    }
                    put_pack(pk, P::down(e));
                }
            }
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0 && (i % kBatch == kBatch - 1 || i + 1 == my_rows)) mbar_arrive(&meta_empty[side]);
    }
    if (!ok && lane == 0) note_timeout(a.timeouts);
    allow_dependents();
}

// ------------------------------------------------------------------------------------------------
// host side

template <class... Ps> int launch_cluster(void (*fn)(Ps...), unsigned grid, int cluster, size_t smem, cudaStream_t st,
                                          const LossArgs& a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, a);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(CTB_ERR_CUDA, std::string("loss rows: ") + cudaGetErrorString(e));
    }
    count_launch();
    return CTB_OK;
}

// How many clusters of `cluster` CTAs are resident at once on the current device (cached). Also opts the
// kernel in to its shared memory there.
int resident_blocks(const void* fn, int threads, int cluster, size_t smem, int* out) {
    static std::mutex mu;
    static std::map<std::tuple<const void*, int, int, size_t>, int> cache;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("loss rows device");
    const auto key = std::make_tuple(fn, dev, cluster, smem);
    std::lock_guard<std::mutex> lock(mu);
    auto it = cache.find(key);
    if (it == cache.end()) {
        // the most that any call may ask for, so that no later call lowers it under a concurrent launch
        if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) != cudaSuccess)
            return check_launch("loss rows smem attribute");
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(cluster));
        cfg.blockDim = dim3(static_cast<unsigned>(threads));
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) return check_launch("loss rows occupancy");
        it = cache.emplace(key, n < 1 ? 1 : n).first;
    }
    *out = it->second;
    return CTB_OK;
}

template <class T, int OP, int E, int CP, int NS, int PER_SM> int hold_typed(const LossArgs& a, int cluster, int* parts, cudaStream_t st) {
    using L = Layout<T, E, CP, NS>;
    const size_t smem = L::bytes(OP, a.top);
    auto fn = loss_rows_kernel<T, OP, E, CP, NS, PER_SM>;
    int n = 0;
    if (int rc = resident_blocks(reinterpret_cast<const void*>(fn), kThreads, cluster, smem, &n)) return rc;
    int64_t clusters = n < a.rows ? n : a.rows;
    if (clusters > kLossMaxCtas) clusters = kLossMaxCtas;
    *parts = static_cast<int>(clusters);
    return launch_cluster(fn, static_cast<unsigned>(clusters * cluster), cluster, smem, st, a);
}

template <class T, int OP> int hold_sized(const LossArgs& a, int* parts, cudaStream_t st) {
    constexpr int VE = PackOf<T>::VE;
    const int64_t packs = a.cols / VE;
    auto need = [&](int e) { return static_cast<int>((packs + static_cast<int64_t>(kCons) * (e / VE) - 1) / (static_cast<int64_t>(kCons) * (e / VE))); };
    if (need(16) <= 1) return hold_typed<T, OP, 16, 16 / VE, 4, OP == kLossDistill ? 3 : 4>(a, 1, parts, st);
    const int c = need(64);
    return hold_typed<T, OP, 64, 4, 6, 2>(a, c, parts, st);
}

// Log-probabilities: a CTA streams a row of any length, so rows are split only where there are too few of
// them to give every SM two, and never below a stage a CTA.
template <class T> int stream_sized(const LossArgs& a, int* parts, cudaStream_t st) {
    const int64_t want = (2 * static_cast<int64_t>(sm_count()) + a.rows - 1) / a.rows;
    const int64_t stages = a.cols / PackOf<T>::VE / (4 * kCons);
    int64_t c = want < stages ? want : stages;
    c = c < 1 ? 1 : c > kMaxCluster ? kMaxCluster : c;
    return hold_typed<T, kLossToken, 4 * PackOf<T>::VE, 4, 6, 2>(a, static_cast<int>(c), parts, st);
}

// Whether the gradient lies over the logits: a row's parts then must not run apart, because each of them
// reads the target's logit, and one of them overwrites it.
bool in_place(const LossArgs& a) {
    auto range = [&](int view, int64_t inner, uintptr_t& lo, uintptr_t& hi) {
        const int64_t size = static_cast<int64_t>(dtype_size(a.dtype[kLrX]));
        int64_t down = inner < 0 ? (a.cols - 1) * inner : 0, up = inner > 0 ? (a.cols - 1) * inner : 0;
        for (int d = 0; d < a.rank; ++d) {
            const int64_t reach = (static_cast<int64_t>(a.ext[d]) - 1) * a.stride[view][d];
            (reach < 0 ? down : up) += reach;
        }
        lo = reinterpret_cast<uintptr_t>(a.ptr[view]) + down * size;
        hi = reinterpret_cast<uintptr_t>(a.ptr[view]) + (up + 1) * size;
    };
    uintptr_t xl, xh, gl, gh;
    range(kLrX, a.x_in, xl, xh);
    range(kLrGrad, a.g_in, gl, gh);
    return xl < gh && gl < xh;
}

template <class T> int pull_typed(const LossArgs& a, cudaStream_t st) {
    constexpr int CP = 4, NS = 6, PER_SM = 2;
    using L = PullLayout<T, CP, NS>;
    auto fn = loss_pull_kernel<T, CP, NS, PER_SM>;
    int resident = 0;
    if (int rc = resident_blocks(reinterpret_cast<const void*>(fn), kCons + 32, 1, L::kBytes, &resident)) return rc;
    // Parts of a row: stages enough that one CTA's last row is a small share of its work.
    const int64_t stages = (a.cols / PackOf<T>::VE + L::kChunkPacks - 1) / L::kChunkPacks;
    int64_t parts = 1;
    if (!in_place(a)) {
        while (parts < 16 && parts * 2 <= stages && (parts * 4 < stages || a.rows * parts < 8 * static_cast<int64_t>(resident))) parts *= 2;
    }
    int64_t groups = (resident + parts - 1) / parts;
    if (groups > a.rows) groups = a.rows;
    launch_dependent(fn, static_cast<unsigned>(groups * parts), kCons + 32, L::kBytes, st, a, static_cast<int>(parts));
    count_launch();
    return check_launch("loss backward");
}

}  // namespace

// Whether the kernels of this file take the call: float32 or bfloat16 rows of unit stride; for a loss with
// its gradient, rows that a cluster can hold.
bool loss_rows_fit(const LossArgs& a, bool held) {
    if (a.dtype[kLrX] != CTB_FLOAT32 && a.dtype[kLrX] != CTB_BFLOAT16) return false;
    if (a.cols > 1 && a.x_in != 1) return false;
    return !held || a.cols <= static_cast<int64_t>(kMaxCluster) * kCons * 64;
}

int loss_backward_fast(const LossArgs& a, cudaStream_t st) {
    return a.dtype[kLrX] == CTB_BFLOAT16 ? pull_typed<__nv_bfloat16>(a, st) : pull_typed<float>(a, st);
}

int loss_rows_fast(const LossPlan& p, int* parts, cudaStream_t st) {
    const LossArgs& a = p.args;
    const bool bf = a.dtype[kLrX] == CTB_BFLOAT16;
    if (p.op == kLossToken) return bf ? stream_sized<__nv_bfloat16>(a, parts, st) : stream_sized<float>(a, parts, st);
    if (p.op == kLossPolicy)
        return bf ? hold_sized<__nv_bfloat16, kLossPolicy>(a, parts, st) : hold_sized<float, kLossPolicy>(a, parts, st);
    return bf ? hold_sized<__nv_bfloat16, kLossDistill>(a, parts, st) : hold_sized<float, kLossDistill>(a, parts, st);
}

}  // namespace ctb
