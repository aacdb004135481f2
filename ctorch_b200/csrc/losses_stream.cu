// losses_stream.cu — log-probabilities of chosen tokens over rows of unit stride (float32, bfloat16), and their
// backward pass: both stream rows through a shared-memory ring (losses_ring.cuh), forward to a sum a row,
// backward through one exponential back to memory.
#include <map>
#include <mutex>
#include <string>
#include <tuple>

#include "losses_ring.cuh"

namespace ctb {

namespace {

constexpr int kConsWarps = 8;
constexpr int kCons = kConsWarps * 32;
constexpr int kProducer = kConsWarps;  // warp numbers
constexpr int kRowWarp = kConsWarps + 1;
constexpr int kThreads = kCons + 64;

// ------------------------------------------------------------------------------------------------
// forward

struct TokenMeta {
    double w, xt;
    long long row;
    int target, head, packs, first, count, pad_;
};

constexpr int kSides = 4;  // rows whose sums may be on their way at once

template <int CP, int NS> struct TokenLayout {
    static constexpr int kChunkPacks = CP * kCons;
    static constexpr size_t kStage = static_cast<size_t>(kChunkPacks) * 16;
    static constexpr size_t kMail = NS * kStage;                                    // uint64 [kSides][kMaxCluster * kConsWarps]
    static constexpr size_t kMeta = kMail + kSides * kMaxCluster * kConsWarps * 8;  // TokenMeta [2][kBatch]
    static constexpr size_t kEdge = kMeta + 2 * kBatch * sizeof(TokenMeta);         // float [2][kBatch][16]
    static constexpr size_t kBars = kEdge + 2 * kBatch * 16 * sizeof(float);
    static constexpr size_t kBytes = kBars + (2 * NS + 4 + kSides + 2) * 8;
};

// A row belongs to a cluster of C CTAs (C = 1 unless there are fewer rows than SMs), a CTA to a slice of it.
// The producer warp streams the slices of the coming rows through the ring; eight consumer warps fold them,
// stage by stage, each with its own maximum, and send (maximum, sum) to every CTA of the cluster (st.async into
// its mailbox, completion counted on its mbarrier); the row warp joins them in float64 and keeps the row's
// sum until the batch's 32 rows are finished together. Nobody waits for it but the row after the next. It takes
// what losses_short.cu does not: B200, [3000, 32768] bf16 44 us, [1000, 131072] bf16 55 us (4.8 TB/s).
template <class T, int CP, int NS, int PER_SM>
__global__ void __launch_bounds__(kThreads, PER_SM) loss_token_kernel(const __grid_constant__ LossArgs a) {
    using L = TokenLayout<CP, NS>;
    using P = PackOf<T>;
    constexpr int VE = P::VE;
    extern __shared__ __align__(128) unsigned char sm[];
    uint64_t* mail = reinterpret_cast<uint64_t*>(sm + L::kMail);
    TokenMeta* metas = reinterpret_cast<TokenMeta*>(sm + L::kMeta);
    float* edges = reinterpret_cast<float*>(sm + L::kEdge);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::kBars);
    uint64_t* empty = full + NS;
    uint64_t* meta_full = empty + NS;
    uint64_t* meta_empty = meta_full + 2;
    uint64_t* mail_full = meta_empty + 2;
    uint64_t* joined = mail_full + kSides;  // the row's side of the mailbox has been read
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank()), size = static_cast<int>(cluster_size());
    const uint32_t mail_bytes = static_cast<uint32_t>(size) * kConsWarps * 8;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kConsWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&meta_full[i], 1);
            mbar_init(&meta_empty[i], kConsWarps + 1);
            mbar_init(&joined[i], 1);
        }
        for (int i = 0; i < kSides; ++i) mbar_init(&mail_full[i], 1);
        mbar_fence_init();
        for (int i = 0; i < kSides; ++i) mbar_arrive_expect_tx(&mail_full[i], mail_bytes);
    }
    __syncthreads();
    cluster_sync();
    dependent_wait();  // the previous kernel in the stream has completed and its writes are visible

    const int64_t cluster = blockIdx.x / size, clusters = gridDim.x / size;
    const int64_t my_rows = cluster < a.rows ? (a.rows - cluster + clusters - 1) / clusters : 0;
    const T* X = static_cast<const T*>(a.ptr[kLrX]);
    bool ok = true;
    uint32_t g = 0;     // stages, of the producer and of each consumer
    uint32_t live = 0;  // rows that count
    if (warp == kProducer) {
        for (int64_t b = 0; b * kBatch < my_rows && ok; ++b) {
            const int side = static_cast<int>(b & 1);
            const int n = static_cast<int>(min(static_cast<int64_t>(kBatch), my_rows - b * kBatch));
            ok = __all_sync(0xffffffffu, wait_phase(&meta_empty[side], ((b >> 1) & 1) ^ 1));
            if (!ok) break;
            int64_t x_off = 0;
            TokenMeta r{};
            if (lane < n) {
                r.row = cluster + (b * kBatch + lane) * clusters;
                r.w = row_weight(a, r.row);
                x_off = loss_offset(a, kLrX, r.row);
                const int64_t head = ((16 - (reinterpret_cast<uintptr_t>(X + x_off) & 15)) & 15) / sizeof(T);
                r.head = static_cast<int>(head < a.cols ? head : a.cols);
                r.packs = static_cast<int>((a.cols - r.head) / VE);
                slice_of(r.packs, rank, size, r.first, r.count);
                r.target = -1;
                if (r.w != 0.0) {
                    const int64_t t = load_index(a.ptr[kLrTarget], a.dtype[kLrTarget], loss_offset(a, kLrTarget, r.row));
                    if (t >= 0 && t < a.cols) {
                        r.target = static_cast<int>(t);
                        r.xt = LossElem<T>::up(X[x_off + t]);
                    } else {
                        note_bad_index(a, t);
                    }
                }
                metas[side * kBatch + lane] = r;
            }
            if (rank == 0) {
                const int behind = r.head + r.packs * VE;
                read_edges(X, x_off, r.w != 0.0 ? edges_of(a, r.head, behind) : 0u, behind, n, lane, edges + side * kBatch * 16);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&meta_full[side]);
            for (int i = 0; i < n && ok; ++i) {
                if (__shfl_sync(0xffffffffu, r.w, i) == 0.0) continue;
                const int64_t off = __shfl_sync(0xffffffffu, x_off, i);
                const int head = __shfl_sync(0xffffffffu, r.head, i);
                const int first = __shfl_sync(0xffffffffu, r.first, i), count = __shfl_sync(0xffffffffu, r.count, i);
                const T* src = X + off + head + static_cast<int64_t>(first) * VE;
                for (int p = 0; p < count; p += L::kChunkPacks, ++g) {
                    const int slot = static_cast<int>(g % NS);
                    ok = __all_sync(0xffffffffu, wait_phase(&empty[slot], ((g / NS) & 1u) ^ 1u));
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
            // the copies in flight land before the CTA's memory goes away
            for (uint32_t i = g > static_cast<uint32_t>(NS) ? g - NS : 0u; i < g; ++i)
                wait_phase(&full[i % NS], (i / NS) & 1u);
        }
    } else if (warp == kRowWarp) {
        // lane i keeps the i-th row of the batch
        double kept_s = 0.0;
        float kept_m = 0.f;
        for (int64_t i = 0; i < my_rows && ok; ++i) {
            const int64_t b = i / kBatch;
            const int side = static_cast<int>(b & 1);
            if (i % kBatch == 0) ok = __all_sync(0xffffffffu, wait_phase(&meta_full[side], (b >> 1) & 1));
            if (!ok) break;
            if (metas[side * kBatch + i % kBatch].w != 0.0) {
                const int ms = static_cast<int>(live % kSides);
                ok = __all_sync(0xffffffffu, wait_phase<true>(&mail_full[ms], (live / kSides) & 1u));
                if (!ok) break;
                const int parts = size * kConsWarps;
                constexpr int kJoin = kMaxCluster * kConsWarps / 32;
                float pm[kJoin], ps[kJoin];
#pragma unroll
                for (int k = 0; k < kJoin; ++k) {
                    const uint64_t v = lane + 32 * k < parts ? mail[ms * kMaxCluster * kConsWarps + lane + 32 * k] : 0xff800000ull;
                    pm[k] = __uint_as_float(static_cast<uint32_t>(v));
                    ps[k] = __uint_as_float(static_cast<uint32_t>(v >> 32));
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive_expect_tx(&mail_full[ms], mail_bytes);  // for the row kSides later
                    mbar_arrive(&joined[live & 1u]);
                }
                float mf = pm[0];
#pragma unroll
                for (int k = 1; k < kJoin; ++k) mf = fmaxf(mf, pm[k]);
                mf = warp_max(mf);
                double s = 0.0;
#pragma unroll
                for (int k = 0; k < kJoin; ++k)
                    if (32 * k < parts)
                        s += pm[k] == -INFINITY ? static_cast<double>(ps[k])  // 0, or NaN
                                                : ps[k] * (pm[k] == mf ? 1.0 : exp((static_cast<double>(pm[k]) - mf) * a.inv_temp));
                s = warp_sum(s);
                if (lane == i % kBatch) {
                    kept_s = mf == INFINITY ? quiet_nan() : s;
                    kept_m = mf;
                }
                ++live;
            }
            if (i % kBatch == kBatch - 1 || i + 1 == my_rows) {
                if (rank == 0 && lane <= i % kBatch) {
                    const TokenMeta& r = metas[side * kBatch + lane];
                    if (r.w == 0.0) {
                        put_empty_row(a, r.row);
                    } else {
                        const double m = kept_m, log_s = log(kept_s);
                        put_row(a, kLrLogp, r.row, r.target >= 0 ? (r.xt - m) * a.inv_temp - log_s : quiet_nan());
                        put_row(a, kLrLse, r.row, m * a.inv_temp + log_s);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&meta_empty[side]);
            }
        }
        if (!ok && lane == 0) note_timeout(a.timeouts);
    } else {
        const int t = threadIdx.x;
        const ExpConst kc = exp_const(a);
        for (int64_t i = 0; i < my_rows && ok; ++i) {
            const int64_t b = i / kBatch;
            const int side = static_cast<int>(b & 1);
            if (i % kBatch == 0) ok = __all_sync(0xffffffffu, wait_phase(&meta_full[side], (b >> 1) & 1));
            if (!ok) break;
            const TokenMeta& r = metas[side * kBatch + i % kBatch];
            if (r.w != 0.0) {
                // The warp keeps one maximum, and its sum is brought down to a new one when that grows (a few times a row).
                const int count = r.count;
                const float xe = rank == 0 && t < 16 ? edges[(side * kBatch + i % kBatch) * 16 + t] : -INFINITY;
                float m = warp_max(xe);
                F2 sum = f2(exp_one(a, xe, m == -INFINITY ? 0.f : m), 0.f);
                for (int p0 = 0; p0 < count; p0 += L::kChunkPacks, ++g) {
                    const int slot = static_cast<int>(g % NS);
                    ok = __all_sync(0xffffffffu, wait_phase(&full[slot], (g / NS) & 1u));
                    if (!ok) break;
                    const uint4* st = reinterpret_cast<const uint4*>(sm + static_cast<size_t>(slot) * L::kStage);
                    uint4 raw[CP];
                    float mx = -INFINITY;
#pragma unroll
                    for (int u = 0; u < CP; ++u) {
                        raw[u] = p0 + u * kCons + t < count ? st[u * kCons + t] : P::lowest();
                        mx = fmaxf(mx, P::max(raw[u]));
                    }
                    mx = warp_max(mx);
                    release_stage(&empty[slot], lane);
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
                // A side of the mailbox is written again four rows later: by then every CTA of the cluster has read it if
                // each warp waits here for its own CTA to have joined the row before the last one.
                if (ok && live >= 2)
                    ok = __all_sync(0xffffffffu, wait_phase(&joined[live & 1u], ((live - 2) >> 1) & 1u));
                if (!ok) break;
                if (lane < size)
                    send8(&mail[(live % kSides * kMaxCluster + rank) * kConsWarps + warp], &mail_full[live % kSides], lane,
                          static_cast<uint64_t>(__float_as_uint(m)) | static_cast<uint64_t>(__float_as_uint(s)) << 32);
                ++live;
            }
            __syncwarp();
            if (lane == 0 && (i % kBatch == kBatch - 1 || i + 1 == my_rows)) mbar_arrive(&meta_empty[side]);
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
// independent. One producer warp, eight consumer warps; bound by the memory (B200, [8192, 50021] f32 557 us,
// 5.9 TB/s in and out). The last rows come first: they are what a forward pass over more than the L2 holds has
// left there.
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
            ok = __all_sync(0xffffffffu, wait_phase(&meta_empty[side], ((b >> 1) & 1) ^ 1));
            if (!ok) break;
            int64_t x_off = 0;
            PullMeta r{};
            if (lane < n) {
                const int64_t row = a.rows - 1 - (group + (b * kBatch + lane) * groups);
                x_off = loss_offset(a, kLrX, row);
                r.g_off = loss_offset(a, kLrGrad, row);
                const int64_t head = ((16 - (reinterpret_cast<uintptr_t>(X + x_off) & 15)) & 15) / sizeof(T);
                r.head = static_cast<int>(head < a.cols ? head : a.cols);
                r.packs = static_cast<int>((a.cols - r.head) / VE);
                const BackwardRow<float> c = backward_row<T>(a, row, X + x_off, row_upstream(a, row));
                r.at = c.at;
                r.shift = c.shift;
                r.a = c.a;
                r.at_target = c.at_target;
                r.target = static_cast<int>(c.target);
                r.zero = c.zero;
                metas[side * kBatch + lane] = r;
            }
            if (rank == 0) {
                const int behind = r.head + r.packs * VE;
                read_edges(X, x_off, lane < n && !r.zero ? edges_of(a, r.head, behind) : 0u, behind, n, lane, edges + side * kBatch * 16);
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
                    ok = __all_sync(0xffffffffu, wait_phase(&empty[slot], ((g / NS) & 1u) ^ 1u));
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
                wait_phase(&full[i % NS], (i / NS) & 1u);
        }
        return;
    }
    const int t = threadIdx.x;
    const F2 c2 = f2(a.c2, a.c2);
    for (int64_t i = 0; i < my_rows; ++i) {
        const int64_t b = i / kBatch;
        const int side = static_cast<int>(b & 1);
        if (i % kBatch == 0) ok = __all_sync(0xffffffffu, wait_phase(&meta_full[side], (b >> 1) & 1));
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
        const int behind = r.head + r.packs * VE;
        const int edge_at = rank == 0 && t < 16 && (edges_of(a, r.head, behind) >> t & 1u) ? edge_column(t, behind) : -1;
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
                ok = __all_sync(0xffffffffu, wait_phase(&full[slot], (g / NS) & 1u));
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

// Log-probabilities: a CTA streams a row of any length, so rows are split only where there are too few of
// them to give every SM two, and never below a stage a CTA.
template <class T> int token_typed(const LossArgs& a, cudaStream_t st) {
    constexpr int CP = 4, NS = 6, PER_SM = 2;
    using L = TokenLayout<CP, NS>;
    const int64_t want = (2 * static_cast<int64_t>(sm_count()) + a.rows - 1) / a.rows;
    const int64_t stages = a.cols / PackOf<T>::VE / L::kChunkPacks;
    int64_t c = want < stages ? want : stages;
    c = c < 1 ? 1 : c > kMaxCluster ? kMaxCluster : c;
    auto fn = loss_token_kernel<T, CP, NS, PER_SM>;
    int n = 0;
    if (int rc = resident_blocks(reinterpret_cast<const void*>(fn), kThreads, static_cast<int>(c), L::kBytes, &n)) return rc;
    const int64_t clusters = n < a.rows ? n : a.rows;
    LossArgs args = a;
    void* argv[1] = {&args};
    return launch_cluster(reinterpret_cast<const void*>(fn), static_cast<unsigned>(clusters * c), kThreads, static_cast<int>(c),
                          L::kBytes, st, argv);
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
    // Rows are split only where there are too few of them for the resident CTAs: parts of a row read its operands
    // each (B200, 2047 rows of 50021 float32: 159 us whole, 168 us in four parts, 184 us in eight).
    const int64_t stages = (a.cols / PackOf<T>::VE + L::kChunkPacks - 1) / L::kChunkPacks;
    int64_t parts = 1;
    while (!in_place(a) && parts * 2 <= stages && parts < 16 && a.rows * parts < 2 * static_cast<int64_t>(resident)) parts *= 2;
    int64_t groups = (resident + parts - 1) / parts;
    if (groups > a.rows) groups = a.rows;
    launch_dependent(fn, static_cast<unsigned>(groups * parts), kCons + 32, L::kBytes, st, a, static_cast<int>(parts));
    count_launch();
    return check_launch("loss backward");
}

}  // namespace

int launch_cluster(const void* fn, unsigned grid, int threads, int cluster, size_t smem, cudaStream_t st, void** args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
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
    const cudaError_t e = cudaLaunchKernelExC(&cfg, fn, args);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(CTB_ERR_CUDA, std::string("loss rows: ") + cudaGetErrorString(e));
    }
    count_launch();
    return CTB_OK;
}

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

// Whether the kernels over rows of unit stride take the call.
bool loss_stream_fit(const LossArgs& a) {
    return (a.dtype[kLrX] == CTB_FLOAT32 || a.dtype[kLrX] == CTB_BFLOAT16) && (a.cols == 1 || a.x_in == 1);
}

int loss_token_stream(const LossArgs& a, cudaStream_t st) {
    return a.dtype[kLrX] == CTB_BFLOAT16 ? token_typed<__nv_bfloat16>(a, st) : token_typed<float>(a, st);
}

int loss_backward_stream(const LossArgs& a, cudaStream_t st) {
    return a.dtype[kLrX] == CTB_BFLOAT16 ? pull_typed<__nv_bfloat16>(a, st) : pull_typed<float>(a, st);
}

}  // namespace ctb
