// losses_short.cu — the losses over rows of unit stride (float32, bfloat16) that a warp takes whole: R rows at a
// time, NP packs of each a lane.
//
// Short rows are bound by what happens once a row, not by their bytes: the ring of losses_stream.cu and
// losses_held.cu hands each of them over between four kinds of warps. Here nothing is handed over. The loads of R rows
// are on their way together, the warp reduces them one after the other, and lanes 0..R-1 do the float64
// arithmetic of a row each, once for R rows. R * NP = 16 packs a lane, two CTAs of eight warps an SM, keep 128 KiB
// of loads on their way, as much as the ring does. A policy row stays in the registers from the first read to the
// gradient; log-probabilities and their backward pass have no second use of it and take longer rows in pieces.
// B200, 16384 bfloat16 rows, us a call against the ring: log-probabilities of 1001 (calls of 15 us are bound by the
// host) 15 against 73, of 4096 32 against 76; with the backward pass 31 against 139 and 110 against 156; policy loss
// of 1024 29 against 64, of 2048 53 against 74, of 4096 85 against 79.
#include "losses_ring.cuh"

namespace ctb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kHeld = 16;  // packs a lane
constexpr int kPull = 3;   // beside LossOp: the backward pass of the log-probabilities

template <class T, int OP, int NP>
__global__ void __launch_bounds__(kThreads, 2) loss_short_kernel(const __grid_constant__ LossArgs a) {
    constexpr int R = kHeld / NP;
    // rows of any length, in pieces of 16 packs a lane
    constexpr bool kChunked = OP != kLossPolicy && R == 1;
    using P = PackOf<T>;
    constexpr int VE = P::VE;
    __shared__ double sums[kWarps];
    dependent_wait();
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarps;
    const T* X = static_cast<const T*>(a.ptr[kLrX]);
    T* G = static_cast<T*>(a.ptr[kLrGrad]);
    const ExpConst kc = exp_const(a);
    double total = 0.0;
    auto get = [&](uint4 (&to)[NP], const T* from, int p0, int packs) {
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            const int p = p0 + u * 32 + lane;
            to[u] = p < packs ? reinterpret_cast<const uint4*>(from)[p] : P::lowest();
        }
    };
    // the backward pass takes the last rows first: they are what a forward pass over more than the L2 holds left there
    auto row_of = [&](int64_t i) { return OP == kPull ? a.rows - 1 - i : i; };
    for (int64_t r0 = (blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5)) * R; r0 < a.rows; r0 += warps * R) {
        const int n = static_cast<int>(min(static_cast<int64_t>(R), a.rows - r0));
        const int64_t row = row_of(r0 + lane);
        // lane r: row r's operands
        int64_t x_off = 0, g_off = 0;
        int head = 0, packs = 0, target = -1;
        double w = 0.0, xt = 0.0;
        float at = 0.f, shift = 0.f, ga = 0.f, at_target = 0.f;
        bool live = false;
        if (lane < n) {
            x_off = loss_offset(a, kLrX, row);
            if (G) g_off = loss_offset(a, kLrGrad, row);
            const int64_t h = ((16 - (reinterpret_cast<uintptr_t>(X + x_off) & 15)) & 15) / sizeof(T);
            head = static_cast<int>(h < a.cols ? h : a.cols);
            packs = static_cast<int>((a.cols - head) / VE);
            w = OP == kPull ? row_upstream(a, row) : row_weight(a, row);
            live = w != 0.0;
        }
        const uint32_t lives = __ballot_sync(0xffffffffu, live);
        uint4 raw[R][NP];
        float edge[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const T* x = X + __shfl_sync(0xffffffffu, x_off, r);
            const int hd = __shfl_sync(0xffffffffu, head, r), pk = __shfl_sync(0xffffffffu, packs, r), behind = hd + pk * VE;
            const bool on = lives >> r & 1u;
            get(raw[r], x + hd, 0, on ? pk : 0);
            edge[r] = -INFINITY;
            if (on && lane < 16 && (edges_of(a, hd, behind) >> lane & 1u)) edge[r] = LossElem<T>::up(x[edge_column(lane, behind)]);
        }
        // the rows are on their way: the other operands, which need more than one load after the other
        double old = 0.0, adv = 0.0, ref = 0.0;
        if (live && OP == kPull) {
            const BackwardRow<float> c = backward_row<T>(a, row, X + x_off, w);
            at = c.at;
            shift = c.shift;
            ga = c.a;
            at_target = c.at_target;
            target = static_cast<int>(c.target);
        } else if (live) {
            if (OP == kLossPolicy) {
                old = row_real(a, kLrOld, row);
                adv = row_real(a, kLrAdv, row);
                if (a.ptr[kLrRef]) ref = row_real(a, kLrRef, row);
            }
            const int64_t t = load_index(a.ptr[kLrTarget], a.dtype[kLrTarget], loss_offset(a, kLrTarget, row));
            if (t >= 0 && t < a.cols) {
                target = static_cast<int>(t);
                xt = LossElem<T>::up(X[x_off + t]);
            } else {
                note_bad_index(a, t);
            }
        }
        if (OP != kPull) {
            float my_m = 0.f, my_s = 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float m = warp_max(edge[r]);
                F2 sum = f2(exp_one(a, edge[r], m == -INFINITY ? 0.f : m), 0.f);
                const T* x = X + __shfl_sync(0xffffffffu, x_off, r) + __shfl_sync(0xffffffffu, head, r);
                const int all = __shfl_sync(0xffffffffu, packs, r), pk = lives >> r & 1u ? all : 0;
                for (int p0 = 0;;) {
                    float mx = m;
#pragma unroll
                    for (int u = 0; u < NP; ++u) mx = fmaxf(mx, P::max(raw[r][u]));
                    mx = warp_max(mx);
                    if (mx > m) {
                        const float down = exp_one(a, m, mx);
                        sum = mul2(sum, f2(down, down));
                        m = mx;
                    }
                    const float from = m == -INFINITY ? 0.f : m;
                    const F2 minus = f2(-from, -from);
                    F2 acc0 = f2(0.f, 0.f), acc1 = f2(0.f, 0.f);
#pragma unroll
                    for (int u = 0; u < NP; ++u) {
                        F2 e[VE / 2];
                        P::up(raw[r][u], e);
#pragma unroll
                        for (int h = 0; h < VE / 2; h += 2) {
                            acc0 = add2(acc0, exp_pair(e[h], minus, kc));
                            acc1 = add2(acc1, exp_pair(e[h + 1], minus, kc));
                        }
                    }
                    sum = add2(sum, add2(acc0, acc1));
                    if constexpr (!kChunked) break;
                    p0 += 32 * NP;
                    if (p0 >= pk) break;
                    get(raw[r], x, p0, pk);
                }
                float s0, s1;
                un(sum, s0, s1);
                const float s = warp_sum(s0 + s1);
                if (lane == r) {
                    my_m = m;
                    my_s = m == INFINITY ? NAN : s;
                }
            }
            if (lane < n && !live) put_empty_row(a, row);
            if (live) {
                const double m = my_m, s = my_s, log_s = log(s);
                const double logp = target >= 0 ? (xt - m) * a.inv_temp - log_s : quiet_nan();
                put_row(a, kLrLogp, row, logp);
                if (OP == kLossToken) {
                    put_row(a, kLrLse, row, m * a.inv_temp + log_s);
                } else {
                    const double d = a.ptr[kLrRef] ? ref - logp : 0.0;
                    const PolicyTerms o = policy_terms(a, w, adv, exp(logp - old), d, a.ptr[kLrRef] ? expm1(d) : 0.0);
                    put_row(a, kLrRowLoss, row, o.loss);
                    put_row(a, kLrKl, row, o.kl);
                    total += w * o.loss;
                    ga = static_cast<float>(-o.g / s);
                    at_target = static_cast<float>(-o.g * expm1(logp));
                    at = my_m;
                }
            }
        }
        if constexpr (OP != kLossToken) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (!G || r >= n) break;
                T* g = G + __shfl_sync(0xffffffffu, g_off, r);
                const int64_t x_r = __shfl_sync(0xffffffffu, x_off, r);
                const int hd = __shfl_sync(0xffffffffu, head, r), pk = __shfl_sync(0xffffffffu, packs, r), behind = hd + pk * VE;
                const int t = __shfl_sync(0xffffffffu, target, r);
                const bool on = lives >> r & 1u;
                const float from = __shfl_sync(0xffffffffu, at, r), by = __shfl_sync(0xffffffffu, shift, r);
                const float fa = __shfl_sync(0xffffffffu, ga, r), ft = __shfl_sync(0xffffffffu, at_target, r);
                const F2 minus = f2(-from, -from), by2 = f2(by, by), fa2 = f2(fa, fa), c2 = f2(a.c2, a.c2);
                const bool whole = a.g_in == 1 && (reinterpret_cast<uintptr_t>(g + hd) & 15) == 0;
                for (int p0 = 0; p0 < pk; p0 += 32 * NP) {
                    if (kChunked && p0 && on) get(raw[r], X + x_r + hd, p0, pk);
                    // without this the compiler keeps the rows' unpacked elements from the sums above, and spills them
#pragma unroll
                    for (int u = 0; u < NP; ++u)
                        asm volatile("" : "+r"(raw[r][u].x), "+r"(raw[r][u].y), "+r"(raw[r][u].z), "+r"(raw[r][u].w));
#pragma unroll
                    for (int u = 0; u < NP; ++u) {
                        const int p = p0 + u * 32 + lane;
                        if (p >= pk) continue;
                        uint4 out = make_uint4(0u, 0u, 0u, 0u);
                        if (on) {
                            const int at_pack = t - hd - p * VE;  // 0..VE-1: the target is in this pack
                            F2 e[VE / 2];
                            P::up(raw[r][u], e);
#pragma unroll
                            for (int h = 0; h < VE / 2; ++h) {
                                F2 y;
                                if (OP == kPull) {
                                    float x0, x1;
                                    un(fma2(add2(e[h], minus), c2, by2), x0, x1);
                                    y = f2(exp2_fast(x0), exp2_fast(x1));
                                } else {
                                    y = exp_pair(e[h], minus, kc);
                                }
                                float y0, y1;
                                un(mul2(y, fa2), y0, y1);
                                if (t >= 0 && at_pack == 2 * h) y0 = ft;
                                if (t >= 0 && at_pack == 2 * h + 1) y1 = ft;
                                e[h] = f2(y0, y1);
                            }
                            out = P::down(e);
                        }
                        if (whole) {
                            reinterpret_cast<uint4*>(g + hd)[p] = out;
                        } else {
                            const T* ov = reinterpret_cast<const T*>(&out);
                            T* dst = g + (hd + p * VE) * a.g_in;
#pragma unroll
                            for (int k = 0; k < VE; ++k) dst[k * a.g_in] = ov[k];
                        }
                    }
                    if (!kChunked) break;
                }
                if (lane < 16 && (edges_of(a, hd, behind) >> lane & 1u)) {
                    const int j = edge_column(lane, behind);
                    const float y = OP == kPull ? row_exp_shifted(a, edge[r], from, by) : exp_one(a, edge[r], from);
                    g[j * a.g_in] = LossElem<T>::down(!on ? 0.f : j == t ? ft : fa * y);
                }
            }
        }
    }
    allow_dependents();
    if (OP == kLossPolicy && a.partials) {
        total = warp_sum(total);
        if (lane == 0) sums[threadIdx.x >> 5] = total;
        __syncthreads();
        if (threadIdx.x == 0) {
            double t = 0.0;
            for (int i = 0; i < kWarps; ++i) t += sums[i];
            a.partials[blockIdx.x] = t;
        }
    }
}

template <class T, int OP, int NP> int sized(const LossArgs& a, int* parts, cudaStream_t st) {
    constexpr int64_t kRows = kWarps * (kHeld / NP);  // rows that a CTA takes at a time
    auto fn = loss_short_kernel<T, OP, NP>;
    const int per_sm = resident_ctas(reinterpret_cast<const void*>(fn), kThreads, 0);
    *parts = static_cast<int>(grid_for((a.rows + kRows - 1) / kRows, per_sm));
    launch_dependent(fn, static_cast<unsigned>(*parts), kThreads, 0, st, a);
    count_launch();
    return check_launch("loss short rows");
}

template <class T, int OP> int typed(const LossArgs& a, int* parts, cudaStream_t st) {
    const int64_t per_lane = (a.cols / PackOf<T>::VE + 31) / 32;
    if (per_lane <= 1) return sized<T, OP, 1>(a, parts, st);
    if (per_lane <= 2) return sized<T, OP, 2>(a, parts, st);
    if (per_lane <= 4) return sized<T, OP, 4>(a, parts, st);
    if constexpr (OP == kLossPolicy) return sized<T, OP, 8>(a, parts, st);
    else return per_lane <= 8 ? sized<T, OP, 8>(a, parts, st) : sized<T, OP, 16>(a, parts, st);
}

template <int OP> int any_type(const LossArgs& a, int* parts, cudaStream_t st) {
    return a.dtype[kLrX] == CTB_BFLOAT16 ? typed<__nv_bfloat16, OP>(a, parts, st) : typed<float, OP>(a, parts, st);
}

}  // namespace

// Which rows a warp takes whole. Policy rows: those of which two fit the registers, 4 KiB (measured above).
// Otherwise rows up to 16 KiB, and longer ones where the last wave of the resident warps is nearly full, since
// each of them is as long as a row (B200, log-probabilities of 32768 bfloat16 against the ring: 4736 rows, two waves,
// 57 us against 64; 8192 rows, 3.5 waves, 100 against 104; 3000 rows, 1.3 waves, 48 against 44). Near the limit of 85%
// the two differ by a few per cent either way; time here over time there, by how full two and three waves are:
//     rows of             78%                      85%                      92%                 100%
//     16384 bfloat16   0.88-0.96, 0.94-0.97   0.88-0.92, 0.91        0.84-0.86, 0.88        0.80-0.82, 0.86-0.87
//     32768            1.02-1.10, 0.99-1.02   0.99-1.05, 0.96-0.97   0.95-0.98, 0.93-0.96   0.92, 0.91-0.96
//     65536            1.06-1.14, 1.01-1.03   1.05-1.07, 0.96-0.97   1.01, 0.92-0.95        0.91-0.95, 0.92-0.93
//     16384 float32    0.99-1.03              0.95-1.00              0.96-0.97              0.92-0.97
// (forward, backward; a single wave is like them forward, 0.93-1.02 backward from 85% on). The
// backward pass of long float32 rows is the ring's (here 1.01-1.12 times as long at every share), which then has the fewer instructions a byte to issue and copies better
// ([8192, 50021] 573 us against 557, [8192, 65536] bfloat16 378 against 384). So are several waves of long rows
// of which some may not count: each wave takes as long as one that counts (the preference loss of 4080 rows of 32768
// bfloat16 at 60%, 180 us against 163).
static bool short_rows(const LossArgs& a, int op) {
    if (!loss_stream_fit(a)) return false;
    const int64_t bytes = a.cols * static_cast<int64_t>(dtype_size(a.dtype[kLrX]));
    if (op == kLossPolicy) return bytes <= 32 * 16 * kHeld / 2;
    if (bytes <= 16384) return true;
    if (op == kPull && a.dtype[kLrX] == CTB_FLOAT32) return false;
    const int64_t wave = static_cast<int64_t>(sm_count()) * 2 * kWarps, waves = (a.rows + wave - 1) / wave;
    const bool some = a.ptr[kLrWeight] || a.offsets;  // rows may not count
    return a.rows * 100 >= waves * wave * 85 && (waves == 1 || !some);
}

bool loss_short_fit(const LossPlan& p) { return p.op != kLossDistill && short_rows(p.args, p.op); }
bool loss_backward_short_fit(const LossArgs& a) { return short_rows(a, kPull); }

int loss_short(const LossPlan& p, int* parts, cudaStream_t st) {
    return p.op == kLossToken ? any_type<kLossToken>(p.args, parts, st) : any_type<kLossPolicy>(p.args, parts, st);
}

int loss_backward_short(const LossArgs& a, cudaStream_t st) {
    int parts = 0;
    return any_type<kPull>(a, &parts, st);
}

}  // namespace ctb
