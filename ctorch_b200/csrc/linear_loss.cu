// linear_loss.cu — the projection to the vocabulary with its cross entropy (include/ctb/ctb.h): checks, the plan of a
// call and its scratch, and the small kernels around the three products (linear_loss_tc.cu for bfloat16,
// linear_loss_f32.cu for float32): the list of rows that count, packed copies, the rows' softmax, the join of split
// sums, the scalar loss.
#include <algorithm>
#include <cmath>

#include <cuda_fp16.h>

#include "linear_loss.cuh"

namespace ctb {

unsigned long long* wait_timeout_counter();  // async.cu

namespace {

constexpr int64_t kHeldBytes = int64_t(2) << 30;  // of a block's logits or exponentials: 8192 rows of 131072 in 16 bits
constexpr int64_t kStatsBytes = int64_t(256) << 20;  // of a block's statistics where nothing is held: 32768 rows of 131072
constexpr int kOrderThreads = 1024;

__device__ __forceinline__ double row_weight(const LinearArgs& a, int64_t row) {
    return a.v.ptr[kLnWeight] ? real_at(a.v.ptr[kLnWeight], a.v.dtype[kLnWeight], row_offset(a.v, kLnWeight, row)) : 1.0;
}

__device__ __forceinline__ void put(const LinearArgs& a, int slot, int64_t row, double x) {
    if (a.v.ptr[slot]) static_cast<float*>(a.v.ptr[slot])[row_offset(a.v, slot, row)] = static_cast<float>(x);
}

// One CTA: the rows that count, then the others, each in their order; results of the others. A thread takes a run of
// rows, so one scan of the threads' counts places them. Bound by its latency (a few microseconds at 8192 rows).
__global__ void __launch_bounds__(kOrderThreads) linear_order(LinearArgs a) {
    dependent_wait();
    allow_dependents();
    __shared__ int64_t counts[kOrderThreads];
    __shared__ float largest[kOrderThreads / 32];
    const int64_t rows = a.v.rows, each = (rows + kOrderThreads - 1) / kOrderThreads;
    const int64_t lo = min(rows, each * threadIdx.x), hi = min(rows, lo + each);
    int64_t mine = 0;
    float top = 0.0f;
    for (int64_t r = lo; r < hi; ++r) {
        const double w = row_weight(a, r);
        if (w != 0.0) {
            ++mine;
            // a divisor in any case; a weight that no float32 holds spoils its own row alone, not what the others are relative to
            const float size = static_cast<float>(fabs(w));
            if (size < INFINITY) top = fmaxf(top, fmaxf(size, 1.17549435e-38f));
        }
    }
    counts[threadIdx.x] = mine;
    for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int d = 1; d < kOrderThreads; d <<= 1) {
        const int64_t before = threadIdx.x >= d ? counts[threadIdx.x - d] : 0;
        __syncthreads();
        counts[threadIdx.x] += before;
        __syncthreads();
    }
    const int64_t n = counts[kOrderThreads - 1];
    int64_t on = counts[threadIdx.x] - mine, off = n + lo - on;
    for (int64_t r = lo; r < hi; ++r) {
        if (row_weight(a, r) != 0.0) {
            a.order[on++] = static_cast<int32_t>(r);
        } else {
            a.order[off++] = static_cast<int32_t>(r);
            a.weighted[r] = 0.0;
            put(a, kLnRowLoss, r, 0.0);
            put(a, kLnLse, r, 0.0);
        }
    }
    if (threadIdx.x == 0) {
        for (int w = 1; w < kOrderThreads / 32; ++w) top = fmaxf(top, largest[w]);
        a.facts->count = static_cast<int32_t>(n);
        a.facts->wmax = top;
    }
}

// Rows as the products want them: contiguous, 16-byte aligned, zero up to the pitch. ORDERED: hidden's rows that
// count, and zeros up to a multiple of 64 rows (they are a product's inner dimension too).
constexpr int kPackThreads = 128;
template <class T, bool ORDERED>
__global__ void __launch_bounds__(kPackThreads) linear_pack(LinearArgs a, Matrix2 from, Matrix2 to, int64_t rows, int64_t cols) {
    dependent_wait();
    const int64_t n = ORDERED && a.order ? a.facts->count : rows;
    const int64_t upto = ORDERED ? min(rows, (n + 63) / 64 * 64) : rows;
    constexpr int kPack = 16 / sizeof(T);
    for (int64_t i = blockIdx.x; i < upto; i += gridDim.x) {
        T* const out = static_cast<T*>(to.ptr) + i * to.row;
        const int64_t r = ORDERED && a.order && i < n ? a.order[i] : i;
        const T* const in = static_cast<const T*>(from.ptr) + (ORDERED ? row_offset(a.v, kLnHidden, r) : r * from.row);
        const bool whole = i < n && from.col == 1 && reinterpret_cast<uintptr_t>(in) % 16 == 0;
        for (int64_t j = static_cast<int64_t>(threadIdx.x) * kPack; j < to.row; j += kPackThreads * kPack) {
            if (whole && j + kPack <= cols) {
                *reinterpret_cast<uint4*>(out + j) = *reinterpret_cast<const uint4*>(in + j);
                continue;
            }
            Pack<T, kPack> v;
#pragma unroll
            for (int q = 0; q < kPack; ++q) v.v[q] = i < n && j + q < cols ? in[(j + q) * from.col] : from_float<T>(0.0f);
            store_pack<T, kPack>(out + j, v);
        }
    }
    allow_dependents();
}

// ------------------------------------------------------------------------------------------------
// the rows' softmax

struct RowResult {
    double lse, loss, w;  // w: weight over the block's factor
    int64_t row, target;
    bool bad;
};

__device__ __forceinline__ RowResult row_result(const LinearArgs& a, int64_t i, double m, double s, double zt) {
    RowResult o;
    o.row = a.order ? a.order[i] : i;
    o.target = index_at(a.v.ptr[kLnTarget], a.v.dtype[kLnTarget], row_offset(a.v, kLnTarget, o.row));
    o.bad = o.target < 0 || o.target >= a.vocab;
    const double w = row_weight(a, o.row), rest = log(s);
    o.lse = m * a.inv_temp + rest;
    o.loss = o.bad ? nan("") : (m - zt) * a.inv_temp + rest + (a.z_coef != 0.0 ? a.z_coef * o.lse * o.lse : 0.0);
    o.w = a.order ? w / static_cast<double>(a.facts->wmax) : 1.0;
    return o;
}

__device__ __forceinline__ void put_row_result(const LinearArgs& a, const RowResult& o) {
    if (o.bad) record_bad_index(a.status, o.target);
    put(a, kLnRowLoss, o.row, o.loss);
    put(a, kLnLse, o.row, o.bad ? nan("") : o.lse);
    a.weighted[o.row] = a.scale * row_weight(a, o.row) * o.loss;
}

__device__ __forceinline__ float exp2_approx(float t) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
    return y;
}

// Joins (maximum, sum) pairs; s is relative to m.
__device__ __forceinline__ void join_sums(float& m, float& s, float om, float os, float c2) {
    const float top = fmaxf(m, om);
    const float at = top == -INFINITY ? 0.0f : top;
    s = s * exp2_approx((m - at) * c2) + os * exp2_approx((om - at) * c2);
    m = om != om || m != m ? NAN : top;
}

template <int THREADS> __device__ __forceinline__ void join_block(float& m, float& s, float c2) {
    __shared__ float sm[THREADS / 32], ss[THREADS / 32];
    for (int d = 16; d >= 1; d >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, d), os = __shfl_xor_sync(0xffffffffu, s, d);
        join_sums(m, s, om, os, c2);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
        sm[threadIdx.x >> 5] = m;
        ss[threadIdx.x >> 5] = s;
    }
    __syncthreads();
    m = sm[0];
    s = ss[0];
    for (int w = 1; w < THREADS / 32; ++w) join_sums(m, s, sm[w], ss[w], c2);
    if (m == INFINITY) s = NAN;
}

// float32: a CTA a row of held logits; statistics, then G in their place. The row's second pass comes from L2.
__global__ void __launch_bounds__(512) linear_rows_f32(LinearArgs a, int64_t first, int grad) {
    dependent_wait();
    const int64_t n = a.order ? linear_block_rows(a, first) : min(a.block, a.v.rows - first);
    for (int64_t b = blockIdx.x; b < n; b += gridDim.x) {
        float* const z = static_cast<float*>(a.held) + b * a.held_pitch;
        float m = -INFINITY, s = 0.0f;
        for (int64_t j = threadIdx.x; j < a.vocab; j += 512) m = z[j] != z[j] ? NAN : m != m ? m : fmaxf(m, z[j]);
        const float at = m == -INFINITY ? 0.0f : m;
        for (int64_t j = threadIdx.x; j < a.vocab; j += 512) s += exp2_approx((z[j] - at) * a.c2);
        join_block<512>(m, s, a.c2);
        const int64_t t0 = index_at(a.v.ptr[kLnTarget], a.v.dtype[kLnTarget],
                                    row_offset(a.v, kLnTarget, a.order ? a.order[first + b] : first + b));
        const bool inside = t0 >= 0 && t0 < a.vocab;
        const float zt = inside ? z[t0] : 0.0f;
        const RowResult o = row_result(a, first + b, m, s, zt);
        __syncthreads();
        if (threadIdx.x == 0) put_row_result(a, o);
        if (!grad) continue;
        const double up = 1.0 + 2.0 * a.z_coef * o.lse;
        const float c = o.bad ? NAN : static_cast<float>(o.w * up / static_cast<double>(s));
        for (int64_t j = threadIdx.x; j < a.held_pitch; j += 512) {
            float g = 0.0f;
            if (j < a.vocab) {
                g = c * exp2_approx((z[j] - m) * a.c2);
                if (j == t0) {
                    const double logp = (static_cast<double>(zt) - m) * a.inv_temp - log(static_cast<double>(s));
                    g = static_cast<float>(o.w * (expm1(logp) + 2.0 * a.z_coef * o.lse * exp(logp)));
                }
            }
            z[j] = g;
        }
    }
    allow_dependents();
}

// bfloat16: a warp a row joins the pieces' maxima and sums and works out the row's results and what its G needs:
//     G_rv = c 2^((m_piece - m) log2(e) / T) held_rv,      at the target: worked out from its own logit
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) linear_rows_tc(LinearArgs a, int64_t first) {
    dependent_wait();
    allow_dependents();
    const int64_t n = a.order ? linear_block_rows(a, first) : min(a.block, a.v.rows - first);
    const int lane = threadIdx.x & 31;
    for (int64_t b = blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5); b < n; b += gridDim.x * (kJoinThreads / 32)) {
        const float2* const stats = a.stats + b * a.tiles;
        float m = -INFINITY, s = 0.0f;
        for (int64_t j = lane; j < a.tiles; j += 32) {
            const float2 o = stats[j];
            join_sums(m, s, o.x, o.y, a.c2);
        }
        for (int d = 16; d >= 1; d >>= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, m, d), os = __shfl_xor_sync(0xffffffffu, s, d);
            join_sums(m, s, om, os, a.c2);
        }
        if (lane != 0) continue;
        if (m == INFINITY) s = NAN;
        const float zt = a.target_z[b];  // of a target outside: not looked at
        const RowResult o = row_result(a, first + b, m, s, zt);
        put_row_result(a, o);
        const double logp = (static_cast<double>(zt) - m) * a.inv_temp - log(static_cast<double>(s));
        LinearRowFactor f;
        f.m = m;
        // 2^-15 belongs to the held exponentials
        f.c = o.bad ? NAN : static_cast<float>(o.w * (1.0 + 2.0 * a.z_coef * o.lse) / static_cast<double>(s) * 0x1p-15);
        f.at_target = static_cast<float>(o.w * (expm1(logp) + 2.0 * a.z_coef * o.lse * exp(logp)));
        f.target = o.bad ? -1 : static_cast<int32_t>(o.target);
        a.factors[b] = f;
    }
}

// Turns the held exponentials (16-bit floats) into G, rounded to bfloat16, in their place; rows behind the last one, up to a
// stage of the products, become zeros. Bound by reading and writing 2 bytes an element, which run at the copy rate only if
// reads stay on their way while results are written: a CTA walks its share of spans of a row (16 KiB each) in order and
// has the next span's vectors under way before it writes this one's. B200, 8192 x 131072 (4.3 GB): 781 us with 16 CTAs
// an SM, four times what is resident (853 with 8, 1119 with 4: the SMs do not all stream alike); without the next span
// under way 802.
constexpr int kScaleThreads = 256, kScaleVecs = 4, kScaleSpan = kScaleThreads * kScaleVecs;  // vectors of 8

struct ScaleSpan {
    uint4 h[kScaleVecs];
    float pm[kScaleVecs];
    LinearRowFactor f;
};

__global__ void __launch_bounds__(kScaleThreads) linear_scale_tc(LinearArgs a, int64_t first) {
    dependent_wait();
    const int64_t limit = min(a.block, a.v.rows - first);
    const int64_t n = a.order ? linear_block_rows(a, first) : limit;
    const int64_t upto = min(limit, (n + 63) / 64 * 64);
    const int packs = static_cast<int>(a.held_pitch / 8), spans = (packs + kScaleSpan - 1) / kScaleSpan;
    const int64_t total = upto * spans, lo = total * blockIdx.x / gridDim.x, hi = total * (blockIdx.x + 1) / gridDim.x;
    if (lo >= hi) return;
    const int tiles = static_cast<int>(a.tiles);
    auto fetch = [&](ScaleSpan& s, int64_t b, int span) {
        if (b >= n) return;
        const uint4* const held = reinterpret_cast<const uint4*>(static_cast<const __half*>(a.held) + b * a.held_pitch);
        const float2* const stats = a.stats + b * tiles;
        s.f = a.factors[b];
#pragma unroll
        for (int q = 0; q < kScaleVecs; ++q) {
            const int j = span * kScaleSpan + q * kScaleThreads + static_cast<int>(threadIdx.x);
            if (j < packs) {
                s.h[q] = held[j];
                s.pm[q] = stats[min(j / (kLinearPiece / 8), tiles - 1)].x;
            }
        }
    };
    int64_t b = lo / spans;
    int span = static_cast<int>(lo - b * spans);
    ScaleSpan next;
    fetch(next, b, span);
    for (int64_t i = lo; i < hi; ++i) {
        ScaleSpan s = next;
        const int64_t row = b;
        const int at = span;
        if (++span == spans) {
            span = 0;
            ++b;
        }
        if (i + 1 < hi) fetch(next, b, span);
        uint4* const held = reinterpret_cast<uint4*>(static_cast<__half*>(a.held) + row * a.held_pitch);
#pragma unroll
        for (int q = 0; q < kScaleVecs; ++q) {
            const int j = at * kScaleSpan + q * kScaleThreads + static_cast<int>(threadIdx.x);
            if (j >= packs) continue;
            if (row >= n) {
                held[j] = make_uint4(0u, 0u, 0u, 0u);
                continue;
            }
            // a piece without a maximum has no mass
            const float c = s.pm[q] == -INFINITY ? s.f.c * 0.0f : s.f.c * exp2_approx((s.pm[q] - s.f.m) * a.c2);
            uint32_t* const u = reinterpret_cast<uint32_t*>(&s.h[q]);
            float g[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 e = __half22float2(*reinterpret_cast<const __half2*>(u + k));
                g[2 * k] = e.x * c;
                g[2 * k + 1] = e.y * c;
            }
            const int hit = s.f.target - j * 8;  // selects, not an index: those would put g into local memory
#pragma unroll
            for (int k = 0; k < 8; ++k) g[k] = hit == k ? s.f.at_target : g[k];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const __nv_bfloat162 y = __floats2bfloat162_rn(g[2 * k], g[2 * k + 1]);
                u[k] = *reinterpret_cast<const uint32_t*>(&y);
            }
            held[j] = s.h[q];
        }
    }
    allow_dependents();
}

// grad_hidden's rows of a block: the splits of dH = G W added in their order, times the factor; zeros where rows do
// not count (with the last block). A CTA takes 512 columns of a row, four a thread.
constexpr int kSumThreads = 128;
template <class T> __global__ void __launch_bounds__(kSumThreads) linear_join(LinearArgs a, int64_t first, int64_t upto) {
    dependent_wait();
    const int64_t n = a.order ? a.facts->count : a.v.rows;
    const double f = linear_factor(a);
    const int64_t inner = a.v.inner[kLnGrad], spans = (a.v.cols + kSumThreads * 4 - 1) / (kSumThreads * 4);
    for (int64_t k = blockIdx.x; k < (upto - first) * spans; k += gridDim.x) {
        const int64_t i = first + k / spans, j = (k % spans) * kSumThreads * 4 + threadIdx.x * 4;
        if (j >= a.v.cols) continue;
        const int64_t r = a.order ? a.order[i] : i;
        T* const out = static_cast<T*>(a.v.ptr[kLnGrad]) + row_offset(a.v, kLnGrad, r) + j * inner;
        const float* const p = a.partial + (i - first) * a.part_pitch + j;
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (i < n) {
#pragma unroll 4
            for (int s = 0; s < a.splits; ++s) {
                const float4 y = *reinterpret_cast<const float4*>(p + s * a.part_rows * a.part_pitch);
                x[0] += y.x;
                x[1] += y.y;
                x[2] += y.z;
                x[3] += y.w;
            }
        }
        T y[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = from_float<T>(static_cast<float>(f * static_cast<double>(x[q])));
        if (inner == 1 && j + 4 <= a.v.cols && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0) {
            Pack<T, 4> v;
#pragma unroll
            for (int q = 0; q < 4; ++q) v.v[q] = y[q];
            store_pack<T, 4>(out, v);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (j + q < a.v.cols) out[q * inner] = y[q];
        }
    }
    allow_dependents();
}

// out = the sum of n numbers in a fixed order, rounded once.
__global__ void __launch_bounds__(1024) linear_total(const double* x, int64_t n, float* out) {
    dependent_wait();
    allow_dependents();
    __shared__ double sm[32];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += x[i];
    for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < 32; ++w) t += sm[w];
        *out = static_cast<float>(t);
    }
}

// ------------------------------------------------------------------------------------------------
// host side

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Whether the products can read a matrix of unit inner stride in place (vector loads and tensor copies start on 16 bytes).
bool in_place(const void* p, int64_t row, int64_t col, int64_t rows, int64_t cols, int dtype, int want) {
    const int64_t size = static_cast<int64_t>(dtype_size(dtype));
    return dtype == want && (col == 1 || cols == 1) && reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
           (rows == 1 || (row * size % 16 == 0 && row >= cols));
}

struct Layout {
    size_t bytes = 0;
    size_t add(int64_t n, int64_t size) {
        const size_t at = bytes;
        bytes += static_cast<size_t>(round_up(n * size, 256));
        return at;
    }
};

struct LinearPlan {
    LinearArgs a{};
    bool grad = false, weighted = false, pack_h = false, pack_w = false;
    int64_t h_row = -1;      // hidden's row stride, where its leading dims are one
    int work = CTB_FLOAT32;  // the products' operand type, hidden's
    int64_t blocks = 0;
    size_t bytes = 0;
    size_t facts, order, weights, target_z, factors, stats, held, partial, acc, h, w;
};

// dH has few tiles and a long sum over the vocabulary: it is split where that fills the GPU's last round of tiles
// better than writing and reading the splits' float32 sums costs.
int splits_of(bool tc, int64_t rows, int64_t dim, int64_t vocab) {
    const int64_t tile = tc ? 256 : 128, units = tc ? sm_count() / 2 : sm_count() * 2;
    const int64_t tiles = (rows + tile - 1) / tile * ((dim + tile - 1) / tile);
    // seconds: a unit's rate, and 6 TB/s for the sums
    const double whole = 2.0 * tile * tile * vocab / (tc ? 2 * 10e12 : 0.2e12);
    const int64_t most = std::min<int64_t>(64, (vocab + 511) / 512);
    int64_t best = 1;
    double least = 1e300;
    for (int64_t s = 1; s <= most; ++s) {
        const double cost = static_cast<double>((tiles * s + units - 1) / units) * whole / s + 8.0 * s * rows * dim / 6e12;
        if (cost < least) {
            least = cost;
            best = s;
        }
    }
    return static_cast<int>(best);
}

// Rows of a block whose rows take `each` of at most `bytes`.
int64_t block_rows(int64_t rows, int64_t bytes, int64_t each) { return std::min(rows, std::max<int64_t>(256, bytes / each / 256 * 256)); }

// The sizes of a call's pieces. Everything here follows from shapes, strides and alignment alone. Without gradients bfloat16
// needs its pieces' statistics alone; `held`: room for the exponentials all the same.
void lay_out(LinearPlan& p, bool held = false) {
    LinearArgs& a = p.a;
    const int64_t rows = a.v.rows, dim = a.v.cols, vocab = a.vocab;
    p.work = a.v.dtype[kLnHidden];
    const bool tc = p.work == CTB_BFLOAT16;
    const int64_t size = static_cast<int64_t>(dtype_size(p.work)), pack = 16 / size;
    const int64_t pitch = round_up(dim, pack);
    a.held_pitch = round_up(vocab, 64);
    a.tiles = (vocab + kLinearPiece - 1) / kLinearPiece;
    held = held || p.grad || !tc;
    a.block = block_rows(rows, held ? kHeldBytes : kStatsBytes, held ? a.held_pitch * size : a.tiles * 8);
    p.blocks = (rows + a.block - 1) / a.block;
    p.pack_h = p.weighted || p.h_row < 0 ||
               !in_place(a.v.ptr[kLnHidden], p.h_row, a.v.inner[kLnHidden], rows, dim, a.v.dtype[kLnHidden], p.work);
    p.pack_w = !in_place(a.weight.ptr, a.weight.row, a.weight.col, vocab, dim, a.weight.dtype, p.work);
    a.splits = splits_of(tc, a.block, dim, vocab);
    a.part_pitch = round_up(dim, 32);
    a.part_rows = round_up(a.block, 256);
    a.acc_pitch = pitch;
    Layout l;
    p.facts = l.add(1, sizeof(LinearFacts));
    p.order = l.add(p.weighted ? rows : 0, 4);
    p.weights = l.add(rows, 8);
    p.target_z = l.add(a.block, 4);
    p.factors = l.add(tc ? a.block : 0, sizeof(LinearRowFactor));
    p.stats = l.add(tc ? a.block * a.tiles : 0, 8);
    p.held = l.add(held ? a.block * a.held_pitch : 0, size);
    p.partial = l.add(p.grad ? a.splits * a.part_rows * a.part_pitch : 0, 4);
    p.acc = l.add(p.grad && p.blocks > 1 ? vocab * a.acc_pitch : 0, 4);
    p.h = l.add(p.pack_h ? rows * pitch : 0, size);
    p.w = l.add(p.pack_w ? vocab * pitch : 0, size);
    p.bytes = l.bytes;
    a.h.row = p.pack_h || rows == 1 ? pitch : p.h_row;  // a single row's stride may be anything
    a.w.row = p.pack_w || vocab == 1 ? pitch : a.weight.row;
    a.h.col = a.w.col = 1;
    a.h.dtype = a.w.dtype = p.work;
}

void place(LinearPlan& p, void* scratch) {
    LinearArgs& a = p.a;
    unsigned char* const s = static_cast<unsigned char*>(scratch);
    a.facts = reinterpret_cast<LinearFacts*>(s + p.facts);
    a.order = p.weighted ? reinterpret_cast<int32_t*>(s + p.order) : nullptr;
    a.weighted = reinterpret_cast<double*>(s + p.weights);
    a.target_z = reinterpret_cast<float*>(s + p.target_z);
    a.stats = reinterpret_cast<float2*>(s + p.stats);
    a.factors = reinterpret_cast<LinearRowFactor*>(s + p.factors);
    a.held = s + p.held;
    a.partial = reinterpret_cast<float*>(s + p.partial);
    a.acc = p.blocks > 1 ? reinterpret_cast<float*>(s + p.acc) : nullptr;
    a.h.ptr = p.pack_h ? static_cast<void*>(s + p.h) : a.v.ptr[kLnHidden];
    a.w.ptr = p.pack_w ? static_cast<void*>(s + p.w) : a.weight.ptr;
}

template <bool ORDERED>
int run_pack(const LinearPlan& p, const Matrix2& from, const Matrix2& to, int64_t rows, cudaStream_t st) {
    auto kernel = p.work == CTB_FLOAT32 ? linear_pack<float, ORDERED> : linear_pack<__nv_bfloat16, ORDERED>;
    launch_dependent(kernel, grid_for(rows, 16), kPackThreads, 0, st, p.a, from, to, rows, p.a.v.cols);
    count_launch();
    return check_launch("linear loss: packing");
}

int linear_run(const LinearPlan& p, const ctb_view* loss, cudaStream_t st) {
    const LinearArgs& a = p.a;
    const int64_t rows = a.v.rows;
    const bool tc = p.work == CTB_BFLOAT16;
    if (rows && p.weighted) {
        launch_dependent(linear_order, 1, kOrderThreads, 0, st, a);
        count_launch();
        CTB_CHECK(check_launch("linear loss: rows"));
    }
    if (p.pack_h) CTB_CHECK(run_pack<true>(p, Matrix2{a.v.ptr[kLnHidden], 0, a.v.inner[kLnHidden], a.v.dtype[kLnHidden]}, a.h, rows, st));
    if (p.pack_w) CTB_CHECK(run_pack<false>(p, a.weight, a.w, a.vocab, st));
    for (int64_t first = 0; first < rows; first += a.block) {
        const int64_t n = std::min(a.block, rows - first);
        CTB_CHECK(tc ? linear_logits_tc(a, first, n, p.grad, st) : linear_logits_f32(a, first, n, st));
        if (tc) launch_dependent(linear_rows_tc, grid_for((n + 7) / 8, 8), kJoinThreads, 0, st, a, first);
        else launch_dependent(linear_rows_f32, grid_for(n, 4), 512, 0, st, a, first, static_cast<int>(p.grad));
        count_launch();
        CTB_CHECK(check_launch("linear loss: rows"));
        if (!p.grad) continue;
        if (tc) {
            launch_dependent(linear_scale_tc, grid_for(n * ((a.held_pitch / 8 + kScaleSpan - 1) / kScaleSpan), 16), kScaleThreads, 0, st, a, first);
            count_launch();
            CTB_CHECK(check_launch("linear loss: rows"));
        }
        CTB_CHECK((tc ? linear_grad_hidden_tc : linear_grad_hidden_f32)(a, first, n, st));
        auto join = a.v.dtype[kLnGrad] == CTB_FLOAT32 ? linear_join<float> : linear_join<__nv_bfloat16>;
        launch_dependent(join, grid_for(n * ((a.v.cols + 4 * kSumThreads - 1) / (4 * kSumThreads)), 16), kSumThreads, 0, st, a, first, first + n);
        count_launch();
        CTB_CHECK(check_launch("linear loss: join"));
        CTB_CHECK((tc ? linear_grad_weight_tc : linear_grad_weight_f32)(a, first, n, first + n == rows, st));
    }
    // without rows the weight's gradient is 0: the float32 product over no rows writes that, whatever the type
    if (rows == 0 && p.grad) CTB_CHECK(linear_grad_weight_f32(a, 0, 0, true, st));
    if (loss) {
        launch_dependent(linear_total, 1, 1024, 0, st, static_cast<const double*>(a.weighted), rows, static_cast<float*>(loss->data));
        count_launch();
        CTB_CHECK(check_launch("linear loss: total"));
    }
    return CTB_OK;
}

}  // namespace
}  // namespace ctb

using namespace ctb;

namespace {

int matrix_of(const ctb_view* v, const char* what, Matrix2& m) {
    CTB_CHECK(check_row_view(v, what));
    CTB_CHECK(check_row_dtype(v, kDtypeMatrix, what));
    if (v->ndim != 2) return fail(CTB_ERR_SHAPE, std::string(what) + " must be [vocabulary, columns of hidden]");
    m = Matrix2{v->data, v->strides[0], v->strides[1], v->dtype};
    return CTB_OK;
}

// The checks that the scratch query shares with the call.
int begin_plan(LinearPlan& p, RowBuilder<kLnViews>& b, const ctb_view* hidden, const ctb_view* weight) {
    CTB_CHECK(b.begin(kLnHidden, hidden, kDtypeMatrix, "hidden"));
    CTB_CHECK(matrix_of(weight, "weight", p.a.weight));
    if (weight->dtype != hidden->dtype) return fail(CTB_ERR_DTYPE, "weight's dtype must equal hidden's");
    if (weight->shape[1] != b.v.cols) return fail(CTB_ERR_SHAPE, "weight must be [vocabulary, columns of hidden]");
    p.a.vocab = weight->shape[0];
    // one stride from row to row, if there is one
    p.h_row = 0;
    int64_t extent = 1;
    for (int d = b.lead - 1; d >= 0 && p.h_row >= 0; --d) {
        if (hidden->shape[d] == 1) continue;
        if (extent == 1) p.h_row = hidden->strides[d];
        else if (hidden->strides[d] != p.h_row * extent) p.h_row = -1;
        extent *= hidden->shape[d];
    }
    if (p.a.vocab < 1) return fail(CTB_ERR_SHAPE, "the vocabulary is empty (a softmax over no entries has no value)");
    if (p.a.vocab >= (int64_t(1) << 31)) return fail(CTB_ERR_SHAPE, "vocabularies of 2^31 or more entries are not supported");
    return CTB_OK;
}

size_t scratch_of(const ctb_view* hidden, const ctb_view* weight, int weighted, int grad, bool held) {
    size_t need = 0;
    c_entry([&]() -> int {
        LinearPlan p;
        RowBuilder<kLnViews> b;
        CTB_CHECK(begin_plan(p, b, hidden, weight));
        b.finish();
        p.a.v = b.v;
        p.weighted = weighted != 0;
        p.grad = grad != 0;
        if (!b.v.rows) return CTB_OK;
        lay_out(p, held);
        need = p.bytes;
        return CTB_OK;
    });
    return need;
}

}  // namespace

extern "C" {

size_t ctb_linear_loss_scratch_bytes(const ctb_view* hidden, const ctb_view* weight, int weighted, int grad) {
    return scratch_of(hidden, weight, weighted, grad, true);
}

size_t ctb_linear_loss_forward_scratch_bytes(const ctb_view* hidden, const ctb_view* weight, int weighted) {
    return scratch_of(hidden, weight, weighted, 0, false);
}

int ctb_linear_cross_entropy(const ctb_view* hidden, const ctb_view* weight, const ctb_view* targets,
                             const ctb_view* weights, double weight_scale, double temperature, double z_coef,
                             const ctb_view* loss, const ctb_view* row_loss, const ctb_view* lse,
                             const ctb_view* grad_hidden, const ctb_view* grad_weight, int32_t* d_status, void* scratch,
                             size_t scratch_bytes, ctb_stream stream) {
    return c_entry([&]() -> int {
        LinearPlan p;
        RowBuilder<kLnViews> b;
        CTB_CHECK(begin_plan(p, b, hidden, weight));
        LinearArgs& a = p.a;
        CTB_CHECK(b.operand(kLnTarget, targets, kDtypeIndex, "targets"));
        if (weights) CTB_CHECK(b.operand(kLnWeight, weights, kDtypeWeight, "weights"));
        CTB_CHECK(b.result(kLnRowLoss, row_loss, 1u << CTB_FLOAT32, "row_loss"));
        CTB_CHECK(b.result(kLnLse, lse, 1u << CTB_FLOAT32, "lse"));
        if (!(temperature >= 1e-30 && temperature <= 1e30))
            return fail(CTB_ERR_ARGUMENT, "temperature must be positive (1e-30 to 1e30)");
        if (!(z_coef >= 0.0 && z_coef <= 1e30)) return fail(CTB_ERR_ARGUMENT, "z_coef must be finite and not negative");
        if (!std::isfinite(weight_scale)) return fail(CTB_ERR_ARGUMENT, "weight_scale must be finite");
        if (loss) {
            CTB_CHECK(check_row_view(loss, "loss"));
            CTB_CHECK(check_row_dtype(loss, 1u << CTB_FLOAT32, "loss"));
            for (int d = 0; d < loss->ndim; ++d)
                if (loss->shape[d] != 1) return fail(CTB_ERR_SHAPE, "loss must hold one element");
        }
        if (!grad_hidden != !grad_weight) return fail(CTB_ERR_ARGUMENT, "both gradients or none");
        p.grad = grad_hidden != nullptr;
        if (p.grad) {
            CTB_CHECK(b.matrix(kLnGrad, grad_hidden, 1u << hidden->dtype, b.v.cols, true, "grad_hidden"));
            CTB_CHECK(matrix_of(grad_weight, "grad_weight", a.grad_weight));
            if (grad_weight->dtype != weight->dtype) return fail(CTB_ERR_DTYPE, "grad_weight's dtype must equal weight's");
            if (grad_weight->shape[0] != weight->shape[0] || grad_weight->shape[1] != weight->shape[1])
                return fail(CTB_ERR_SHAPE, "grad_weight's shape must equal weight's");
            CTB_CHECK(check_written(grad_weight, "grad_weight"));
        }
        CTB_CHECK(check_row_status(d_status));
        b.finish();
        a.v = b.v;
        a.scale = weight_scale;
        a.inv_temp = 1.0 / temperature;
        a.c2 = static_cast<float>(1.4426950408889634 * a.inv_temp);
        a.z_coef = z_coef;
        a.status = d_status;
        a.timeouts = wait_timeout_counter();
        p.weighted = weights != nullptr;
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (a.v.rows == 0) {  // no rows: a loss of 0 and a weight gradient of 0
            a.block = 0;
        } else {
            lay_out(p);
            CTB_CHECK(check_row_scratch(scratch, scratch_bytes, p.bytes, 256));
            place(p, scratch);
        }
        return linear_run(p, loss, st);
    });
}

}  // extern "C"
