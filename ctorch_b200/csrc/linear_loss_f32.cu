// linear_loss_f32.cu — the three products of the projection with its cross entropy in float32.
//
// The tensor cores take float32 operands with 10 bits (tf32), which is not what a float32 caller asks for (operands split
// into three bfloat16 parts each, six products of parts, would keep 23 bits; not built), so these run on the FMA pipe: 128 x 128 tiles, 16 of the inner dimension a step through double-buffered shared memory, 8 x 8
// sums a thread as packed pairs (fma.rn.f32x2: half the instructions of single ones, so the shared-memory loads fit
// beside them). Sums are float32, one rounding a step. B200, 509 x 517 x 10007: 160, 143 and 160 us, 33 to 37 TFLOP/s, about
// half of the pipe's rate; with single FMA instructions 8% slower.
#include "linear_loss.cuh"

namespace ctb {

namespace {

constexpr int kBM = 128, kBN = 128, kBK = 16, kThreads = 256;

enum Product : int { kLogits = 0, kGradHidden = 1, kGradWeight = 2 };

struct ProductF32 {
    const float *x, *y;
    int64_t ldx, ldy;
    int64_t m, n, k;  // of the block at most
    int64_t first;    // the block's first row
    int last;
};

__device__ __forceinline__ void fma2(float2& d, float2 x, float2 y) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;"
        : "+l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(x)), "l"(reinterpret_cast<const unsigned long long&>(y)));
}

constexpr int kLd = kBM + 4;  // of a tile in shared memory, [kBK][kLd]

__device__ __forceinline__ void copy16(float* to, const float* from, int elements) {  // the rest becomes 0
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from),
                 "r"(elements * 4)
                 : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// This thread's share of the tiles of an operand: two vectors of 4, whose addresses move on by a step at a time. Where the
// product's outer dimension is contiguous they go to shared memory as they lie, asynchronously; where the inner one is
// (INNER: rows of the matrix are rows of the tile) they pass through registers to be laid out the other way. Elements
// outside are 0.
template <bool INNER> struct Share {
    const float* at;   // of the first vector; the second one is `apart` behind
    int64_t apart, step;
    int left[2];       // elements of a vector that exist along the contiguous dimension; INNER: whether its row exists
    int rest;          // inner indexes left
    float4 r[INNER ? 2 : 1];

    __device__ __forceinline__ Share(const float* p, int64_t ld, int64_t outer0, int64_t outers, int64_t k0, int64_t k1) {
        rest = static_cast<int>(k1 - k0);
        if (INNER) {
            const int64_t row = outer0 + (threadIdx.x >> 2);
            apart = 64 * ld;
            step = kBK;
            left[0] = row < outers;
            left[1] = row + 64 < outers;
            at = p + row * ld + k0 + (threadIdx.x & 3) * 4;
        } else {
            const int64_t col = outer0 + (threadIdx.x & 31) * 4;
            apart = 8 * ld;
            step = kBK * ld;
            left[0] = left[1] = static_cast<int>(col + 4 <= outers ? 4 : col < outers ? outers - col : 0);
            at = p + (k0 + (threadIdx.x >> 5)) * ld + col;
        }
    }

    // Sets the next tile's vectors on their way: into `sm`, or into registers until put().
    __device__ __forceinline__ void fetch(float* sm) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (INNER) {
                const int n = left[i] ? rest - static_cast<int>(threadIdx.x & 3) * 4 : 0;
                const float* const q = at + i * apart;
                r[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (n >= 4) {
                    r[i] = *reinterpret_cast<const float4*>(q);
                } else if (n > 0) {
                    r[i].x = q[0];
                    if (n > 1) r[i].y = q[1];
                    if (n > 2) r[i].z = q[2];
                }
            } else {
                const int k = static_cast<int>(threadIdx.x >> 5) + 8 * i, n = k < rest ? left[i] : 0;
                copy16(sm + k * kLd + (threadIdx.x & 31) * 4, n ? at + i * apart : at - (threadIdx.x & 31) * 4, n);
            }
        }
        at += step;
        rest -= kBK;
    }

    __device__ __forceinline__ void put(float* sm) {
        if constexpr (INNER) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = static_cast<int>(threadIdx.x >> 2) + 64 * i, k = (threadIdx.x & 3) * 4;
                sm[(k + 0) * kLd + row] = r[i].x;
                sm[(k + 1) * kLd + row] = r[i].y;
                sm[(k + 2) * kLd + row] = r[i].z;
                sm[(k + 3) * kLd + row] = r[i].w;
            }
        }
    }
};

template <int P> __global__ void __launch_bounds__(kThreads, 2) linear_product_f32(LinearArgs a, ProductF32 p) {
    dependent_wait();
    __shared__ __align__(16) float sx[2][kBK * kLd], sy[2][kBK * kLd];
    constexpr bool kXInner = P != kGradWeight, kYInner = P == kLogits;
    const int64_t rows = a.order ? linear_block_rows(a, p.first) : (P == kGradWeight ? p.k : p.m);
    const int64_t m = P == kGradWeight ? p.m : rows, k = P == kGradWeight ? rows : p.k;
    const int64_t tm = (p.m + kBM - 1) / kBM, tn = (p.n + kBN - 1) / kBN;
    int64_t tile = blockIdx.x;
    const int64_t i0 = tile % tm * kBM;
    tile /= tm;
    const int64_t j0 = tile % tn * kBN;
    const int64_t split = tile / tn;
    if (i0 >= m) return;
    int64_t k0 = 0, k1 = k;
    if (P == kGradHidden) {
        const int64_t each = ((k + a.splits - 1) / a.splits + kBK - 1) / kBK * kBK;
        k0 = min(k, split * each);
        k1 = min(k, k0 + each);
    }
    float2 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = make_float2(0.f, 0.f);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    Share<kXInner> share_x(p.x, p.ldx, i0, m, k0, k1);
    Share<kYInner> share_y(p.y, p.ldy, j0, p.n, k0, k1);
    if (k0 < k1) {
        share_x.fetch(sx[0]);
        share_y.fetch(sy[0]);
        share_x.put(sx[0]);
        share_y.put(sy[0]);
        copies_done();
    }
    __syncthreads();
    int at = 0;
    for (int steps = static_cast<int>((k1 - k0 + kBK - 1) / kBK); steps > 0; --steps) {
        const bool more = steps > 1;
        if (more) {
            share_x.fetch(sx[at ^ 1]);
            share_y.fetch(sy[at ^ 1]);
        }
#pragma unroll 2
        for (int q = 0; q < kBK; ++q) {
            const float* const xs = sx[at] + q * kLd;
            const float* const ys = sy[at] + q * kLd;
            const float4 x0 = *reinterpret_cast<const float4*>(xs + ty * 4), x1 = *reinterpret_cast<const float4*>(xs + 64 + ty * 4);
            const float4 y0 = *reinterpret_cast<const float4*>(ys + tx * 4), y1 = *reinterpret_cast<const float4*>(ys + 64 + tx * 4);
            const float xv[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
            const float2 yv[4] = {{y0.x, y0.y}, {y0.z, y0.w}, {y1.x, y1.y}, {y1.z, y1.w}};
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) fma2(acc[i][j], make_float2(xv[i], xv[i]), yv[j]);
        }
        if (more) {
            share_x.put(sx[at ^ 1]);
            share_y.put(sy[at ^ 1]);
            copies_done();
        }
        __syncthreads();
        at ^= 1;
    }
    allow_dependents();
    const double f = P == kGradWeight ? linear_factor(a) : 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = i0 + (i >> 2) * 64 + ty * 4 + (i & 3);
        if (row >= m) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t col = j0 + (j >> 1) * 64 + tx * 4 + (j & 1) * 2;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (col + h >= p.n) continue;
                float x = h ? acc[i][j].y : acc[i][j].x;
                if (P == kLogits) {
                    static_cast<float*>(a.held)[row * a.held_pitch + col + h] = x;
                } else if (P == kGradHidden) {
                    a.partial[(split * a.part_rows + row) * a.part_pitch + col + h] = x;
                } else {
                    if (a.acc && p.first > 0) x += a.acc[row * a.acc_pitch + col + h];
                    if (!p.last) {
                        a.acc[row * a.acc_pitch + col + h] = x;
                        continue;
                    }
                    const float y = static_cast<float>(f * static_cast<double>(x));
                    const int64_t to = row * a.grad_weight.row + (col + h) * a.grad_weight.col;
                    if (a.grad_weight.dtype == CTB_FLOAT32) static_cast<float*>(a.grad_weight.ptr)[to] = y;
                    else static_cast<__nv_bfloat16*>(a.grad_weight.ptr)[to] = __float2bfloat16_rn(y);
                }
            }
        }
    }
}

template <int P> int launch(const LinearArgs& a, const ProductF32& p, int64_t splits, cudaStream_t st) {
    const int64_t tiles = (p.m + kBM - 1) / kBM * ((p.n + kBN - 1) / kBN) * splits;
    if (tiles == 0) return CTB_OK;
    if (tiles >= (int64_t(1) << 31)) return fail(CTB_ERR_SHAPE, "linear loss: too many tiles");
    launch_dependent(linear_product_f32<P>, static_cast<unsigned>(tiles), kThreads, 0, st, a, p);
    count_launch();
    return check_launch("linear loss: product");
}

}  // namespace

int linear_logits_f32(const LinearArgs& a, int64_t first, int64_t rows, cudaStream_t st) {
    ProductF32 p{};
    p.x = static_cast<const float*>(a.h.ptr) + first * a.h.row;
    p.y = static_cast<const float*>(a.w.ptr);
    p.ldx = a.h.row;
    p.ldy = a.w.row;
    p.m = rows;
    p.n = a.vocab;
    p.k = a.v.cols;
    p.first = first;
    return launch<kLogits>(a, p, 1, st);
}

int linear_grad_hidden_f32(const LinearArgs& a, int64_t first, int64_t rows, cudaStream_t st) {
    ProductF32 p{};
    p.x = static_cast<const float*>(a.held);
    p.y = static_cast<const float*>(a.w.ptr);
    p.ldx = a.held_pitch;
    p.ldy = a.w.row;
    p.m = rows;
    p.n = a.v.cols;
    p.k = a.vocab;
    p.first = first;
    return launch<kGradHidden>(a, p, a.splits, st);
}

int linear_grad_weight_f32(const LinearArgs& a, int64_t first, int64_t rows, bool last, cudaStream_t st) {
    ProductF32 p{};
    p.x = static_cast<const float*>(a.held);
    p.y = static_cast<const float*>(a.h.ptr) + first * a.h.row;
    p.ldx = a.held_pitch;
    p.ldy = a.h.row;
    p.m = a.vocab;
    p.n = a.v.cols;
    p.k = rows;
    p.first = first;
    p.last = last;
    return launch<kGradWeight>(a, p, 1, st);
}

}  // namespace ctb
