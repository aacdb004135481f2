// linear_loss_tc.cu — the three products of the projection with its cross entropy in bfloat16, on the tensor cores.
//
// One kernel for all three: pairs of CTAs, one pair per two SMs, walk over 256 x 256 tiles. In each CTA one warp brings
// stages of 64 of the inner dimension (32 KiB a CTA) into a ring of shared memory, one thread of the pair issues the
// products, and eight warps take finished tiles out of tensor memory (two tiles' worth, so the next tile's products run
// meanwhile), each 32 rows by 128 columns, and do what the product is for:
//   z = H W^T      (maximum, sum of exponentials) of every 128 columns of a row, the target's z, and for the gradients
//                  exp(z - maximum) in 16 bits
//   dH = G W       float32 sums, split along the vocabulary where there are few tiles
//   dW = G^T H     rounded once, or added up in float32 over the blocks of rows
// H and G have the inner dimension of z = H W^T and dH = G W contiguous; the other operands their outer one, which the
// tensor cores read as it lies.
//
// Why these tiles: a pair's 256 x 256 tile needs 64 bytes of operands a clock and SM at the tensor cores' full rate, half of what
// a 128 x 256 tile of one CTA would, and two of them fit tensor memory, so a tile's results leave while the next one is
// computed. Bound by the tensor cores and, in long runs, by power: B200, 3686 x 2048 x 32768: 365 (z, with the
// exponentials written), 356 (dH, in four splits) and 319 us (dW), 1.36 to 1.55 PFLOP/s, the tensor pipe 74 to 84% busy; 8192 x 4096 x 131072 6.8 to 7.6 ms each,
// 1.15 to 1.3 PFLOP/s. Results as 16-byte stores of a thread took 364, 353 and 328 us, and 7.4 to 7.8 ms (z in one stretch).
#include <cuda_fp16.h>

#include "linear_loss.cuh"
#include "tensor_core.cuh"

namespace ctb {

namespace {

constexpr int kTile = 256, kHalf = 128, kK = 64, kStages = 6;
constexpr int kStageBytes = 2 * kHalf * kK * 2;  // of one CTA: its halves of both operands
constexpr int kEpilogueWarps = 8, kThreads = 32 * (kEpilogueWarps + 2);
constexpr int kBoxBytes = 32 * 128;  // of results on their way out, one a warp
constexpr int kSmem = kStages * kStageBytes + kEpilogueWarps * kBoxBytes + 1024;
constexpr int kLogitsStretch = 12, kFewRows = 8, kFewStretch = 4, kGradStretch = 256;  // stages summed in tensor memory at a time
constexpr int kGroup = 8;  // tiles of rows walked together, so that both operands are met again in L2 (2 to 32: within 5%)

enum Product : int { kLogits = 0, kLogitsOnly = 1, kGradHidden = 2, kGradWeight = 3 };

struct ProductArgs {
    int64_t m, n, k;  // of the block at most
    int64_t first;    // the block's first row
    int last;         // the last block
    int boxes;        // dW leaves as boxes
    int stretch;      // stages that tensor memory sums at a time
};

struct Bars {
    uint64_t full[kStages], empty[kStages], done[2], free[2];
    uint32_t tmem;
};

struct Work {
    int64_t m, n;      // tile
    int64_t kb0, kbs;  // stages of the inner dimension
    int64_t split;
};

template <int P> struct Schedule {
    int64_t tm, tn, kblocks, splits, total;
    __device__ Schedule(const LinearArgs& a, const ProductArgs& p, int64_t rows) {
        const int64_t m = P == kGradWeight ? p.m : rows, k = P == kGradWeight ? rows : p.k;
        tm = (m + kTile - 1) / kTile;
        tn = (p.n + kTile - 1) / kTile;
        kblocks = (k + kK - 1) / kK;
        splits = P == kGradHidden ? a.splits : 1;
        total = tm * tn * splits;
    }
    // Groups of kGroup tiles of m, the columns of tiles after one another within a group, splits last.
    __device__ Work at(int64_t w) const {
        Work o;
        o.split = w / (tm * tn);
        w -= o.split * tm * tn;
        const int64_t group = w / (kGroup * tn), m0 = group * kGroup, size = min(static_cast<int64_t>(kGroup), tm - m0);
        w -= group * kGroup * tn;
        o.n = w / size;
        o.m = m0 + w % size;
        const int64_t each = (kblocks + splits - 1) / splits;
        o.kb0 = min(kblocks, o.split * each);
        o.kbs = min(kblocks, o.kb0 + each) - o.kb0;
        return o;
    }
};

__device__ __forceinline__ float exp2_approx(float t) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
    return y;
}

// Two numbers in one word of 16-bit floats, the first one low.
__device__ __forceinline__ uint32_t two_halves(float x, float y) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t two_bf16(float x, float y) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}

// The tensor cores truncate a float32 sum at every step of 16 products, so a long one comes out short by a share of itself (one
// that grows evenly by about 1.6e-8 a step; an exact one by nothing). So they sum a stretch of stages, and the stretches are
// added in registers, rounded to nearest: a logit loses 8e-7 of itself at most on average, however long, and an exact one
// nothing. Every stretch costs the products about half a microsecond, and short ones wait for the rows' exponentials. B200,
// 3686 x 2048 x 32768 (32 stages), z and the log-sum-exp's error: one stretch 349 us and 1.3e-6 (at twice the columns), 16
// stages 356 and 3.6e-7, 12 stages 363 and 2.4e-7, 8 stages 380 and 1.7e-7, 4 stages 450 and 8e-8. A few rows' losses have
// no others to average with: their stretches are of 4 stages (1 row: 46.7 -> 51.8 us, the loss's error 3.0e-7 -> 1.0e-7 at the
// median, 2.6e-6 -> 4.2e-7 at most; 4 rows 44.2 -> 46.5). Gradients are rounded to 16 bits or of such terms, and 1.6e-5 of a
// stretch is far below that.
int logits_stretch(const LinearArgs& a) { return a.v.rows <= kFewRows ? kFewStretch : kLogitsStretch; }

// 128 columns of a row of logits: their maximum and the sum of exp((z - max) / T), the target's z, and with HOLD
// 2^15 exp((z - max) / T) in 16 bits: 11 bits of precision down to 2^-29 of the largest, nothing below 2^-40.
struct Out {  // where a warp's results leave through
    const CUtensorMap* map;
    uint32_t box;
    int row;  // of its 32 rows, the first
};

// Gives the warp's box to the copy engine (every lane has written its row of it).
__device__ __forceinline__ void send_box(const Out& o, int64_t col) {
    proxy_fence();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tensor_store(o.map, static_cast<int>(col), o.row, o.box);
}
__device__ __forceinline__ void box_free() {
    if ((threadIdx.x & 31) == 0) tensor_stores_read();
    __syncwarp();
}

template <bool HOLD>
__device__ __forceinline__ void logits_row(const LinearArgs& a, float (&z)[kHalf], int64_t i, int64_t col, int64_t target, bool live,
                                           const Out& out) {
    const int64_t left = a.vocab - col;
    if (left < kHalf) {
#pragma unroll
        for (int j = 0; j < kHalf; ++j)
            if (j >= left) z[j] = -INFINITY;
    }
    const int64_t t = target - col;
    const bool here = live && t >= 0 && t < kHalf && t < left;
    if (__any_sync(0xffffffffu, here)) {
        float zt = 0.0f;
#pragma unroll
        for (int j = 0; j < kHalf; ++j)
            if (j == t) zt = z[j];
        if (here) a.target_z[i] = zt;
    }
    float m = z[0];
#pragma unroll
    for (int j = 1; j < kHalf; ++j) m = fmaxf(m, z[j]);
    const float at = m == -INFINITY ? 0.0f : m;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < kHalf; ++j) {
        z[j] = exp2_approx(fmaf(z[j] - at, a.c2, 15.0f));
        s[j & 3] += z[j];
    }
    if (live) a.stats[i * a.tiles + col / kHalf] = make_float2(m, ((s[0] + s[1]) + (s[2] + s[3])) * 3.0517578125e-05f);
    if (!HOLD) return;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (h * 64 >= left) break;
        box_free();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float* const e = z + h * 64 + q * 8;
            store_shared16(swizzled_piece(out.box, lane, q), two_halves(e[0], e[1]), two_halves(e[2], e[3]), two_halves(e[4], e[5]),
                           two_halves(e[6], e[7]));
        }
        send_box(out, col + h * 64);
    }
}

constexpr int kChunk = 32;  // columns of a gradient that a thread has in hand at a time

__device__ __forceinline__ void grad_hidden_rows(const float* x, int64_t col, const Out& out) {
    box_free();
#pragma unroll
    for (int q = 0; q < 8; ++q)
        store_shared16(swizzled_piece(out.box, threadIdx.x & 31, q), __float_as_uint(x[4 * q]), __float_as_uint(x[4 * q + 1]),
                       __float_as_uint(x[4 * q + 2]), __float_as_uint(x[4 * q + 3]));
    send_box(out, col);
}

// 32 columns of dW into half of the warp's box, which leaves with every second piece.
__device__ __forceinline__ void grad_weight_rows(const float* x, int64_t col, float factor, int piece, const Out& out) {
    if ((piece & 1) == 0) box_free();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float* const y = x + 8 * q;
        store_shared16(swizzled_piece(out.box, threadIdx.x & 31, (piece & 1) * 4 + q), two_bf16(y[0] * factor, y[1] * factor),
                       two_bf16(y[2] * factor, y[3] * factor), two_bf16(y[4] * factor, y[5] * factor), two_bf16(y[6] * factor, y[7] * factor));
    }
    if ((piece & 1) == 1) send_box(out, col - kChunk);
}

// The same for any layout of dW, and where the blocks before are added.
__device__ __forceinline__ void grad_weight_row(const LinearArgs& a, const ProductArgs& p, float* x, int64_t v, int64_t col,
                                                int64_t cols, float factor) {
    if (a.acc) {
        float* const acc = a.acc + v * a.acc_pitch + col;
#pragma unroll
        for (int q = 0; q < kChunk / 4; ++q) {
            if (col + q * 4 >= cols) continue;
            float4* const to = reinterpret_cast<float4*>(acc + q * 4);
            if (p.first > 0) {
                const float4 y = *to;
                x[4 * q] += y.x;
                x[4 * q + 1] += y.y;
                x[4 * q + 2] += y.z;
                x[4 * q + 3] += y.w;
            }
            if (!p.last) *to = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
        }
        if (!p.last) return;
    }
    __nv_bfloat16* const out = static_cast<__nv_bfloat16*>(a.grad_weight.ptr) + v * a.grad_weight.row + col * a.grad_weight.col;
#pragma unroll
    for (int j = 0; j < kChunk; ++j)
        if (col + j < cols) out[j * a.grad_weight.col] = __float2bfloat16_rn(x[j] * factor);
}

template <int P>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    linear_product_tc(const __grid_constant__ LinearArgs a, const __grid_constant__ ProductArgs p,
                      const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                      const __grid_constant__ CUtensorMap map_out) {
    extern __shared__ unsigned char raw[];
    __shared__ Bars bars;
    unsigned char* const smem = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
    constexpr bool kAOuter = P == kGradWeight, kBOuter = P == kGradHidden || P == kGradWeight;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&bars.full[s], 1);
            mbar_init(&bars.empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bars.done[s], 1);
            mbar_init(&bars.free[s], 2 * kEpilogueWarps);
        }
        mbar_fence_init();
    }
    if (warp == kEpilogueWarps) tmem_alloc_pair(&bars.tmem, 2 * kTile);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = bars.tmem;
    dependent_wait();

    const int64_t rows = a.order ? linear_block_rows(a, p.first) : (P == kGradWeight ? p.k : p.m);
    const Schedule<P> plan(a, p, rows);
    const int64_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    bool ok = true;

    if (warp == kEpilogueWarps) {
        // brings this CTA's halves: 128 of the tile's rows of the left operand, 128 of its columns of the right one
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            for (int64_t w = pair; ok && w < plan.total; w += pairs) {
                const Work o = plan.at(w);
                const int64_t i0 = o.m * kTile + rank * kHalf, j0 = o.n * kTile + rank * kHalf;
                for (int64_t kb = 0; kb < o.kbs; ++kb) {
                    if (!mbar_wait(&bars.empty[stage], phase ^ 1u)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) mbar_arrive_expect_tx(&bars.full[stage], 2 * kStageBytes);
                    const uint32_t bar = in_first_cta(&bars.full[stage]);
                    const uint32_t sa = smem_addr(smem + stage * kStageBytes), sb = sa + kStageBytes / 2;
                    const int k0 = static_cast<int>((o.kb0 + kb) * kK);
                    if (kAOuter) {
                        tensor_load_pair(sa, &map_a, static_cast<int>(i0), k0, bar);
                        tensor_load_pair(sa + 8192, &map_a, static_cast<int>(i0) + 64, k0, bar);
                    } else {
                        const int64_t base = P == kLogits || P == kLogitsOnly ? p.first : 0;
                        tensor_load_pair(sa, &map_a, k0, static_cast<int>(base + i0), bar);
                    }
                    if (kBOuter) {
                        const int kb_row = k0 + static_cast<int>(P == kGradWeight ? p.first : 0);
                        tensor_load_pair(sb, &map_b, static_cast<int>(j0), kb_row, bar);
                        tensor_load_pair(sb + 8192, &map_b, static_cast<int>(j0) + 64, kb_row, bar);
                    } else {
                        tensor_load_pair(sb, &map_b, k0, static_cast<int>(j0), bar);
                    }
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // no copy or arrival is on its way to this CTA once its last stages are given back (unused ones count as such)
            for (int s = 0; ok && s < kStages; ++s) {
                if (!mbar_wait(&bars.empty[stage], phase ^ 1u)) ok = false;
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == kEpilogueWarps + 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t kInstruction = instruction_bf16(kTile, kTile, kAOuter, kBOuter);
            constexpr uint32_t kAStep = kAOuter ? 2048 : 32, kBStep = kBOuter ? 2048 : 32;  // bytes of 16 of the inner dimension
            uint32_t stage = 0, phase = 0;
            int acc = 0;
            uint32_t acc_phase = 0;
            for (int64_t w = pair; ok && w < plan.total; w += pairs) {
                const Work o = plan.at(w);
                for (int64_t left = o.kbs; ok && left > 0; left -= p.stretch) {
                    if (!mbar_wait(&bars.free[acc], acc_phase ^ 1u)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem + acc * kTile;
                    const int stages = static_cast<int>(min(left, static_cast<int64_t>(p.stretch)));
                    for (int kb = 0; kb < stages; ++kb) {
                        if (!mbar_wait(&bars.full[stage], phase)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t sa = smem_addr(smem + stage * kStageBytes), sb = sa + kStageBytes / 2;
#pragma unroll
                        for (int k = 0; k < kK / 16; ++k)
                            mma_pair(d, matrix_descriptor(sa + k * kAStep, 8192, 1024), matrix_descriptor(sb + k * kBStep, 8192, 1024),
                                     kInstruction, kb > 0 || k > 0);
                        mma_commit_pair(&bars.empty[stage]);
                        if (++stage == kStages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                    mma_commit_pair(&bars.done[acc]);
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1u;
                }
            }
        }
    } else {
        const int quarter = warp & 3, half = warp >> 2;
        int acc = 0;
        uint32_t acc_phase = 0;
        const float factor = P == kGradWeight ? static_cast<float>(linear_factor(a)) : 1.0f;
        const int64_t m = P == kGradWeight ? p.m : rows;
        Out out = {&map_out, smem_addr(smem + kStages * kStageBytes + warp * kBoxBytes), 0};
        for (int64_t w = pair; ok && w < plan.total; w += pairs) {
            const Work o = plan.at(w);
            const int64_t i0 = o.m * kTile + rank * kHalf + quarter * 32, i = i0 + lane, col = o.n * kTile + half * kHalf;
            out.row = static_cast<int>(i0 + (P == kGradHidden ? o.split * a.part_rows : 0));
            int64_t target = -1;
            if ((P == kLogits || P == kLogitsOnly) && i < m) {
                const int64_t r = a.order ? a.order[p.first + i] : p.first + i;
                target = index_at(a.v.ptr[kLnTarget], a.v.dtype[kLnTarget], row_offset(a.v, kLnTarget, r));
            }
            float x[kHalf];
            for (int64_t kb = 0; kb < o.kbs; kb += p.stretch) {
                ok = __all_sync(0xffffffffu, mbar_wait(&bars.done[acc], acc_phase));
                if (!ok) break;
                tc_fence_after();
                const uint32_t from = tmem + acc * kTile + half * kHalf + (static_cast<uint32_t>(quarter * 32) << 16);
                if (i0 >= m) {
                    // no rows here: the sums stay where they are (loads of tensor memory take the products' time at it)
                } else if (kb == 0) {
#pragma unroll
                    for (int c = 0; c < kHalf / 32; ++c) tmem_load32(x + c * 32, from + c * 32);
                    tmem_load_wait();
                } else {
#pragma unroll
                    for (int c = 0; c < kHalf / 16; ++c) {
                        float y[16];
                        tmem_load16(y, from + c * 16);
                        tmem_load_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[c * 16 + j] += y[j];
                    }
                }
                // the sums are in registers: the tensor memory goes back to the products
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(in_first_cta(&bars.free[acc]));
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
            if (!ok) break;
            if (o.kbs == 0) {
#pragma unroll
                for (int j = 0; j < kHalf; ++j) x[j] = 0.0f;
            }
            if constexpr (P == kLogits || P == kLogitsOnly) {
                if (col < p.n && i0 < m) logits_row<P == kLogits>(a, x, i, col, target, i < m, out);
            } else {
#pragma unroll
                for (int c = 0; c < kHalf / kChunk; ++c) {
                    const int64_t at = col + c * kChunk;
                    if (P == kGradHidden) {
                        if (i0 < m && at < p.n) grad_hidden_rows(x + c * kChunk, at, out);
                    } else if (p.boxes) {
                        if (i0 < m && col + (c & ~1) * kChunk < p.n) grad_weight_rows(x + c * kChunk, at, factor, c, out);
                    } else if (i < m && at < p.n) {
                        grad_weight_row(a, p, x + c * kChunk, i, at, p.n, factor);
                    }
                }
            }
        }
        if (lane == 0) tensor_stores_done();
    }
    __syncwarp();
    if (!ok) {
        // a wait ran out: count it, and leave the copies and products in flight time to land before the memory goes
        note_timeout(a.timeouts);
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 2000000ull) __nanosleep(1000);
    }
    __syncwarp();
    allow_dependents();
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == kEpilogueWarps) {
        tc_fence_after();
        tmem_free_pair(tmem, 2 * kTile);
    }
}

template <int P>
int launch(const LinearArgs& a, const ProductArgs& p, const CUtensorMap& map_a, const CUtensorMap& map_b,
           const CUtensorMap& map_out, cudaStream_t st) {
    auto kernel = linear_product_tc<P>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(CTB_ERR_CUDA, std::string("linear loss: ") + cudaGetErrorString(e));
    }
    launch_dependent(kernel, static_cast<unsigned>(sm_count() / 2 * 2), kThreads, kSmem, st, a, p, map_a, map_b, map_out);
    count_launch();
    return check_launch("linear loss: product");
}

int no_map() { return fail(CTB_ERR_CUDA, "linear loss: the driver refused a tensor map"); }

}  // namespace

int linear_logits_tc(const LinearArgs& a, int64_t first, int64_t rows, bool hold, cudaStream_t st) {
    CUtensorMap h, w, e;
    if (!encode_matrix_map(&h, a.h.ptr, a.v.rows, a.v.cols, a.h.row, kHalf) ||
        !encode_matrix_map(&w, a.w.ptr, a.vocab, a.v.cols, a.w.row, kHalf) ||
        !encode_matrix_map(&e, hold ? a.held : a.h.ptr, rows, hold ? a.vocab : 1, hold ? a.held_pitch : a.h.row, 32))
        return no_map();
    const ProductArgs p{rows, a.vocab, a.v.cols, first, 0, 0, logits_stretch(a)};
    return hold ? launch<kLogits>(a, p, h, w, e, st) : launch<kLogitsOnly>(a, p, h, w, e, st);
}

int linear_grad_hidden_tc(const LinearArgs& a, int64_t first, int64_t rows, cudaStream_t st) {
    CUtensorMap g, w, out;
    if (!encode_matrix_map(&g, a.held, rows, a.vocab, a.held_pitch, kHalf) ||
        !encode_matrix_map(&w, a.w.ptr, a.vocab, a.v.cols, a.w.row, kK) ||
        !encode_matrix_map(&out, a.partial, a.splits * a.part_rows, a.v.cols, a.part_pitch, 32, 4))
        return no_map();
    return launch<kGradHidden>(a, ProductArgs{rows, a.v.cols, a.vocab, first, 0, 0, kGradStretch}, g, w, out, st);
}

int linear_grad_weight_tc(const LinearArgs& a, int64_t first, int64_t rows, bool last, cudaStream_t st) {
    CUtensorMap g, h, out;
    // a dW that a tensor map can describe, whole at once, leaves as boxes
    const Matrix2& d = a.grad_weight;
    const bool boxes = !a.acc && d.col == 1 && reinterpret_cast<uintptr_t>(d.ptr) % 16 == 0 && d.row % 8 == 0 && d.row >= a.v.cols;
    if (!encode_matrix_map(&g, a.held, rows, a.vocab, a.held_pitch, kK) ||
        !encode_matrix_map(&h, a.h.ptr, a.v.rows, a.v.cols, a.h.row, kK) ||
        !(boxes ? encode_matrix_map(&out, d.ptr, a.vocab, a.v.cols, d.row, 32) : encode_matrix_map(&out, a.held, rows, a.vocab, a.held_pitch, 32)))
        return no_map();
    return launch<kGradWeight>(a, ProductArgs{a.vocab, a.v.cols, rows, first, last ? 1 : 0, boxes ? 1 : 0, kGradStretch}, g, h, out, st);
}

}  // namespace ctb
