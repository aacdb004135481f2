// losses_ring.cuh — what the loss kernels over rows of unit stride share: a row cut into 16-byte packs and the
// few elements around them, exponentials of pairs of floats, clusters, and the copies in and out of a
// shared-memory ring (async_copy.cuh).
//
// Accuracy of the sums. log2(e)/T as one float32 is off by up to 6e-8 relative, and so is every t = d log2(e)/T
// and with it, one-sidedly, the sum; a sequence's log-probabilities add that up. So t is taken with log2(e)/T in two
// parts, rounded once, and raised by the mean error of the hardware's 2^t (log-probabilities on B200, [4000, 32768]
// at T = 0.8, 1, 2: mean error 8e-9, 5e-9, 9e-9 and less; 4e-8 to 8e-8 without either). The gradients of the losses use it
// too; the backward pass of the log-probabilities does without (row_exp_shifted). Long sums are taken in two levels, a stage's share of a
// thread and then the stages, so that small terms are not lost against a grown sum ([2048, 131072] logits of
// standard deviation 4 in one level: 1.7e-7 low on average).
#pragma once

#include "async_copy.cuh"
#include "losses.cuh"

namespace ctb {

constexpr int kMaxCluster = 8;
constexpr int kBatch = 32;  // rows whose operands a producer warp reads together, one a lane
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

// The hardware's 2^t is 5.0e-8 low on average (measured on B200 over t in [-30, -1], 2^24 points; 2.9e-8 over [-1, 0]):
// t is raised by that before it is rounded. 2^0 stays 1.
constexpr float kExpBias = 7.2e-8f;  // 5.0e-8 log2(e)

// exp of pairs: t = d c + d rho, the first product and the sum rounded once together, with c = log2(e)/T rounded
// down and rho its rest. rho is positive, so that d = -inf stays -inf.
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
    const F2 d = add2(x, minus_m);
    const F2 t = fma2(d, k.c, fma2(d, k.rho, f2(kExpBias, kExpBias)));
    float a, b;
    un(t, a, b);
    return f2(exp2_fast(a), exp2_fast(b));
}
__device__ __forceinline__ float exp_one(const LossArgs& a, float x, float m) {
    const float d = x - m;
    return exp2_fast(fmaf(d, a.c2_down, fmaf(d, a.c2_rest, kExpBias)));
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

// Waits as mbar_wait does, but asks the hardware to suspend the warp between looks: two helper warps and the
// consumers that wait poll a quarter of a kernel's instructions away otherwise. CLUSTER: threads of other CTAs
// of the cluster contribute to the phase.
template <bool CLUSTER = false> __device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity) {
    constexpr uint32_t kSuspendNs = 20000;
    uint64_t t0 = 0;
    for (;;) {
        uint32_t done;
        if (CLUSTER)
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(done)
                : "r"(smem_addr(bar)), "r"(parity), "r"(kSuspendNs)
                : "memory");
        else
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(done)
                : "r"(smem_addr(bar)), "r"(parity), "r"(kSuspendNs)
                : "memory");
        if (done) return true;
        const uint64_t now = global_ns();
        if (t0 == 0) t0 = now;
        else if (now - t0 > kWaitLimitNs) return false;
    }
}

// Rank r's share of a row's packs.
__device__ __forceinline__ void slice_of(int packs, int rank, int size, int& first, int& count) {
    first = static_cast<int>(static_cast<int64_t>(packs) * rank / size);
    count = static_cast<int>(static_cast<int64_t>(packs) * (rank + 1) / size) - first;
}

// The elements around a row's whole packs, as a mask: bits 0..7 for columns 0, 1, ... before them, bits 8..15 for
// columns `behind`, `behind` + 1, ... behind them.
__device__ __forceinline__ uint32_t edges_of(const LossArgs& a, int head, int behind) {
    return ((1u << head) - 1u) | ((1u << (static_cast<int>(a.cols) - behind)) - 1u) << 8;
}
__device__ __forceinline__ int edge_column(int l, int behind) { return l < 8 ? l : behind + l - 8; }

// Reads the edges of up to 32 rows, lane i's being row i: to[16 i + l], -inf where there is none. Sixteen rows' loads
// are on their way at once; one row after the other took 10 us for 32.
template <class T>
__device__ __forceinline__ void read_edges(const T* x, int64_t x_off, uint32_t edges, int behind, int n, int lane, float* to) {
    const int l = lane & 15;
    for (int i0 = 0; i0 < n; i0 += 16) {
        T raw[8];
        uint32_t have = 0u;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = i0 + 2 * u + (lane >> 4);
            const uint32_t m = __shfl_sync(0xffffffffu, edges, i);
            const int64_t off = __shfl_sync(0xffffffffu, x_off, i);
            const int tail = __shfl_sync(0xffffffffu, behind, i);
            if (i < n && (m >> l & 1u)) {
                raw[u] = x[off + edge_column(l, tail)];
                have |= 1u << u;
            }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = i0 + 2 * u + (lane >> 4);
            if (i < n) to[16 * i + l] = have >> u & 1u ? LossElem<T>::up(raw[u]) : -INFINITY;
        }
    }
}

// ------------------------------------------------------------------------------------------------
// host side (losses_stream.cu)

// Starts `fn` with clusters of `cluster` CTAs, as a programmatic dependent of the kernel before it.
int launch_cluster(const void* fn, unsigned grid, int threads, int cluster, size_t smem, cudaStream_t st, void** args);

// How many clusters of `cluster` CTAs of `fn` are resident at once on the current device (cached). Also opts
// the kernel in to its shared memory there.
int resident_blocks(const void* fn, int threads, int cluster, size_t smem, int* out);

}  // namespace ctb
