// tensor_core.cuh — the pieces of a product on the 5th-generation tensor cores by pairs of CTAs: tensor copies into
// swizzled shared memory, matrix descriptors, tcgen05.mma by one thread, accumulators in tensor memory.
//
// A pair (cluster of two CTAs, cta_group::2) computes one 256 x 256 tile: each CTA brings 128 rows of the left operand
// and 128 of the right one's, and the first CTA's thread issues the products over both. All waits are the bounded ones
// of async_copy.cuh. No copy uses cluster multicast.
#pragma once

#include "async_copy.cuh"

namespace ctb {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The address of the pair's first CTA's copy of a shared variable.
__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(p)));
    return a;
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// A box of a matrix into this CTA's shared memory; the bytes are counted on a barrier of either CTA of the pair.
// x times the element size is a multiple of 16 bytes; what lies outside the matrix arrives as zeros.
__device__ __forceinline__ void tensor_load_pair(uint32_t smem_dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::
            "r"(smem_dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* smem_dst, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(smem_dst)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}

__device__ __forceinline__ void tmem_free_pair(uint32_t address, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}

__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle, tile of 64 inner elements (128 bytes) a row, base on 1024 bytes.
//   inner dimension contiguous: rows of 128 bytes, `group` = 1024 bytes between groups of 8 rows (`atom` unused);
//   outer dimension contiguous: a row of 128 bytes is 64 outer elements of one inner index, `group` = 1024 bytes
//   between groups of 8 inner indexes, `atom` bytes between pieces of 64 outer elements.
__device__ __forceinline__ uint64_t matrix_descriptor(uint32_t address, uint32_t atom, uint32_t group) {
    return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | static_cast<uint64_t>(atom >> 4) << 16 |
           static_cast<uint64_t>(group >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}

// Instruction descriptor: bfloat16 operands, float32 sums.
constexpr uint32_t instruction_bf16(int m, int n, bool a_outer, bool b_outer) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (a_outer ? 1u << 15 : 0u) | (b_outer ? 1u << 16 : 0u) |
           static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
}

__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(instruction), "r"(static_cast<uint32_t>(add))
        : "memory");
}

// Arrives on the barrier at this offset in both CTAs once all products issued so far are done.
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}

// 32 columns of this warp's quarter of the lanes: thread t gets lane t's.
__device__ __forceinline__ void tmem_load32(float* r, uint32_t address) {
    uint32_t* const u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
          "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
          "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(address));
}

// The same of 16 columns.
__device__ __forceinline__ void tmem_load16(float* r, uint32_t address) {
    uint32_t* const u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(address));
}

__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// A box out of shared memory (swizzled as the map says) into a matrix; what lies outside the matrix is left out. One thread
// issues it, after proxy_fence() by the threads that wrote the box and a barrier among them.
__device__ __forceinline__ void tensor_store(const CUtensorMap* map, int x, int y, uint32_t smem_src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(smem_src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Until the boxes stored so far have been read, or have been written.
__device__ __forceinline__ void tensor_stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tensor_stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// 16 bytes of a row of 128 in a box of 32 rows, swizzled: the rows' same pieces lie in different banks.
__device__ __forceinline__ uint32_t swizzled_piece(uint32_t box, int row, int piece) {
    return box + static_cast<uint32_t>(row * 128 + ((piece ^ (row & 7)) << 4));
}
__device__ __forceinline__ void store_shared16(uint32_t to, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// A 2-D map of a row-major matrix [rows, cols] of 2- or 4-byte elements with `pitch` elements from row to row, for boxes of
// 128 bytes (one swizzled row each) by box_rows rows; false where the driver refuses it.
bool encode_matrix_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows,
                       int size = 2);  // async.cu

}  // namespace ctb
