// tcgen05.cuh -- PTX glue of the paired-CTA tensor-core kernels: mbarriers in
// a cluster of two, TMA tile copies that signal the leader's
// barrier, tcgen05 allocation, products and commits with cta_group::2.
#pragma once

#include "common.cuh"

namespace jlb {
namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The address in CTA `rank` of the cluster of this CTA's shared address.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// A cluster barrier before which every operation of this CTA is performed, its
// arrivals on the other CTA's barriers among them.
__device__ __forceinline__ void cluster_sync_released() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A cluster barrier that orders no memory of its own: callers publish nothing
// by it but what they have fenced (a releasing one waits for every store of
// the epilogue, about 1 us at a kernel's end).
__device__ __forceinline__ void cluster_sync_relaxed() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
        : "memory");
}
__device__ __forceinline__ void mbar_arrive_elect(uint32_t bar, uint32_t count) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e mbarrier.arrive.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(count)
        : "memory");
}
// Stores one word in a CTA of the cluster and counts its 4 bytes on a barrier
// there (both shared::cluster addresses).
__device__ __forceinline__ void store_remote(uint32_t addr, uint32_t value, uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(addr), "r"(value),
                 "r"(bar)
                 : "memory");
}
// `count` arrivals on a barrier of this CTA.
__device__ __forceinline__ void mbar_arrive_count(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
// Arrives on a barrier of any CTA of the cluster (shared::cluster address).
// What it reports is done and fenced before (TMEM reads by tcgen05.fence, row
// copies by a proxy fence), so the default CTA-scope release is enough; a
// cluster-scope release took about 1 us an arrival here.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}

// Copies whose completion is counted on `bar`, a barrier of either CTA of the
// pair (shared::cluster address); the destination is in this CTA.  Issued, like
// the arrivals below, by one elected lane of a converged warp, so that their
// operands stay in uniform registers (from a branch of one lane each product
// took some 75 cycles to issue).
__device__ __forceinline__ void tma_2d(uint32_t dst, const void *map, uint32_t bar, int x, int y) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const void *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];\n\t}" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const void *map, uint32_t bar, int x, int y, int z, int w) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];\n\t}" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// Arrives, once the elected lane's products so far are done, on the barrier at
// this offset in both CTAs of the pair; called by a converged warp.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void alloc_pair(uint32_t smem_dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc_pair(uint32_t tmem, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle: start address, leading
// and stride byte offsets in 16-byte units, descriptor version 1.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 |
           (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// bf16 x bf16 -> fp32, M x N; *_mn: the operand's outer dimension is
// contiguous in shared memory (else its inner one).
__device__ __forceinline__ uint32_t instr_desc(uint32_t m, uint32_t n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           ((n >> 3) << 17) | ((m >> 4) << 24);
}

// Four products of 16 inner elements each, issued by one elected lane of a
// converged warp: the descriptors' low (address) words advance by a_step and
// b_step (16-byte units, no carry: addresses stay below 256 KB).  first == 0
// overwrites D.
template <int A_STEP, int B_STEP>
__device__ __forceinline__ void mma_pair_k64(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                             uint32_t idesc, uint32_t first) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\t.reg .b32 t, u;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %6, p;\n\t"
        "add.u32 t, %1, %7;\n\tadd.u32 u, %3, %8;\n\t"
        "mov.b64 a, {t, %2};\n\tmov.b64 b, {u, %4};\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %6, 1;\n\t"
        "add.u32 t, t, %7;\n\tadd.u32 u, u, %8;\n\t"
        "mov.b64 a, {t, %2};\n\tmov.b64 b, {u, %4};\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %6, 1;\n\t"
        "add.u32 t, t, %7;\n\tadd.u32 u, u, %8;\n\t"
        "mov.b64 a, {t, %2};\n\tmov.b64 b, {u, %4};\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %6, 1;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(first), "r"(idesc), "n"(A_STEP), "n"(B_STEP)
        : "memory");
}

#define JLB_TC_LD32(taddr, r)                                                                \
    asm volatile(                                                                            \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "                                            \
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"                            \
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"          \
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),           \
          "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),         \
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),     \
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),     \
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),     \
          "=r"(r[30]), "=r"(r[31])                                                           \
        : "r"(taddr)                                                                         \
        : "memory")
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

}  // namespace tc
}  // namespace jlb
