// The sm_100a instructions of the 8-bit product: tensor-map copies into
// swizzled shared memory, matrix instructions into tensor memory and the reads
// back.  Every wait has a time limit.
#pragma once

#include "bulk_copy.cuh"

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace mdsoap {
namespace tc {

using bulk::smem_u32;

// 2-D tile load; x (bytes here) must be a multiple of 16, out-of-range elements arrive as zero.
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
            "r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}

// The same into this CTA's shared memory, completing on the pair's first CTA's barrier.
__device__ __forceinline__ void load_tile_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// 2-D tile store out of shared memory; parts outside the matrix are cut off, along a row at whole 16 bytes.
__device__ __forceinline__ void store_tile(const CUtensorMap* map, int x, int y, const void* src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x),
                 "r"(y), "r"(smem_u32(src))
                 : "memory");
}
// Ends a group of this thread's stores; a group may be empty.
__device__ __forceinline__ void end_stores() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// Until all but the last LEFT groups have read their shared memory.
template <int LEFT>
__device__ __forceinline__ void wait_store_reads() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory");
}

// ------------------------------------------------------------ clusters

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Cluster-wide address of a shared variable of CTA `rank`.
__device__ __forceinline__ uint32_t map_shared(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// Arrives on a barrier of any CTA of the cluster.  It hands on no data in memory
// (a release at cluster scope would wait for the thread's loads and stores).
__device__ __forceinline__ void arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float load_shared_at(uint32_t address) {
    float f;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(address) : "memory");
    return f;
}

__device__ __forceinline__ int load_int_at(uint32_t address) {
    int i;
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(i) : "r"(address) : "memory");
    return i;
}
__device__ __forceinline__ void store_shared_at(uint32_t address, int value) {
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(address), "r"(value) : "memory");
}
// Counts bytes on a barrier of this CTA that were announced and no copy will bring.
__device__ __forceinline__ void complete_bytes(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// One warp allocates `columns` of tensor memory (a power of two from 32 on) and
// the same warp frees them.
template <int GROUP>
__device__ __forceinline__ void alloc(uint32_t* address, uint32_t columns) {
    if constexpr (GROUP == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(address)),
                     "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(address)),
                     "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int GROUP>
__device__ __forceinline__ void dealloc(uint32_t address, uint32_t columns) {
    if constexpr (GROUP == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
}

__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// Descriptor of a K-major operand in 128-byte swizzled shared memory: rows of
// 128 bytes, groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(const void* tile) {
    return (uint64_t)((smem_u32(tile) & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// Instruction word: e4m3 x e4m3 into float32, M x N.
__host__ __device__ constexpr uint32_t instruction(int m, int n) { return 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24; }

// D (+)= A B^T over 32 bytes of K; issued by one thread.  GROUP 2: by the first
// CTA of a pair, each CTA holding half of A's and B's rows at the same
// addresses and half of D's rows.
template <int GROUP>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t word, bool add) {
    if constexpr (GROUP == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(word), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(word), "r"((uint32_t)add)
            : "memory");
}

// Arrives on `bar` (GROUP 2: on both CTAs' barriers at this address) once the
// matrix instructions this thread issued so far are done.
template <int GROUP>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if constexpr (GROUP == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                     : "memory");
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
}

// 32 columns of the warp's 32 lanes of tensor memory; complete after wait_loads.
__device__ __forceinline__ void load32(uint32_t address, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(address)
        : "memory");
}
__device__ __forceinline__ void load(uint32_t address, uint32_t (&r)[32]) { load32(address, r); }
__device__ __forceinline__ void load(uint32_t address, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(address)
                 : "memory");
}
__device__ __forceinline__ void load(uint32_t address, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(address)
        : "memory");
}
__device__ __forceinline__ void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Waits for a barrier phase; false (and *gave_up set) once a second has passed
// or another thread of the CTA gave up.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
    if (bulk::try_wait(bar, parity) || (!*gave_up && bulk::try_wait(bar, parity))) return true;
    const uint64_t start = bulk::global_ns();
    while (!bulk::try_wait(bar, parity)) {
        if (*gave_up) return false;
        if (bulk::global_ns() - start > 1000000000ull) {
            *gave_up = 1;
            return false;
        }
    }
    return true;
}

// Whether `x` is non-zero in any of the `threads` threads that meet at barrier `id`.
__device__ __forceinline__ bool any_of(int id, int threads, int x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.s32 p, %3, 0;\n\t"
        "bar.red.or.pred q, %1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(id), "r"(threads), "r"(x)
        : "memory");
    return r != 0;
}

// Registers a thread of the calling warpgroup (all four warps): fewer, or more
// out of what others of the CTA gave up.
template <int COUNT>
__device__ __forceinline__ void give_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(COUNT));
}
template <int COUNT>
__device__ __forceinline__ void take_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(COUNT));
}

// ------------------------------------------------------------ pairs of floats

__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void split_pair(uint64_t p, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

}  // namespace tc
}  // namespace mdsoap
