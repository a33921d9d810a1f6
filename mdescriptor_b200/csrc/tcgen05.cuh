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

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// One warp allocates `columns` of tensor memory (a power of two from 32 on) and
// the same warp frees them.
__device__ __forceinline__ void alloc(uint32_t* address, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(address)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc(uint32_t address, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
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

// D (+)= A B^T over 32 bytes of K; issued by one thread.
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t word, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(word), "r"((uint32_t)add)
        : "memory");
}

// Arrives on `bar` once the matrix instructions this thread issued so far are done.
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
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
__device__ __forceinline__ void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Waits for a barrier phase; false (and *gave_up set) once a second has passed
// or another thread of the CTA gave up.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
    if (bulk::try_wait(bar, parity)) return true;
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

}  // namespace tc
}  // namespace mdsoap
