// bf16x_umma.cuh -- the tcgen05 pieces that the GEMMs and the prompt attention
// share: shared-memory descriptors, commits, fences and the swizzled offset.
#pragma once

#include "bf16x_common.cuh"

namespace bf16x {

__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t smem_addr) {
    // K-major, 128-byte swizzle: rows of 128 bytes, 8-row atoms 1024 bytes apart
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3FFFu);          // start address
    d |= (uint64_t)1u << 16;                               // leading byte offset (unused for swizzled K-major)
    d |= (uint64_t)(1024u >> 4) << 32;                     // stride byte offset
    d |= (uint64_t)1u << 46;                               // descriptor version (sm100)
    d |= (uint64_t)2u << 61;                               // layout: SWIZZLE_128B
    return d;
}

__device__ __forceinline__ void umma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 :: "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Byte offset of element (row, col) inside a 128-row x 64-column K-major
// 128-byte-swizzled tile (16-byte chunk index XOR row % 8).
__device__ __forceinline__ uint32_t sw128_offset(uint32_t row, uint32_t col) {
    return row * 128u + ((((col >> 3) ^ row) & 7u) << 4) + ((col & 7u) << 1);
}

}  // namespace bf16x
