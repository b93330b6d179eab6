/*  p2hip_async.h – direct loads from global memory into LDS and the waits for them.
 */
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace p2k {

/* Direct global → LDS loads (16 bytes per lane into 16-byte lane slots at lds + 16·lane). Issued from inline
 * assembly so that the compiler adds no waits of its own for them: the GEMM waits for them explicitly (wait_vm),
 * and the compiler's waits for its own loads stay correct since the vector-memory counter retires in order. */
__device__ __forceinline__ void dma_16(const void *src, const void *lds)
{
    const uint32_t a = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(a) : "memory", "m0");
}

/* s_waitcnt vmcnt(N) alone (expcnt and lgkmcnt left open); a compiler barrier for memory operations */
template <int N>
__device__ __forceinline__ void wait_vm()
{
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | (0x7 << 4) | (0xF << 8) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}

/* this wave's LDS reads complete, then the workgroup barrier; no wait on vector memory */
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

/* dma_16 from a base that is the same for all lanes and an offset of each, and the same of 4 bytes per lane (at lds +
 * 4·lane) from an address of each */
__device__ __forceinline__ void dma_16(const void *base, uint32_t offset, const void *lds)
{
    const uint32_t a = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(a)
                 : "memory", "m0");
}
__device__ __forceinline__ void dma_4(const void *src, const void *lds)
{
    const uint32_t a = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(a) : "memory", "m0");
}

/* dma_16 through a buffer descriptor: a byte offset per lane from its base; lanes whose bytes end past its size read
 * nothing. */
__device__ __forceinline__ void dma_16(__amdgpu_buffer_rsrc_t from, uint32_t offset, const void *lds)
{
    const uint32_t a = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(from), "s"(a)
                 : "memory", "m0");
}

}  // namespace p2k
