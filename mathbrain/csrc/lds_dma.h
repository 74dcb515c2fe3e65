// Loads from memory straight into LDS, and what goes with them.
#pragma once

#include "common.h"

namespace mb {

// 16 (or 4) bytes a lane from base + voff to LDS at lds + 16 (or 4) * lane.  M0 holds the LDS address; the compiler
// reserves it for its own instructions, which set it before they use it, warns of the clobber for that reason, and
// has to know of it so that it keeps no value there from one of them to the next.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ inline void dma16(uint32_t lds, uint32_t voff, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds), "v"(voff), "s"(base)
                 : "memory", "m0");
}
__device__ inline void dma4(uint32_t lds, uint32_t voff, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :
                 : "s"(lds), "v"(voff), "s"(base)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
// Waits until at most N of the wave's loads are on their way, and for the other waves.
template <int N>
__device__ inline void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

__device__ inline int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ inline uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

}  // namespace mb
