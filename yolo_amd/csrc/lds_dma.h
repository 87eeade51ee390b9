// LDS-DMA (loads that go from memory straight to LDS) and the waits for it, for the gfx950 kernels
// that stage their tiles by hand.
#pragma once
#include "common.h"

namespace yolo_amd {

// One LDS-DMA instruction: 16 bytes per lane from gsrc (per lane) to lds_dst (wave-uniform) +
// 16 * lane.  Issued as inline assembly rather than through the builtin: once the compiler
// sees an LDS-DMA instruction it stops trusting the order in which LDS reads return and puts a
// full `s_waitcnt lgkmcnt(0)` in front of the first use of ANY ds_read result, which serialises
// "eight fragment reads, then twelve MFMAs" where counted waits let the first MFMAs start
// after the first reads.  The loads' own completion is tracked by hand anyway (wait_vmcnt).
#ifndef YOLO_AMD_ASM_DMA
#define YOLO_AMD_ASM_DMA 1
#endif
__device__ __forceinline__ void lds_dma16(const void* gsrc, char* lds_dst) {
#if YOLO_AMD_ASM_DMA
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds_dst;
    // (m0 is named as clobbered on purpose -- nothing else in these kernels uses it)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :
                 : "v"(gsrc), "s"(base)
                 : "memory", "m0");
#pragma clang diagnostic pop
#else
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)gsrc,
                                     (__attribute__((address_space(3))) void*)lds_dst, 16, 0, 0);
#endif
}

// The same with the address split into a wave-uniform base (a scalar register pair) and a
// 32-bit per-lane byte offset, plus OFF constant bytes (the instruction's offset field, which the
// hardware adds to the source address AND to the LDS address): the form for a source whose per-lane part
// never changes (weights: one offset register for the whole kernel, the walk over taps and
// channel chunks done in scalar arithmetic, no vector instruction per load -- the vector
// instructions of the tap loop compete with the MFMAs of the other waves for issue slots).
template <int OFF = 0>
__device__ __forceinline__ void lds_dma16_sv(const void* sbase, uint32_t lane_bytes, char* lds_dst) {
    static_assert(OFF >= 0 && OFF < 4096, "13-bit signed instruction offset");
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds_dst;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%3"
                 :
                 : "v"(lane_bytes), "s"(sbase), "s"(base), "n"(OFF)
                 : "memory", "m0");
#pragma clang diagnostic pop
}

// The same from a raw buffer: 16 bytes per lane from (descriptor base + soff + voff) to lds_dst + 16 * lane.
// The per-lane part is one 32-bit byte offset, the walk over a tensor goes through the scalar offset, and a
// lane whose offset lies beyond the descriptor's size reads as zero: padding needs no zero page, no select
// and no 64-bit address per lane.
__device__ __forceinline__ void lds_dma16_buf(__amdgpu_buffer_rsrc_t rsrc, uint32_t voff, uint32_t soff, char* lds_dst) {
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds_dst;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :
                 : "v"(voff), "s"(rsrc), "s"(soff), "s"(base)
                 : "memory", "m0");
#pragma clang diagnostic pop
}
constexpr uint32_t kRawBufferWord3 = 0x00020000u;  // untyped 32-bit raw buffer descriptor word 3
constexpr uint32_t kBufferNowhere = 0xFFFFFF00u;   // a byte offset beyond any descriptor these kernels build

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

}  // namespace yolo_amd
