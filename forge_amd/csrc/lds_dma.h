// LDS DMA of 16 (or 2) bytes a lane, lane l's to lds + 16 l (4 l, zero-extended), as in mfma_tile.h but written out:
// the compiler makes every transposing LDS read wait for all DMAs that it knows of, and counts the
// loads of a loop only where each of its paths has the same ones; either would end a prefetch. Nothing is returned
// in registers; the callers wait by count (wait_vmcnt), and their kernels' own loads are waited for in order with
// these, which is never too short. M0 has no other use in these kernels. The wait
// states that the compiler keeps for its own instructions are written out as well: one between M0 and the DMA that
// reads it, five between a vector instruction's scalar result (an address that was kept in a vector register, or a
// reloaded one) and a memory instruction that takes it.
#pragma once

#include "mfma_tile.h"

namespace forge_amd {

// s_waitcnt lgkmcnt(0) only.
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xC07F); }

__device__ __forceinline__ uint32_t lds_address(const int8_t* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const int8_t*)p));
}
__device__ __forceinline__ void dma16_rows(v4i rsrc, uint32_t voff, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(lds) : "memory");
#endif
}
__device__ __forceinline__ void dma16_at(const void* p, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "memory");
#endif
}
// A raw buffer resource over `bytes` from p, both wave-uniform.
__device__ __forceinline__ v4i row_rsrc(const void* p, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return v4i{__builtin_amdgcn_readfirstlane(static_cast<int>(a)),
               __builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32) & 0xFFFF), static_cast<int>(bytes), 0x00020000};
}
// From `off` bytes past a uniform base.
__device__ __forceinline__ void dma16_off(const void* base, uint32_t off, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
#endif
}
__device__ __forceinline__ void dma2_off(const void* base, uint32_t off, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_ushort %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
#endif
}

}  // namespace forge_amd
