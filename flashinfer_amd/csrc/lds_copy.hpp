// Global -> LDS copies, their wait, and the LDS row swizzles of the tiled
// kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mimoe {

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// LDS byte address of a pointer into __shared__ memory.
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(size_t)(lds_ptr_t)p;
}

// 16-byte global -> LDS copy: lane l's 16 bytes land at lds_base + 16 * l
// (lds_base must be wave-uniform; gfx950 global_load_lds_dwordx4).
//
// Written as inline asm on purpose: the compiler cannot tell that a copy into
// one LDS stage does not alias reads of the other stage, and would put a
// vmcnt(0) wait in front of every LDS read, serialising copy and compute.
// The kernels using these place their own vmcnt waits before each barrier.
// One wait state between the M0 write and the LDS DMA is required.
__device__ __forceinline__ void g2l16(const void* gsrc, void* lds_base) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :
                 : "v"(gsrc), "s"(lds_addr(lds_base))
                 : "memory", "m0");
}

// 4-byte global -> LDS copy: lane l's dword lands at lds_base + 4 * l.
__device__ __forceinline__ void g2l4(const void* gsrc, void* lds_base) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
                 :
                 : "v"(gsrc), "s"(lds_addr(lds_base))
                 : "memory", "m0");
}

// The same two copies with a wave-uniform 64-bit base in SGPRs and a 32-bit
// per-lane byte offset (the saddr form: address = sbase + voff): one VGPR per
// copy instead of a 64-bit address per lane.
__device__ __forceinline__ void g2l16s(const void* sbase, uint32_t voff, void* lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(voff), "s"(sbase), "s"(lds_addr(lds_base))
                 : "memory", "m0");
}

// g2l16s for data that nothing reads again: it leaves nothing in the caches.
__device__ __forceinline__ void g2l16s_once(const void* sbase, uint32_t voff, void* lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                 :
                 : "v"(voff), "s"(sbase), "s"(lds_addr(lds_base))
                 : "memory", "m0");
}

__device__ __forceinline__ void g2l4s(const void* sbase, uint32_t voff, void* lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
                 :
                 : "v"(voff), "s"(sbase), "s"(lds_addr(lds_base))
                 : "memory", "m0");
}

__device__ __forceinline__ void wait_vmem() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// XOR swizzle of the 16-byte chunk index inside a 128-byte LDS row: 16
// consecutive rows reading the same logical chunk hit 16 distinct 16-byte
// bank groups (conflict-free for 32- and 64-bank LDS).
__device__ __forceinline__ int swz8(int row) { return (row & 7) ^ ((row >> 3) & 1); }

// Swizzle of a 128-byte row whose reads are also conflict-free when 32 lanes
// (16 rows x two adjacent chunks) are serviced together: for the four rows
// r, r+4, r+8, r+12 that share a bank group the values differ in their upper
// two bits, so chunks c and c^1 of those rows land on 8 distinct positions;
// 16 rows at one chunk still take 16 distinct bank groups. A copy of 8 rows
// x 8 chunks still reads each row's 128 bytes whole.
__device__ __forceinline__ int swzq(int row) { return (((row >> 2) & 3) << 1) | ((row >> 1) & 1); }

// Same for a 256-byte row of 16 chunks.
__device__ __forceinline__ int swz16(int row) { return row & 15; }

}  // namespace mimoe
