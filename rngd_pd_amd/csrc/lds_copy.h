// Copies from memory straight into LDS (gfx950), for rings of tiles that are read
// while younger ones are under way.
#pragma once

#include "pdk_common.h"

namespace pdk {

typedef __attribute__((address_space(3))) const void lds_ptr;

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(lds_ptr*)p;
}

// 16 bytes a lane from `base` (uniform) + `at` bytes (per lane) to LDS address `to`
// (uniform) + 16 * lane. The compiler's builtin makes it wait for all copies under way
// before any LDS read that it cannot tell from their targets; of a statement it knows
// nothing, so the waits are the caller's: copies_done before a tile is read. There is
// no output register, and a compiler's own wait for a vector load counts fewer loads than
// are under way, so that it can only wait for too many (a kernel's own loads are best
// consumed before its loop: settle). One wait state lies between M0's write and the
// copy that reads it.
__device__ __forceinline__ void copy16(const void* base, uint32_t at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(at), "s"(base), "s"(to)
               : "memory", "m0");
}

// The same with 4 bytes a lane.
__device__ __forceinline__ void copy4(const void* base, uint32_t at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(at), "s"(base), "s"(to)
               : "memory", "m0");
}

// The loads of x have arrived from here on.
__device__ __forceinline__ void settle(v8& x) {
  asm volatile("" : "+v"(x.w[0]), "+v"(x.w[1]), "+v"(x.w[2]), "+v"(x.w[3]));
}

// All but the youngest N of this wavefront's loads have arrived and its LDS reads are
// done; then the workgroup's barrier.
template <int N>
__device__ __forceinline__ void copies_done() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

}  // namespace pdk
