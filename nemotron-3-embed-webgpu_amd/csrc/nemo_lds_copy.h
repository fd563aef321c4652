// Copies from memory into LDS without registers between, and the barrier that
// goes with them (gfx950).
#pragma once

#include "nemo_common.h"

namespace nemo {

typedef __attribute__((address_space(3))) void lds_void;

// Copies of 16 bytes a lane into LDS at `to` + 16 lane, from a buffer's range
// (zeros past its end) or an address. The compiler, which knows of the builtin for this that
// it writes LDS, waits for every copy in flight before each transposed read;
// written as here it has no register to be waited for, and the loops wait
// for their images themselves. (m0 is reserved: the compiler sets it where it
// uses it itself.)
__device__ __forceinline__ uint32_t lds_address(const uint8_t* to) { return (uint32_t)(uintptr_t)(lds_void*)to; }
__device__ __forceinline__ void copy_range(u32x4 range, uint32_t offset, const uint8_t* to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds_address(to)), "v"(offset), "s"(range)
               : "memory");
}
__device__ __forceinline__ void copy_address(const void* from, const uint8_t* to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds_address(to)), "v"(from)
               : "memory");
}
// A barrier that waits for none of the wave's work in flight; no access of
// memory is moved over it.
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace nemo
