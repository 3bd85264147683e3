// svb_opaque.h -- a register that the optimiser may not look through.
//
// A value that is cheap to recompute from a register (an unpacked bf16, a centred input) is kept alive by the compiler from its first
// use to its last once it has computed it.  Where the last use lies behind a barrier, making the source opaque there forces the cheap
// recomputation instead of the second register.  No instruction is emitted.
// Included as <svb_opaque.h>: tests/emu/include/ holds the lane emulator's stand-in.
#pragma once
#include <hip/hip_runtime.h>

__device__ __forceinline__ void svb_opaque(unsigned& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void svb_opaque(float& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void svb_opaque(long long& v) { asm volatile("" : "+v"(v)); }      // (an offset: an opaque pointer would be a flat one)
__device__ __forceinline__ void svb_opaque_uniform(long long& v) { asm volatile("" : "+s"(v)); }      // (the same in every lane)
