// Direct global -> LDS loads: shared by the int8 GEMM and the first product of the adapters.
#pragma once

#include "i8f_common.hpp"

namespace i8f {
namespace gemm {

typedef int v4i __attribute__((ext_vector_type(4)));

// chunk swizzle: a function of the low 5 bits of the row only
template <int CPR>
__device__ __forceinline__ int swz(int r) {
    if constexpr (CPR == 4) return ((r >> 1) & 3) ^ ((r >> 3) & 1);
    else return (r ^ ((r >> 3) & 3)) & 7;
}

__device__ __forceinline__ constexpr int waitcnt_vm(int n) {
    // gfx9 encoding: vmcnt[3:0] | expcnt[6:4] | lgkmcnt[11:8] | vmcnt_hi[15:14]; others left at "no wait"
    return (n & 0xf) | (0x7 << 4) | (0xf << 8) | (((n >> 4) & 0x3) << 14);
}

typedef __attribute__((address_space(3))) void *lds_ptr_t;

// One wave-wide global -> LDS load of 16 bytes per lane (lane l lands at lds_base + 16 l), issued
// from inline assembly on purpose: the compiler knows nothing of an LDS write in flight, so it does
// not put a full vmcnt(0) wait in front of every later LDS read (it cannot prove that the reads
// touch another stage).  The waits for these loads are the explicit s_waitcnt of the main loop.
__device__ __forceinline__ void dma16(v4i rsrc, uint32_t lds_base, uint32_t voffset, int soffset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds_base), "v"(voffset), "s"(rsrc), "s"(soffset)
                 : "memory", "m0");
}

__device__ __forceinline__ v4i make_rsrc(const void *p, uint32_t bytes) {
    const uint64_t a = (uint64_t)p;
    v4i r = {(int)(uint32_t)a, (int)((uint32_t)(a >> 32) & 0xffffu), (int)bytes, 0x00020000};
    return r;
}

}  // namespace gemm
}  // namespace i8f
