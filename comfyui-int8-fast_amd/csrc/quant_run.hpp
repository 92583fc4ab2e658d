// The int8 rounding of rows of 16-bit values: shared by the quantisers and by what quantises its own result.
#pragma once

#include "i8f_common.hpp"

namespace i8f {
namespace {

// the sum over the wave in a fixed order (the same in every lane)
__device__ __forceinline__ float wave_sum_all(float v) {
#pragma unroll
    for (int b = 1; b < 64; b <<= 1) v += __shfl_xor(v, b, 64);
    return v;
}

__device__ __forceinline__ float max3_abs(float m, float a, float b) {
    float r;
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(m), "v"(a), "v"(b));
    return r;
}

// scale = max(amax / 127, 1e-30) and inv = 1 / scale, both correctly rounded, for an amax that is a value of a 16-bit
// dtype, without the division sequence (22 instructions of a wave's fixed work become 8):
//   amax / 127 = fma(r, y, q) with y = RN(1 / 127), q = RN(amax y), r = amax - 127 q (exact): Markstein's correction,
//     which gives the correctly rounded quotient for every finite bfloat16 and binary16 amax whose quotient is not
//     below the 1e-30 floor (every such value is checked on the host by the test suite);
//   1 / scale = fma(e, y0, y0) with y0 the hardware reciprocal (1 ulp) and e = 1 - scale y0: correctly rounded unless
//     the significand of scale is all ones (Markstein), which takes the division.
// MIXED: the lanes hold scales of several rows (else one scale, tested as a scalar)
template <bool MIXED = false>
__device__ __forceinline__ void scale_and_inverse16(float amax, float &scale, float &inv) {
    const float y = 0x1.020408p-7f;  // RN(1 / 127)
    const float q = amax * y;
    const float r = __builtin_fmaf(-127.0f, q, amax);
    float s = __builtin_fmaf(r, y, q);
    s = s < 1e-30f ? 1e-30f : s;
    const float y0 = __builtin_amdgcn_rcpf(s);
    const float e = __builtin_fmaf(-s, y0, 1.0f);
    float iv = __builtin_fmaf(e, y0, y0);
    // (a branch that is practically never taken)
    const bool ones = MIXED ? __builtin_amdgcn_ballot_w64((__float_as_uint(s) & 0x7fffffu) == 0x7fffffu) != 0
                            : (__builtin_amdgcn_readfirstlane(__float_as_uint(s)) & 0x7fffffu) == 0x7fffffu;
    if (__builtin_expect(ones, 0)) iv = 1.0f / s;
    scale = s;
    inv = iv;
}

// Sixteen values of one run to sixteen int8 in four dwords.  p + 1.5 * 2^23 leaves the rounded integer in the low byte
// of the sum; the additions after the first of each dword write that byte straight into its place (an SDWA destination
// select with the other bytes preserved), so nothing is left to shuffle: 32 instructions per run instead of 44.  An
// instruction that writes part of a register must not be followed at once by a reader of that register: the four dwords
// are worked on in turn, which puts three instructions between any two that touch the same one.
// inv: the inverse scale of the first eight, inv2 that of the others.
__device__ __forceinline__ uint4 quant16_magic(const float (&v)[16], float inv, float inv2) {
    float p[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) p[j] = v[j] * (j < 8 ? inv : inv2);
    const float M = 12582912.0f;
    uint32_t o0, o1, o2, o3;
#define I8F_SDWA_ADD(d, s, b) "v_add_f32_sdwa %" #d ", %" #s ", %20 dst_sel:BYTE_" #b " dst_unused:UNUSED_PRESERVE src0_sel:DWORD src1_sel:DWORD\n\t"
    asm("v_add_f32 %0, %4, %20\n\tv_add_f32 %1, %8, %20\n\tv_add_f32 %2, %12, %20\n\tv_add_f32 %3, %16, %20\n\t"
        I8F_SDWA_ADD(0, 5, 1) I8F_SDWA_ADD(1, 9, 1) I8F_SDWA_ADD(2, 13, 1) I8F_SDWA_ADD(3, 17, 1)
        I8F_SDWA_ADD(0, 6, 2) I8F_SDWA_ADD(1, 10, 2) I8F_SDWA_ADD(2, 14, 2) I8F_SDWA_ADD(3, 18, 2)
        I8F_SDWA_ADD(0, 7, 3) I8F_SDWA_ADD(1, 11, 3) I8F_SDWA_ADD(2, 15, 3) I8F_SDWA_ADD(3, 19, 3)
        "s_nop 0"
        : "=&v"(o0), "=&v"(o1), "=&v"(o2), "=&v"(o3)
        : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7]), "v"(p[8]), "v"(p[9]),
          "v"(p[10]), "v"(p[11]), "v"(p[12]), "v"(p[13]), "v"(p[14]), "v"(p[15]), "v"(M));
#undef I8F_SDWA_ADD
    return make_uint4(o0, o1, o2, o3);
}
__device__ __forceinline__ uint4 quant16_magic(const float (&v)[16], float inv) { return quant16_magic(v, inv, inv); }

}  // namespace
}  // namespace i8f
