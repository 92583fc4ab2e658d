// The 128-point Hadamard rotation of 16-bit rows with 16 consecutive elements (a run) to a lane: shared by the quantiser and
// the small-batch kernel.
#pragma once

#include "i8f_common.hpp"

namespace i8f {
namespace {

template <int DT>
__device__ __forceinline__ void expand16(const uint4 &a, const uint4 &b, float (&v)[16]) {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (DT == I8F_BF16) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
            v[2 * j] = f16_bits_to_f32(w[j] & 0xffffu);
            v[2 * j + 1] = f16_bits_to_f32(w[j] >> 16);
        }
    }
}

// v[j] += sign * (v[j] of the partner lane) for 16 registers: v_fmac_f32 with a DPP source.  The
// compiler does not fold a DPP move into a fused multiply-add, hence the assembly.  A DPP read of a
// register needs two wait states after a vector write of it, which the compiler cannot see inside
// the block: the s_nop covers the instruction in front of it, and inside it every instruction
// touches another register.
#define I8F_DPP_FMAC(n, ctrl) "v_fmac_f32_dpp %" #n ", %" #n ", %16 " ctrl " row_mask:0xf bank_mask:0xf bound_ctrl:0\n\t"
#define I8F_DPP_FMAC16(ctrl)                                                                                       \
    asm volatile("s_nop 1\n\t" I8F_DPP_FMAC(0, ctrl) I8F_DPP_FMAC(1, ctrl) I8F_DPP_FMAC(2, ctrl) I8F_DPP_FMAC(3, ctrl)  \
                 I8F_DPP_FMAC(4, ctrl) I8F_DPP_FMAC(5, ctrl) I8F_DPP_FMAC(6, ctrl) I8F_DPP_FMAC(7, ctrl)             \
                 I8F_DPP_FMAC(8, ctrl) I8F_DPP_FMAC(9, ctrl) I8F_DPP_FMAC(10, ctrl) I8F_DPP_FMAC(11, ctrl)           \
                 I8F_DPP_FMAC(12, ctrl) I8F_DPP_FMAC(13, ctrl) I8F_DPP_FMAC(14, ctrl) I8F_DPP_FMAC(15, ctrl)         \
                 : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]), "+v"(v[4]), "+v"(v[5]), "+v"(v[6]), "+v"(v[7]),  \
                   "+v"(v[8]), "+v"(v[9]), "+v"(v[10]), "+v"(v[11]), "+v"(v[12]), "+v"(v[13]), "+v"(v[14]),         \
                   "+v"(v[15])                                                                                     \
                 : "v"(sign))
template <int STAGE>
__device__ __forceinline__ void dpp_fmac16(float (&v)[16], float sign) {
    if constexpr (STAGE == 0) I8F_DPP_FMAC16("quad_perm:[1,0,3,2]");
    else if constexpr (STAGE == 1) I8F_DPP_FMAC16("quad_perm:[2,3,0,1]");
    else I8F_DPP_FMAC16("row_half_mirror");
}

template <int DT>
__device__ __forceinline__ void rotate_run16(float (&v)[16], float s0, float s1, float s2) {
#pragma unroll
    for (int s = 1; s < 16; s <<= 1) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if ((j & s) == 0) {
                const float lo = v[j], hi = v[j + s];
                v[j] = lo + hi;
                v[j + s] = lo - hi;
            }
        }
    }
    // Across lanes a stage is own + sign * other: the lower lane gets own + other, the upper lane
    // own - other, which is the negative of the butterfly's other - own.  Negation is exact and
    // commutes with every rounding, both lanes of a later pair carry the same accumulated sign, and
    // the product of the three signs is folded into the final multiplication (hs = +-h).  One
    // fused multiply-add with a DPP operand per element and stage; the product by +-1 is exact, so
    // the sum is rounded once, as an addition would be.
    dpp_fmac16<0>(v, s0);   // quad_perm [1,0,3,2]
    dpp_fmac16<1>(v, s1);   // quad_perm [2,3,0,1]
    dpp_fmac16<2>(v, s2);   // row_half_mirror
    const float h = hadamard_entry<DT>() * (s0 * s1 * s2);
    // bfloat16: the packed conversion with a zero in the low half leaves the rounded value in the high half, which IS its
    // binary32 form: one instruction rounds and widens (two values per conversion would need two more instructions to pull
    // them apart again).  binary16: two values to a conversion, one more each to widen them.
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
        if constexpr (DT == I8F_BF16) {
            v[j] = __uint_as_float(f32x2_to_bf16x2_bits(0.0f, v[j] * h));
            v[j + 1] = __uint_as_float(f32x2_to_bf16x2_bits(0.0f, v[j + 1] * h));
        } else if constexpr (DT == I8F_F16) {
            const half2v a = f32x2_to_half2(v[j] * h, v[j + 1] * h);
            v[j] = (float)a.x, v[j + 1] = (float)a.y;
        } else {
            v[j] *= h, v[j + 1] *= h;
        }
    }
}

// binary32 rows: a 128-block is 32 chunks of 4 elements, held by an aligned group of 32 lanes.  Strides 1, 2 of the
// butterfly stay inside a lane; strides 4 ... 32 pair chunks c and c ^ 1, c ^ 2, c ^ 4, c ^ 8, which DPP reaches as lanes
// l ^ 1, l ^ 2 (quad permutes), l ^ 7 (mirror of 8 lanes) and l ^ 15 (mirror of a row of 16) if lane l holds chunk
//   c(l) = (l & 3) ^ (7 if bit 2 of l) ^ (12 if bit 3 of l)     (linear over GF(2): c(l ^ 7) = c(l) ^ 4, c(l ^ 15) = c(l) ^ 8)
// of its group of 16; stride 64 pairs the two rows of 16 of the group through one lane exchange.  As in rotate_run16 a
// DPP stage is own + sign * other (one fused multiply-add whose product is exact), which leaves the upper chunk of a
// pair with the negative of the butterfly's value; both lanes of every later pair carry the same accumulated sign, and
// the product of the four signs is folded into the final multiplication.  Same fixed-order butterfly, 4 of the 5
// cross-lane stages without an LDS round trip.
__device__ __forceinline__ int chunk_of_lane16(int l) { return (l & 3) ^ ((l & 4) ? 7 : 0) ^ ((l & 8) ? 12 : 0); }

#define I8F_DPP_FMAC4(ctrl)                                                                                              \
    asm volatile("s_nop 1\n\t"                                                                                           \
                 "v_fmac_f32_dpp %0, %0, %4 " ctrl " row_mask:0xf bank_mask:0xf bound_ctrl:0\n\t"                        \
                 "v_fmac_f32_dpp %1, %1, %4 " ctrl " row_mask:0xf bank_mask:0xf bound_ctrl:0\n\t"                        \
                 "v_fmac_f32_dpp %2, %2, %4 " ctrl " row_mask:0xf bank_mask:0xf bound_ctrl:0\n\t"                        \
                 "v_fmac_f32_dpp %3, %3, %4 " ctrl " row_mask:0xf bank_mask:0xf bound_ctrl:0\n\t"                        \
                 : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3])                                                       \
                 : "v"(sign))
template <int STAGE>
__device__ __forceinline__ void dpp_fmac4(float (&v)[4], float sign) {
    if constexpr (STAGE == 0) I8F_DPP_FMAC4("quad_perm:[1,0,3,2]");
    else if constexpr (STAGE == 1) I8F_DPP_FMAC4("quad_perm:[2,3,0,1]");
    else if constexpr (STAGE == 2) I8F_DPP_FMAC4("row_half_mirror");
    else I8F_DPP_FMAC4("row_mirror");
}

// v: the chunk chunk_of_lane16(lane % 16) + 16 (lane / 16 % 2) of the lane's 128-block
__device__ __forceinline__ void rotate_chunk_f32(float (&v)[4], int lane) {
#pragma unroll
    for (int s = 1; s < 4; s <<= 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if ((j & s) == 0) {
                const float lo = v[j], hi = v[j + s];
                v[j] = lo + hi;
                v[j + s] = lo - hi;
            }
        }
    }
    const int c = chunk_of_lane16(lane & 15);
    const float s0 = (c & 1) ? -1.0f : 1.0f, s1 = (c & 2) ? -1.0f : 1.0f, s2 = (c & 4) ? -1.0f : 1.0f, s3 = (c & 8) ? -1.0f : 1.0f;
    dpp_fmac4<0>(v, s0);
    dpp_fmac4<1>(v, s1);
    dpp_fmac4<2>(v, s2);
    dpp_fmac4<3>(v, s3);
    const bool upper = (lane & 16) != 0;   // both lanes of this pair carry the same accumulated sign
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float other = __shfl_xor(v[j], 16, 64);
        v[j] = upper ? (other - v[j]) : (v[j] + other);
    }
    const float h = hadamard_entry<I8F_F32>() * (s0 * s1 * s2 * s3);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = v[j] * h;
}

// A wave that holds one 128-block, two elements to a lane (any alignment).
template <int DT>
__device__ __forceinline__ void rotate128_wave(float &e0, float &e1, int lane) {
    // the wave holds one 128-block: lane l has elements l (e0) and l + 64 (e1)
#pragma unroll
    for (int b = 1; b < 64; b <<= 1) {
        const bool upper = (lane & b) != 0;
        const float o0 = __shfl_xor(e0, b, 64);
        const float o1 = __shfl_xor(e1, b, 64);
        e0 = upper ? (o0 - e0) : (e0 + o0);
        e1 = upper ? (o1 - e1) : (e1 + o1);
    }
    const float lo = e0, hi = e1;
    e0 = lo + hi;
    e1 = lo - hi;
    const float h = hadamard_entry<DT>();
    e0 = round_to_dtype<DT>(e0 * h);
    e1 = round_to_dtype<DT>(e1 * h);
}

}  // namespace
}  // namespace i8f
