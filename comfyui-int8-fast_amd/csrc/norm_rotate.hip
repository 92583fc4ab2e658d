// Queries and keys between their projection and the attention: the norm of every head and the rotation by the token's positions, in one
// pass (include/i8f_attention.h has the formula).
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "divisor.hpp"
#include "extents.hpp"
#include "i8f_common.hpp"

#include "../../include/i8f_attention.h"

namespace i8f {
namespace {

struct Groups {
    i8f_heads g[I8F_MAX_HEAD_GROUPS];
    int n;
};

__device__ __forceinline__ double position_at(const void *p, int type, int64_t i) {
    switch (type) {
    case I8F_POSITION_I32: return (double)((const int32_t *)p)[i];
    case I8F_POSITION_I64: return (double)((const int64_t *)p)[i];
    case I8F_POSITION_F32: return (double)((const float *)p)[i];
    default: return ((const double *)p)[i];
    }
}

// Cosine and sine of pair j's angle at the token's positions.  The turns are a product in binary64 (rounded by half a unit of 2^-53 of its
// size: a position of 2^31 leaves 2^-24 turns) and what is left of them behind the whole ones is at most a half, so that binary32 holds it to 2^-26.
// The hardware's functions take turns: over all of -1/2 ... 1/2 in steps of 2^-25 they are within 1.26e-7 (2^-22.9) of sine and cosine.  That is
// far below the steps of 16 bits.  For heads in binary32 quarters are taken off, so that what is left of the angle, at most pi/4, is off by 2^-25, and
// the series of sine and cosine, to x^9 and x^10, are within 2^-23.4 together with it.
template <int DT>
__device__ __forceinline__ void turn(const i8f_norm_rotate_args &a, const double (&pos)[I8F_MAX_AXES], int j, float &c, float &s) {
    double p = pos[0];
#pragma unroll
    for (int x = 1; x < I8F_MAX_AXES; ++x) p = x < a.axes && j >= a.first_pair[x] ? pos[x] : p;
    const double t = p * a.rates[j];
    if constexpr (DT != I8F_F32) {
        const float left = (float)(t - __builtin_rint(t));
        c = __builtin_amdgcn_cosf(left), s = __builtin_amdgcn_sinf(left);
    } else {
        const double quarters = __builtin_rint(4.0 * t);
        const float x = (float)(__builtin_fma(quarters, -0.25, t) * 6.283185307179586476925), z = x * x;
        const float quarter = (float)(quarters - 4.0 * __builtin_rint(0.25 * quarters));   // -2 ... 2
        float sine = __builtin_fmaf(z, 1.0f / 362880, -1.0f / 5040), cosine = __builtin_fmaf(z, -1.0f / 3628800, 1.0f / 40320);
        sine = __builtin_fmaf(__builtin_fmaf(sine, z, 1.0f / 120), z, -1.0f / 6);
        cosine = __builtin_fmaf(__builtin_fmaf(cosine, z, -1.0f / 720), z, 1.0f / 24);
        sine = __builtin_fmaf(x * z, sine, x), cosine = __builtin_fmaf(z, __builtin_fmaf(z, cosine, -0.5f), 1.0f);
        const bool odd = fabsf(quarter) == 1.0f, back = fabsf(quarter) == 2.0f;
        c = odd ? sine : cosine, s = odd ? cosine : sine;
        c = quarter == 1.0f || back ? -c : c, s = quarter == -1.0f || back ? -s : s;
    }
}

__device__ __forceinline__ void token_positions(const i8f_norm_rotate_args &a, unsigned b, unsigned t, double (&pos)[I8F_MAX_AXES]) {
    const int64_t at = b * a.position_batch + t * a.position_token;
#pragma unroll
    for (int x = 0; x < I8F_MAX_AXES; ++x) pos[x] = x < a.axes ? position_at(a.positions, a.positions_type, at + x * a.position_axis) : 0.0;
}

// A lane holds eight elements of a head: neighbours, or of pairs that lie apart four elements of either half.  They move in 16 or 8 bytes from
// whatever address they have.  The last lane of a width or of a half that is no multiple begins further back, in elements that the lane before
// it has too, which it computes again and leaves out of the sum (SHIFTED); where that would tear pairs of neighbours or leave the head
// its elements move one by one (SINGLE).
enum { FULL, SHIFTED, SINGLE };
typedef v4u_t any4_t __attribute__((aligned(2)));
typedef v2u_t any2_t __attribute__((aligned(2)));
template <int DT>
struct Eight {
    v4u_t v[DT == I8F_F32 ? 2 : 1];
};
template <int DT, bool APART>
__device__ __forceinline__ Eight<DT> load_eight(const char *p, int e0, int e1) {
    Eight<DT> r;
    if constexpr (DT == I8F_F32) {
        r.v[0] = *(const any4_t *)(p + e0 * 4), r.v[1] = *(const any4_t *)(p + e1 * 4);
    } else if constexpr (APART) {
        const v2u_t lo = *(const any2_t *)(p + e0 * 2), hi = *(const any2_t *)(p + e1 * 2);
        r.v[0] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3);
    } else {
        r.v[0] = *(const any4_t *)(p + e0 * 2);
    }
    return r;
}
// the first n of each four (of a lane's pairs that lie apart), or of eight neighbours; the others are zeros
template <int DT>
__device__ __forceinline__ Eight<DT> load_some(const char *p, int e0, int e1, int n0, int n1) {
    Eight<DT> r = {};
    uint32_t *w = (uint32_t *)&r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (e % 4 >= (e < 4 ? n0 : n1)) continue;
        const int at = (e < 4 ? e0 : e1) + e % 4;
        if constexpr (DT == I8F_F32) w[e] = *(const uint32_t *)(p + at * 4);
        else w[e / 2] |= (uint32_t)*(const uint16_t *)(p + at * 2) << (16 * (e % 2));
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void expand_eight(const Eight<DT> &r, float (&v)[8]) {
    if constexpr (DT == I8F_F32) {
        __builtin_memcpy(v, &r, 32);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = r.v[0][i];
            v[2 * i] = DT == I8F_BF16 ? __uint_as_float(w << 16) : f16_bits_to_f32(w & 0xffffu);
            v[2 * i + 1] = DT == I8F_BF16 ? __uint_as_float(w & 0xffff0000u) : f16_bits_to_f32(w >> 16);
        }
    }
}
template <int DT>
__device__ __forceinline__ Eight<DT> round_eight(const float (&v)[8]) {
    Eight<DT> r;
    if constexpr (DT == I8F_F32) {
        __builtin_memcpy(&r, v, 32);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[0][i] = DT == I8F_BF16 ? f32x2_to_bf16x2_bits(v[2 * i], v[2 * i + 1]) : f32x2_to_f16x2_bits(v[2 * i], v[2 * i + 1]);
    }
    return r;
}
template <int DT, bool APART>
__device__ __forceinline__ void store_eight(char *p, int e0, int e1, const Eight<DT> &r) {
    if constexpr (DT == I8F_F32) {
        __builtin_nontemporal_store(r.v[0], (any4_t *)(p + e0 * 4)), __builtin_nontemporal_store(r.v[1], (any4_t *)(p + e1 * 4));
    } else if constexpr (APART) {
        __builtin_nontemporal_store(__builtin_shufflevector(r.v[0], r.v[0], 0, 1), (any2_t *)(p + e0 * 2));
        __builtin_nontemporal_store(__builtin_shufflevector(r.v[0], r.v[0], 2, 3), (any2_t *)(p + e1 * 2));
    } else {
        __builtin_nontemporal_store(r.v[0], (any4_t *)(p + e0 * 2));
    }
}
template <int DT>
__device__ __forceinline__ void store_some(char *p, int e0, int e1, int n0, int n1, const Eight<DT> &r) {
    const uint32_t *w = (const uint32_t *)&r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (e % 4 >= (e < 4 ? n0 : n1)) continue;
        const int at = (e < 4 ? e0 : e1) + e % 4;
        if constexpr (DT == I8F_F32) *(uint32_t *)(p + at * 4) = w[e];
        else *(uint16_t *)(p + at * 2) = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
    }
}
// a sum over LPH neighbouring lanes, in every one of them
template <int LPH>
__device__ __forceinline__ float sum_of_lanes(float v) {
    auto add = [&](auto ctrl) __attribute__((always_inline)) {
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    using std::integral_constant;
    if constexpr (LPH > 1) add(integral_constant<int, 0xb1>{});     // quad_perm [1,0,3,2]
    if constexpr (LPH > 2) add(integral_constant<int, 0x4e>{});     // quad_perm [2,3,0,1]
    if constexpr (LPH > 4) add(integral_constant<int, 0x141>{});    // row_half_mirror
    if constexpr (LPH > 8) add(integral_constant<int, 0x140>{});    // row_mirror
    if constexpr (LPH > 16) v += __shfl_xor(v, 16);
    if constexpr (LPH > 32) v += __shfl_xor(v, 32);
    return v;
}

// Memory bounds it: a head is read once and written once, its elements stay in registers between, the sum goes over the lanes that hold them,
// and what a token's heads share (positions, sine and cosine, the norm's weights) is made once for the passes of a wave.  32760 tokens of 40 + 40 heads
// of 128 222 to 225 us, 6.0 TB/s (256 us when each launch starts on its own; a copy of 2 GiB 4.97 TB/s); 4096 of 30 + 30 23 us, 5.5; 8192 of 32 x 64 in
// binary32 23.2 us, 5.8; 4071 of 16 heads of 72, pairs apart, 8 to 9 us, 2.2 (10 of 16 lanes hold elements); a few tokens 4 to 5 us, a launch and the
// chain of position, angle and head.  Eight elements to a lane, so that a head of 128 in 16 bits is one
// 16-byte access of 16 lanes.  Measured and not kept: everything that a wave reads requested before the first of it is used (4.1 us for 2 tokens as
// now, 300 for the 32760).
constexpr int DEEP = 4;   // passes that a wave requests at a time
// A wave takes `per` passes of one token, a pass being 64 / LPH heads: the angles are the same for all of them.
template <int DT, int LPH, bool APART, int ENDS>
__global__ __launch_bounds__(256) void norm_rotate_kernel(const unsigned first, const unsigned tokens, const unsigned chunks, const int per, const Divisor by_chunks,
                                                          const Divisor by_tokens, const i8f_norm_rotate_args a, const Groups groups) {
    constexpr int HPP = 64 / LPH, SIZE = DT == I8F_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, sub = lane / LPH, l = lane % LPH;
    const unsigned id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = by_chunks(id);
    if (at >= tokens) return;
    const unsigned bt = first + at, b = by_tokens(bt), t = bt - b * (unsigned)a.tokens;
    const int start = (int)(id - at * chunks) * per;
    const int width = (int)a.width, pairs = a.axes ? a.first_pair[a.axes] : 0;
    const int lows = (pairs + 3) / 4;
    const bool low = APART && l < lows;   // (lanes behind the turned pairs hold eight neighbours in either form)
    int e0 = !APART ? 8 * l : low ? 4 * l : 2 * pairs + 8 * (l - lows), e1 = low ? pairs + 4 * l : e0 + 4;
    int n0 = low ? pairs - 4 * l : width - e0, n1 = low ? n0 : n0 - 4;   // elements from e0 and e1 on, up to four of them the lane's
    const bool in = n0 > 0;
    int pair = low || !APART ? 4 * l : pairs, again = 0;   // the lane's first pair; elements (of each four, or of eight) of the lane before
    if constexpr (ENDS != FULL) {
        const int need = low ? 4 : 8, back = need - n0, begin = APART && !low ? 2 * pairs : 0;
        if (in && back > 0 && back <= e0 - begin && (APART || back % 2 == 0)) {
            again = back, e0 -= back, e1 -= back, n0 = 4, n1 = 4;
            if (low) pair -= back;
            else if (!APART) pair -= back / 2;
        }
    }
    const bool whole = ENDS != SINGLE || (n0 >= 4 && n1 >= 4);
    float c[4], s[4];
    if (pairs) {
        double pos[I8F_MAX_AXES];
        token_positions(a, b, t, pos);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (pair + i < pairs) turn<DT>(a, pos, pair + i, c[i], s[i]);
    }
    int before = 0;
    for (int g = 0; g < groups.n; ++g) {
        const i8f_heads &h = groups.g[g];
        const int passes = ((int)h.heads + HPP - 1) / HPP, lo = start - before > 0 ? start - before : 0, hi = start + per - before < passes ? start + per - before : passes;
        before += passes;
        if (lo >= hi) continue;
        float w[8];
        if (h.weight && in) {
            const char *p = (const char *)h.weight;
            if (DT == I8F_F32 || h.weight_dtype == I8F_F32) expand_eight<I8F_F32>(whole ? load_eight<I8F_F32, APART>(p, e0, e1) : load_some<I8F_F32>(p, e0, e1, n0, n1), w);
            else expand_eight<DT>(whole ? load_eight<DT, APART>(p, e0, e1) : load_some<DT>(p, e0, e1, n0, n1), w);
        }
        const char *x = (const char *)h.x + (b * h.batch_stride + t * h.token_stride) * SIZE;
        char *out = (char *)h.out + (int64_t)bt * h.heads * width * SIZE;
        for (int pass = lo; pass < hi; pass += DEEP) {
            Eight<DT> raw[DEEP];
#pragma unroll
            for (int i = 0; i < DEEP; ++i) {
                const int head = (pass + i) * HPP + sub;
                raw[i] = {};
                if (pass + i < hi && in && head < h.heads) {
                    if (whole) raw[i] = load_eight<DT, APART>(x + head * h.head_stride * SIZE, e0, e1);
                    else raw[i] = load_some<DT>(x + head * h.head_stride * SIZE, e0, e1, n0, n1);
                }
            }
#pragma unroll
            for (int i = 0; i < DEEP; ++i) {
                if (pass + i >= hi) break;
                const int head = (pass + i) * HPP + sub;
                float v[8];
                expand_eight<DT>(raw[i], v);
                if (a.norm) {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum = ENDS != FULL && (low ? e % 4 : e) < again ? sum : __builtin_fmaf(v[e], v[e], sum);
                    const float rstd = 1.0f / sqrtf(sum_of_lanes<LPH>(sum) / (float)width + a.eps);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= rstd;
                    if (h.weight) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] *= w[e];
                    }
                }
                if (pairs) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float &v0 = v[APART ? e : 2 * e], &v1 = v[APART ? e + 4 : 2 * e + 1];
                        const float y0 = __builtin_fmaf(v0, c[e], -(v1 * s[e])), y1 = __builtin_fmaf(v0, s[e], v1 * c[e]);
                        if (pair + e < pairs) v0 = y0, v1 = y1;   // (the others as they are: 0 times an infinity is none)
                    }
                }
                if (in && head < h.heads) {
                    if (whole) store_eight<DT, APART>(out + (int64_t)head * width * SIZE, e0, e1, round_eight<DT>(v));
                    else store_some<DT>(out + (int64_t)head * width * SIZE, e0, e1, n0, n1, round_eight<DT>(v));
                }
            }
        }
    }
}

template <int DT, int LPH, bool APART, int ENDS>
int launch_passes(const i8f_norm_rotate_args &a, const Groups &groups, hipStream_t st) {
    int64_t passes = 0;
    for (int i = 0; i < groups.n; ++i) passes += (groups.g[i].heads + 64 / LPH - 1) / (64 / LPH);
    if (passes > 0x7fffffff) return I8F_ERR_UNSUPPORTED;
    // As many passes to a wave as it requests at a time: us for 4096 tokens of 30 + 30 heads of 128 and 32760 of 40 + 40, 1 pass 35.4 and 464, 2 24.0 and
    // 281, 4 23.0 and 224, 8 23.6 and 233, a whole token 23.2 and 248.  Fewer where the waves would be few: 4071 tokens of 16 heads of 72 10.4 with one
    // pass, 7.7 with four.
    const int64_t tokens = a.batch * a.tokens, total = tokens * passes;
    int64_t per = total / 2048;
    per = per < 1 ? 1 : per > DEEP ? DEEP : per;
    const int64_t chunks = (passes + per - 1) / per;
    per = (passes + chunks - 1) / chunks;
    const int64_t most = ((int64_t)4 << 23) / chunks;   // tokens to a launch, which has fewer than 2^32 threads
    if (most < 1) return I8F_ERR_UNSUPPORTED;
    for (int64_t t = 0; t < tokens; t += most) {
        const int64_t n = tokens - t < most ? tokens - t : most;
        hipLaunchKernelGGL((norm_rotate_kernel<DT, LPH, APART, ENDS>), dim3((unsigned)((n * chunks + 3) / 4)), dim3(256), 0, st, (unsigned)t, (unsigned)n,
                           (unsigned)chunks, (int)per, Divisor((uint32_t)chunks), Divisor((uint32_t)a.tokens), a, groups);
        if (int rc = check_launch()) return rc;
    }
    return I8F_OK;
}
template <int DT, int LPH, bool APART>
int launch_ends(const i8f_norm_rotate_args &a, const Groups &groups, hipStream_t st) {
    const int64_t pairs = APART ? a.first_pair[a.axes] : 0, rest = a.width - 2 * pairs;
    if (pairs % 4 == 0 && rest % 8 == 0) return launch_passes<DT, LPH, APART, FULL>(a, groups, st);
    const bool halves = pairs % 4 == 0 || pairs >= 4, end = rest % 8 == 0 || (rest >= 8 && (APART || rest % 2 == 0));
    return halves && end ? launch_passes<DT, LPH, APART, SHIFTED>(a, groups, st) : launch_passes<DT, LPH, APART, SINGLE>(a, groups, st);
}
template <int DT, bool APART>
int launch_lanes(const i8f_norm_rotate_args &a, const Groups &groups, hipStream_t st) {
    const int64_t pairs = APART ? a.first_pair[a.axes] : 0, lanes = (pairs + 3) / 4 + (a.width - 2 * pairs + 7) / 8;   // (33 at the most)
    if (lanes <= 8) return launch_ends<DT, 8, APART>(a, groups, st);
    if (lanes <= 16) return launch_ends<DT, 16, APART>(a, groups, st);
    if (lanes <= 32) return launch_ends<DT, 32, APART>(a, groups, st);
    return launch_ends<DT, 64, APART>(a, groups, st);
}
template <int DT>
int launch(const i8f_norm_rotate_args &a, const Groups &groups, hipStream_t st) {
    return a.axes && a.apart ? launch_lanes<DT, true>(a, groups, st) : launch_lanes<DT, false>(a, groups, st);
}

int validate(const i8f_norm_rotate_args &a, const i8f_heads *groups, int n) {
    if (a.batch < 0 || a.tokens < 0 || a.width < 1 || !valid_dtype(a.dtype) || n < 0 || (n && !groups)) return I8F_ERR_INVALID;
    if (a.norm && !(a.eps >= 0.0f)) return I8F_ERR_INVALID;
    if (a.axes < 0) return I8F_ERR_INVALID;
    if (a.axes > I8F_MAX_AXES || n > I8F_MAX_HEAD_GROUPS || a.width > 256) return I8F_ERR_UNSUPPORTED;
    if (a.batch > 0x7fffffff || a.tokens > 0x7fffffff || (a.batch && a.tokens > 0x7fffffff / a.batch)) return I8F_ERR_UNSUPPORTED;
    const bool any = a.batch && a.tokens;
    const int64_t position_size = a.positions_type == I8F_POSITION_I32 || a.positions_type == I8F_POSITION_F32 ? 4 : 8;
    int64_t positions = 0, rates = 0;   // elements
    if (a.axes) {
        if (a.positions_type < I8F_POSITION_I32 || a.positions_type > I8F_POSITION_F64 || a.first_pair[0] != 0) return I8F_ERR_INVALID;
        for (int x = 0; x < a.axes; ++x)
            if (a.first_pair[x + 1] <= a.first_pair[x]) return I8F_ERR_INVALID;
        if (2 * (int64_t)a.first_pair[a.axes] > a.width) return I8F_ERR_INVALID;
        if (any && (!a.rates || !a.positions)) return I8F_ERR_INVALID;
        if (a.position_batch < 0 || a.position_token < 0 || a.position_axis < 0) return I8F_ERR_INVALID;
        if ((uintptr_t)a.positions % position_size || (uintptr_t)a.rates % 8) return I8F_ERR_INVALID;
        positions = extent({{a.batch, a.position_batch}, {a.tokens, a.position_token}, {a.axes, a.position_axis}}), rates = a.first_pair[a.axes];
        if (positions < 0) return I8F_ERR_UNSUPPORTED;
    }
    const int64_t size = (int64_t)dtype_size(a.dtype);
    int64_t in[I8F_MAX_HEAD_GROUPS], out[I8F_MAX_HEAD_GROUPS];
    for (int i = 0; i < n; ++i) {
        const i8f_heads &g = groups[i];
        if (g.heads < 0 || g.batch_stride < 0 || g.token_stride < 0 || g.head_stride < 0) return I8F_ERR_INVALID;
        if (g.heads > 0x7fffffff) return I8F_ERR_UNSUPPORTED;
        if (g.weight && (!a.norm || (g.weight_dtype != a.dtype && g.weight_dtype != I8F_F32))) return I8F_ERR_INVALID;
        in[i] = extent({{a.batch, g.batch_stride}, {a.tokens, g.token_stride}, {g.heads, g.head_stride}, {a.width, 1}});
        out[i] = extent({{a.batch, a.tokens * g.heads * a.width}, {a.tokens, g.heads * a.width}, {g.heads, a.width}, {a.width, 1}});
        if (in[i] < 0 || out[i] < 0) return I8F_ERR_UNSUPPORTED;
        if (in[i] && (!g.x || !g.out)) return I8F_ERR_INVALID;
        if (((uintptr_t)g.x | (uintptr_t)g.out) % size || (g.weight && (uintptr_t)g.weight % dtype_size(g.weight_dtype))) return I8F_ERR_INVALID;
    }
    for (int i = 0; i < n; ++i) {     // (a head is written while other waves read)
        if (overlap(groups[i].out, out[i] * size, a.positions, positions * position_size) || overlap(groups[i].out, out[i] * size, a.rates, rates * 8)) return I8F_ERR_INVALID;
        for (int j = 0; j < n; ++j) {
            const int64_t weight = groups[j].weight ? a.width * (int64_t)dtype_size(groups[j].weight_dtype) : 0;
            if (overlap(groups[i].out, out[i] * size, groups[j].weight, weight)) return I8F_ERR_INVALID;
            if (overlap(groups[i].out, out[i] * size, groups[j].x, in[j] * size) || (i != j && overlap(groups[i].out, out[i] * size, groups[j].out, out[j] * size)))
                return I8F_ERR_INVALID;
        }
    }
    return I8F_OK;
}

}  // namespace
}  // namespace i8f

extern "C" int i8f_norm_rotate(const i8f_norm_rotate_args *args, const i8f_heads *heads, int n_groups, void *stream) {
    using namespace i8f;
    if (!args) return I8F_ERR_INVALID;
    if (int rc = validate(*args, heads, n_groups)) return rc;
    Groups groups = {};
    for (int i = 0; i < n_groups; ++i)
        if (heads[i].heads > 0) groups.g[groups.n++] = heads[i];
    if (!groups.n || !args->batch || !args->tokens) return I8F_OK;
    if (int rc = check_device()) return rc;
    switch (args->dtype) {
    case I8F_BF16: return launch<I8F_BF16>(*args, groups, (hipStream_t)stream);
    case I8F_F16: return launch<I8F_F16>(*args, groups, (hipStream_t)stream);
    default: return launch<I8F_F32>(*args, groups, (hipStream_t)stream);
    }
}
