// Queries and keys between their projection and the attention: the norm of every head and the rotation by the token's positions, in one
// pass (include/i8f_attention.h has the formula).
#include <initializer_list>
#include <type_traits>
#include <utility>

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
__device__ __forceinline__ void turn(const i8f_norm_rotate_args &a, const double (&pos)[I8F_MAX_AXES], int j, float &c, float &s) {
    double p = pos[0];
#pragma unroll
    for (int x = 1; x < I8F_MAX_AXES; ++x) p = x < a.axes && j >= a.first_pair[x] ? pos[x] : p;
    const double t = p * a.rates[j];
    sincospif((float)(2.0 * (t - __builtin_rint(t))), &s, &c);
}

__device__ __forceinline__ void token_positions(const i8f_norm_rotate_args &a, int64_t bt, double (&pos)[I8F_MAX_AXES]) {
    const int64_t at = bt / a.tokens * a.position_batch + bt % a.tokens * a.position_token;
#pragma unroll
    for (int x = 0; x < I8F_MAX_AXES; ++x) pos[x] = x < a.axes ? position_at(a.positions, a.positions_type, at + x * a.position_axis) : 0.0;
}

// ---- any width, alignment and pairing: a wave to a token, a lane to every 64th pair -----------------------------------------------
// (elements behind the turned ones go in pairs too, which are not turned; the last may be one element)
template <int DT, int NP>
__global__ __launch_bounds__(256) void norm_rotate_any_kernel(const int64_t first, const i8f_norm_rotate_args a, const Groups groups) {
    const int lane = threadIdx.x & 63;
    const int64_t bt = first + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (bt >= a.batch * a.tokens) return;
    const int width = (int)a.width, pairs = a.axes ? a.first_pair[a.axes] : 0;
    double pos[I8F_MAX_AXES];
    token_positions(a, bt, pos);
    float c[NP], s[NP];
    int e0[NP], e1[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int j = i * 64 + lane;
        c[i] = 1.0f, s[i] = 0.0f;
        e0[i] = j >= pairs || !a.apart ? 2 * j : j;
        e1[i] = j >= pairs || !a.apart ? 2 * j + 1 : j + pairs;
        if (j < pairs) turn(a, pos, j, c[i], s[i]);
    }
    for (int g = 0; g < groups.n; ++g) {
        const i8f_heads &h = groups.g[g];
        const int64_t xb = bt / a.tokens * h.batch_stride + bt % a.tokens * h.token_stride;
        for (int64_t head = 0; head < h.heads; ++head) {
            float v0[NP], v1[NP], sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                v0[i] = e0[i] < width ? load_as_f32<DT>(h.x, xb + head * h.head_stride + e0[i]) : 0.0f;
                v1[i] = e1[i] < width ? load_as_f32<DT>(h.x, xb + head * h.head_stride + e1[i]) : 0.0f;
                sum = __builtin_fmaf(v0[i], v0[i], __builtin_fmaf(v1[i], v1[i], sum));
            }
            if (a.norm) {
#pragma unroll
                for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x);
                const float rstd = 1.0f / sqrtf(sum / (float)width + a.eps);
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    v0[i] *= rstd, v1[i] *= rstd;
                    if (h.weight) {
                        const bool wide = DT == I8F_F32 || h.weight_dtype == I8F_F32;
                        if (e0[i] < width) v0[i] *= wide ? ((const float *)h.weight)[e0[i]] : load_as_f32<DT>(h.weight, e0[i]);
                        if (e1[i] < width) v1[i] *= wide ? ((const float *)h.weight)[e1[i]] : load_as_f32<DT>(h.weight, e1[i]);
                    }
                }
            }
            const int64_t ob = (bt * h.heads + head) * width;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const bool turned = i * 64 + lane < pairs;   // (the others as they are: 0 times an infinity is none)
                const float y0 = turned ? __builtin_fmaf(v0[i], c[i], -(v1[i] * s[i])) : v0[i], y1 = turned ? __builtin_fmaf(v0[i], s[i], v1[i] * c[i]) : v1[i];
                if (e0[i] < width) store_from_f32<DT>(h.out, ob + e0[i], y0);
                if (e1[i] < width) store_from_f32<DT>(h.out, ob + e1[i], y1);
            }
        }
    }
}

template <int DT, int NP>
int launch_any(const i8f_norm_rotate_args &a, const Groups &groups, hipStream_t st) {
    const int64_t rows = a.batch * a.tokens, most = (int64_t)4 << 23;   // (a launch has fewer than 2^32 threads)
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t n = rows - r < most ? rows - r : most;
        hipLaunchKernelGGL((norm_rotate_any_kernel<DT, NP>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, r, a, groups);
        if (int rc = check_launch()) return rc;
    }
    return I8F_OK;
}

// ---- heads of whole aligned pieces: a lane holds eight elements of a head, LPH lanes a head ------------------------------------------
// Pairs that lie apart are in one lane as well: it takes four elements of either half.
template <int DT>
struct Eight {
    uint4 v[DT == I8F_F32 ? 2 : 1];
};
template <int DT, bool APART>
__device__ __forceinline__ Eight<DT> load_eight(const char *p, int e0, int e1) {
    Eight<DT> r;
    if constexpr (DT == I8F_F32) {
        r.v[0] = *(const uint4 *)(p + e0 * 4), r.v[1] = *(const uint4 *)(p + e1 * 4);
    } else if constexpr (APART) {
        const uint2 lo = *(const uint2 *)(p + e0 * 2), hi = *(const uint2 *)(p + e1 * 2);
        r.v[0] = make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else {
        r.v[0] = *(const uint4 *)(p + e0 * 2);
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void expand_eight(const Eight<DT> &r, float (&v)[8]) {
    if constexpr (DT == I8F_F32) {
        __builtin_memcpy(v, &r, 32);
    } else {
        const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = DT == I8F_BF16 ? __uint_as_float(w[i] << 16) : f16_bits_to_f32(w[i] & 0xffffu);
            v[2 * i + 1] = DT == I8F_BF16 ? __uint_as_float(w[i] & 0xffff0000u) : f16_bits_to_f32(w[i] >> 16);
        }
    }
}
template <int DT, bool APART>
__device__ __forceinline__ void store_eight(char *p, int e0, int e1, const float (&v)[8]) {
    if constexpr (DT == I8F_F32) {
        uint4 lo, hi;
        __builtin_memcpy(&lo, v, 16);
        __builtin_memcpy(&hi, v + 4, 16);
        stream_store16(p + e0 * 4, lo), stream_store16(p + e1 * 4, hi);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = DT == I8F_BF16 ? f32x2_to_bf16x2_bits(v[2 * i], v[2 * i + 1]) : f32x2_to_f16x2_bits(v[2 * i], v[2 * i + 1]);
        if constexpr (APART) stream_store8(p + e0 * 2, make_uint2(w[0], w[1])), stream_store8(p + e1 * 2, make_uint2(w[2], w[3]));
        else stream_store16(p + e0 * 2, make_uint4(w[0], w[1], w[2], w[3]));
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

constexpr int DEEP = 4;   // passes that a wave requests at a time
// A wave takes `per` passes of one token, a pass being 64 / LPH heads: the angles are the same for all of them.
template <int DT, int LPH, bool APART>
__global__ __launch_bounds__(256) void norm_rotate_kernel(const int64_t first, const unsigned chunks, const int per, const i8f_norm_rotate_args a, const Groups groups) {
    constexpr int HPP = 64 / LPH, SIZE = DT == I8F_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, sub = lane / LPH, l = lane % LPH;
    const int64_t id = first + (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t bt = id / chunks;
    if (bt >= a.batch * a.tokens) return;
    const int start = (int)(id % chunks) * per;
    const int64_t b = bt / a.tokens, t = bt % a.tokens;
    const int width = (int)a.width, pairs = a.axes ? a.first_pair[a.axes] : 0;
    const bool low = APART && l < pairs / 4;   // (lanes behind the turned pairs hold eight neighbours in either form)
    const int e0 = !APART ? 8 * l : low ? 4 * l : 2 * pairs + 8 * (l - pairs / 4), e1 = low ? pairs + 4 * l : e0 + 4;
    const bool in = e0 < width;
    float c[4], s[4];
    if (pairs) {
        double pos[I8F_MAX_AXES];
        token_positions(a, bt, pos);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * l + i < pairs) turn(a, pos, 4 * l + i, c[i], s[i]);
    }
    int before = 0;
    for (int g = 0; g < groups.n; ++g) {
        const i8f_heads &h = groups.g[g];
        const int passes = ((int)h.heads + HPP - 1) / HPP, lo = start - before > 0 ? start - before : 0, hi = start + per - before < passes ? start + per - before : passes;
        before += passes;
        if (lo >= hi) continue;
        float w[8];
        if (h.weight && in) {
            if (DT == I8F_F32 || h.weight_dtype == I8F_F32) expand_eight<I8F_F32>(load_eight<I8F_F32, APART>((const char *)h.weight, e0, e1), w);
            else expand_eight<DT>(load_eight<DT, APART>((const char *)h.weight, e0, e1), w);
        }
        const char *x = (const char *)h.x + (b * h.batch_stride + t * h.token_stride) * SIZE;
        char *out = (char *)h.out + bt * h.heads * width * SIZE;
        for (int pass = lo; pass < hi; pass += DEEP) {
            Eight<DT> raw[DEEP];
#pragma unroll
            for (int i = 0; i < DEEP; ++i) {
                const int head = (pass + i) * HPP + sub;
                if (pass + i < hi && in && head < h.heads) raw[i] = load_eight<DT, APART>(x + head * h.head_stride * SIZE, e0, e1);
                else raw[i] = {};
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
                    for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(v[e], v[e], sum);
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
                        if (4 * l + e < pairs) v0 = y0, v1 = y1;   // (the others as they are: 0 times an infinity is none)
                    }
                }
                if (in && head < h.heads) store_eight<DT, APART>(out + (int64_t)head * width * SIZE, e0, e1, v);
            }
        }
    }
}

// All operands in 16-byte pieces, and with pairs that lie apart the turned and the other elements in whole lanes.
bool in_pieces(const i8f_norm_rotate_args &a, const Groups &groups) {
    const int64_t per16 = 16 / (int64_t)dtype_size(a.dtype);
    if (a.width % 8 || (a.axes && a.apart && a.first_pair[a.axes] % 4)) return false;
    for (int i = 0; i < groups.n; ++i) {
        const i8f_heads &g = groups.g[i];
        if (((uintptr_t)g.x | (uintptr_t)g.weight | (uintptr_t)g.out) % 16 || g.batch_stride % per16 || g.token_stride % per16 || g.head_stride % per16) return false;
    }
    return true;
}

template <int DT, int LPH, bool APART>
int launch_pieces(const i8f_norm_rotate_args &a, const Groups &groups, hipStream_t st) {
    int64_t passes = 0;
    for (int i = 0; i < groups.n; ++i) passes += (groups.g[i].heads + 64 / LPH - 1) / (64 / LPH);
    if (passes > 0x7fffffff) return I8F_ERR_UNSUPPORTED;
    // As many passes to a wave as it requests at a time: us for 4096 tokens of 30 + 30 heads of 128 and 32760 of 40 + 40, 1 pass 45 and 239, 4 or 5
    // 24.1 and 238, 8 24.6 and 246, a whole token 24.8 and 248.  Fewer where the waves would be few.
    const int64_t tokens = a.batch * a.tokens, total = tokens * passes;
    int64_t per = total / 4096;
    per = per < 1 ? 1 : per > DEEP ? DEEP : per;
    const int64_t chunks = (passes + per - 1) / per;
    per = (passes + chunks - 1) / chunks;
    const int64_t waves = tokens * chunks, most = (int64_t)4 << 23;   // (a launch has fewer than 2^32 threads)
    for (int64_t w = 0; w < waves; w += most) {
        const int64_t n = waves - w < most ? waves - w : most;
        hipLaunchKernelGGL((norm_rotate_kernel<DT, LPH, APART>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, w, (unsigned)chunks, (int)per, a, groups);
        if (int rc = check_launch()) return rc;
    }
    return I8F_OK;
}
template <int DT, bool APART>
int launch_lanes(const i8f_norm_rotate_args &a, const Groups &groups, hipStream_t st) {
    if (a.width <= 64) return launch_pieces<DT, 8, APART>(a, groups, st);
    if (a.width <= 128) return launch_pieces<DT, 16, APART>(a, groups, st);
    if (a.width <= 256) return launch_pieces<DT, 32, APART>(a, groups, st);
    return launch_pieces<DT, 64, APART>(a, groups, st);
}

template <int DT>
int launch(const i8f_norm_rotate_args &a, const Groups &groups, hipStream_t st) {
    if (in_pieces(a, groups)) return a.axes && a.apart ? launch_lanes<DT, true>(a, groups, st) : launch_lanes<DT, false>(a, groups, st);
    const int64_t pairs = (a.width + 1) / 2;
    if (pairs <= 64) return launch_any<DT, 1>(a, groups, st);
    if (pairs <= 128) return launch_any<DT, 2>(a, groups, st);
    return launch_any<DT, 4>(a, groups, st);
}

// The elements that a strided tensor reaches to from its first one, -1 past 2^62.
int64_t extent(std::initializer_list<std::pair<int64_t, int64_t>> dims) {
    __int128 last = 0;
    for (auto [size, stride] : dims) {
        if (size < 1) return 0;
        last += (__int128)(size - 1) * stride;
    }
    return last >= ((__int128)1 << 62) ? -1 : (int64_t)last + 1;
}

bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    return na > 0 && nb > 0 && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

int validate(const i8f_norm_rotate_args &a, const i8f_heads *groups, int n) {
    if (a.batch < 0 || a.tokens < 0 || a.width < 1 || !valid_dtype(a.dtype) || n < 0 || (n && !groups)) return I8F_ERR_INVALID;
    if (a.norm && !(a.eps >= 0.0f)) return I8F_ERR_INVALID;
    if (a.axes < 0) return I8F_ERR_INVALID;
    if (a.axes > I8F_MAX_AXES || n > I8F_MAX_HEAD_GROUPS || a.width > 512) return I8F_ERR_UNSUPPORTED;
    if (a.batch > 0x7fffffff || a.tokens > 0x7fffffff || (a.batch && a.tokens > ((int64_t)1 << 40) / a.batch)) return I8F_ERR_UNSUPPORTED;
    const bool any = a.batch && a.tokens;
    if (a.axes) {
        if (a.positions_type < I8F_POSITION_I32 || a.positions_type > I8F_POSITION_F64 || a.first_pair[0] != 0) return I8F_ERR_INVALID;
        for (int x = 0; x < a.axes; ++x)
            if (a.first_pair[x + 1] <= a.first_pair[x]) return I8F_ERR_INVALID;
        if (2 * (int64_t)a.first_pair[a.axes] > a.width) return I8F_ERR_INVALID;
        if (any && (!a.rates || !a.positions)) return I8F_ERR_INVALID;
        if (a.position_batch < 0 || a.position_token < 0 || a.position_axis < 0) return I8F_ERR_INVALID;
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
    }
    for (int i = 0; i < n; ++i)
        for (int j = 0; j < n; ++j)   // (a head is written while other waves read)
            if (overlap(groups[i].out, out[i] * size, groups[j].x, in[j] * size) || (i != j && overlap(groups[i].out, out[i] * size, groups[j].out, out[j] * size)))
                return I8F_ERR_INVALID;
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
