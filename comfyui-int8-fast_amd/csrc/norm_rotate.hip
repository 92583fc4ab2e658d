// Queries and keys between their projection and the attention: the norm of every head and the rotation by the token's positions, in one
// pass (include/i8f_attention.h has the formula).
#include <initializer_list>
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

template <int DT>
int launch(const i8f_norm_rotate_args &a, const Groups &groups, hipStream_t st) {
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
