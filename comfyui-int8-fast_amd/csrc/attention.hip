// Attention over an encoder's states (include/i8f_attention.h has the formula).
#include <initializer_list>
#include <utility>

#include "i8f_common.hpp"

#include "../../include/i8f_attention.h"

namespace i8f {
namespace {

// Whether state j of batch b counts, and its addend.
__device__ __forceinline__ bool counts(const i8f_attention_args &a, int64_t b, int64_t j, float &m) {
    m = 0.0f;
    if (!a.key_mask) return true;
    const int64_t at = b * a.mask_batch + j * a.mask_key;
    switch (a.mask_type) {
    case I8F_MASK_BYTES: return ((const uint8_t *)a.key_mask)[at] != 0;
    case I8F_MASK_BF16: m = load_as_f32<I8F_BF16>(a.key_mask, at); return !(m <= -3.3895313892515355e38f);
    case I8F_MASK_F16: m = load_as_f32<I8F_F16>(a.key_mask, at); return !(m <= -65504.0f);
    default: m = ((const float *)a.key_mask)[at]; return !(m <= -3.4028234663852886e38f);
    }
}

// A wave to a query's head: 64 states at a time, a lane to a state for the scores and a lane to every 64th element for the result.
template <int DT>
__global__ __launch_bounds__(256) void attention_kernel(const i8f_attention_args a) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.batch * a.queries * a.heads) return;
    const int64_t h = row % a.heads, i = row / a.heads % a.queries, b = row / a.heads / a.queries, g = h / (a.heads / a.kv_heads);
    const int64_t qb = b * a.q_batch + i * a.q_token + h * a.q_head, kb = b * a.k_batch + g * a.k_head, vb = b * a.v_batch + g * a.v_head;
    int64_t n = a.keys;
    if (a.key_lengths) {
        const int64_t given = a.lengths_type ? ((const int64_t *)a.key_lengths)[b] : ((const int32_t *)a.key_lengths)[b];
        n = given < 0 ? 0 : given < n ? given : n;
    }
    const float to_log2 = 1.4426950408889634f;
    float top = -3.4028234663852886e38f, total = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t j0 = 0; j0 < n; j0 += 64) {
        float s = -__builtin_inff(), m;
        const int64_t j = j0 + lane;
        const bool in = j < n && counts(a, b, j, m);
        if (in) {
            float dot = 0.0f;
            for (int e = 0; e < a.width; ++e) dot = __builtin_fmaf(load_as_f32<DT>(a.q, qb + e), load_as_f32<DT>(a.k, kb + j * a.k_token + e), dot);
            s = __builtin_fmaf(dot, a.scale * to_log2, m * to_log2);
        }
        const float new_top = fmaxf(top, wave_max(s)), fade = __builtin_amdgcn_exp2f(top - new_top);
        const float p = in ? __builtin_amdgcn_exp2f(s - new_top) : 0.0f;
        top = new_top, total = total * fade + p;
        for (int e = 0; e < 4; ++e) o[e] *= fade;
        for (uint64_t left = __ballot(in); left; left &= left - 1) {
            const int x = __builtin_ctzll(left);
            const float px = round_to_dtype<DT>(__shfl(p, x));
            for (int e = 0; e < 4; ++e)
                if (e * 64 + lane < a.width) o[e] = __builtin_fmaf(px, load_as_f32<DT>(a.v, vb + (j0 + x) * a.v_token + e * 64 + lane), o[e]);
        }
    }
    for (int x = 1; x < 64; x *= 2) total += __shfl_xor(total, x);
    for (int e = 0; e < 4; ++e)
        if (e * 64 + lane < a.width) store_from_f32<DT>(a.out, row * a.width + e * 64 + lane, total > 0.0f ? o[e] / total : total);
}

// The elements that a strided tensor reaches to from its first one, 0 for one without elements, -1 past 2^62.
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

int validate(const i8f_attention_args &a) {
    if (a.batch < 0 || a.queries < 0 || a.keys < 0 || a.heads < 0 || a.kv_heads < 0 || a.width < 1) return I8F_ERR_INVALID;
    if (a.dtype != I8F_BF16 && a.dtype != I8F_F16) return valid_dtype(a.dtype) ? I8F_ERR_UNSUPPORTED : I8F_ERR_INVALID;
    if (a.heads && (!a.kv_heads || a.heads % a.kv_heads)) return I8F_ERR_INVALID;
    if (!(a.scale > 0.0f) || !(a.scale <= 3.4028234663852886e38f)) return I8F_ERR_INVALID;
    if (a.width > 256) return I8F_ERR_UNSUPPORTED;
    for (int64_t s : {a.q_batch, a.q_token, a.q_head, a.k_batch, a.k_token, a.k_head, a.v_batch, a.v_token, a.v_head})
        if (s < 0) return I8F_ERR_INVALID;
    for (int64_t n : {a.batch, a.queries, a.keys, a.heads})
        if (n > 0x7fffffff) return I8F_ERR_UNSUPPORTED;
    const int64_t rows = a.batch * a.queries;
    if (rows && a.heads > ((int64_t)1 << 33) / rows) return I8F_ERR_UNSUPPORTED;
    if (a.key_lengths && a.lengths_type != 0 && a.lengths_type != 1) return I8F_ERR_INVALID;
    if (a.key_mask && (a.mask_type < I8F_MASK_BYTES || a.mask_type > I8F_MASK_F32 || a.mask_batch < 0 || a.mask_key < 0)) return I8F_ERR_INVALID;
    const int64_t out = rows * a.heads * a.width, q = extent({{a.batch, a.q_batch}, {a.queries, a.q_token}, {a.heads, a.q_head}, {a.width, 1}});
    const int64_t k = extent({{a.batch, a.k_batch}, {a.keys, a.k_token}, {a.kv_heads, a.k_head}, {a.width, 1}});
    const int64_t v = extent({{a.batch, a.v_batch}, {a.keys, a.v_token}, {a.kv_heads, a.v_head}, {a.width, 1}});
    if (q < 0 || k < 0 || v < 0) return I8F_ERR_UNSUPPORTED;
    if (!out) return I8F_OK;   // (nothing to write: the pointers may be NULL)
    if (!a.q || !a.out || (a.keys && (!a.k || !a.v))) return I8F_ERR_INVALID;
    if (overlap(a.out, 2 * out, a.q, 2 * q) || overlap(a.out, 2 * out, a.k, 2 * k) || overlap(a.out, 2 * out, a.v, 2 * v)) return I8F_ERR_INVALID;
    return I8F_OK;
}

}  // namespace
}  // namespace i8f

extern "C" int64_t i8f_attention_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

extern "C" int i8f_attention(const i8f_attention_args *args, void *stream) {
    using namespace i8f;
    if (!args) return I8F_ERR_INVALID;
    const i8f_attention_args &a = *args;
    if (int rc = validate(a)) return rc;
    const int64_t rows = a.batch * a.queries * a.heads;
    if (!rows) return I8F_OK;
    if (!grid_fits((rows + 3) / 4, 256)) return I8F_ERR_UNSUPPORTED;
    if (int rc = check_device()) return rc;
    if (a.dtype == I8F_BF16) hipLaunchKernelGGL((attention_kernel<I8F_BF16>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((attention_kernel<I8F_F16>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch();
}
