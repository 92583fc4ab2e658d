// What the kernels around a shared projection take of the adapters (include/i8f_blocks.h).
#pragma once

#include "i8f_common.hpp"

#include "../../include/i8f_blocks.h"

namespace i8f {

// Adapter of row m, or -1: numbers outside [0, count) are rows without one, so that no address is formed from them.
__device__ __forceinline__ int adapter_of(const i8f_adapters &ad, int64_t m) {
    const int a = ad.ids[(uint32_t)m / (uint32_t)ad.rows_per_id];   // (M < 2^31)
    return (uint32_t)a < (uint32_t)ad.count ? a : -1;
}

// sum_j t[m,j] B_a[n,j] over the adapter's padded ranks from 8 k on, every 8 of `of` eights, pairs of 16-bit values at a time, in binary32
template <int DT>
__device__ __forceinline__ float adapter_term(const i8f_adapters &ad, const void *t, int64_t m, int64_t n, int64_t N, int a, int k = 0, int of = 1) {
    const int first = ad.first_rank[a], r = ad.first_rank[a + 1] - first;
    const char *tp = (const char *)t + m * ad.max_rank * 2, *bp = (const char *)ad.up + (N * first + n * r) * 2;
    float sum = 0.0f;
    for (int j = 8 * k; j < r; j += 8 * of) {
        const uint4 tv = *(const uint4 *)(tp + j * 2), bv = *(const uint4 *)(bp + j * 2);
        const uint32_t tw[4] = {tv.x, tv.y, tv.z, tv.w}, bw[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (DT == I8F_BF16) {
                sum = __builtin_fmaf(bf16_bits_to_f32(tw[e] & 0xffffu), bf16_bits_to_f32(bw[e] & 0xffffu), sum);
                sum = __builtin_fmaf(bf16_bits_to_f32(tw[e] >> 16), bf16_bits_to_f32(bw[e] >> 16), sum);
            } else {
                sum = __builtin_fmaf(f16_bits_to_f32(tw[e] & 0xffffu), f16_bits_to_f32(bw[e] & 0xffffu), sum);
                sum = __builtin_fmaf(f16_bits_to_f32(tw[e] >> 16), f16_bits_to_f32(bw[e] >> 16), sum);
            }
        }
    }
    return sum;
}

// 16 x 16 x 32 product of two fragments of 16-bit values, eight of each to a lane, into binary32
template <int DT, class V, class F>
__device__ __forceinline__ F factor_mfma(V a, V b, F c) {
    typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
    typedef _Float16 v8h __attribute__((ext_vector_type(8)));
    if constexpr (DT == I8F_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// The adapters of up to four layers, of one ids and rows_per_id, and where their first products go
struct DownLayers {
    i8f_adapters ad[I8F_MAX_ADAPTED_LAYERS];
    char *t[I8F_MAX_ADAPTED_LAYERS];
    float *side[I8F_MAX_ADAPTED_LAYERS];
    int64_t N[I8F_MAX_ADAPTED_LAYERS];
    int first_block[I8F_MAX_ADAPTED_LAYERS + 1];   // (rows form: first workgroup of each layer behind the quantiser's; [n] = all)
    int first_column[I8F_MAX_ADAPTED_LAYERS + 1];  // (partial sums: first column of each layer, max_rank of them; [n] = all)
    int n;
};
// Elements of a row of the adapters' first factors in memory: K, padded with zeros to a multiple of eight
__host__ __device__ inline int64_t factor_width(int64_t K) { return (K + 7) / 8 * 8; }
// A copy of x's rows with that width
inline int64_t adapters_copy_bytes(int64_t M, int64_t K) { return (M * factor_width(K) * 2 + 255) / 256 * 256; }
int adapters_copy_rows(const void *x, int64_t M, int64_t K, int64_t ldx, void *to, hipStream_t st);
// Many rows (adapters_down.hip; K a multiple of eight, aligned rows): slices of the columns that a launch for M rows is split into, and the
// launch.  One slice leaves t; more leave partial, [slices, M, first_column[n]] float, which adapters_combine makes t of.
int adapters_down_slices(int64_t M, int64_t K);
int adapters_down_partial(const void *x, int dtype, int64_t M, int64_t K, int64_t ldx, const DownLayers &g, float *partial, int slices, hipStream_t st);

// Host: whether the structure can be used on M rows of 16-bit type `dtype` at all (I8F_OK), before any pointer in it is.
inline int validate_adapters(const i8f_adapters *ad, int dtype, int64_t M) {
    if (!ad || ad->count < 0 || ad->count > 0x7fffffff || ad->max_rank < 0 || ad->max_rank % 16 || ad->rows_per_id <= 0) return I8F_ERR_INVALID;
    if (dtype != I8F_BF16 && dtype != I8F_F16) return I8F_ERR_INVALID;
    if (M == 0) return I8F_OK;
    if (!ad->ids || (ad->count > 0 && (!ad->first_rank || !ad->scale))) return I8F_ERR_INVALID;
    if (ad->max_rank > 0 && (!ad->down || !ad->up)) return I8F_ERR_INVALID;
    if (((uintptr_t)ad->down | (uintptr_t)ad->up) % 16) return I8F_ERR_INVALID;
    return M > 0x7fffffff || ad->max_rank > 65536 ? I8F_ERR_UNSUPPORTED : I8F_OK;
}
// The same of the layers of a call, and of what else they name
inline int validate_layers(const i8f_adapted_layer *layers, int n, int dtype, int64_t M) {
    if (M < 0 || n < 0 || (n > 0 && !layers)) return I8F_ERR_INVALID;
    if (n > I8F_MAX_ADAPTED_LAYERS) return I8F_ERR_UNSUPPORTED;
    for (int i = 0; i < n; ++i) {
        const i8f_adapted_layer &l = layers[i];
        if (int rc = validate_adapters(&l.adapters, dtype, M)) return rc;
        if (l.N < 0 || (l.bias && !valid_dtype(l.bias_dtype)) || (l.scale_mode != I8F_SCALE_TENSOR && l.scale_mode != I8F_SCALE_ROW)) return I8F_ERR_INVALID;
        if (l.adapters.ids != layers[0].adapters.ids || l.adapters.rows_per_id != layers[0].adapters.rows_per_id) return I8F_ERR_INVALID;
        if (M > 0 && l.adapters.max_rank > 0 && l.adapters.count > 0 && (!l.t || (uintptr_t)l.t % 16)) return I8F_ERR_INVALID;
        if ((l.side != nullptr) != (layers[0].side != nullptr) || (uintptr_t)l.side % 16) return I8F_ERR_INVALID;
    }
    return I8F_OK;
}
// A copy whose rows_per_id fits 32 bits (M does)
inline i8f_adapters for_kernel(const i8f_adapters &ad) {
    i8f_adapters k = ad;
    if (k.rows_per_id > 0x7fffffff) k.rows_per_id = 0x7fffffff;
    return k;
}

}  // namespace i8f
