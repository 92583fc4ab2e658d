// Between two blocks: the norm behind a block, its gate and the scales of branch and residual stream, and the norm and modulation in
// front of the next block, in one pass over the two rows that it takes (include/i8f_blocks.h has the formula).
#include "i8f_common.hpp"
#include "quant_run.hpp"
#include "rotate_run.hpp"

#include "../../include/i8f_blocks.h"

namespace i8f {
namespace {

enum { H_NONE, H_STORED, H_INT8, H_INT8_ROTATED };   // what becomes of h

// tanh(u) = (1 - e) / (1 + e) with e = exp(-2 |u|) on the hardware's exp2 and reciprocal: within 2e-7 of tanh, which 16-bit results do
// not see; binary32 rows take the library's function.
template <int DT>
__device__ __forceinline__ float gate_tanh(float u) {
    if constexpr (DT == I8F_F32) return tanhf(u);
    const float e = __builtin_amdgcn_exp2f(fabsf(u) * -2.8853900817779268f);
    return copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), u);
}

template <int DT>
__device__ __forceinline__ float norm_operand(const void *p, int dtype, int64_t k) {
    return DT == I8F_F32 || dtype == I8F_F32 ? ((const float *)p)[k] : load_as_f32<DT>(p, k);
}

// ---- any width, any alignment: 256 threads to a row, which is read again for every statistic (from cache) ------------------
template <int DT, int H>
__global__ __launch_bounds__(256) void block_norm_generic_kernel(const i8f_block_norm_args a) {
    __shared__ float red[4];
    const int64_t m = blockIdx.x, K = a.K;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t yb = m * a.ldy, rb = m * a.ldr;
    const int64_t gb = a.gate ? m / a.rows_per_gate * K : 0, sb = a.mod_scale ? m / a.rows_per_scale * K : 0;
    const int64_t tb = a.mod_shift ? m / a.rows_per_shift * K : 0;
    auto sum_over_row = [&](auto value) {
        float s = 0.0f;
        for (int64_t k = tid; k < K; k += 256) s += value(k);
        s = wave_sum_all(s);
        __syncthreads();   // (the slots of the sum before have been read)
        if (lane == 0) red[wave] = s;
        __syncthreads();
        return (red[0] + red[1]) + (red[2] + red[3]);
    };
    auto statistics = [&](int norm, float eps, auto value, float &mean, float &rstd) {
        mean = 0.0f, rstd = 1.0f;
        if (norm == I8F_NORM_NONE) return;
        if (norm == I8F_NORM_LAYER) mean = sum_over_row(value) / (float)K;
        const float mu = mean;
        rstd = 1.0f / sqrtf(sum_over_row([&](int64_t k) { const float d = value(k) - mu; return d * d; }) / (float)K + eps);
    };
    auto affine = [&](float v, int64_t k, const void *w, const void *b, int dtype) {
        if (w) v *= norm_operand<DT>(w, dtype, k);
        if (b) v += norm_operand<DT>(b, dtype, k);
        return v;
    };
    float mean1, rstd1, mean2, rstd2;
    statistics(a.post_norm, a.post_eps, [&](int64_t k) { return load_as_f32<DT>(a.y, yb + k); }, mean1, rstd1);
    auto x_of = [&](int64_t k) {
        const float n = affine((load_as_f32<DT>(a.y, yb + k) - mean1) * rstd1, k, a.post_weight, a.post_bias, a.post_dtype);
        float g = a.branch_scale;
        if (a.gate) {
            const float u = load_as_f32<DT>(a.gate, gb + k);
            g *= a.gate_tanh ? gate_tanh<DT>(u) : u;
        }
        return __builtin_fmaf(n, g, a.residual_scale * load_as_f32<DT>(a.residual, rb + k));
    };
    for (int64_t k = tid; k < K; k += 256) store_from_f32<DT>(a.x_out, m * K + k, x_of(k));
    if constexpr (H == H_NONE) return;
    statistics(a.pre_norm, a.pre_eps, x_of, mean2, rstd2);
    auto h_of = [&](int64_t k) {
        float h = affine((x_of(k) - mean2) * rstd2, k, a.pre_weight, a.pre_bias, a.pre_dtype);
        if (a.mod_scale) h *= 1.0f + load_as_f32<DT>(a.mod_scale, sb + k);
        if (a.mod_shift) h += load_as_f32<DT>(a.mod_shift, tb + k);
        return round_to_dtype<DT>(h);
    };
    if constexpr (H == H_STORED) {
        for (int64_t k = tid; k < K; k += 256) store_from_f32<DT>(a.h, m * K + k, h_of(k));
    } else {   // i8f_quant_rowwise's arithmetic on the rounded h
        float amax = 0.0f;
        auto over_blocks = [&](auto use) {   // a wave holds a 128-block
            for (int64_t b = wave; b < K / 128; b += 4) {
                float e0 = h_of(b * 128 + lane), e1 = h_of(b * 128 + 64 + lane);
                rotate128_wave<DT>(e0, e1, lane);
                use(b * 128 + lane, e0), use(b * 128 + 64 + lane, e1);
            }
        };
        auto most = [&](int64_t, float v) { amax = fmaxf(amax, fabsf(v)); };
        if constexpr (H == H_INT8_ROTATED) over_blocks(most);
        else
            for (int64_t k = tid; k < K; k += 256) most(k, h_of(k));
        amax = wave_max(amax);
        __syncthreads();
        if (lane == 0) red[wave] = amax;
        __syncthreads();
        amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        float s = amax / 127.0f;
        s = s < 1e-30f ? 1e-30f : s;
        const float inv = 1.0f / s;
        auto store = [&](int64_t k, float v) { a.q[m * K + k] = (int8_t)quant_i8(v * inv); };
        if constexpr (H == H_INT8_ROTATED) over_blocks(store);
        else
            for (int64_t k = tid; k < K; k += 256) store(k, h_of(k));
        if (tid == 0) a.scale[m] = s;
    }
}

template <int DT, int H>
int launch(const i8f_block_norm_args &a, hipStream_t st) {
    hipLaunchKernelGGL((block_norm_generic_kernel<DT, H>), dim3((unsigned)a.M), dim3(256), 0, st, a);
    return check_launch();
}

template <int DT>
int dispatch(const i8f_block_norm_args &a, hipStream_t st) {
    if (a.h) return launch<DT, H_STORED>(a, st);
    if (!a.q) return launch<DT, H_NONE>(a, st);
    return a.rotate_block ? launch<DT, H_INT8_ROTATED>(a, st) : launch<DT, H_INT8>(a, st);
}

int validate(const i8f_block_norm_args &a) {
    if (a.M < 0 || a.K < 0 || !valid_dtype(a.dtype)) return I8F_ERR_INVALID;
    if (a.rotate_block != 0 && a.rotate_block != 128) return I8F_ERR_UNSUPPORTED;
    if (a.rotate_block && (a.K % 128 || !a.q)) return I8F_ERR_INVALID;
    if ((a.h && a.q) || (a.q != nullptr) != (a.scale != nullptr)) return I8F_ERR_INVALID;
    auto norm = [&](int kind, float eps, const void *w, const void *b, int dtype) {
        if (kind != I8F_NORM_NONE && kind != I8F_NORM_RMS && kind != I8F_NORM_LAYER) return false;
        if (kind == I8F_NORM_NONE) return !w && !b;
        return eps >= 0.0f && ((!w && !b) || dtype == a.dtype || dtype == I8F_F32);
    };
    if (!norm(a.post_norm, a.post_eps, a.post_weight, a.post_bias, a.post_dtype) || !norm(a.pre_norm, a.pre_eps, a.pre_weight, a.pre_bias, a.pre_dtype))
        return I8F_ERR_INVALID;
    if ((a.gate && a.rows_per_gate <= 0) || (a.mod_scale && a.rows_per_scale <= 0) || (a.mod_shift && a.rows_per_shift <= 0)) return I8F_ERR_INVALID;
    if (a.M == 0 || a.K == 0) return I8F_OK;   // (an empty tensor's outputs may be NULL)
    if (!a.h && !a.q && (a.pre_norm != I8F_NORM_NONE || a.mod_scale || a.mod_shift)) return I8F_ERR_INVALID;
    if (!a.y || !a.residual || !a.x_out || a.ldy < a.K || a.ldr < a.K) return I8F_ERR_INVALID;
    return a.M > 0x7fffffff || a.K > 0x7fffffff ? I8F_ERR_UNSUPPORTED : I8F_OK;
}

}  // namespace
}  // namespace i8f

extern "C" int i8f_block_norm(const i8f_block_norm_args *args, void *stream) {
    using namespace i8f;
    if (!args) return I8F_ERR_INVALID;
    const i8f_block_norm_args &a = *args;
    if (int rc = validate(a)) return rc;
    if (a.M == 0 || a.K == 0) return I8F_OK;
    if (int rc = check_device()) return rc;
    hipStream_t st = (hipStream_t)stream;
    switch (a.dtype) {
    case I8F_BF16: return dispatch<I8F_BF16>(a, st);
    case I8F_F16: return dispatch<I8F_F16>(a, st);
    default: return dispatch<I8F_F32>(a, st);
    }
}
