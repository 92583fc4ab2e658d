// Between two blocks: the norm behind a block, its gate and the scales of branch and residual stream, and the norm and modulation in
// front of the next block, in one pass over the two rows that it takes (include/i8f_blocks.h has the formula).
#include <type_traits>

#include "i8f_common.hpp"
#include "quant_run.hpp"
#include "rotate_run.hpp"

#include "../../include/i8f_blocks.h"

namespace i8f {
namespace {

enum { H_NONE, H_STORED, H_INT8, H_INT8_ROTATED };   // what becomes of h

// tanh(u) = (1 - e) / (1 + e) with e = exp(-2 |u|) on the hardware's exp2 and reciprocal, within 2e-7 of it, and the first terms of the series
// near zero (the next one, 17 u^7 / 315, is below 4e-9 u there): 4e-6 relative at the most, which 16-bit results do not see.  binary32 rows
// take the library's function.
template <int DT>
__device__ __forceinline__ float gate_tanh(float u) {
    if constexpr (DT == I8F_F32) return tanhf(u);
    const float e = __builtin_amdgcn_exp2f(fabsf(u) * -2.8853900817779268f), u2 = u * u;
    const float near = __builtin_fmaf(u * u2, __builtin_fmaf(u2, 0.13333333f, -0.33333333f), u);   // (u - u^3 / 3 + 2 u^5 / 15: 1 - e cancels there)
    return fabsf(u) < 0.0625f ? near : copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), u);
}

template <int DT>
__device__ __forceinline__ float norm_operand(const void *p, int dtype, int64_t k) {
    return DT == I8F_F32 || dtype == I8F_F32 ? ((const float *)p)[k] : load_as_f32<DT>(p, k);
}

// ---- rows of less than a run, or too wide for registers (more than 16384 elements): 256 threads to a row, which is read again for every statistic
// (from cache) ----------------
template <int DT, int H>
__global__ __launch_bounds__(256) void block_norm_generic_kernel(const int64_t first_row, const i8f_block_norm_args a) {
    __shared__ float red[4];
    const int64_t m = first_row + blockIdx.x, K = a.K;
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

// ---- rows that stay in registers --------------------------------------------------------------------------------------------
// Both rows are read once, the sums are taken over registers: 7 or 8 bytes an element in 16 bits, which is what bounds it.  16384 x 5120 in
// bfloat16 153 us (149 to 159 from card to card), 4.4 TB/s, where a copy of 4 GiB runs at 4.75; 2048 x 3840 13.7 us, 4.6 TB/s;
// 4096 x 2048 in binary32 23.8 us, 5.6 TB/s, part of it from the last-level cache; 4096 x 3840 with int8 rows out 29 us.  A launch of two rows is
// 2.8 to 3.4 us, 4.5 in a row, of dependent loads.
// WPR waves share a row, a lane holds NCH runs of RUN consecutive elements (32 bytes of a 16-bit row, 16 of a binary32 one).  How many waves
// a row gets depends on its width alone, so that a row's bits depend neither on the rows beside it nor on what becomes of h.
template <int DT>
struct Run {
    static constexpr int N = DT == I8F_F32 ? 4 : 16;
};

// a lane's sum over the wave, in a fixed order: within quads, halves of rows and rows of 16 lanes, then across rows (as wave_max)
__device__ __forceinline__ float wave_sum_dpp(float v) {
    auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        const int moved = __builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
        v += __int_as_float(moved);
    };
    using std::integral_constant;
    add(integral_constant<int, 0xb1>{}, integral_constant<int, 0xf>{});    // quad_perm [1,0,3,2]
    add(integral_constant<int, 0x4e>{}, integral_constant<int, 0xf>{});    // quad_perm [2,3,0,1]
    add(integral_constant<int, 0x141>{}, integral_constant<int, 0xf>{});   // row_half_mirror
    add(integral_constant<int, 0x140>{}, integral_constant<int, 0xf>{});   // row_mirror
    add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});   // row_bcast 15 into rows 1 and 3
    add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});   // row_bcast 31 into rows 2 and 3
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

template <int DT>
struct Raw {
    uint4 v[DT == I8F_F32 ? 1 : 2];
};
// ANY: from whatever address it has
template <int DT, bool ANY>
__device__ __forceinline__ Raw<DT> load_run(const char *p) {
    Raw<DT> r;
    if constexpr (ANY) {
        __builtin_memcpy(&r, p, sizeof(r));
    } else {
        r.v[0] = *(const uint4 *)p;
        if constexpr (DT != I8F_F32) r.v[1] = *(const uint4 *)(p + 16);
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void expand(const Raw<DT> &r, float (&v)[Run<DT>::N]) {
    if constexpr (DT == I8F_F32) v[0] = __uint_as_float(r.v[0].x), v[1] = __uint_as_float(r.v[0].y), v[2] = __uint_as_float(r.v[0].z), v[3] = __uint_as_float(r.v[0].w);
    else expand16<DT>(r.v[0], r.v[1], v);
}
template <int DT, bool ANY>
__device__ __forceinline__ void store_run(char *p, const float (&v)[Run<DT>::N]) {
    constexpr int N = Run<DT>::N;
    uint32_t o[DT == I8F_F32 ? 4 : 8];
#pragma unroll
    for (int e = 0; e < (DT == I8F_F32 ? 4 : 8); ++e)
        o[e] = DT == I8F_F32 ? __float_as_uint(v[e % N]) : DT == I8F_BF16 ? f32x2_to_bf16x2_bits(v[2 * e % N], v[(2 * e + 1) % N]) : f32x2_to_f16x2_bits(v[2 * e % N], v[(2 * e + 1) % N]);
    if constexpr (ANY) {
        __builtin_memcpy(p, o, sizeof(o));
    } else {
        stream_store16(p, make_uint4(o[0], o[1], o[2], o[3]));
        if constexpr (DT != I8F_F32) stream_store16(p + 16, make_uint4(o[4], o[5], o[6], o[7]));
    }
}
// the run of a weight or bias that starts at element k
template <int DT, bool ANY>
__device__ __forceinline__ void operand_run(const void *p, int dtype, int64_t k, float (&v)[Run<DT>::N]) {
    if (DT != I8F_F32 && dtype == I8F_F32) {
#pragma unroll
        for (int e = 0; e < Run<DT>::N; e += 4) {
            float f[4];
            expand<I8F_F32>(load_run<I8F_F32, ANY>((const char *)((const float *)p + k + e)), f);
            v[e] = f[0], v[e + 1] = f[1], v[e + 2] = f[2], v[e + 3] = f[3];
        }
    } else {
        expand<DT>(load_run<DT, ANY>((const char *)p + k * (DT == I8F_F32 ? 4 : 2)), v);
    }
}

// ANY: rows of any width (a run at least) and alignment.  A row's last run then ends with it and begins in the run before, whose elements it
// computes again and leaves out of the sums, which are the same ones in the same order.
template <int DT, int H, int WPR, int NCH, bool ANY>
__global__ __launch_bounds__(256) void block_norm_kernel(const int64_t first_row, const i8f_block_norm_args a) {
    constexpr int N = Run<DT>::N, TPR = 64 * WPR, ROWS = 4 / WPR, SIZE = DT == I8F_F32 ? 4 : 2;
    __shared__ float red[5][ROWS][WPR];
    const int t = threadIdx.x % TPR, rb = threadIdx.x / TPR, lane = threadIdx.x & 63;
    const int64_t K = a.K;
    const int runs = (int)((K + N - 1) / N);
    const int64_t own = first_row + (int64_t)blockIdx.x * ROWS + rb;
    const bool ok = own < a.M;
    const int64_t m = ok ? own : a.M - 1;   // (a wave past the last row computes it again and stores nothing)
    // which of its runs a lane holds: its own, or where the rotation pairs lanes by DPP the one that it wants there (rotate_run16,
    // rotate_chunk_f32); the sums pair the same runs either way
    const int p = H != H_INT8_ROTATED ? t : DT == I8F_F32 ? (t & ~15) | chunk_of_lane16(t & 15) : t ^ (((t >> 2) & 1) * 3);
    auto sum_over_row = [&](float part, int slot) {
        part = wave_sum_dpp(part);
        if constexpr (WPR > 1) {   // (a slot for each sum: nobody waits for its readers)
            if (lane == 0) red[slot][rb][t / 64] = part;
            __syncthreads();
            part = red[slot][rb][0];
#pragma unroll
            for (int w = 1; w < WPR; ++w) part += red[slot][rb][w];
        }
        return part;
    };
    int64_t at[NCH];   // first element of each run; a lane without one takes the row's first and leaves it out of the sums
    bool in[NCH];
    int skip[NCH];     // ANY: elements that belong to the run before
    Raw<DT> yr[NCH], rr[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        in[i] = i * TPR + p < runs;
        at[i] = in[i] ? (int64_t)(i * TPR + p) * N : 0;
        skip[i] = 0;
        if (ANY && at[i] > K - N) skip[i] = (int)(at[i] - (K - N)), at[i] = K - N;
        yr[i] = load_run<DT, ANY>((const char *)a.y + (m * a.ldy + at[i]) * SIZE);
        rr[i] = load_run<DT, ANY>((const char *)a.residual + (m * a.ldr + at[i]) * SIZE);
    }
    float x[NCH][N];
#pragma unroll
    for (int i = 0; i < NCH; ++i) expand<DT>(yr[i], x[i]);
    // (x - mean) * rstd * weight + bias of the rows in x, in place
    auto normalise = [&](int norm, float eps, const void *w, const void *b, int dtype, int slot) __attribute__((always_inline)) {
        if (norm == I8F_NORM_NONE) return;
        if (norm == I8F_NORM_LAYER) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) sum += in[i] && (!ANY || e >= skip[i]) ? x[i][e] : 0.0f;
            const float mean = sum_over_row(sum, slot) / (float)K;
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) x[i][e] -= mean;
        }
        float squares = 0.0f;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < N; ++e) s = ANY && e < skip[i] ? s : __builtin_fmaf(x[i][e], x[i][e], s);
            squares += in[i] ? s : 0.0f;
        }
        const float rstd = 1.0f / sqrtf(sum_over_row(squares, slot + 1) / (float)K + eps);
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            float v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) x[i][e] *= rstd;
            if (w) {
                operand_run<DT, ANY>(w, dtype, at[i], v);
#pragma unroll
                for (int e = 0; e < N; ++e) x[i][e] *= v[e];
            }
            if (b) {
                operand_run<DT, ANY>(b, dtype, at[i], v);
#pragma unroll
                for (int e = 0; e < N; ++e) x[i][e] += v[e];
            }
        }
    };
    auto vector_of = [&](const void *v, int64_t rows_per) { return (const char *)v + (int64_t)((uint32_t)m / (uint32_t)rows_per) * K * SIZE; };
    normalise(a.post_norm, a.post_eps, a.post_weight, a.post_bias, a.post_dtype, 0);
    const char *gate = a.gate ? vector_of(a.gate, a.rows_per_gate) : nullptr;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        float r[N], g[N];
        expand<DT>(rr[i], r);
        if (gate) {
            expand<DT>(load_run<DT, ANY>(gate + at[i] * SIZE), g);
            if (a.gate_tanh) {
#pragma unroll
                for (int e = 0; e < N; ++e) g[e] = gate_tanh<DT>(g[e]);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) x[i][e] = __builtin_fmaf(x[i][e], g[e] * a.branch_scale, a.residual_scale * r[e]);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) x[i][e] = __builtin_fmaf(x[i][e], a.branch_scale, a.residual_scale * r[e]);
        }
        if (ok && in[i]) store_run<DT, ANY>((char *)a.x_out + (m * K + at[i]) * SIZE, x[i]);
    }
    if constexpr (H == H_NONE) return;
    normalise(a.pre_norm, a.pre_eps, a.pre_weight, a.pre_bias, a.pre_dtype, 2);
    const char *ms = a.mod_scale ? vector_of(a.mod_scale, a.rows_per_scale) : nullptr, *mt = a.mod_shift ? vector_of(a.mod_shift, a.rows_per_shift) : nullptr;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        float v[N];
        if (ms) {
            expand<DT>(load_run<DT, ANY>(ms + at[i] * SIZE), v);
#pragma unroll
            for (int e = 0; e < N; ++e) x[i][e] *= 1.0f + v[e];
        }
        if (mt) {
            expand<DT>(load_run<DT, ANY>(mt + at[i] * SIZE), v);
#pragma unroll
            for (int e = 0; e < N; ++e) x[i][e] += v[e];
        }
        if constexpr (H == H_STORED) {
            if (ok && in[i]) store_run<DT, ANY>((char *)a.h + (m * K + at[i]) * SIZE, x[i]);
        } else {   // i8f_quant_rowwise's arithmetic on the rounded h
#pragma unroll
            for (int e = 0; e < N; ++e) x[i][e] = in[i] ? round_to_dtype<DT>(x[i][e]) : 0.0f;
            if constexpr (H == H_INT8_ROTATED) {
                if constexpr (DT == I8F_F32) rotate_chunk_f32(x[i], t);
                else rotate_run16<DT>(x[i], (p & 1) ? -1.0f : 1.0f, (p & 2) ? -1.0f : 1.0f, (p & 4) ? -1.0f : 1.0f);
            }
#pragma unroll
            for (int e = 0; e < N; e += 2) amax = max3_abs(amax, x[i][e], x[i][e + 1]);
        }
    }
    if constexpr (H == H_INT8 || H == H_INT8_ROTATED) {
        amax = wave_max(amax);
        if constexpr (WPR > 1) {
            if (lane == 0) red[4][rb][t / 64] = amax;
            __syncthreads();
            amax = red[4][rb][0];
#pragma unroll
            for (int w = 1; w < WPR; ++w) amax = fmaxf(amax, red[4][rb][w]);
        }
        // (as i8f_quant_rowwise does with rows of this width: the short forms differ from these in what becomes of a value that is not finite)
        const bool saturating = DT == I8F_F32 || (ANY && K % 16 != 0);
        float s, inv;
        if (saturating) {
            s = amax / 127.0f;
            s = s < 1e-30f ? 1e-30f : s;
            inv = 1.0f / s;
        } else {
            scale_and_inverse16(amax, s, inv);
        }
        if (!ok) return;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            if (!in[i]) continue;
            int8_t *dst = a.q + m * K + at[i];
            if (saturating) {
                uint32_t w[N / 4];
#pragma unroll
                for (int e = 0; e < N; ++e) w[e / 4] = (e % 4 ? w[e / 4] : 0u) | ((uint32_t)quant_i8(x[i][e] * inv) & 0xffu) << (8 * (e % 4));
                __builtin_memcpy(dst, w, N);
            } else if constexpr (DT != I8F_F32) {
                const uint4 o = quant16_magic(x[i], inv);
                if constexpr (ANY) __builtin_memcpy(dst, &o, 16);
                else stream_store16(dst, o);
            }
        }
        if (t == 0) a.scale[m] = s;
    }
}

// ROWS rows to a workgroup, in as many launches as it takes: one has fewer than 2^32 threads
// (the first row comes ahead of the structure, among the arguments that are in registers when a wave starts: 2048 x 3840 13.7 us, 14.1 behind it)
template <int ROWS, class KERNEL>
int launch_ranges(KERNEL kernel, const i8f_block_norm_args &a, hipStream_t st) {
    constexpr int64_t MOST = (int64_t)ROWS << 23;
    for (int64_t m0 = 0; m0 < a.M; m0 += MOST) {
        const int64_t rows = a.M - m0 < MOST ? a.M - m0 : MOST;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + ROWS - 1) / ROWS)), dim3(256), 0, st, m0, a);
        if (int rc = check_launch()) return rc;
    }
    return I8F_OK;
}
template <int DT, int H, int WPR, int NCH, bool ANY>
int launch_rows(const i8f_block_norm_args &a, hipStream_t st) {
    return launch_ranges<4 / WPR>(block_norm_kernel<DT, H, WPR, NCH, ANY>, a, st);
}

// Aligned rows of whole runs; 16-byte pieces of every operand
bool whole_runs(const i8f_block_norm_args &a, int run) {
    const uintptr_t all = (uintptr_t)a.y | (uintptr_t)a.residual | (uintptr_t)a.post_weight | (uintptr_t)a.post_bias | (uintptr_t)a.pre_weight |
                          (uintptr_t)a.pre_bias | (uintptr_t)a.gate | (uintptr_t)a.mod_scale | (uintptr_t)a.mod_shift | (uintptr_t)a.x_out |
                          (uintptr_t)a.h | (uintptr_t)a.q;
    const int64_t per16 = 16 / (int64_t)dtype_size(a.dtype);
    return all % 16 == 0 && a.K % run == 0 && a.ldy % per16 == 0 && a.ldr % per16 == 0;
}

// Waves to a row by its width, us for 2, 512, 4096 and 32768 rows with both norms, a tanh gate and a scale:
//     1024 x 16 bits  one wave          4.1   4.9   9.6   58      four, half of them idle   4.4   5.3  19.7  128
//     2048            two, a run each   4.4   5.3  16.0  110      one, two runs             6.3   7.5  16.7  112     four  4.3  5.5  21.8  147
//     4096            four, a run each  4.5   6.9  27.9  217      two, two runs             6.8   8.7  29.9  212     one  10.5  12.8  35.5  251
//     512 x 32 bits   one, two runs     4.1   4.6   8.4   54      two, a run each           3.2   3.7   8.7   58
//     1024            four, a run each  3.4   4.2  15.0  108      two, two runs             4.3   5.1  13.9  100
template <int DT, int H, bool ANY>
int launch_width(const i8f_block_norm_args &a, int64_t runs, hipStream_t st) {
    if (runs <= 64) return launch_rows<DT, H, 1, 1, ANY>(a, st);
    if (runs <= 128) return launch_rows<DT, H, DT == I8F_F32 ? 1 : 2, DT == I8F_F32 ? 2 : 1, ANY>(a, st);
    if (runs <= 256) return launch_rows<DT, H, 4, 1, ANY>(a, st);
    if (runs <= 512) return launch_rows<DT, H, 4, 2, ANY>(a, st);
    if (runs <= 768) return launch_rows<DT, H, 4, 3, ANY>(a, st);
    if (DT != I8F_F32 || runs <= 1024) return launch_rows<DT, H, 4, 4, ANY>(a, st);
    if constexpr (DT == I8F_F32) {   // (runs of four elements: as many registers as half of that in 16 bits)
        if (runs <= 1536) return launch_rows<DT, H, 4, 6, ANY>(a, st);
        if (runs <= 2048) return launch_rows<DT, H, 4, 8, ANY>(a, st);
    }
    return launch_rows<DT, H, 4, DT == I8F_F32 ? 16 : 4, ANY>(a, st);
}

template <int DT, int H>
int launch(const i8f_block_norm_args &a, hipStream_t st) {
    constexpr int N = Run<DT>::N;
    const int64_t runs = (a.K + N - 1) / N;
    if (runs <= (DT == I8F_F32 ? 4096 : 1024) && a.K >= N) return whole_runs(a, N) ? launch_width<DT, H, false>(a, runs, st) : launch_width<DT, H, true>(a, runs, st);
    return launch_ranges<1>(block_norm_generic_kernel<DT, H>, a, st);
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
    for (const void *in : {a.y, a.residual})
        if (a.x_out == in || a.h == in || (const void *)a.q == in) return I8F_ERR_INVALID;   // (a row is written while other waves read it)
    if (a.x_out == a.h || a.x_out == (void *)a.q) return I8F_ERR_INVALID;
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
    i8f_block_norm_args k = a;   // (M is below 2^31, and so are the rows of a vector then)
    for (int64_t *rows : {&k.rows_per_gate, &k.rows_per_scale, &k.rows_per_shift}) *rows = *rows < 1 ? 1 : *rows > 0x7fffffff ? 0x7fffffff : *rows;
    switch (k.dtype) {
    case I8F_BF16: return dispatch<I8F_BF16>(k, st);
    case I8F_F16: return dispatch<I8F_F16>(k, st);
    default: return dispatch<I8F_F32>(k, st);
    }
}
