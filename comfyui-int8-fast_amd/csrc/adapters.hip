// Low-rank adapters that differ from row to row, beside a projection that all rows share (include/i8f_blocks.h):
//   t = scale_a A_a x        i8f_adapters_down
//   out = base + B_a t       i8f_adapters_up, or the epilogue of the layer's own kernel
#include "adapters.hpp"
#include "quant_run.hpp"

namespace i8f {
namespace {

// ---- t = scale_a A_a x: any width and alignment, one wave to a rank of a row ------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void adapters_down_kernel(const char *__restrict__ x, int64_t K, int64_t ldx, const i8f_adapters ad, char *__restrict__ t) {
    const int64_t m = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int a = adapter_of(ad, m);
    if (a < 0) return;
    const int first = ad.first_rank[a], r = ad.first_rank[a + 1] - first;
    const float s = ad.scale[a];
    for (int j = wave; j < r; j += 4) {
        float sum = 0.0f;
        for (int64_t k = lane; k < K; k += 64) sum = __builtin_fmaf(load_as_f32<DT>(x, m * ldx + k), load_as_f32<DT>(ad.down, (first + j) * K + k), sum);
        sum = wave_sum_all(sum);
        if (lane == 0) store_from_f32<DT>(t, m * ad.max_rank + j, sum * s);
    }
}

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ v4f down_mfma(v4u a, v4u b, v4f c) {
    if constexpr (DT == I8F_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ float dot8(v4u a, v4u b, float sum) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (DT == I8F_BF16) {
            sum = __builtin_fmaf(bf16_bits_to_f32(a[e] & 0xffffu), bf16_bits_to_f32(b[e] & 0xffffu), sum);
            sum = __builtin_fmaf(__uint_as_float(a[e] & 0xffff0000u), __uint_as_float(b[e] & 0xffff0000u), sum);
        } else {
            sum = __builtin_fmaf(f16_bits_to_f32(a[e] & 0xffffu), f16_bits_to_f32(b[e] & 0xffffu), sum);
            sum = __builtin_fmaf(f16_bits_to_f32(a[e] >> 16), f16_bits_to_f32(b[e] >> 16), sum);
        }
    }
    return sum;
}

// The same with 16-byte loads (K % 8 == 0, aligned rows), eight of each operand under way at once: few rows, so that what counts is that
// every rank of every row is a wave of its own.
template <int DT>
__global__ __launch_bounds__(256) void adapters_down_rows_kernel(const char *__restrict__ x, int K, int64_t ldx, const i8f_adapters ad, char *__restrict__ t) {
    const int64_t m = blockIdx.x;
    const int lane = threadIdx.x & 63, j = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int a = adapter_of(ad, m);
    if (a < 0) return;
    const int first = ad.first_rank[a];
    if (j >= ad.first_rank[a + 1] - first) return;
    const char *xp = x + m * ldx * 2, *ap = (const char *)ad.down + (int64_t)(first + j) * K * 2;
    float sum = 0.0f;
    for (int k0 = lane * 8; k0 < K; k0 += 8 * 512) {
        v4u xv[8], av[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int k = k0 + c * 512;
            xv[c] = k < K ? *(const v4u *)(xp + (int64_t)k * 2) : (v4u)0u;
            av[c] = k < K ? *(const v4u *)(ap + (int64_t)k * 2) : (v4u)0u;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) sum = dot8<DT>(xv[c], av[c], sum);
    }
    sum = wave_sum_all(sum);
    if (lane == 0) store_from_f32<DT>(t, m * ad.max_rank + j, sum * ad.scale[a]);
}

// Many rows: 16 of them to a workgroup, the matrix unit multiplies 16 rows by 16 ranks, up to 64 ranks at a time.  Eight waves share the
// columns: wave w takes blocks w, w + 8, ... of 64 columns.  Eight neighbouring lanes load the 128 bytes of a row, of x and of A
// alike, and the tiles change to the matrix unit's layout in LDS of the wave's own; the next block's loads are under way meanwhile.
// An adapter that occurs among the rows is a pass over the columns for all of them; its products are stored for its own rows.
template <int DT>
__global__ __launch_bounds__(512) void adapters_down_tiles_kernel(const char *__restrict__ x, int M, int K, int64_t ldx, const i8f_adapters ad, char *__restrict__ t) {
    constexpr int RT = 4;
    __shared__ union {
        v4u tile[8][1 + RT][128];  // [wave][x, A...][row * 8 + (16-byte chunk ^ row & 7)]
        v4f sum[8][RT][64];
    } sh;
    const int tid = threadIdx.x, lane = tid & 63, r = lane >> 3, c = lane & 7, fr = lane & 15, fg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row0 = blockIdx.x * 16, blocks = (K + 63) / 64;
    const int my_row = row0 + fr;
    const int id = my_row < M ? adapter_of(ad, my_row) : -1;
    uint64_t left = __builtin_amdgcn_ballot_w64(id >= 0);
    const char *x0 = x + (int64_t)min(row0 + r, M - 1) * ldx * 2 + c * 16, *x1 = x + (int64_t)min(row0 + r + 8, M - 1) * ldx * 2 + c * 16;
    v4u(*tile)[128] = sh.tile[wave];
    const int put = r * 8 + (c ^ r);
    while (left) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        left &= ~__builtin_amdgcn_ballot_w64(id == a);
        const int first = __builtin_amdgcn_readfirstlane(ad.first_rank[a]), rank = __builtin_amdgcn_readfirstlane(ad.first_rank[a + 1]) - first;
        const float s = ad.scale[a];
        for (int j0 = 0; j0 < rank; j0 += 16 * RT) {
            const int tiles = min(RT, (rank - j0) / 16);
            const char *ap = (const char *)ad.down + (int64_t)(first + j0 + r) * K * 2 + c * 16;
            v4f acc[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) acc[i] = (v4f)0.0f;
            v4u xv[2], av[RT][2];
            auto fetch = [&](int b) __attribute__((always_inline)) {
                const bool in = b < blocks && b * 64 + c * 8 < K;   // (K % 8 == 0)
                const int64_t off = in ? (int64_t)b * 128 : -c * 16;
                xv[0] = *(const v4u *)(x0 + off), xv[1] = *(const v4u *)(x1 + off);
                if (!in) xv[0] = xv[1] = (v4u)0u;
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    if (i < tiles) {
                        av[i][0] = *(const v4u *)(ap + (int64_t)(16 * i) * K * 2 + off), av[i][1] = *(const v4u *)(ap + (int64_t)(16 * i + 8) * K * 2 + off);
                        if (!in) av[i][0] = av[i][1] = (v4u)0u;
                    }
                }
            };
            fetch(wave);
            for (int b = wave; b < blocks; b += 8) {
                tile[0][put] = xv[0], tile[0][put + 64] = xv[1];
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    if (i < tiles) tile[1 + i][put] = av[i][0], tile[1 + i][put + 64] = av[i][1];
                fetch(b + 8);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int get = fr * 8 + ((4 * h + fg) ^ (fr & 7));
                    const v4u xf = tile[0][get];
#pragma unroll
                    for (int i = 0; i < RT; ++i)
                        if (i < tiles) acc[i] = down_mfma<DT>(tile[1 + i][get], xf, acc[i]);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
            __syncthreads();   // (the tiles are done with)
#pragma unroll
            for (int i = 0; i < RT; ++i) sh.sum[wave][i][lane] = acc[i];
            __syncthreads();
            if (wave < tiles && id == a) {   // the waves' sums, in wave order: ranks j0 + 16 wave + 4 fg ... of the lane's row
                v4f sum = sh.sum[0][wave][lane];
#pragma unroll
                for (int w = 1; w < 8; ++w) sum += sh.sum[w][wave][lane];
                uint2 o;
                if constexpr (DT == I8F_BF16) o = make_uint2(f32x2_to_bf16x2_bits(sum.x * s, sum.y * s), f32x2_to_bf16x2_bits(sum.z * s, sum.w * s));
                else o = make_uint2(f32x2_to_f16x2_bits(sum.x * s, sum.y * s), f32x2_to_f16x2_bits(sum.z * s, sum.w * s));
                *(uint2 *)(t + ((int64_t)my_row * ad.max_rank + j0 + 16 * wave + 4 * fg) * 2) = o;
            }
            __syncthreads();   // (the sums are read before the next tiles)
        }
    }
}

// out = round(base + B_a t): one thread to an output
template <int DT, int BASE>
__global__ __launch_bounds__(256) void adapters_up_kernel(const void *base, const i8f_adapters ad, const void *__restrict__ t, void *out, int64_t N, int64_t m0) {
    const int64_t m = m0 + blockIdx.y, n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    const int a = adapter_of(ad, m);
    float v = load_as_f32<BASE>(base, m * N + n);
    if (a >= 0) v += adapter_term<DT>(ad, t, m, n, N, a);
    store_from_f32<DT>(out, m * N + n, v);
}

template <int DT, int BASE>
int launch_up(const void *base, const i8f_adapters &ad, const void *t, void *out, int64_t M, int64_t N, hipStream_t st) {
    for (int64_t m0 = 0; m0 < M; m0 += 65535) {   // (the second dimension of a grid ends there)
        const dim3 grid((unsigned)((N + 255) / 256), (unsigned)(M - m0 < 65535 ? M - m0 : 65535));
        hipLaunchKernelGGL((adapters_up_kernel<DT, BASE>), grid, dim3(256), 0, st, base, ad, t, out, N, m0);
        if (int rc = check_launch()) return rc;
    }
    return I8F_OK;
}

constexpr int64_t DOWN_ROWS = 256;   // rows up to which a rank of a row is a wave of its own

template <int DT>
int launch_down(const void *x, int64_t M, int64_t K, int64_t ldx, const i8f_adapters &ad, void *t, hipStream_t st) {
    if (K % 8 == 0 && (uintptr_t)x % 16 == 0 && ldx % 8 == 0 && K < (1ll << 30)) {
        if (M <= DOWN_ROWS)
            hipLaunchKernelGGL((adapters_down_rows_kernel<DT>), dim3((unsigned)M, (unsigned)(ad.max_rank / 4)), dim3(256), 0, st, (const char *)x, (int)K, ldx, ad, (char *)t);
        else
            hipLaunchKernelGGL((adapters_down_tiles_kernel<DT>), dim3((unsigned)((M + 15) / 16)), dim3(512), 0, st, (const char *)x, (int)M, (int)K, ldx, ad, (char *)t);
        return check_launch();
    }
    hipLaunchKernelGGL((adapters_down_kernel<DT>), dim3((unsigned)M), dim3(256), 0, st, (const char *)x, K, ldx, ad, (char *)t);
    return check_launch();
}

}  // namespace
}  // namespace i8f

extern "C" int i8f_adapters_down(const void *x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const i8f_adapters *adapters, void *t, void *stream) {
    using namespace i8f;
    if (M < 0 || K < 0) return I8F_ERR_INVALID;
    if (int rc = validate_adapters(adapters, x_dtype, M)) return rc;
    if (M == 0 || adapters->max_rank == 0 || adapters->count == 0) return I8F_OK;
    if (!t || ldx < K || (K > 0 && !x) || (uintptr_t)t % 16) return I8F_ERR_INVALID;
    if (K > 0x7fffffff) return I8F_ERR_UNSUPPORTED;
    if (int rc = check_device()) return rc;
    const i8f_adapters ad = for_kernel(*adapters);
    return x_dtype == I8F_BF16 ? launch_down<I8F_BF16>(x, M, K, ldx, ad, t, (hipStream_t)stream) : launch_down<I8F_F16>(x, M, K, ldx, ad, t, (hipStream_t)stream);
}

extern "C" int i8f_adapters_up(const void *base, int base_dtype, const i8f_adapters *adapters, const void *t, void *out, int out_dtype, int64_t M,
                               int64_t N, void *stream) {
    using namespace i8f;
    if (M < 0 || N < 0 || (base_dtype != I8F_F32 && base_dtype != out_dtype)) return I8F_ERR_INVALID;
    if (int rc = validate_adapters(adapters, out_dtype, M)) return rc;
    if (M == 0 || N == 0) return I8F_OK;
    if (!base || !out || (adapters->max_rank > 0 && (!t || (uintptr_t)t % 16))) return I8F_ERR_INVALID;
    if (base == out && base_dtype != out_dtype) return I8F_ERR_INVALID;
    if (N > 0x7fffffff) return I8F_ERR_UNSUPPORTED;
    if (int rc = check_device()) return rc;
    const i8f_adapters ad = for_kernel(*adapters);
    hipStream_t st = (hipStream_t)stream;
    if (out_dtype == I8F_BF16)
        return base_dtype == I8F_F32 ? launch_up<I8F_BF16, I8F_F32>(base, ad, t, out, M, N, st) : launch_up<I8F_BF16, I8F_BF16>(base, ad, t, out, M, N, st);
    return base_dtype == I8F_F32 ? launch_up<I8F_F16, I8F_F32>(base, ad, t, out, M, N, st) : launch_up<I8F_F16, I8F_F16>(base, ad, t, out, M, N, st);
}
