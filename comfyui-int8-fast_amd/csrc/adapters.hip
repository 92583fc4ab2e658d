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

template <int DT>
int launch_down(const void *x, int64_t M, int64_t K, int64_t ldx, const i8f_adapters &ad, void *t, hipStream_t st) {
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

extern "C" int64_t i8f_linear_w8a8_adapters_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    (void)K;
    return M > 0 && N > 0 ? M * N * 4 : 0;
}

extern "C" int i8f_linear_w8a8_adapters(const int8_t *a, const float *a_scale, const int8_t *w, const float *w_scale, float w_scale_host, int scale_mode,
                                        const void *bias, int bias_dtype, const i8f_adapters *adapters, const void *t, void *out, int out_dtype,
                                        int64_t M, int64_t N, int64_t K, void *workspace, int64_t workspace_bytes, void *stream) {
    using namespace i8f;
    if (M < 0 || N < 0 || K < 0) return I8F_ERR_INVALID;
    if (int rc = validate_adapters(adapters, out_dtype, M)) return rc;
    if (M == 0 || N == 0) return I8F_OK;
    if (!out || (adapters->max_rank > 0 && !t)) return I8F_ERR_INVALID;
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < i8f_linear_w8a8_adapters_workspace_bytes(M, N, K)) return I8F_ERR_INVALID;
    // the projection in binary32, then the adapters' share and the one rounding
    if (int rc = i8f_linear_w8a8(a, a_scale, w, w_scale, w_scale_host, scale_mode, bias, bias_dtype, workspace, I8F_F32, M, N, K, I8F_EPI_FUSED, stream))
        return rc;
    return i8f_adapters_up(workspace, I8F_F32, adapters, t, out, out_dtype, M, N, stream);
}
