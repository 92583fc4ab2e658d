// The second product of low-rank adapters that differ from row to row, beside a projection that is there already
// (include/i8f_blocks.h; quant_adapters.hpp has the first product, the layers' own kernels add the second themselves).
#include "adapters.hpp"

namespace i8f {
namespace {

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

}  // namespace
}  // namespace i8f

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
