// The second product of low-rank adapters that differ from row to row, beside a projection that is there already
// (include/i8f_blocks.h; quant_adapters.hpp has the first product, the layers' own kernels add the second themselves).
#include "adapters.hpp"

namespace i8f {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// out = round(base + B_a t): a wave takes 16 rows and 32 columns.  The matrix unit's 16 x 16 x 32 form has the rows' t as one operand and 16
// rows of the factor as the other; an adapter that occurs among the 16 rows is a product for all of them, and a row takes its own (a select:
// zeros in t instead would let an adapter that is not finite into every row).  Loads of base and stores bound it where rows share adapters,
// the trips to memory for one factor after the other where they do not: 2382 x 292 with 43 requests of ranks up to 91 6.2 us, 333 x 1001 with
// five of up to 13 4.4 (a thread to an output: 22.8 and 3.4).
template <int DT, int BASE>
__global__ __launch_bounds__(256) void adapters_up_kernel(const void *base, const i8f_adapters ad, const void *__restrict__ t, void *out, int64_t M, int64_t N,
                                                          int64_t m_first) {
    constexpr int BLOCKS = 2;   // of 16 columns
    const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
    const int64_t m0 = m_first + (int64_t)blockIdx.y * 16, m = m0 + l16;   // the row whose t the lane fetches; its results are of rows 4 lq + e
    const int64_t n0 = ((int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * (16 * BLOCKS);
    if (n0 >= N) return;
    const int id = m < M ? adapter_of(ad, m) : -1;
    const int first = id >= 0 ? ad.first_rank[id] : 0, rank = id >= 0 ? ad.first_rank[id + 1] - first : 0;
    const char *tp = (const char *)t + m * ad.max_rank * 2;
    float v[BLOCKS][4];
    v4f sum[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        sum[b] = (v4f)0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t row = m0 + 4 * lq + e, n = n0 + 16 * b + l16;
            v[b][e] = row < M && n < N ? load_as_f32<BASE>(base, row * N + n) : 0.0f;
        }
    }
    int whose[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) whose[e] = __shfl(id, 4 * lq + e);
    uint64_t left = __builtin_amdgcn_ballot_w64(rank > 0);
    while (left) {
        const int row = __builtin_ctzll(left), a = __builtin_amdgcn_readlane(id, row), r = __builtin_amdgcn_readlane(rank, row);
        const char *up = (const char *)ad.up + N * __builtin_amdgcn_readlane(first, row) * 2;
        left &= ~__builtin_amdgcn_ballot_w64(id == a);
#pragma unroll 2
        for (int k = 8 * lq; k - 8 * lq < r; k += 32) {
            const bool in = k < r;   // (ranks come in sixteens: the last step may be half a one)
            const v4u tv = in && id == a ? *(const v4u *)(tp + k * 2) : (v4u)0u;
            v4u bv[BLOCKS];
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const int64_t n = n0 + 16 * b + l16 < N ? n0 + 16 * b + l16 : N - 1;
                bv[b] = in ? *(const v4u *)(up + (n * r + k) * 2) : (v4u)0u;
            }
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const v4f d = factor_mfma<DT>(tv, bv[b], sum[b]);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[b][e] = whose[e] == a ? d[e] : sum[b][e];
            }
        }
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t row = m0 + 4 * lq + e, n = n0 + 16 * b + l16;
            if (row < M && n < N) store_from_f32<DT>(out, row * N + n, v[b][e] + sum[b][e]);
        }
}

template <int DT, int BASE>
int launch_up(const void *base, const i8f_adapters &ad, const void *t, void *out, int64_t M, int64_t N, hipStream_t st) {
    if (!grid_fits((N + 127) / 128, 256)) return I8F_ERR_UNSUPPORTED;
    constexpr int64_t MOST = 16 * 65535;   // (the second dimension of a grid ends there)
    for (int64_t m0 = 0; m0 < M; m0 += MOST) {
        const dim3 grid((unsigned)((N + 127) / 128), (unsigned)(((M - m0 < MOST ? M - m0 : MOST) + 15) / 16));
        hipLaunchKernelGGL((adapters_up_kernel<DT, BASE>), grid, dim3(256), 0, st, base, ad, t, out, M, N, m0);
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
