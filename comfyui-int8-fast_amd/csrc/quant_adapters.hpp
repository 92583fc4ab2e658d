// The first product of low-rank adapters that differ from row to row, t = scale_a A_a x, of all layers that read x, and the quantiser of
// x beside it (included by quant_rowwise.hip; include/i8f_blocks.h has the interface).
#include "adapters.hpp"

namespace i8f {
namespace {

template <int DT>
__device__ __forceinline__ float dot8(v4u a, v4u b, float sum) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (DT == I8F_BF16) {
            sum = __builtin_fmaf(__uint_as_float(a[e] << 16), __uint_as_float(b[e] << 16), sum);
            sum = __builtin_fmaf(__uint_as_float(a[e] & 0xffff0000u), __uint_as_float(b[e] & 0xffff0000u), sum);
        } else {
            sum = __builtin_fmaf(f16_bits_to_f32(a[e] & 0xffffu), f16_bits_to_f32(b[e] & 0xffffu), sum);
            sum = __builtin_fmaf(f16_bits_to_f32(a[e] >> 16), f16_bits_to_f32(b[e] >> 16), sum);
        }
    }
    return sum;
}

// ---- few rows: every rank of every row (or two of them) is a wave of its own, with 16-byte loads, eight of each operand under way at once; what counts is
// the one trip to memory.  The first quant_blocks workgroups quantise a row of x each (RUNS > 0).
// ANY: x of any width and alignment (a row's last eight elements, where it has fewer of them, are fetched one by one; the factors' rows
// are padded).
template <int DT, bool ROT, int RUNS, bool ANY, int PER>
__global__ __launch_bounds__(256) void adapters_rows_kernel(const char *__restrict__ x, int64_t M, int K, int64_t ldx, int8_t *__restrict__ q,
                                                            float *__restrict__ scale, int quant_blocks, const DownLayers g) {
    if constexpr (RUNS > 0) {
        if ((int)blockIdx.x < quant_blocks) {
            const Prologue none{};
            quant16_body<DT, ROT, 4, RUNS, false, I8F_PRO_NONE, 1>(x, M, K, ldx * 2, q, scale, none, (int64_t)blockIdx.x);
            return;
        }
    }
    const int block = (int)blockIdx.x - quant_blocks;
    int l = 0;
#pragma unroll
    for (int i = 1; i < I8F_MAX_ADAPTED_LAYERS; ++i)
        if (i < g.n && block >= g.first_block[i]) l = i;
    l = __builtin_amdgcn_readfirstlane(l);
    const i8f_adapters &ad = g.ad[l];
    const uint32_t groups = (uint32_t)ad.max_rank / (4 * PER), at = (uint32_t)(block - g.first_block[l]);   // a workgroup takes 4 PER ranks of a row
    const int64_t m = at / groups;
    const int lane = threadIdx.x & 63, j = ((int)(at % groups) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * PER;
    const int a = __builtin_amdgcn_readfirstlane(adapter_of(ad, m));
    if (a < 0) return;
    const int first = ad.first_rank[a];
    if (j >= ad.first_rank[a + 1] - first) return;
    const char *xp = x + m * ldx * 2, *ap = (const char *)ad.down + (int64_t)(first + j) * factor_width(K) * 2;
    float sum[PER] = {};
    for (int k0 = lane * 8; k0 < K; k0 += 8 * 512) {
        v4u xv[8], av[PER][8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int k = k0 + c * 512;
            if constexpr (ANY) {
                xv[c] = (v4u)0u;
                if (k + 8 <= K) __builtin_memcpy(&xv[c], xp + (int64_t)k * 2, 16);
            } else {
                xv[c] = k < K ? *(const v4u *)(xp + (int64_t)k * 2) : (v4u)0u;
            }
#pragma unroll
            for (int i = 0; i < PER; ++i) av[i][c] = k < K ? *(const v4u *)(ap + (i * factor_width(K) + k) * 2) : (v4u)0u;
        }
        if constexpr (ANY) {
            const int c = (K - k0) / 512, k = k0 + c * 512;   // the piece that holds the row's end, if it is this lane's
            if (K % 8 && c < 8 && K - k < 8) {
                v4u end = (v4u)0u;
                for (int e = 0; e < K - k; ++e) end[e / 2] |= (uint32_t)((const uint16_t *)xp)[k + e] << (16 * (e % 2));
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i == c) xv[i] = end;
            }
        }
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int i = 0; i < PER; ++i) sum[i] = dot8<DT>(xv[c], av[i][c], sum[i]);
    }
    const float s = ad.scale[a];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        sum[i] = wave_sum_all(sum[i]);
        if (lane == 0) store_from_f32<DT>(g.t[l], m * ad.max_rank + j + i, sum[i] * s);
    }
}

// ---- many rows, the sums of the slices of K (adapters_down.hip): t = scale_a (the slices' sums, in order), rounded: four ranks of a row to a thread
template <int DT>
__device__ __forceinline__ void adapters_combine(const float *__restrict__ partial, int64_t M, int slices, int64_t block, const DownLayers &g) {
    const uint32_t columns = (uint32_t)g.first_column[g.n], quads = columns / 4;
    const int64_t at = block * 256 + threadIdx.x;
    const int64_t m = at / quads;
    if (m >= M) return;
    const int col = (int)(at % quads) * 4;
    int l = 0;
#pragma unroll
    for (int k = 1; k < I8F_MAX_ADAPTED_LAYERS; ++k)
        if (k < g.n && col >= g.first_column[k]) l = k;
    const int a = adapter_of(g.ad[l], m), j = col - g.first_column[l];
    if (a < 0 || j >= g.ad[l].first_rank[a + 1] - g.ad[l].first_rank[a]) return;
    const float *p = partial + m * columns + col;
    v4f sum = *(const v4f *)p;
    for (int z = 1; z < slices; ++z) sum += *(const v4f *)(p + z * M * columns);
    const float s = g.ad[l].scale[a];
    uint2 o;
    if constexpr (DT == I8F_BF16) o = make_uint2(f32x2_to_bf16x2_bits(sum.x * s, sum.y * s), f32x2_to_bf16x2_bits(sum.z * s, sum.w * s));
    else o = make_uint2(f32x2_to_f16x2_bits(sum.x * s, sum.y * s), f32x2_to_f16x2_bits(sum.z * s, sum.w * s));
    *(uint2 *)(g.t[l] + (m * g.ad[l].max_rank + j) * 2) = o;
}
// and the quantiser of x beside it, by the workgroups behind (RUNS > 0, WPR waves to a row): alone the sums take 5 us, most of them the way
// into and out of a kernel.
template <int DT, bool ROT, int WPR, int RUNS>
__global__ __launch_bounds__(256) void adapters_combine_kernel(const float *__restrict__ partial, int64_t M, int slices, int combine_blocks,
                                                               const char *__restrict__ x, int64_t K, int64_t ldx, int8_t *__restrict__ q,
                                                               float *__restrict__ scale, const DownLayers g) {
    if constexpr (RUNS > 0) {
        if ((int)blockIdx.x >= combine_blocks) {
            const Prologue none{};
            quant16_body<DT, ROT, WPR, RUNS, false, I8F_PRO_NONE, 1>(x, M, K, ldx * 2, q, scale, none, (int64_t)((int)blockIdx.x - combine_blocks) * (4 / WPR));
            return;
        }
    }
    adapters_combine<DT>(partial, M, slices, blockIdx.x, g);
}

template <int DT, bool ROT, int WPR, int RUNS>
int launch_combine(const float *partial, int64_t M, int slices, const void *x, int64_t K, int64_t ldx, int8_t *q, float *scale, const DownLayers &g, hipStream_t st) {
    const int64_t combine = (M * (g.first_column[g.n] / 4) + 255) / 256, quant = RUNS > 0 ? (M + 4 / WPR - 1) / (4 / WPR) : 0;
    if (!grid_fits(combine + quant, 256)) return I8F_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((adapters_combine_kernel<DT, ROT, WPR, RUNS>), dim3((unsigned)(combine + quant)), dim3(256), 0, st, partial, M, slices, (int)combine, (const char *)x,
                       K, ldx, q, scale, g);
    return check_launch();
}
template <int DT, bool ROT>
int pick_combine(const float *partial, int64_t M, int slices, const void *x, int64_t K, int64_t ldx, int8_t *q, float *scale, const DownLayers &g, hipStream_t st) {
    const auto go = [&](auto WPR, auto RUNS) { return launch_combine<DT, ROT, decltype(WPR)::value, decltype(RUNS)::value>(partial, M, slices, x, K, ldx, q, scale, g, st); };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, 3> three;
    const std::integral_constant<int, 4> four;
    if (!q) return go(one, std::integral_constant<int, 0>{});
    switch ((K / 16 + 63) / 64) {   // (a wave holds 64 runs of 16 values at a time; the most four times, then the row goes to four waves)
    case 1: return go(one, one);
    case 2: return go(one, two);
    case 3: return go(one, three);
    case 4: return go(one, four);
    case 5: case 6: case 7: case 8: return go(four, two);
    case 9: case 10: case 11: case 12: return go(four, three);
    default: return go(four, four);
    }
}

// Where a rank of a row is a wave of its own: few rows, whatever adapters they have, or few of those waves; x and a factor's row are fetched
// again for each, so that beyond it rows share the factors (adapters_down.hip), which costs a pass for every adapter that occurs among 64
// rows.  K = 4096 with the quantiser, us, rows of one adapter, of eight requests and of 32 in turn:
//     rows x ranks   128 x 16   4.3   4.3   4.3 by waves,  11   16   60 by tiles       512 x 16    7.7   7.8   7.8 and  12   12   61
//                    128 x 128 11.5  11.4  14.1            14   27  147               1024 x 16   12    13    12        12   12   62
//                    256 x 128  20    20    24             15   19  146                512 x 128  42    41    46        17   17   61
// (the tiles' figures but the last ones are of passes that one workgroup took; dealt over idle ones they cost about half where they are many)
inline bool down_by_rows(int64_t M, int64_t K, int64_t ranks) {
    return M <= 128 || (M <= 256 && M * ranks <= 1 << 15) || (M < (1 << 14) && M * ranks <= 1 << 14) || K >= (1 << 23);   // (32-bit offsets within 64 rows)
}

template <int DT, bool ROT, int RUNS, bool ANY, int PER>
int launch_rows_of(const void *x, int64_t M, int64_t K, int64_t ldx, int8_t *q, float *scale, DownLayers &g, hipStream_t st) {
    const int64_t quant_blocks = RUNS > 0 ? M : 0;
    int64_t first = 0;
    for (int i = 0; i < g.n; ++i) g.first_block[i] = (int)first, first += M * (g.ad[i].max_rank / (4 * PER));
    for (int i = g.n; i <= I8F_MAX_ADAPTED_LAYERS; ++i) g.first_block[i] = (int)first;
    if (quant_blocks + first == 0) return I8F_OK;
    if (!grid_fits(quant_blocks + first, 256)) return I8F_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((adapters_rows_kernel<DT, ROT, RUNS, ANY, PER>), dim3((unsigned)(quant_blocks + first)), dim3(256), 0, st, (const char *)x, M, (int)K, ldx, q, scale,
                       (int)quant_blocks, g);
    return check_launch();
}

template <int DT, bool ROT, int RUNS, bool ANY = false>
int launch_rows_form(const void *x, int64_t M, int64_t K, int64_t ldx, int8_t *q, float *scale, DownLayers &g, hipStream_t st) {
    // two ranks to a wave, which share the row of x, where there are waves enough: K = 4096, 128 x 128 12.6 and 11.5 us, 1024 x 16 14.2 and 12.0;
    // 128 x 16 4.3 and 4.7
    return M * g.first_column[g.n] >= 1 << 14 ? launch_rows_of<DT, ROT, RUNS, ANY, 2>(x, M, K, ldx, q, scale, g, st)
                                           : launch_rows_of<DT, ROT, RUNS, ANY, 1>(x, M, K, ldx, q, scale, g, st);
}

// ---- few rows with a side each: then their share of the result, B_a t, by a launch of its own that fills the chip, where the tiles of the
// projection are too few to fetch as many different factors as there are rows.  A wave takes 256 columns of a row: the matrix unit's 16 x 16
// x 32 form reads 16 rows of the factor in whole pieces, t stands in all columns of its other operand, and lane column b keeps block b's
// result, so that a store is 1 KB in one piece.  64 rows x 6144 columns, ranks of 8 to 64: 12 us, 4 of them the factors' bytes, the rest the way
// to a row's number, its factor and back.
template <int DT>
__global__ __launch_bounds__(256) void adapters_side_kernel(const DownLayers g) {
    int l = 0;
#pragma unroll
    for (int i = 1; i < I8F_MAX_ADAPTED_LAYERS; ++i)
        if (i < g.n && (int)blockIdx.x >= g.first_block[i]) l = i;
    l = __builtin_amdgcn_readfirstlane(l);
    const i8f_adapters &ad = g.ad[l];
    const int64_t N = g.N[l];
    const uint32_t at = blockIdx.x - g.first_block[l], pieces = (uint32_t)((N + 1023) / 1024);
    const int64_t m = at / pieces;
    const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
    const int64_t n0 = (int64_t)(at % pieces) * 1024 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 256;
    if (n0 >= N) return;
    const int a = __builtin_amdgcn_readfirstlane(adapter_of(ad, m));
    const int first = a < 0 ? 0 : ad.first_rank[a], rank = a < 0 ? 0 : ad.first_rank[a + 1] - first;
    const char *t = g.t[l] + m * ad.max_rank * 2, *up = (const char *)ad.up + N * first * 2;
    v4f keep = (v4f)0.0f;
    for (int k = 8 * lq; k - 8 * lq < rank; k += 32) {
        const bool in = k < rank;   // (ranks come in sixteens: the last step may be half a one)
        const v4u tv = in ? *(const v4u *)(t + k * 2) : (v4u)0u;
        v4u bv[16];
#pragma unroll
        for (int b = 0; b < 16; ++b) {
            const int64_t row = n0 + 16 * b + l16 < N ? n0 + 16 * b + l16 : N - 1;
            bv[b] = in ? *(const v4u *)(up + (row * rank + k) * 2) : (v4u)0u;
        }
#pragma unroll
        for (int b = 0; b < 16; ++b) {
            const v4f d = factor_mfma<DT>(bv[b], tv, (v4f)0.0f);
#pragma unroll
            for (int e = 0; e < 4; ++e) keep[e] = l16 == b ? keep[e] + d[e] : keep[e];
        }
    }
    const int64_t n = n0 + 16 * l16 + 4 * lq;   // the four columns that the lane kept (N comes in eights)
    if (n < N) *(v4f *)(g.side[l] + m * N + n) = keep;
}

template <int DT>
int launch_side(int64_t M, DownLayers &g, hipStream_t st) {
    int64_t first = 0;
    for (int i = 0; i < g.n; ++i) g.first_block[i] = (int)first, first += M * ((g.N[i] + 1023) / 1024);
    for (int i = g.n; i <= I8F_MAX_ADAPTED_LAYERS; ++i) g.first_block[i] = (int)first;
    if (first == 0) return I8F_OK;
    hipLaunchKernelGGL((adapters_side_kernel<DT>), dim3((unsigned)first), dim3(256), 0, st, g);
    return check_launch();
}

inline bool side_in_place(int64_t M, int64_t N) { return N % 8 == 0 && M * ((N + 1023) / 1024) < (1ll << 22); }   // (four layers in a grid)
inline bool down_in_place(const void *x, int64_t K, int64_t ldx) { return K % 8 == 0 && (uintptr_t)x % 16 == 0 && ldx % 8 == 0 && ldx < (1ll << 23); }

template <int DT>
int launch_first(const void *x, int64_t M, int64_t K, int64_t ldx, DownLayers &g, int rotate_block, int8_t *q, float *scale, void *workspace,
                int64_t workspace_bytes, hipStream_t st) {
    const int64_t ranks = g.first_column[g.n];
    const bool in_place = down_in_place(x, K, ldx), by_rows = down_by_rows(M, K, ranks);
    if (by_rows && in_place && q && K % 16 == 0 && K <= 16384 && (uintptr_t)q % 16 == 0) {   // the quantiser in the same launch
        const int64_t runs = (K / 16 + 255) / 256;
        auto go = [&](auto ROT) {
            switch (runs) {
            case 1: return launch_rows_form<DT, decltype(ROT)::value, 1>(x, M, K, ldx, q, scale, g, st);
            case 2: return launch_rows_form<DT, decltype(ROT)::value, 2>(x, M, K, ldx, q, scale, g, st);
            case 3: return launch_rows_form<DT, decltype(ROT)::value, 3>(x, M, K, ldx, q, scale, g, st);
            default: return launch_rows_form<DT, decltype(ROT)::value, 4>(x, M, K, ldx, q, scale, g, st);
            }
        };
        return rotate_block ? go(std::true_type{}) : go(std::false_type{});
    }
    const int64_t copy = in_place ? 0 : adapters_copy_bytes(M, K);
    int slices = adapters_down_slices(M, K);
    if (!workspace || workspace_bytes < copy + slices * M * ranks * 4) slices = 1;
    const bool beside = in_place && !by_rows && ranks > 0 && slices > 1 && K % 16 == 0 && K <= 16384 && (uintptr_t)q % 16 == 0;   // the quantiser goes along with the sums
    if (q && !beside)
        if (int rc = i8f_quant_rowwise(x, DT, M, K, ldx, rotate_block, q, scale, st)) return rc;
    if (ranks == 0) return I8F_OK;
    if (by_rows)
        return in_place ? launch_rows_form<DT, false, 0>(x, M, K, ldx, q, scale, g, st) : launch_rows_form<DT, false, 0, true>(x, M, K, ldx, q, scale, g, st);
    // rows that the direct loads do not take are copied first, padded like the factors
    if (copy) {
        if (!workspace || workspace_bytes < copy) return launch_rows_form<DT, false, 0, true>(x, M, K, ldx, q, scale, g, st);
        if (int rc = adapters_copy_rows(x, M, K, ldx, workspace, st)) return rc;
        x = workspace, K = ldx = factor_width(K);
    }
    const float *partial = (const float *)((char *)workspace + copy);
    if (int rc = adapters_down_partial(x, DT, M, K, ldx, g, (float *)partial, slices, st)) return rc;
    if (slices == 1) return I8F_OK;
    if (!beside) q = nullptr;
    return rotate_block ? pick_combine<DT, true>(partial, M, slices, x, K, ldx, q, scale, g, st) : pick_combine<DT, false>(partial, M, slices, x, K, ldx, q, scale, g, st);
}

template <int DT>
int launch_down(const void *x, int64_t M, int64_t K, int64_t ldx, DownLayers &g, int rotate_block, int8_t *q, float *scale, void *workspace,
                int64_t workspace_bytes, hipStream_t st) {
    const int rc = launch_first<DT>(x, M, K, ldx, g, rotate_block, q, scale, workspace, workspace_bytes, st);
    return rc || !g.n || !g.side[0] ? rc : launch_side<DT>(M, g, st);
}

}  // namespace
}  // namespace i8f

extern "C" int i8f_adapters_down(const void *x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const i8f_adapted_layer *layers, int n_layers,
                                 int rotate_block, int8_t *q, float *scale, void *workspace, int64_t workspace_bytes, void *stream) {
    using namespace i8f;
    if (workspace && (uintptr_t)workspace % 16) return I8F_ERR_INVALID;
    if (K < 0 || (q != nullptr) != (scale != nullptr)) return I8F_ERR_INVALID;
    if (rotate_block != 0 && rotate_block != 128) return I8F_ERR_UNSUPPORTED;
    if (rotate_block && K % 128) return I8F_ERR_INVALID;
    if (x_dtype != I8F_BF16 && x_dtype != I8F_F16) return I8F_ERR_INVALID;
    if (int rc = validate_layers(layers, n_layers, x_dtype, M)) return rc;
    if (M == 0) return I8F_OK;
    if (ldx < K || (K > 0 && !x)) return I8F_ERR_INVALID;
    if (M > 0x7fffffff || K > (1 << 30)) return I8F_ERR_UNSUPPORTED;   // (a lane's column is 32 bits, and goes a few steps past the row)
    if (int rc = check_device()) return rc;
    DownLayers g{};
    for (int i = 0; i < n_layers; ++i)
        if (layers[i].side || (layers[i].adapters.count > 0 && layers[i].adapters.max_rank > 0)) {
            if (layers[i].side && !side_in_place(M, layers[i].N)) return I8F_ERR_UNSUPPORTED;
            g.ad[g.n] = for_kernel(layers[i].adapters), g.t[g.n] = (char *)layers[i].t, g.side[g.n] = layers[i].side, g.N[g.n] = layers[i].N;
            if (layers[i].adapters.max_rank == 0) g.ad[g.n].count = 0;
            g.first_column[g.n + 1] = g.first_column[g.n] + (int)layers[i].adapters.max_rank;   // (four of up to 65536)
            ++g.n;
        }
    return x_dtype == I8F_BF16 ? launch_down<I8F_BF16>(x, M, K, ldx, g, rotate_block, q, scale, workspace, workspace_bytes, (hipStream_t)stream)
                               : launch_down<I8F_F16>(x, M, K, ldx, g, rotate_block, q, scale, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int64_t i8f_adapters_down_workspace_bytes(int64_t M, int64_t K, int64_t ranks, int x_aligned) {
    using namespace i8f;
    if (M <= 0 || K <= 0 || ranks <= 0 || M > 0x7fffffff || K > (1 << 30) || down_by_rows(M, K, ranks)) return 0;
    const int slices = adapters_down_slices(M, K);
    return (x_aligned && K % 8 == 0 ? 0 : adapters_copy_bytes(M, K)) + (slices < 2 ? 0 : slices * M * ranks * 4);
}

extern "C" int i8f_adapters_by_side(int64_t M, int64_t N, int64_t K, int64_t rows_per_id) {
    // Up to 16 rows are another kernel's, and widths that the tiled kernels do not take go by way of i8f_adapters_up.  64 tokens of as many
    // requests, 4096 -> 4096 + 1024 + 1024, ranks of 8 to 64: 33.5 us by side and 37.6 with the factors fetched by the 96 tiles; of one
    // request the tiles' way is the faster one (64 x 4096 -> 4096, rank 64: 3 us more than without adapters, and 10 by side).
    return rows_per_id > 0 && M / rows_per_id > 16 && M <= 128 && i8f::side_in_place(M, N) && i8f_linear_w8a8_adapters_workspace_bytes(M, N, K) == 0;
}
