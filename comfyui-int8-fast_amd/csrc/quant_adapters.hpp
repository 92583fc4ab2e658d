// The first product of low-rank adapters that differ from row to row, t = scale_a A_a x, of all layers that read x, and the quantiser of
// x beside it (included by quant_rowwise.hip; include/i8f_blocks.h has the interface).
#include "adapters.hpp"

namespace i8f {
namespace {

// The adapters of up to four layers, of one ids and rows_per_id
struct DownLayers {
    i8f_adapters ad[I8F_MAX_ADAPTED_LAYERS];
    char *t[I8F_MAX_ADAPTED_LAYERS];
    int first_block[I8F_MAX_ADAPTED_LAYERS + 1];   // (rows form: first workgroup of each layer behind the quantiser's; [n] = all)
    int n;
};

// ---- any width and alignment: one wave to a rank of a row --------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void adapters_down_kernel(const char *__restrict__ x, int64_t K, int64_t ldx, const DownLayers g) {
    const int64_t m = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int l = 0; l < g.n; ++l) {
        const i8f_adapters &ad = g.ad[l];
        const int a = adapter_of(ad, m);
        if (a < 0) continue;
        const int first = ad.first_rank[a], r = ad.first_rank[a + 1] - first;
        const float s = ad.scale[a];
        for (int j = wave; j < r; j += 4) {
            float sum = 0.0f;
            for (int64_t k = lane; k < K; k += 64) sum = __builtin_fmaf(load_as_f32<DT>(x, m * ldx + k), load_as_f32<DT>(ad.down, (first + j) * K + k), sum);
            sum = wave_sum_all(sum);
            if (lane == 0) store_from_f32<DT>(g.t[l], m * ad.max_rank + j, sum * s);
        }
    }
}

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

// ---- few rows (K % 8 == 0, aligned): every rank of every row is a wave of its own, with 16-byte loads, eight of each operand under way at
// once; what counts is the one trip to memory.  The first quant_blocks workgroups quantise a row of x each (RUNS > 0).
template <int DT, bool ROT, int RUNS>
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
    const uint32_t quads = (uint32_t)ad.max_rank / 4, at = (uint32_t)(block - g.first_block[l]);   // a workgroup takes four ranks of a row
    const int64_t m = at / quads;
    const int lane = threadIdx.x & 63, j = (int)(at % quads) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int a = __builtin_amdgcn_readfirstlane(adapter_of(ad, m));
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
    if (lane == 0) store_from_f32<DT>(g.t[l], m * ad.max_rank + j, sum * ad.scale[a]);
}

// ---- many rows: 16 G of them to a workgroup, the matrix unit multiplies 16 rows by 16 ranks, RT such tiles of ranks at a time.  Eight waves
// share the columns: wave w takes blocks w, w + 8, ... of 64 columns.  Eight neighbouring lanes load the 128 bytes of a row, of x and
// of A alike, and the tiles change to the matrix unit's layout in LDS of the wave's own; RING blocks are under way.
// Every workgroup reads the whole factors, so what bounds it is what the CUs draw from L2: more rows to a workgroup where there are enough.
// An adapter that occurs among the rows is a pass over the columns for all of them, with its ranks in all layers; its products are stored
// for its own rows (a row of t depends on its own row of x alone).
template <int DT, int G, int RT, int RING>
__global__ __launch_bounds__(512) void adapters_tiles_kernel(const char *__restrict__ x, int M, int K, int64_t ldx, const DownLayers g) {
    __shared__ union {
        v4u tile[8][G + RT][128];  // [wave][x..., A...][row * 8 + (16-byte chunk ^ row & 7)]
        v4f sum[8][G * RT][64];
    } sh;
    const int tid = threadIdx.x, lane = tid & 63, r = lane >> 3, c = lane & 7, fr = lane & 15, fg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row0 = blockIdx.x * (16 * G), blocks = (K + 63) / 64;
    int64_t most = 0;
    for (int l = 0; l < g.n; ++l) most = g.ad[l].count > most ? g.ad[l].count : most;
    int id[G];
    uint64_t left[G];
#pragma unroll
    for (int i = 0; i < G; ++i) {
        const int m = row0 + 16 * i + fr;
        const int a = g.ad[0].ids[(uint32_t)min(m, M - 1) / (uint32_t)g.ad[0].rows_per_id];
        id[i] = m < M && (uint32_t)a < (uint32_t)most ? a : -1;
        left[i] = __builtin_amdgcn_ballot_w64(id[i] >= 0);
    }
    // (a lane's offsets from addresses that are the workgroup's: rows past the last one repeat it)
    const char *xbase = x + (int64_t)row0 * ldx * 2;
    uint32_t xo[2 * G];
#pragma unroll
    for (int i = 0; i < 2 * G; ++i) xo[i] = (uint32_t)min(8 * i + r, M - 1 - row0) * (uint32_t)(ldx * 2) + c * 16;
    const uint32_t ao = (uint32_t)r * (uint32_t)(K * 2) + c * 16;
    v4u(*tile)[128] = sh.tile[wave];
    const int put = r * 8 + (c ^ r);
    const uint32_t eight = 16u * (uint32_t)K;  // bytes of eight rows of A
    while (true) {
        int a = -1;
#pragma unroll
        for (int i = G - 1; i >= 0; --i)
            if (left[i]) a = __builtin_amdgcn_readlane(id[i], __builtin_ctzll(left[i]));
        if (a < 0) break;
#pragma unroll
        for (int i = 0; i < G; ++i) left[i] &= ~__builtin_amdgcn_ballot_w64(id[i] == a);
        // its tiles of 16 ranks, layer after layer
        int first[I8F_MAX_ADAPTED_LAYERS], until[I8F_MAX_ADAPTED_LAYERS], all = 0;
#pragma unroll
        for (int l = 0; l < I8F_MAX_ADAPTED_LAYERS; ++l) {
            first[l] = 0;
            if (l < g.n && a < g.ad[l].count) {
                first[l] = __builtin_amdgcn_readfirstlane(g.ad[l].first_rank[a]);
                all += (__builtin_amdgcn_readfirstlane(g.ad[l].first_rank[a + 1]) - first[l]) / 16;
            }
            until[l] = all;
        }
        for (int t0 = 0; t0 < all; t0 += RT) {
            // (the last tiles of a pass may be none: they repeat the last one and are not stored)
            const char *ap[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int n = min(t0 + i, all - 1);
                int l = 0, before = 0, at = first[0];
#pragma unroll
                for (int k = 0; k + 1 < I8F_MAX_ADAPTED_LAYERS; ++k)
                    if (n >= until[k]) l = k + 1, before = until[k], at = first[k + 1];
                ap[i] = (const char *)g.ad[l].down + (int64_t)(at + (n - before) * 16) * K * 2;
            }
            v4f acc[G][RT];
#pragma unroll
            for (int i = 0; i < G; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j) acc[i][j] = (v4f)0.0f;
            v4u xv[RING][2 * G], av[RING][RT][2];
            auto fetch = [&](int b, int s) __attribute__((always_inline)) {
                const bool in = b < blocks && b * 64 + c * 8 < K;   // (K % 8 == 0; what is not there is the row's first piece, unused)
                const uint32_t off = in ? (uint32_t)b * 128u : 0u - c * 16u;
#pragma unroll
                for (int i = 0; i < 2 * G; ++i) xv[s][i] = *(const v4u *)(xbase + (xo[i] + off));
#pragma unroll
                for (int i = 0; i < RT; ++i) av[s][i][0] = *(const v4u *)(ap[i] + (ao + off)), av[s][i][1] = *(const v4u *)(ap[i] + (ao + eight + off));
            };
#pragma unroll
            for (int s = 0; s < RING; ++s) fetch(wave + 8 * s, s);
            for (int b0 = wave; b0 < blocks; b0 += 8 * RING) {
#pragma unroll
                for (int s = 0; s < RING; ++s) {
                    const int b = b0 + 8 * s;
                    const bool in = b < blocks && b * 64 + c * 8 < K;
                    const v4u zero = (v4u)0u;
#pragma unroll
                    for (int i = 0; i < G; ++i) tile[i][put] = in ? xv[s][2 * i] : zero, tile[i][put + 64] = in ? xv[s][2 * i + 1] : zero;
#pragma unroll
                    for (int i = 0; i < RT; ++i) tile[G + i][put] = in ? av[s][i][0] : zero, tile[G + i][put + 64] = in ? av[s][i][1] : zero;
                    fetch(b + 8 * RING, s);
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int get = fr * 8 + ((4 * h + fg) ^ (fr & 7));
                        v4u xf[G];
#pragma unroll
                        for (int i = 0; i < G; ++i) xf[i] = tile[i][get];
#pragma unroll
                        for (int j = 0; j < RT; ++j) {
                            const v4u af = tile[G + j][get];
#pragma unroll
                            for (int i = 0; i < G; ++i) acc[i][j] = lora_mfma<DT>(af, xf[i], acc[i][j]);
                        }
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                }
            }
            __syncthreads();   // (the tiles are done with)
#pragma unroll
            for (int i = 0; i < G; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j) sh.sum[wave][i * RT + j][lane] = acc[i][j];
            __syncthreads();
            // the waves' sums, in wave order: four ranks of the lane's row of a group, a tile of a group to a wave
#pragma unroll
            for (int i = 0; i < G; ++i) {
                for (int j = (wave - i * RT % 8 + 8) % 8; j < RT; j += 8) {
                    if (t0 + j >= all || id[i] != a) continue;
                    v4f sum = sh.sum[0][i * RT + j][lane];
#pragma unroll
                    for (int w = 1; w < 8; ++w) sum += sh.sum[w][i * RT + j][lane];
                    const int n = t0 + j;
                    int l = 0, before = 0;
#pragma unroll
                    for (int k = 0; k + 1 < I8F_MAX_ADAPTED_LAYERS; ++k)
                        if (n >= until[k]) l = k + 1, before = until[k];
                    const float s = g.ad[l].scale[a];
                    uint2 o;
                    if constexpr (DT == I8F_BF16) o = make_uint2(f32x2_to_bf16x2_bits(sum.x * s, sum.y * s), f32x2_to_bf16x2_bits(sum.z * s, sum.w * s));
                    else o = make_uint2(f32x2_to_f16x2_bits(sum.x * s, sum.y * s), f32x2_to_f16x2_bits(sum.z * s, sum.w * s));
                    *(uint2 *)(g.t[l] + ((int64_t)(row0 + 16 * i + fr) * g.ad[l].max_rank + (n - before) * 16 + 4 * fg) * 2) = o;
                }
            }
            __syncthreads();   // (the sums are read before the next tiles)
        }
    }
}

constexpr int64_t DOWN_ROWS = 256;   // rows up to which a rank of a row is a wave of its own

template <int DT, bool ROT, int RUNS>
int launch_rows_form(const void *x, int64_t M, int64_t K, int64_t ldx, int8_t *q, float *scale, DownLayers &g, hipStream_t st) {
    const int64_t quant_blocks = RUNS > 0 ? M : 0;
    int64_t first = 0;
    for (int i = 0; i < g.n; ++i) g.first_block[i] = (int)first, first += M * (g.ad[i].max_rank / 4);
    for (int i = g.n; i <= I8F_MAX_ADAPTED_LAYERS; ++i) g.first_block[i] = (int)first;
    if (quant_blocks + first == 0) return I8F_OK;
    hipLaunchKernelGGL((adapters_rows_kernel<DT, ROT, RUNS>), dim3((unsigned)(quant_blocks + first)), dim3(256), 0, st, (const char *)x, M, (int)K, ldx, q, scale,
                       (int)quant_blocks, g);
    return check_launch();
}

template <int DT>
int launch_down(const void *x, int64_t M, int64_t K, int64_t ldx, DownLayers &g, int rotate_block, int8_t *q, float *scale, hipStream_t st) {
    const bool vectors = K % 8 == 0 && (uintptr_t)x % 16 == 0 && ldx % 8 == 0 && K > 0 && ldx < (1ll << 24);   // (32-bit offsets within 64 rows)
    int64_t ranks = 0;
    for (int i = 0; i < g.n; ++i) ranks += g.ad[i].max_rank;
    if (vectors && M <= DOWN_ROWS && M * ranks < (1ll << 30)) {
        if (q && K % 16 == 0 && K <= 16384 && (uintptr_t)q % 16 == 0) {   // the quantiser in the same launch
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
        if (q)
            if (int rc = i8f_quant_rowwise(x, DT, M, K, ldx, rotate_block, q, scale, st)) return rc;
        return launch_rows_form<DT, false, 0>(x, M, K, ldx, q, scale, g, st);
    }
    if (q)
        if (int rc = i8f_quant_rowwise(x, DT, M, K, ldx, rotate_block, q, scale, st)) return rc;
    if (ranks == 0) return I8F_OK;
    if (vectors) {
        auto go = [&](auto kernel, int rows) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((M + rows - 1) / rows)), dim3(512), 0, st, (const char *)x, (int)M, (int)K, ldx, g);
            return check_launch();
        };
        if (M >= 8192) return ranks <= 32 ? go(adapters_tiles_kernel<DT, 4, 2, 2>, 64) : go(adapters_tiles_kernel<DT, 4, 4, 1>, 64);
        if (M >= 2048) return ranks <= 32 ? go(adapters_tiles_kernel<DT, 2, 2, 3>, 32) : ranks <= 64 ? go(adapters_tiles_kernel<DT, 2, 4, 2>, 32) : go(adapters_tiles_kernel<DT, 2, 6, 2>, 32);
        return ranks <= 32 ? go(adapters_tiles_kernel<DT, 1, 2, 4>, 16) : go(adapters_tiles_kernel<DT, 1, 4, 3>, 16);
    }
    hipLaunchKernelGGL((adapters_down_kernel<DT>), dim3((unsigned)M), dim3(256), 0, st, (const char *)x, K, ldx, g);
    return check_launch();
}

}  // namespace
}  // namespace i8f

extern "C" int i8f_adapters_down(const void *x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const i8f_adapted_layer *layers, int n_layers,
                                 int rotate_block, int8_t *q, float *scale, void *stream) {
    using namespace i8f;
    if (K < 0 || (q != nullptr) != (scale != nullptr)) return I8F_ERR_INVALID;
    if (rotate_block != 0 && rotate_block != 128) return I8F_ERR_UNSUPPORTED;
    if (rotate_block && K % 128) return I8F_ERR_INVALID;
    if (x_dtype != I8F_BF16 && x_dtype != I8F_F16) return I8F_ERR_INVALID;
    if (int rc = validate_layers(layers, n_layers, x_dtype, M)) return rc;
    if (M == 0) return I8F_OK;
    if (ldx < K || (K > 0 && !x)) return I8F_ERR_INVALID;
    if (M > 0x7fffffff || K > 0x7fffffff) return I8F_ERR_UNSUPPORTED;
    if (int rc = check_device()) return rc;
    DownLayers g{};
    for (int i = 0; i < n_layers; ++i)
        if (layers[i].adapters.count > 0 && layers[i].adapters.max_rank > 0) g.ad[g.n] = for_kernel(layers[i].adapters), g.t[g.n++] = (char *)layers[i].t;
    return x_dtype == I8F_BF16 ? launch_down<I8F_BF16>(x, M, K, ldx, g, rotate_block, q, scale, (hipStream_t)stream)
                               : launch_down<I8F_F16>(x, M, K, ldx, g, rotate_block, q, scale, (hipStream_t)stream);
}
