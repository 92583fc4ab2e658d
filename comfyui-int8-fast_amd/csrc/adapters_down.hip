// The first product of low-rank adapters for many rows: t = scale_a A_a x of all layers that read x (include/i8f_blocks.h).
//
// A product of M rows by a few dozen to a few hundred ranks over a long K.  What bounds it is what the CUs draw from L2 (about 35 bytes a
// cycle each when all of them do): a workgroup reads its rows of x and the whole of the factors' slice, so 64 rows share the factors, and the
// columns are dealt over `slices` workgroups, whose sums meet in memory (adapters_combine, quant_adapters.hpp), until every CU has two.
// 64 rows and up to 128 ranks at a time: four waves of 16 rows by all the ranks, K-tiles of 64 columns (128 bytes of a row) in LDS, fetched
// by direct loads a few tiles ahead, with the 16-byte chunks of a row permuted by the row so that the 16 rows of a fragment are
// read from different banks.  One barrier per K-tile: behind it the tile has landed for everyone, and everyone is done with the tile
// whose stage the next loads go to.
// An adapter that occurs among the 64 rows is a pass over the slice for all of them, with its ranks in all layers; the products are stored
// for its own rows (a row of t depends on its own row of x alone).  The passes run into one another: 512 rows of 4096 columns with 64 adapters
// of rank 64 in every block 213 us with a drained pipeline between them and 174 now; seven requests in 1357 rows 10.0 and 9.1 us.
#include "adapters.hpp"
#include "dma.hpp"

namespace i8f {
namespace {

using gemm::dma16;
using gemm::make_rsrc;
using gemm::swz;
using gemm::v4i;
using gemm::waitcnt_vm;

typedef float v4f __attribute__((ext_vector_type(4)));

// column n of an adapter's tiles: its layer, and the tile within the layer
struct Tiles {
    int first[I8F_MAX_ADAPTED_LAYERS], until[I8F_MAX_ADAPTED_LAYERS], all;   // first rank of the adapter in each layer; tiles up to each layer
};
__device__ __forceinline__ int layer_of_tile(const Tiles &t, int n, int &within) {
    int l = 0, before = 0;
#pragma unroll
    for (int k = 0; k + 1 < I8F_MAX_ADAPTED_LAYERS; ++k)
        if (n >= t.until[k]) l = k + 1, before = t.until[k];
    within = n - before;
    return l;
}

// All loads of this wave but the YOUNGER last ones have landed and its LDS reads have returned, for every wave
template <int YOUNGER>
__device__ __forceinline__ void stage_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(YOUNGER) & 0xF0FF);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

constexpr int ROWS = 64, BK = 64;   // rows of a workgroup, columns of a K-tile

template <int DT, int RT, int STAGES>
__global__ __launch_bounds__(256) void adapters_partial_kernel(const char *__restrict__ x, int M, int K, int ldx_bytes, float *__restrict__ partial, int slices,
                                                               int per_slice, int parts, const DownLayers g) {
    constexpr int STAGE = (ROWS + 16 * RT) * 128, XL = 2, AL = RT / 2, LOADS = XL + AL;   // bytes of a stage; loads of a wave for a K-tile
    static_assert(RT % 2 == 0 && STAGE * STAGES <= 80 * 1024, "two workgroups to a CU");
    __shared__ __attribute__((aligned(1024))) char smem[STAGE * STAGES];
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // (the slices of a block of rows are neighbours in the launch; with eight of them an XCD has the same slice of the factors for all rows)
    const int slice = blockIdx.x % slices, part = blockIdx.x / slices % parts, block = blockIdx.x / slices / parts, m0 = block * ROWS;
    const int kt_first = slice * per_slice, KT = min(per_slice, (K + BK - 1) / BK - kt_first);
    const uint32_t OOB = 0x7ffffff0u, smem_base = (uint32_t)(uintptr_t)smem;
    int64_t most = 0;
    for (int l = 0; l < g.n; ++l) most = g.ad[l].count > most ? g.ad[l].count : most;
    int id = m0 + lane < M ? g.ad[0].ids[(uint32_t)(m0 + lane) / (uint32_t)g.ad[0].rows_per_id] : -1;   // of row m0 + lane
    id = (uint32_t)id < (uint32_t)most ? id : -1;
    const int mine = __shfl(id, 16 * wave + l16);   // of the row whose products this lane gets
    int first_of[I8F_MAX_ADAPTED_LAYERS], tiles_in[I8F_MAX_ADAPTED_LAYERS];   // of the adapter of row m0 + lane, in each layer
#pragma unroll
    for (int l = 0; l < I8F_MAX_ADAPTED_LAYERS; ++l) {
        first_of[l] = tiles_in[l] = 0;
        if (l < g.n && id >= 0 && id < g.ad[l].count) first_of[l] = g.ad[l].first_rank[id], tiles_in[l] = (g.ad[l].first_rank[id + 1] - first_of[l]) / 16;
    }
    uint64_t left = __builtin_amdgcn_ballot_w64(id >= 0);

    // load t of a wave: t < XL rows 8 (4 t + wave) ... of x, else half a tile of ranks; lane l takes 16-byte chunk (l % 8) ^ swz of row l / 8
    const int lr = lane >> 3, lc = lane & 7;
    const int rows = min(ROWS, M - m0);
    const v4i rx = make_rsrc(x + (int64_t)m0 * ldx_bytes, (uint32_t)(rows - 1) * (uint32_t)ldx_bytes + (uint32_t)K * 2u);
    uint32_t xo[XL], xc[XL], ac[AL], ao[AL];
#pragma unroll
    for (int t = 0; t < XL; ++t) {
        const int row = (4 * t + wave) * 8 + lr;
        xc[t] = (uint32_t)(lc ^ swz<8>(row)) * 16u;
        xo[t] = row < rows ? (uint32_t)row * (uint32_t)ldx_bytes + xc[t] : OOB;
    }
#pragma unroll
    for (int t = 0; t < AL; ++t) {
        const int row = ROWS + (4 * t + wave) * 8 + lr;
        ac[t] = (uint32_t)(lc ^ swz<8>(row)) * 16u;
        ao[t] = (uint32_t)((wave & 1) * 8 + lr) * (uint32_t)(K * 2) + ac[t];
    }
    // A pass takes RT tiles of ranks of an adapter through the slice.  The passes are one stream of K-tiles: while one ends, the loads of the
    // next are under way (its slice has to be as long as they reach ahead; the row's last one may be too short, and drains).
    struct Pass {
        int a, t0;
        Tiles tl;
        v4i ra[AL];   // (tiles past the adapter's last one are empty buffers: they load zeros)
    };
    Pass now, next;
    int number = parts - part;   // passes are dealt over the parts in turn: this workgroup takes the next one at `parts`
    auto advance = [&](Pass &p) __attribute__((always_inline)) {   // (a -1 behind the last)
        p.t0 += RT;
        while (p.t0 >= p.tl.all || number != parts) {
            if (p.t0 < p.tl.all) {   // another workgroup's
                p.t0 += RT, ++number;
                continue;
            }
            p.a = -1;
            if (!left) return;
            const int row = __builtin_ctzll(left);
            p.a = __builtin_amdgcn_readlane(id, row);
            left &= ~__builtin_amdgcn_ballot_w64(id == p.a);
            p.t0 = p.tl.all = 0;
#pragma unroll
            for (int l = 0; l < I8F_MAX_ADAPTED_LAYERS; ++l) {
                p.tl.first[l] = __builtin_amdgcn_readlane(first_of[l], row);
                p.tl.until[l] = p.tl.all += __builtin_amdgcn_readlane(tiles_in[l], row);
            }
        }
        number = 1;
#pragma unroll
        for (int t = 0; t < AL; ++t) {
            const int n = p.t0 + 2 * t + (wave >> 1);
            int within;
            const int l = layer_of_tile(p.tl, min(n, p.tl.all - 1), within);
            int first = p.tl.first[0];
#pragma unroll
            for (int k = 1; k < I8F_MAX_ADAPTED_LAYERS; ++k) first = l == k ? p.tl.first[k] : first;
            p.ra[t] = make_rsrc((const char *)g.ad[l].down + (int64_t)(first + within * 16) * K * 2, n < p.tl.all ? (uint32_t)K * 32u : 0u);
        }
    };
    int base = 0;   // the stage of the pass's first tile
    auto issue = [&](const Pass &p, int kt, int stage, bool live) __attribute__((always_inline)) {   // (not live: the loads move nothing, but are counted)
        const uint32_t st = smem_base + (uint32_t)(stage % STAGES) * STAGE + wave * 1024;
        const uint32_t kb = (uint32_t)(kt_first + kt) * (BK * 2);
#pragma unroll
        for (int t = 0; t < LOADS; ++t) {
            const bool is_x = t < XL;
            const uint32_t ck = is_x ? xc[t % XL] : ac[is_x ? 0 : t - XL], off = is_x ? xo[t % XL] : ao[is_x ? 0 : t - XL];
            v4i r = is_x ? rx : p.ra[is_x ? 0 : t - XL];
            r.z = live ? r.z : 0;
            dma16(r, st + t * 4096, kb + ck < (uint32_t)K * 2u && off != OOB ? off + kb : OOB, 0);
        }
    };
    auto fill = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) issue(now, s, base + s, s < KT);
    };
    const bool stream = KT >= STAGES - 1;
    now.t0 = 0, now.tl.all = 0;
    advance(now);
    if (now.a < 0) return;
    fill();
    while (true) {
        next = now;
        advance(next);
        v4f acc[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[j] = (v4f)0.0f;
        for (int kt = 0; kt < KT; ++kt) {
            stage_barrier<(STAGES - 2) * LOADS>();
            const int ahead = kt + STAGES - 1;
            if (ahead < KT || !stream) issue(now, ahead, base + ahead, ahead < KT);
            else issue(next, ahead - KT, base + ahead, next.a >= 0);
            const char *st = smem + (base + kt) % STAGES * STAGE;
            const int xrow = 16 * wave + l16;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v4i xf = *(const v4i *)(st + xrow * 128 + ((4 * h + lq) ^ swz<8>(xrow)) * 16);
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    const int arow = ROWS + 16 * j + l16;
                    acc[j] = factor_mfma<DT>(*(const v4i *)(st + arow * 128 + ((4 * h + lq) ^ swz<8>(arow)) * 16), xf, acc[j]);
                }
            }
        }
        base = (base + KT) % STAGES;
        if (mine == now.a) {   // (stores count with the loads that a barrier waits for: it waits for more of those then, not for fewer)
            const int m = m0 + 16 * wave + l16;
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                if (now.t0 + j >= now.tl.all) break;
                int within;
                const int l = layer_of_tile(now.tl, now.t0 + j, within);
                const int col = within * 16 + 4 * lq;
                if (slices > 1) {
                    *(v4f *)(partial + ((int64_t)slice * M + m) * g.first_column[g.n] + g.first_column[l] + col) = acc[j];
                } else {
                    const float s = g.ad[l].scale[now.a];
                    uint2 o;
                    if constexpr (DT == I8F_BF16) o = make_uint2(f32x2_to_bf16x2_bits(acc[j].x * s, acc[j].y * s), f32x2_to_bf16x2_bits(acc[j].z * s, acc[j].w * s));
                    else o = make_uint2(f32x2_to_f16x2_bits(acc[j].x * s, acc[j].y * s), f32x2_to_f16x2_bits(acc[j].z * s, acc[j].w * s));
                    *(uint2 *)(g.t[l] + ((int64_t)m * g.ad[l].max_rank + col) * 2) = o;
                }
            }
        }
        if (next.a < 0) break;
        now = next;
        if (!stream) {
            stage_barrier<0>();   // (the stages are free for the next pass)
            fill();
        }
    }
    stage_barrier<0>();
}

// rows of 16-bit values to rows of a multiple of eight of them, zeros behind: eight to a thread
__global__ __launch_bounds__(256) void copy_rows_kernel(const uint16_t *__restrict__ x, int64_t pieces, int K, int64_t ldx, int per_row, char *__restrict__ to) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= pieces) return;
    const int64_t m = at / per_row;
    const int k = (int)(at % per_row) * 8;
    const uint16_t *p = x + m * ldx + k;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k + 8 <= K) {
        __builtin_memcpy(&v, p, 16);
    } else {
        uint16_t e[8] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < K) e[i] = p[i];
        __builtin_memcpy(&v, e, 16);
    }
    *(uint4 *)(to + at * 16) = v;
}

template <int DT>
int launch(const char *x, int M, int K, int ldx_bytes, const DownLayers &g, float *partial, int slices, hipStream_t st) {
    const int per = ((K + BK - 1) / BK + slices - 1) / slices, ranks = g.first_column[g.n];
    // where the rows' slices leave CUs idle, the passes of a block of rows are dealt over workgroups too (471 x 2080, 29 requests with three
    // layers of rank 68: 52 us in one, 19 in eight; 188 x 1141, 85 requests, rank 82: 43 in eight, 22 in 32); those without a pass end at once
    const unsigned units = (unsigned)((M + ROWS - 1) / ROWS) * slices;
    const int parts = units >= 512 ? 1 : units <= 16 ? 32 : (int)(512 / units);
    if (!grid_fits((int64_t)units * parts, 256)) return I8F_ERR_UNSUPPORTED;
    const dim3 grid(units * parts);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, x, M, K, ldx_bytes, partial, slices, per, parts, g); };
    if (ranks <= 32) go(adapters_partial_kernel<DT, 2, 5>);
    else if (ranks <= 64) go(adapters_partial_kernel<DT, 4, 5>);
    else if (ranks <= 96) go(adapters_partial_kernel<DT, 6, 4>);
    else go(adapters_partial_kernel<DT, 8, 3>);
    return check_launch();
}

}  // namespace

// Two workgroups to a CU, slices of at least four K-tiles, none of them empty
int adapters_down_slices(int64_t M, int64_t K) {
    const int64_t blocks = (M + ROWS - 1) / ROWS, tiles = (factor_width(K) + BK - 1) / BK;
    int64_t s = 512 / blocks;
    if (s > tiles / 4) s = tiles / 4;
    if (s > 16) s = 16;
    if (s < 2) return 1;
    const int64_t per = (tiles + s - 1) / s;
    return (int)((tiles + per - 1) / per);
}

int adapters_copy_rows(const void *x, int64_t M, int64_t K, int64_t ldx, void *to, hipStream_t st) {
    const int64_t per_row = factor_width(K) / 8, pieces = M * per_row;
    if (!grid_fits((pieces + 255) / 256, 256)) return I8F_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(copy_rows_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, st, (const uint16_t *)x, pieces, (int)K, ldx, (int)per_row, (char *)to);
    return check_launch();
}

int adapters_down_partial(const void *x, int dtype, int64_t M, int64_t K, int64_t ldx, const DownLayers &g, float *partial, int slices, hipStream_t st) {
    if ((M + ROWS - 1) / ROWS * slices > 0x7fffffff || M * (g.first_column[g.n] / 4) / 256 >= 0x7fffffff) return I8F_ERR_UNSUPPORTED;
    return dtype == I8F_BF16 ? launch<I8F_BF16>((const char *)x, (int)M, (int)K, (int)ldx * 2, g, partial, slices, st)
                             : launch<I8F_F16>((const char *)x, (int)M, (int)K, (int)ldx * 2, g, partial, slices, st);
}

}  // namespace i8f
