// Attention over an encoder's states (include/i8f_attention.h has the formula).
//
// A wave takes 32 rows and goes over the states in tiles, keeping the running maximum and sum of a softmax.  A row is a query of one of the
// heads that share a head of the states, so that one token's 32 heads over 8 fill eight waves' rows by fours and every state is read once.
// Both products are computed transposed: S^T = K Q^T leaves a lane with 16 scores of ONE row in every 32 x 32 block, so that maximum and sum are
// in-lane but for one exchange of wave halves, and rounded to 16 bits the scores' weights already are the second operand of
// O^T = V^T P^T, the contraction index being free to run in the order in which a lane happens to hold the states; the first operand comes
// out of row-major V by LDS reads that transpose (ds_read_b64_tr_b16).
//
// What bounds it.  Long calls the matrix unit and the other vector instructions one after the other: for 8192 x 8192, 40 heads of 128, a wave's 64
// states take 1930 cycles of its SIMD, 1024 of them 32 matrix instructions, 755 the other 156 vector instructions (32 exponentials among them),
// which hardly run beside the products of the SIMD's other wave; the LDS is read in 27 % of them.  The clock is at 1.9 of 2.4 GHz besides.  1243 to
// 1340 us over cards and runs, 1.03 to 1.11 PFLOP/s; 1.58 is what a large library product reaches.  Calls over few states have the traffic of their rows on
// top, at the start and the end of a workgroup, when it multiplies nothing: 32760 x 512 408 to 446 us (0.77 to 0.84 PFLOP/s), over 64 states 171 to
// 181 us, 3.8 TB/s.  One token memory: 65536 states of 8 heads 58 us with the join, 4.6 TB/s; small ones the latencies of a launch (5 us).  Widths
// above 128 one workgroup of four waves to a CU: 4096 x 1024, 16 heads of 256, 92 to 97 us (0.71 to 0.75 PFLOP/s).  Widths that are no whole pieces
// the copies in front on top: 4096 x 4096, 40 heads of 100, 378 us (0.71 PFLOP/s; heads of 128 in
// binary16, whole pieces, 350 to 357: 0.97), one query over 257 states, 16 heads of 37, 10.4 us.
// Measured and not kept: 64 rows to a wave, which halve the LDS reads but leave one wave to a SIMD and a third of the vector instructions
// moving scores between register files (1450 us for 8192 x 8192); tiles of 32 states with three waves to a SIMD (405 against 419 us for 32768 x 512,
// 1320 against 1290 for 8192 x 8192, 82 to 107 for 1024 x 4096 of 32 heads); LDS reads three products ahead of their use in a fixed order (no
// faster); two steps unrolled so that addresses are constants (registers spilled); the rows of the workgroup to come requested into the L2
// (408 for 415 us at 32760 x 512, 2 to 5 % more everywhere else).
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "divisor.hpp"
#include "dma.hpp"
#include "extents.hpp"
#include "i8f_common.hpp"

#include "../../include/i8f_attention.h"

namespace i8f {
namespace {

using gemm::dma16;
using gemm::make_rsrc;
using gemm::v4i;

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr float LOWEST = -3.4028234663852886e38f, TO_LOG2 = 1.4426950408889634f;
constexpr float NONE = -__builtin_inff();   // a maximum of no scores

struct Launch {
    i8f_attention_args a;
    uint32_t share, rows;        // heads to one of the states', rows = queries * share to (batch, state head)
    uint32_t row_tiles, splits;  // of a (batch, state head)
    uint32_t tiles;              // of a split, in tiles of the kernel
    uint32_t loaded;             // elements of a row in memory, whole pieces of eight
    uint32_t wide_out;           // rows of the result are whole aligned pieces
    Divisor by_share, by_row_tiles, by_splits, by_kv_heads;
    float *partial;             // splits > 1: [batch * kv_heads, splits, rows, padded width], then [.., rows, 2]: maximum and sum
    float *stats;
};

template <int DT>
__device__ __forceinline__ v16f mfma(v8s a, v8s b, v16f c) {
    if constexpr (DT == I8F_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
// Two weights rounded to the type, and their sum as they were rounded added to `sum`.  The matrix unit takes operands of 16 bits: with u half a step
// each weight is off by u of itself at the most, either way, and what is divided by is the sum of what was multiplied, so that equal values stay what they are.
// Weights in 32 bits would be a second product with the remainders: 16 more matrix instructions to a step's 32.
template <int DT>
__device__ __forceinline__ uint32_t round_weights(float lo, float hi, float &sum) {
    if constexpr (DT == I8F_BF16) {
        const uint32_t w = f32x2_to_bf16x2_bits(lo, hi);
        sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, w), __builtin_bit_cast(v2bf, 0x3f803f80u), sum, false);
        return w;
    } else {
        const uint32_t w = f32x2_to_f16x2_bits(lo, hi);
        sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, w), __builtin_bit_cast(half2v, 0x3c003c00u), sum, false);
        return w;
    }
}
// the other half of the wave's value beside the own
__device__ __forceinline__ float max_of_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_of_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// What a score is multiplied by in the exponential: the scale and log2 e, or log2 e where addends were put on top of scaled scores (not in units
// of log 2: addends reach to the ends of binary32).
__device__ __forceinline__ float exponents_of(const i8f_attention_args &a) {
    return a.key_mask && a.mask_type != I8F_MASK_BYTES ? TO_LOG2 : a.scale * TO_LOG2;
}

// What weights under one maximum become under a larger or the same one (which may be that of no scores).
__device__ __forceinline__ float fading(float from, float to, float unit) { return from == to ? 1.0f : __builtin_amdgcn_exp2f((from - to) * unit); }

// A state's element of the mask as it is in memory, and whether it counts by it, with its addend.
__device__ __forceinline__ uint32_t mask_bits(const i8f_attention_args &a, int64_t b, int64_t j) {
    const int64_t at = b * a.mask_batch + j * a.mask_key;
    switch (a.mask_type) {
    case I8F_MASK_BYTES: return ((const uint8_t *)a.key_mask)[at];
    case I8F_MASK_F32: return ((const uint32_t *)a.key_mask)[at];
    default: return ((const uint16_t *)a.key_mask)[at];
    }
}
__device__ __forceinline__ bool counts(int type, uint32_t bits, float &add) {
    add = 0.0f;
    if (type == I8F_MASK_BYTES) return bits != 0;
    const float m = type == I8F_MASK_BF16 ? bf16_bits_to_f32(bits) : type == I8F_MASK_F16 ? f16_bits_to_f32(bits) : __uint_as_float(bits);
    const float lowest = type == I8F_MASK_BF16 ? -3.3895313892515355e38f : type == I8F_MASK_F16 ? -65504.0f : LOWEST;
    if (m <= lowest) return false;
    add = m;
    return true;
}

// The 16-byte pieces of a row are exchanged within it by a function of the row, so that the lanes of an LDS read are spread over the banks.
// K is read by 32 rows' same piece at a time (ds_read_b128): sixteen rows that differ in their number's last four bits are on different
// banks.  V is read by four rows' same 64 bytes (ds_read_b64_tr_b16); rows of 192 bytes lie three quarters of the banks apart by themselves.
template <int DP>
__device__ __forceinline__ int k_piece(int row, int piece) {
    if constexpr (DP == 96) return piece ^ ((row >> 2) & 3);
    else if constexpr (DP % 128 == 0) return piece ^ (row & 15);
    else return piece ^ ((row >> 1) & 7);
}
template <int DP>
__device__ __forceinline__ int v_quad(int row) {   // what the number of a row's 64-byte quarter is exchanged by
    if constexpr (DP == 96) return 0;
    else if constexpr (DP % 128 == 0) return row & 3;
    else return (row >> 1) & 1;
}

// DP: the width, padded.  WAVES of a workgroup; APART: they have the same 32 rows and a tile of 32 states each, by themselves; otherwise 32 rows
// each and a tile of 64 states together.
template <int DT, int DP, int WAVES, bool APART, bool MASK>
struct Shape {
    static constexpr int KT = APART ? 32 : 64, PIECES = DP / 8, TILE = KT * DP * 2;
    static constexpr int LOADS = KT * PIECES / 64 / (APART ? 1 : WAVES);       // a wave's of a tile of K, or of V
    static_assert(KT * PIECES % (64 * (APART ? 1 : WAVES)) == 0, "");
    static constexpr int SETS = APART ? WAVES : 1, LDS = SETS * 4 * TILE;      // two stages of K and V
    static constexpr int ROWS = APART ? 32 : 32 * WAVES;
    static constexpr int PER_SIMD = WAVES == 8 || LDS <= 80 * 1024 ? 2 : 1;    // waves
};

template <int DT, int DP, int WAVES, bool APART, bool MASK>
__global__ __launch_bounds__(WAVES * 64, (Shape<DT, DP, WAVES, APART, MASK>::PER_SIMD)) void attention_kernel(const Launch p) {
    using S = Shape<DT, DP, WAVES, APART, MASK>;
    constexpr int KT = S::KT, KB = KT / 32, NK = DP / 16, ND = DP / 32;
    __shared__ __attribute__((aligned(16))) char lds[S::LDS + (MASK ? WAVES * 128 * 4 : 0)];
    const i8f_attention_args &a = p.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the workgroups of an XCD (number mod 8) take consecutive row tiles of the same states
    const unsigned per = gridDim.x / 8, extra = gridDim.x % 8, xcd = blockIdx.x % 8;
    const unsigned id = xcd * per + (xcd < extra ? xcd : extra) + blockIdx.x / 8, set = p.by_row_tiles(id), row_tile = id - set * p.row_tiles;
    const unsigned bg = p.by_splits(set), split = set - bg * p.splits;
    const int64_t b = p.by_kv_heads(bg), g = bg - (unsigned)b * (unsigned)a.kv_heads;
    int n = (int)a.keys;
    if (a.key_lengths) {
        const int64_t given = a.lengths_type ? ((const int64_t *)a.key_lengths)[b] : ((const int32_t *)a.key_lengths)[b];
        n = given < 0 ? 0 : given < n ? (int)given : n;
    }
    const int from_tile = (int)(split * p.tiles) + (APART ? wave : 0), all_tiles = (n - 1 + KT) / KT, to_tile = (int)((split + 1) * p.tiles);
    const int last_tile = all_tiles < to_tile ? all_tiles : to_tile;
    constexpr int STEP = APART ? WAVES : 1;   // (apart, every WAVES-th tile is a wave's)

    // where a lane's pieces of a tile come from: LDS is filled in order, 16 bytes a lane
    constexpr uint32_t NOWHERE = 0x80000000u;   // (behind the buffer's end: such a piece is zeros)
    uint32_t from_k[S::LOADS], from_v[S::LOADS];
    auto piece_at = [&](int i) { return (APART ? i : i * WAVES + wave) * 64 + lane; };
#pragma unroll
    for (int i = 0; i < S::LOADS; ++i) {
        const int at = piece_at(i), r = at / S::PIECES, c = at % S::PIECES;
        const unsigned ck = k_piece<DP>(r, c), cv = c ^ (v_quad<DP>(r) << 2);
        from_k[i] = ck * 8 < p.loaded ? ((uint32_t)r * (uint32_t)a.k_token + ck * 8) * 2u : NOWHERE;
        from_v[i] = cv * 8 < p.loaded ? ((uint32_t)r * (uint32_t)a.v_token + cv * 8) * 2u : NOWHERE;
    }
    const uint16_t *kp = (const uint16_t *)a.k + b * a.k_batch + g * a.k_head, *vp = (const uint16_t *)a.v + b * a.v_batch + g * a.v_head;
    const uint32_t lds_at = (uint32_t)(uintptr_t)(gemm::lds_ptr_t)lds + (APART ? wave * 4 * S::TILE : 0);   // stage s: K at s * 2 * TILE, V behind it

    // A tile, which of its states count (bit j for its state j) and with a mask a lane's own addend.
    struct Tile {
        int at;
        uint64_t on;
        float add;
    };
    constexpr uint64_t ALL = KT == 64 ? ~0ull : 0xffffffffull;
    // a lane's state of a tile in the mask; it is asked for a step before it is looked at
    auto peek = [&](int at) -> uint32_t {
        const int j = at * KT + lane;
        return MASK && at < last_tile && lane < KT && j < n ? mask_bits(a, b, j) : 0u;
    };
    auto tile_from = [&](int at, uint32_t bits) {   // the first tile from `at` on (whose mask is there) with a state that counts, or one past the last
        Tile t = {at, ALL, 0.0f};
        for (; t.at < last_tile; t.at += STEP) {
            const int left = n - t.at * KT;
            if constexpr (!MASK) {
                if (left < KT) t.on = (1ull << left) - 1;
                break;
            } else {
                if (t.at != at) bits = peek(t.at);
                const bool on = counts(a.mask_type, bits, t.add) && lane < KT && lane < left;
                if ((t.on = __ballot(on)) != 0) break;
            }
        }
        return t;
    };
    // the wave's pieces of a tile of K (or of V) on their way into a stage; those of states that do not count are zeros
    auto request = [&](const Tile &t, const uint16_t *x, int64_t token, const uint32_t (&from)[S::LOADS], uint32_t to) {
        if (t.at >= last_tile) return;
        const v4i r = make_rsrc(x + (int64_t)t.at * KT * token, 0x7ffffff0u);
        if (t.on == ALL) {
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) dma16(r, to + i * (APART ? 1 : WAVES) * 1024, from[i], 0);
        } else {
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) dma16(r, to + i * (APART ? 1 : WAVES) * 1024, t.on >> (piece_at(i) / S::PIECES) & 1 ? from[i] : NOWHERE, 0);
        }
    };
    const uint32_t lds_to = lds_at + (APART ? 0 : wave * 1024);
    auto request_k = [&](const Tile &t, int stage) { request(t, kp, a.k_token, from_k, lds_to + stage * 2 * S::TILE); };
    auto request_v = [&](const Tile &t, int stage) { request(t, vp, a.v_token, from_v, lds_to + stage * 2 * S::TILE + S::TILE); };
    auto all_here = [&]() {   // what was requested has arrived, and (together) everyone has read what may now be overwritten
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if constexpr (!APART) __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    Tile now = tile_from(from_tile, peek(from_tile)), next = tile_from(now.at + STEP, peek(now.at + STEP));
    uint32_t ahead = peek(next.at + STEP);
    request_k(now, 0), request_v(now, 0), request_k(next, 1);

    // a wave's 32 rows, a lane's in both halves
    const unsigned first_row = row_tile * S::ROWS + (APART ? 0 : wave * 32);
    v8s q[NK];
    {
        const unsigned row = first_row + (lane & 31), real = row < p.rows ? row : p.rows - 1, query = p.by_share(real);
        const uint16_t *qp = (const uint16_t *)a.q + b * a.q_batch + query * a.q_token + (g * p.share + (real - query * p.share)) * a.q_head;
#pragma unroll
        for (int e = 0; e < NK; ++e) {
            const unsigned at = e * 16 + half * 8;
            q[e] = at < p.loaded ? *(const v8s *)(qp + at) : v8s{};
        }
    }
    v16f o[ND], s[KB];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = v16f{};
    float top = NONE, sum = 0.0f, most = NONE;   // (the maxima in the scores' own unit)
    // The largest weight of a row lies between 2^RAISE and 2^(RAISE + 8) (see below).  Binary16's fixed step below 2^-14 asks for 2^14; bfloat16 has the
    // exponents of binary32, and weights up to 1 leave the sums of their products with values the whole of its range.
    constexpr float RAISE = DT == I8F_F16 ? 6.0f : -8.0f;
    // A weight is 2^(unit x - unit top), one fused operation on x with unit top rounded beforehand.  That rounding is the same for all weights under
    // one reference, but weights of other tiles were formed under others, and in the end it would leave the type's range: at 2^28 binary16's, at
    // 2^33 bfloat16's.  Below 2^12 it is 2^-13 at the most, less than half of what binary16 rounds a weight by.  A row that is beyond has its
    // maximum taken off the scores first, exactly where they are close to it, and scales them afterwards; the wave's other rows get what they
    // would have had (a few more operations a score for all of them).  A row whose scores so far are all -inf or NaN has no reference.
    constexpr float FAR = 4096.0f;
    const float unit = exponents_of(a);
    const float allowed = 8.0f / unit;   // growth of the maximum that `top` need not follow, while its own steps are small beside that
    auto beyond = [&]() { return fabsf(top) < __builtin_inff() && !(fabsf(top * unit) < FAR); };
    auto off = [&]() { return top == NONE ? RAISE : __builtin_fmaf(-top, unit, RAISE); };
    bool far = false;                                  // a row of the wave is beyond
    float limit = NONE, factor = unit, from = RAISE;   // `top`'s; the exponents are factor x + from

    // where a lane reads: K row (lane & 31) of a block, V's four rows from 4 half on by 16 elements
    char *const tiles = lds + (APART ? wave * 4 * S::TILE : 0);
    const int k_row = (lane & 31) * DP * 2;
    const int v_row = (4 * half + ((lane >> 2) & 3)) * DP * 2 + (2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) * 16 + (lane & 1) * 8;
    const int v_x = v_quad<DP>((lane >> 2) & 3);
    // With a mask the scores' sums begin at 0 or, of states that do not count, at -inf: their K is zeros, so that is what they stay, without a
    // vector instruction.  A lane has states 8 (i / 4) + 4 half + i % 4 of a block.
    float *const begins = (float *)(lds + S::LDS) + wave * 128, *const adds = begins + 64;
    auto begin = [&](const Tile &t, int k) {
        v16f x = {};
        if constexpr (MASK) {
            if (k == 0) begins[lane] = t.on >> lane & 1 ? 0.0f : -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 y = *(const float4 *)(begins + k * 32 + 8 * i + 4 * half);
                x[4 * i] = y.x, x[4 * i + 1] = y.y, x[4 * i + 2] = y.z, x[4 * i + 3] = y.w;
            }
        }
        return x;
    };
    auto k_part = [&](const char *ks, int e, int k) { return *(const v8s *)(ks + k * 32 * DP * 2 + k_row + k_piece<DP>(lane & 31, 2 * e + half) * 16); };
    auto largest = [&](const v16f (&x)[KB]) {   // (of the wave half's states)
        float m = x[0][0];
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int i = 0; i < 16; ++i) m = __builtin_elementwise_maximum(m, x[k][i]);
        return m;
    };

    all_here();
    // (the rows have arrived as well: without this the compiler waits for them, and with them for the tiles under way, in every step)
#pragma unroll
    for (int e = 0; e < NK; ++e) asm volatile("" : "+v"(q[e]));
    if (now.at < last_tile) {
#pragma unroll
        for (int e = 0; e < NK; ++e)
#pragma unroll
            for (int k = 0; k < KB; ++k) s[k] = mfma<DT>(k_part(tiles, e, k), q[e], e ? s[k] : begin(now, k));
        most = largest(s);
    }
    // One tile: its scores and their maximum are there; the next tile's scores are formed on the matrix unit (MORE) while the vector units have
    // this one's exponentials, and their maximum beside this one's last products.
    int stage = 0;
    auto step = [&](auto more) __attribute__((always_inline)) {
        constexpr bool MORE = decltype(more)::value;
        if constexpr (MASK) {
            if (a.mask_type != I8F_MASK_BYTES) {   // (scaled here, since addends come on top)
                adds[lane] = now.add;
#pragma unroll
                for (int k = 0; k < KB; ++k)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[k][i] = __builtin_fmaf(s[k][i], a.scale, adds[k * 32 + 8 * (i / 4) + 4 * half + i % 4]);
                most = largest(s);
            }
        } else if (now.on != ALL) {   // (the last tile)
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                uint32_t mine = (uint32_t)(now.on >> (32 * k)) >> (4 * half);
                asm volatile("" : "+v"(mine));   // (keeps what follows in this branch)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[k][i] = mine >> (8 * (i / 4) + i % 4) & 1 ? s[k][i] : -__builtin_inff();
            }
            most = largest(s);
        }
        most = max_of_halves(most);
        // The reference of the exponentials follows the maximum only where that has grown by 2^8: the weights are below 2^8 times 2^RAISE then, which
        // costs no bits, and the result is divided by their sum either way.
        if (__any(most > limit)) {
            const float to = most > limit ? most : top, fade = fading(top, to, unit);   // (a row's bits do not depend on the rows beside it)
            top = to;
            const bool mine = beyond();
            far = __any(mine);
            limit = mine ? top : top + allowed, factor = far ? 1.0f : unit, from = !far ? off() : mine ? RAISE : 0.0f;
            sum *= fade;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= fade;
        }
        if (far) {
            const bool mine = beyond();
            const float near = off();
#pragma unroll
            for (int k = 0; k < KB; ++k)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[k][i] = mine ? (s[k][i] - top) * unit : __builtin_fmaf(s[k][i], unit, near);
        }
        all_here();   // the tile's V and the next one's K
        const Tile after = MORE ? tile_from(next.at + STEP, ahead) : next;
        if constexpr (MORE) request_k(after, stage), request_v(next, stage ^ 1), ahead = peek(after.at + STEP);
        const char *vs = tiles + stage * 2 * S::TILE + S::TILE, *ks = tiles + (stage ^ 1) * 2 * S::TILE;
        v16f t[KB];
        constexpr int PARTS = 2 * KB;   // of 16 states
        auto score = [&](int part) __attribute__((always_inline)) {
            if constexpr (MORE) {
#pragma unroll
                for (int e = NK * part / PARTS; e < NK * (part + 1) / PARTS; ++e)
#pragma unroll
                    for (int k = 0; k < KB; ++k) t[k] = mfma<DT>(k_part(ks, e, k), q[e], e ? t[k] : begin(next, k));
            }
        };
        auto weigh = [&](int part) __attribute__((always_inline)) {
            const v16f &x = s[part / 2];
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = round_weights<DT>(__builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * (part % 2) + 2 * i], factor, from)),
                                         __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * (part % 2) + 2 * i + 1], factor, from)), sum);
            return __builtin_bit_cast(v8s, (v4i){(int)w[0], (int)w[1], (int)w[2], (int)w[3]});
        };
        score(0);
        v8s weights = weigh(0);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            const v8s mine = weights;
            if (part + 1 < PARTS) score(part + 1), weights = weigh(part + 1);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                typedef __attribute__((address_space(3))) v4s *v4s_lds;
                const char *at = vs + part * 16 * DP * 2 + v_row + (d ^ v_x) * 64;
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s_lds)(gemm::lds_ptr_t)at);
                const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s_lds)(gemm::lds_ptr_t)(at + 8 * DP * 2));
                o[d] = mfma<DT>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), mine, o[d]);
            }
        }
        if constexpr (MORE) {
            most = largest(t);
#pragma unroll
            for (int k = 0; k < KB; ++k) s[k] = t[k];
        }
        now = next, next = after, stage ^= 1;
    };
    while (next.at < last_tile) step(std::integral_constant<bool, true>{});
    if (now.at < last_tile) step(std::integral_constant<bool, false>{});

    // a lane has elements 32 d + 8 (i / 4) + 4 half + i % 4 of its row
    sum = sum_of_halves(sum);
    if constexpr (APART) {   // the waves' results meet in LDS, in the place of their tiles
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __syncthreads();
        float *const others = (float *)lds;   // [WAVES][32][DP + 4]
        constexpr int PITCH = DP + 4;
        static_assert(WAVES * 32 * (PITCH + 2) * 4 <= S::LDS, "");
        float *const heads = others + WAVES * 32 * PITCH;   // [WAVES][32][2]
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float4 v = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
                *(float4 *)(others + (wave * 32 + (lane & 31)) * PITCH + 32 * d + 8 * i + 4 * half) = v;
            }
        if (half == 0) heads[(wave * 32 + lane) * 2] = top, heads[(wave * 32 + lane) * 2 + 1] = sum;
        __syncthreads();
        constexpr int QUADS = DP / 4;
        for (int at = threadIdx.x; at < 32 * QUADS; at += WAVES * 64) {
            const int r = at / QUADS, e = at % QUADS * 4;
            const unsigned own = row_tile * 32 + r;
            if (own >= p.rows) continue;
            float best = NONE, total = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) best = fmaxf(best, heads[(w * 32 + r) * 2]);
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float f = fading(heads[(w * 32 + r) * 2], best, unit);
                total = __builtin_fmaf(heads[(w * 32 + r) * 2 + 1], f, total);
                const float4 x = *(const float4 *)(others + (w * 32 + r) * PITCH + e);
                v[0] = __builtin_fmaf(x.x, f, v[0]), v[1] = __builtin_fmaf(x.y, f, v[1]), v[2] = __builtin_fmaf(x.z, f, v[2]), v[3] = __builtin_fmaf(x.w, f, v[3]);
            }
            if (p.splits > 1) {
                const int64_t at_row = ((int64_t)bg * p.splits + split) * p.rows + own;
                *(float4 *)(p.partial + at_row * DP + e) = make_float4(v[0], v[1], v[2], v[3]);
                if (e == 0) p.stats[at_row * 2] = best, p.stats[at_row * 2 + 1] = total;
            } else {
                const int64_t to = ((b * a.queries + p.by_share(own)) * a.heads + g * p.share + (own - p.by_share(own) * p.share)) * a.width;
                for (int i = 0; i < 4; ++i)
                    if (e + i < a.width) store_from_f32<DT>(a.out, to + e + i, total == 0.0f ? 0.0f : v[i] / total);
            }
        }
    } else {
        if (p.splits > 1) {
            const unsigned row = first_row + (lane & 31);
            if (row >= p.rows) return;
            const int64_t at_row = ((int64_t)bg * p.splits + split) * p.rows + row;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *(float4 *)(p.partial + at_row * DP + 32 * d + 8 * i + 4 * half) = make_float4(o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
            if (half == 0) p.stats[at_row * 2] = top, p.stats[at_row * 2 + 1] = sum;
            return;
        }
        // A lane has pieces of one row, memory wants whole lines: the rows change places in LDS.  The stage that the last tile is not in has been
        // read by everyone and nothing is under way to it; it holds the rows of four waves, those of eight take both.
        static_assert(WAVES * 32 * DP * 2 <= (WAVES == 8 ? S::LDS : 2 * S::TILE), "");
        if constexpr (WAVES == 8) __syncthreads();
        char *const mine = lds + (WAVES == 8 ? 0 : stage * 2 * S::TILE) + wave * 32 * DP * 2;
        const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = o[d][4 * i] * by, y = o[d][4 * i + 1] * by, z = o[d][4 * i + 2] * by, w = o[d][4 * i + 3] * by;
                const uint2 v = DT == I8F_BF16 ? make_uint2(f32x2_to_bf16x2_bits(x, y), f32x2_to_bf16x2_bits(z, w)) : make_uint2(f32x2_to_f16x2_bits(x, y), f32x2_to_f16x2_bits(z, w));
                *(uint2 *)(mine + k_row + k_piece<DP>(lane & 31, 4 * d + i) * 16 + half * 8) = v;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < 32 * S::PIECES / 64; ++i) {
            const int at = i * 64 + lane, x = at / S::PIECES, c = at % S::PIECES;
            const unsigned own = first_row + x;
            if (own >= p.rows || c * 8 >= a.width) continue;
            const uint4 v = *(const uint4 *)(mine + x * DP * 2 + k_piece<DP>(x, c) * 16);
            const unsigned query = p.by_share(own);
            uint16_t *const to = (uint16_t *)a.out + ((b * a.queries + query) * a.heads + g * p.share + (own - query * p.share)) * a.width + c * 8;
            if (p.wide_out) {
                stream_store16(to, v);
            } else {
                uint16_t e[8];
                __builtin_memcpy(e, &v, 16);
                for (int j = 0; j < 8; ++j)
                    if (c * 8 + j < a.width) to[j] = e[j];
            }
        }
    }
}

// The splits' results of a row joined: a workgroup to a row, its threads by four elements and by splits, so that all of them are requested at once
// (4 us for 32 rows of 32 splits; a wave to a row, split after split, was 25).
constexpr int MOST_SPLITS = 256;
template <int DT, int DP>
__global__ __launch_bounds__(256) void join_kernel(const Launch p) {
    constexpr int QUADS = DP / 4, PARTS = 256 / QUADS;
    __shared__ float weight[MOST_SPLITS], red[4];
    __shared__ float4 sums[PARTS][QUADS];
    const i8f_attention_args &a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, quad = tid % QUADS, part = tid / QUADS, splits = (int)p.splits;
    const unsigned row = blockIdx.x % p.rows;
    const int64_t bg = blockIdx.x / p.rows, b = bg / a.kv_heads, g = bg % a.kv_heads, first = bg * p.splits * p.rows + row;
    const bool mine = tid < splits;
    const float2 own = mine ? *(const float2 *)(p.stats + 2 * (first + (int64_t)tid * p.rows)) : make_float2(NONE, 0.0f);
    float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    const float top = wave_max(own.x);
    if (lane == 0) red[wave] = top;
    __syncthreads();
    const float best = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float f = mine ? fading(own.x, best, exponents_of(a)) : 0.0f;
    weight[tid] = f;
    float total = own.y * f;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) total += __shfl_xor(total, x);
    __syncthreads();
    if (lane == 0) red[wave] = total;
    if (part < PARTS) {
#pragma unroll 8
        for (int s = part; s < splits; s += PARTS) {
            const float4 x = *(const float4 *)(p.partial + (first + (int64_t)s * p.rows) * DP + quad * 4);
            const float w = weight[s];
            v.x = __builtin_fmaf(x.x, w, v.x), v.y = __builtin_fmaf(x.y, w, v.y), v.z = __builtin_fmaf(x.z, w, v.z), v.w = __builtin_fmaf(x.w, w, v.w);
        }
        sums[part][quad] = v;
    }
    __syncthreads();
    if (tid >= QUADS) return;
    total = (red[0] + red[1]) + (red[2] + red[3]);
    v = sums[0][tid];
#pragma unroll
    for (int i = 1; i < PARTS; ++i) v.x += sums[i][tid].x, v.y += sums[i][tid].y, v.z += sums[i][tid].z, v.w += sums[i][tid].w;
    const unsigned query = p.by_share(row);
    const int64_t to = ((b * a.queries + query) * a.heads + g * p.share + (row - query * p.share)) * a.width + tid * 4;
    const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (tid * 4 + i < a.width) store_from_f32<DT>(a.out, to + i, total == 0.0f ? 0.0f : o[i] / total);
}

// [batch, tokens, heads, width] of any strides and alignment as rows of whole 16-byte pieces, the rest of them zeros, in the same order; or with
// a head's tokens side by side where a tile's rows would lie farther apart than the kernel's 32-bit offsets reach.
struct Pack {
    const uint16_t *x;
    uint16_t *out;
    int64_t rows, tokens, heads, batch_stride, token_stride, head_stride;
    int64_t out_token, out_head;
    int width, padded;
};
struct Packs {
    Pack p[3];
};
__global__ __launch_bounds__(256) void pack_kernel(const Packs packs) {
    const Pack &p = packs.p[blockIdx.y];
    const int pieces = p.padded / 8;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < p.rows * pieces; at += (int64_t)gridDim.x * 256) {
        const int64_t row = at / pieces, h = row % p.heads, t = row / p.heads % p.tokens, b = row / p.heads / p.tokens;
        const int e = (int)(at % pieces) * 8;
        const uint16_t *x = p.x + b * p.batch_stride + t * p.token_stride + h * p.head_stride + e;
        uint16_t v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = e + i < p.width ? x[i] : (uint16_t)0;
        uint4 o;
        __builtin_memcpy(&o, v, 16);
        *(uint4 *)(p.out + b * p.tokens * p.heads * p.padded + t * p.out_token + h * p.out_head + e) = o;
    }
}

// No states at all: zeros.
__global__ __launch_bounds__(256) void zeros_kernel(uint16_t *out, const int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = 0;
}

// ---- how a call is cut ------------------------------------------------------------------------------------------------------------
struct Plan {
    int padded;               // width of the kernels
    bool apart;               // the waves of a workgroup take the states in turn
    int waves;                // of a workgroup
    int64_t row_tiles, splits, tiles;
    int64_t partials;         // floats of the splits' results, behind which two to a row are their statistics
    int64_t partial_bytes;    // of both, whole pieces of 16 (the copies lie behind them)
};
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

Plan plan_of(int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t width) {
    Plan p = {};
    p.padded = width <= 64 ? 64 : width <= 96 ? 96 : width <= 128 ? 128 : width <= 192 ? 192 : 256;
    const int64_t rows = queries * (heads / kv_heads), sets = batch * kv_heads;
    // Apart, four waves to 32 rows, where 128 rows together leave waves idle or CUs.  us together and apart: 16 heads of 64, 64 rows over 512 states
    // 10.3 and 6.5, 96 over 512 10.8 and 6.0, over 4096 13.9 and 13.5, over 32768 36 and 40; 32 heads of 128, 96 rows over 512 16.2 and 9.3, over
    // 4096 28 and 35; 256 heads of 64, 77 rows over 512 11.7 and 15.0.
    p.apart = rows <= 32 || (sets * ((rows + 31) / 32) <= 128 && keys <= 2048);
    p.waves = p.apart && p.padded > 128 ? 2 : 4;
    // Eight waves read the states half as often, which is energy, and the card runs at its power limit in long calls; but theirs is the CU's only
    // workgroup, so that rows filled up to 256 and a last round of few workgroups cost more than that.  us with four and eight, heads of 128, (batch,
    // head) pairs x rows x states: 8 x 32768 x 4096 517 and 503, 32 x 8192 x 8192 1022 and 1005, 40 x 8192 x 8192 1270 and 1258, 4096 x 200 x 4096 2509 and
    // 2462; 40 x 32768 x 2048 1333 and 1333, 40 x 32768 x 512 419 and 449; with 5.5 rounds, 176 x 2048 x 4096, 739 and 757; with 16.03, 456 x 2300 x 4096,
    // 2156 and 2210; filled up, 2048 x 300 x 4096 1757 and 2189, 1024 x 64 x 4096 401 and 571.  Heads of 64: 40 x 8192 x 8192 746 and 773.
    const int64_t wide = sets * ((rows + 255) / 256);
    if (!p.apart && p.padded == 128 && keys >= 4096 && wide >= 1024 && round_up(rows, 256) == round_up(rows, 128) && (round_up(wide, 256) - wide) * 32 <= wide) p.waves = 8;
    const int64_t to_group = p.apart ? 32 : 32 * p.waves;
    p.row_tiles = (rows + to_group - 1) / to_group;
    const int64_t tile = p.apart ? 32 : 64, all = (keys + tile - 1) / tile, groups = sets * p.row_tiles;
    // as many splits as make a workgroup to a CU (one token over 65536 states of 8 heads: 256 workgroups 59 us, 512 81), of at least 4 tiles to a wave
    const int64_t least = 4 * (p.apart ? p.waves : 1);
    p.splits = groups >= 256 || all < 2 * least ? 1 : (256 + groups - 1) / groups;
    if (p.splits > all / least) p.splits = all / least;
    if (p.splits < 1) p.splits = 1;
    p.tiles = round_up((all + p.splits - 1) / p.splits, p.apart ? p.waves : 1);
    if (p.tiles < 1) p.tiles = 1;
    p.splits = all ? (all + p.tiles - 1) / p.tiles : 1;
    const int64_t results = p.splits > 1 ? sets * p.splits * rows : 0;
    p.partials = results * p.padded, p.partial_bytes = round_up((p.partials + 2 * results) * 4, 16);
    return p;
}

// The kernels read 16-byte pieces, and a tile's rows by 32-bit offsets.
constexpr int64_t MOST_STRIDE = 1 << 22;
bool in_pieces(const void *x, int64_t width, std::initializer_list<int64_t> strides, int64_t token) {
    if ((uintptr_t)x % 16 || width % 8 || token > MOST_STRIDE) return false;
    for (int64_t s : strides)
        if (s % 8) return false;
    return true;
}
// Which of q, k and v (bits 0 to 2) have to be copied into whole pieces first, and the bytes of the copies.
int to_pack(const i8f_attention_args &a, int64_t (&bytes)[3]) {
    const bool in[3] = {in_pieces(a.q, a.width, {a.q_batch, a.q_token, a.q_head}, 0), in_pieces(a.k, a.width, {a.k_batch, a.k_token, a.k_head}, a.k_token),
                        in_pieces(a.v, a.width, {a.v_batch, a.v_token, a.v_head}, a.v_token)};
    const int64_t states = a.batch * a.keys * a.kv_heads, rows[3] = {a.batch * a.queries * a.heads, states, states};
    int which = 0;
    for (int i = 0; i < 3; ++i) bytes[i] = in[i] ? 0 : rows[i] * round_up(a.width, 8) * 2, which |= in[i] ? 0 : 1 << i;
    return which;
}

template <int DT, int DP, int WAVES, bool APART, bool MASK>
int launch_tiles(const Launch &p, int64_t groups, hipStream_t st) {
    if (!grid_fits(groups, WAVES * 64)) return I8F_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((attention_kernel<DT, DP, WAVES, APART, MASK>), dim3((unsigned)groups), dim3(WAVES * 64), 0, st, p);
    return check_launch();
}
template <int DT, int DP, bool MASK>
int launch_masked(const Launch &p, const Plan &plan, int64_t groups, hipStream_t st) {
    if (plan.apart) return launch_tiles<DT, DP, DP <= 128 ? 4 : 2, true, MASK>(p, groups, st);
    if constexpr (DP == 128) {
        if (plan.waves == 8) return launch_tiles<DT, DP, 8, false, MASK>(p, groups, st);
    }
    return launch_tiles<DT, DP, 4, false, MASK>(p, groups, st);
}
template <int DT, int DP>
int launch_form(const Launch &p, const Plan &plan, int64_t groups, hipStream_t st) {
    return p.a.key_mask ? launch_masked<DT, DP, true>(p, plan, groups, st) : launch_masked<DT, DP, false>(p, plan, groups, st);
}
template <int DT, int DP>
int launch_width(const Launch &p, const Plan &plan, hipStream_t st) {
    const int64_t sets = p.a.batch * p.a.kv_heads;
    const int rc = launch_form<DT, DP>(p, plan, sets * p.row_tiles * p.splits, st);
    if (rc || p.splits == 1) return rc;
    if (!grid_fits(sets * p.rows, 256)) return I8F_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((join_kernel<DT, DP>), dim3((unsigned)(sets * p.rows)), dim3(256), 0, st, p);
    return check_launch();
}
template <int DT>
int launch(const Launch &p, const Plan &plan, hipStream_t st) {
    switch (plan.padded) {
    case 64: return launch_width<DT, 64>(p, plan, st);
    case 96: return launch_width<DT, 96>(p, plan, st);
    case 128: return launch_width<DT, 128>(p, plan, st);
    case 192: return launch_width<DT, 192>(p, plan, st);
    default: return launch_width<DT, 256>(p, plan, st);
    }
}

int validate(const i8f_attention_args &a) {
    if (a.batch < 0 || a.queries < 0 || a.keys < 0 || a.heads < 0 || a.kv_heads < 0 || a.width < 1) return I8F_ERR_INVALID;
    if (a.dtype != I8F_BF16 && a.dtype != I8F_F16) return valid_dtype(a.dtype) ? I8F_ERR_UNSUPPORTED : I8F_ERR_INVALID;
    if (a.heads && (!a.kv_heads || a.heads % a.kv_heads)) return I8F_ERR_INVALID;
    if (!(a.scale > 0.0f) || !(a.scale <= 0x1p126f)) return I8F_ERR_INVALID;   // (times log2 e it stays finite)
    if (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) % 2) return I8F_ERR_INVALID;
    if (a.width > 256) return I8F_ERR_UNSUPPORTED;
    for (int64_t s : {a.q_batch, a.q_token, a.q_head, a.k_batch, a.k_token, a.k_head, a.v_batch, a.v_token, a.v_head})
        if (s < 0) return I8F_ERR_INVALID;
    for (int64_t n : {a.batch, a.queries, a.keys, a.heads})
        if (n > 1 << 30) return I8F_ERR_UNSUPPORTED;
    const int64_t rows = a.batch * a.queries;
    if (rows && a.heads > 0x7fffffff / rows) return I8F_ERR_UNSUPPORTED;   // (rows are counted in 32 bits)
    const int length_size = a.lengths_type ? 8 : 4, mask_size = a.mask_type == I8F_MASK_BYTES ? 1 : a.mask_type == I8F_MASK_F32 ? 4 : 2;
    if (a.key_lengths && ((a.lengths_type != 0 && a.lengths_type != 1) || (uintptr_t)a.key_lengths % length_size)) return I8F_ERR_INVALID;
    if (a.key_mask && ((uintptr_t)a.key_mask % mask_size || a.mask_type < I8F_MASK_BYTES || a.mask_type > I8F_MASK_F32 || a.mask_batch < 0 || a.mask_key < 0)) return I8F_ERR_INVALID;
    const int64_t out = rows * a.heads * a.width, q = extent({{a.batch, a.q_batch}, {a.queries, a.q_token}, {a.heads, a.q_head}, {a.width, 1}});
    const int64_t k = extent({{a.batch, a.k_batch}, {a.keys, a.k_token}, {a.kv_heads, a.k_head}, {a.width, 1}});
    const int64_t v = extent({{a.batch, a.v_batch}, {a.keys, a.v_token}, {a.kv_heads, a.v_head}, {a.width, 1}});
    // (expanded operands have few elements and states without end, whose copies are counted in 64 bits)
    if ((__int128)a.batch * a.keys * a.kv_heads * 512 > (__int128)1 << 58) return I8F_ERR_UNSUPPORTED;
    const int64_t mask = a.key_mask ? extent({{a.batch, a.mask_batch}, {a.keys, a.mask_key}}) : 0;
    if (q < 0 || k < 0 || v < 0 || mask < 0) return I8F_ERR_UNSUPPORTED;
    if (!out) return I8F_OK;   // (nothing to write: the pointers may be NULL)
    if (!a.q || !a.out || (a.keys && (!a.k || !a.v))) return I8F_ERR_INVALID;
    if (overlap(a.out, 2 * out, a.q, 2 * q) || overlap(a.out, 2 * out, a.k, 2 * k) || overlap(a.out, 2 * out, a.v, 2 * v)) return I8F_ERR_INVALID;
    if ((a.key_lengths && overlap(a.out, 2 * out, a.key_lengths, length_size * a.batch)) || overlap(a.out, 2 * out, a.key_mask, mask_size * mask)) return I8F_ERR_INVALID;
    return I8F_OK;
}

}  // namespace
}  // namespace i8f

extern "C" int64_t i8f_attention_workspace_bytes(const i8f_attention_args *args) {
    using namespace i8f;
    if (!args || validate(*args) || !args->batch || !args->queries || !args->keys || !args->heads) return 0;
    const i8f_attention_args &a = *args;
    int64_t bytes[3];
    to_pack(a, bytes);
    return plan_of(a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.width).partial_bytes + bytes[0] + bytes[1] + bytes[2];
}

// How a call of these arguments is cut, for tests to know which form they reach: waves of a workgroup, whether they take the states apart, splits
// of the states, the kernel's width.
extern "C" int i8f_internal_attention_plan(const i8f_attention_args *args, int64_t *waves, int64_t *apart, int64_t *splits, int64_t *padded) {
    using namespace i8f;
    if (!args || !waves || !apart || !splits || !padded) return I8F_ERR_INVALID;
    const i8f_attention_args &a = *args;
    if (int rc = validate(a)) return rc;
    if (!a.batch || !a.queries || !a.keys || !a.heads) return I8F_ERR_INVALID;   // (nothing is cut)
    const Plan p = plan_of(a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.width);
    *waves = p.waves, *apart = p.apart, *splits = p.splits, *padded = p.padded;
    return I8F_OK;
}

extern "C" int i8f_attention(const i8f_attention_args *args, void *stream) {
    using namespace i8f;
    if (!args) return I8F_ERR_INVALID;
    const i8f_attention_args &a = *args;
    if (int rc = validate(a)) return rc;
    if (!a.batch || !a.queries || !a.heads) return I8F_OK;
    const int64_t need = i8f_attention_workspace_bytes(args);
    if (need && (!a.workspace || a.workspace_bytes < need || (uintptr_t)a.workspace % 16)) return I8F_ERR_INVALID;
    const Plan plan = plan_of(a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.width);
    const int64_t share = a.heads / a.kv_heads;
    if (int rc = check_device()) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (!a.keys) {
        const int64_t n = a.batch * a.queries * a.heads * a.width, blocks = (n + 2047) / 2048;
        hipLaunchKernelGGL(zeros_kernel, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, (uint16_t *)a.out, n);
        return check_launch();
    }
    Launch p = {a, (uint32_t)share, (uint32_t)(a.queries * share), (uint32_t)plan.row_tiles, (uint32_t)plan.splits, (uint32_t)plan.tiles, (uint32_t)round_up(a.width, 8)};
    p.wide_out = a.width % 8 == 0 && (uintptr_t)a.out % 16 == 0;
    p.by_share = Divisor(p.share), p.by_row_tiles = Divisor(p.row_tiles), p.by_splits = Divisor(p.splits), p.by_kv_heads = Divisor((uint32_t)a.kv_heads);
    p.partial = (float *)a.workspace;
    p.stats = p.partial ? p.partial + plan.partials : nullptr;
    int64_t bytes[3];
    const int which = to_pack(a, bytes);
    if (which) {
        Packs packs = {};
        char *at = (char *)a.workspace + plan.partial_bytes;
        int count = 0;
        int64_t most = 0;
        auto pack = [&](int i, const void *&x, int64_t tokens, int64_t heads, int64_t &batch_stride, int64_t &token_stride, int64_t &head_stride) {
            if (!(which >> i & 1)) return;
            const int64_t padded = round_up(a.width, 8);
            const bool apart = heads * padded > MOST_STRIDE;
            const int64_t out_token = apart ? padded : heads * padded, out_head = apart ? tokens * padded : padded;
            packs.p[count++] = {(const uint16_t *)x, (uint16_t *)at, a.batch * tokens * heads, tokens, heads, batch_stride, token_stride, head_stride, out_token, out_head, (int)a.width, (int)padded};
            x = at, head_stride = out_head, token_stride = out_token, batch_stride = tokens * heads * padded;
            most = bytes[i] > most ? bytes[i] : most;
            at += bytes[i];
        };
        pack(0, p.a.q, a.queries, a.heads, p.a.q_batch, p.a.q_token, p.a.q_head);
        pack(1, p.a.k, a.keys, a.kv_heads, p.a.k_batch, p.a.k_token, p.a.k_head);
        pack(2, p.a.v, a.keys, a.kv_heads, p.a.v_batch, p.a.v_token, p.a.v_head);
        const int64_t blocks = (most / 16 + 255) / 256;
        hipLaunchKernelGGL(pack_kernel, dim3((unsigned)(blocks < 8192 ? blocks : 8192), count), dim3(256), 0, st, packs);
        if (int rc = check_launch()) return rc;
    }
    return a.dtype == I8F_BF16 ? launch<I8F_BF16>(p, plan, st) : launch<I8F_F16>(p, plan, st);
}
