/*
 * The operators around a quantised projection when one model serves many requests, beside the layers of i8f.h and with its
 * conventions (device pointers owned by the caller, row-major matrices, the caller's stream, negative i8f_status on errors, arguments
 * checked on the host before anything is launched): low-rank adapters that differ from row to row, and what lies between two blocks of
 * a model that normalises a block's output.
 */
#ifndef I8F_BLOCKS_H
#define I8F_BLOCKS_H

#include "i8f.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * The adapters of one layer and which of them each row takes.  Adapter a has rank r_a, padded with zeros to a multiple of 16 in
 * memory: its padded ranks are first_rank[a] ... first_rank[a + 1] - 1.  Row m takes adapter ids[m / rows_per_id], none where that is
 * not one of 0 ... count - 1.  All pointers are device pointers; the factors have the type of the activations (bfloat16 or binary16).
 */
typedef struct i8f_adapters {
    const void *down;          /* [first_rank[count], K]: the adapters' A one below the other, each row padded with zeros to a multiple of
                                  eight elements in memory */
    const void *up;            /* adapter a: B as [N, padded r_a] from element N * first_rank[a] on */
    const float *scale;        /* [count] multiplies A x */
    const int32_t *first_rank; /* [count + 1], multiples of 16, first_rank[0] = 0 */
    const int32_t *ids;        /* [ceil(M / rows_per_id)] */
    int64_t rows_per_id;
    int64_t count;
    int64_t max_rank;          /* the largest padded rank: a multiple of 16, the row stride of t */
} i8f_adapters;

/*
 * A layer and its adapters.  Layers of one call read the same rows, and their adapters have the same ids and rows_per_id.
 */
#define I8F_MAX_ADAPTED_LAYERS 4
typedef struct i8f_adapted_layer {
    const int8_t *w;           /* [N,K] int8, with w_scale [N] float (I8F_SCALE_ROW) or one scale: w_scale[0], or w_scale_host where it is NULL */
    const float *w_scale;
    float w_scale_host;
    int scale_mode;
    const void *bias;          /* [N] of bias_dtype or NULL */
    int bias_dtype;
    int64_t N;
    i8f_adapters adapters;
    void *t;                   /* [M, max_rank] of the activations' type: the adapters' first product */
    float *side;               /* NULL, or [M,N]: the adapters' whole share of the result, see i8f_adapters_down */
    void *out;                 /* [M,N] of the activations' type */
} i8f_adapted_layer;

/*
 * Whether M rows of a W8A8 layer with K inputs and N outputs are better served by way of `side` (few rows, which may all have different
 * adapters: their share is then computed by a launch of its own that fills the chip).
 */
int i8f_adapters_by_side(int64_t M, int64_t N, int64_t K, int64_t rows_per_id);

/*
 * t[m, 0 ... r) = scale_a * A_a x[m] of every layer, for the adapter a of row m and its padded rank r: sums in binary32, one rounding to
 * x's type (what the matrix unit multiplies with in the second product; binary16 ends at 65504 and has fewer bits below 2^-14, so a
 * caller lets the largest element of B be about 1 there and puts the rest into the scale); ranks beyond r and rows without an adapter are
 * left as they are.  Of the layers only adapters, t, side and, with it, N are looked at.
 * Layers with a side get side[m,n] = sum_j t[m,j] B_a[n,j] in binary32 besides (zeros for rows without an adapter); i8f_linear_w8a8_adapters
 * then adds that instead of reading t.  N is then a multiple of 8.  All layers of a call or none.  x_dtype I8F_BF16 or I8F_F16, n_layers up to I8F_MAX_ADAPTED_LAYERS.
 * q, scale: NULL, or the int8 rows of x and their scales besides, as i8f_quant_rowwise with rotate_block leaves them (the adapters take
 * x as it is).
 * workspace: any contents; i8f_adapters_down_workspace_bytes(M, K, the sum of the layers' max_rank, x_aligned) bytes let many rows' columns
 * be dealt over more workgroups, and rows that are not 16-byte aligned (x_aligned 0: x, or ldx in elements, is no multiple of 16 bytes) be
 * copied; less, or NULL, is slower there and rounds otherwise in the last place of the binary32 sums.
 */
int64_t i8f_adapters_down_workspace_bytes(int64_t M, int64_t K, int64_t ranks, int x_aligned);
int i8f_adapters_down(const void *x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const i8f_adapted_layer *layers, int n_layers,
                      int rotate_block, int8_t *q, float *scale, void *workspace, int64_t workspace_bytes, void *stream);

/*
 * out[m,n] = round(base[m,n] + sum_j t[m,j] B_a[n,j]); base [M,N] of base_dtype, which is I8F_F32 or out_dtype; out may be base then.
 */
int i8f_adapters_up(const void *base, int base_dtype, const i8f_adapters *adapters, const void *t, void *out, int out_dtype, int64_t M,
                    int64_t N, void *stream);

/*
 * i8f_linear_w8a8 of every layer with its adapters' second product in the epilogue, in the operation order I8F_EPI_FUSED and rounded once:
 *   out[m,n] = round(acc * (a_scale[m] * w_scale[n]) + bias[n] + sum_j t[m,j] B_a[n,j])
 * t as i8f_adapters_down leaves it; out_dtype is the factors'.  Rows without an adapter get i8f_linear_w8a8's result in that order, bit
 * for bit.  workspace: any contents, at least i8f_linear_w8a8_adapters_workspace_bytes(M, N, K) for the layer that needs most (shapes
 * that the tiled kernels do not take; 0 else).  I8F_ERR_UNSUPPORTED for operands of the other shapes that are not 16-byte aligned: the
 * caller then takes i8f_linear_w8a8 in binary32 and i8f_adapters_up.
 */
int64_t i8f_linear_w8a8_adapters_workspace_bytes(int64_t M, int64_t N, int64_t K);
int i8f_linear_w8a8_adapters(const int8_t *a, const float *a_scale, const i8f_adapted_layer *layers, int n_layers, int out_dtype, int64_t M,
                             int64_t K, void *workspace, int64_t workspace_bytes, void *stream);

/*
 * i8f_linear_w8a16_small_m (M <= 16) of every layer with its adapters' second product added before its one rounding.  x_dtype is the
 * factors' type.
 */
int i8f_linear_w8a16_small_m_adapters(const void *x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const i8f_adapted_layer *layers,
                                      int n_layers, void *stream);

/*
 * From a block's output y and the residual stream r to the residual stream x behind the block and the input h of the next one:
 *   x = residual_scale * r + branch_scale * g * norm_post(y)        g = gate, tanh(gate) or 1
 *   h = norm_pre(x) * (1 + mod_scale) + mod_shift                   each part where it is given
 * with norm(z) = z / sqrt(sum z^2 / K + eps) * weight + bias (I8F_NORM_RMS), the same of z - sum z / K (I8F_NORM_LAYER) or z
 * (I8F_NORM_NONE).  Everything in binary32 from the first load on, the statistics of x before its rounding among it; x and h are
 * rounded once, when they are stored.
 *   y, residual   [M,K] of dtype, row strides ldy, ldr      x_out   [M,K], contiguous
 *   h        [M,K] or NULL
 *   q, scale [M,K] int8 and [M] or NULL: i8f_quant_rowwise of the rounded h with rotate_block, without h in memory (where h is not
 *            given).  At most one of h and q.  pre_norm must be I8F_NORM_NONE, and the modulation absent, where both are NULL.
 *   weights and biases [K] of dtype or I8F_F32 (post_dtype, pre_dtype), each NULL when absent; an I8F_NORM_NONE has neither
 *   gate, mod_scale, mod_shift   [ceil(M / rows_per_...), K] of dtype or NULL; row m uses vector m / rows_per_...
 * The outputs may overlap neither the inputs nor one another.
 */
typedef enum i8f_norm { I8F_NORM_NONE = 0, I8F_NORM_RMS = 1, I8F_NORM_LAYER = 2 } i8f_norm;
typedef struct i8f_block_norm_args {
    const void *y, *residual;
    int64_t M, K, ldy, ldr;
    int dtype;
    int post_norm, post_dtype, pre_norm, pre_dtype;
    float post_eps, pre_eps;
    const void *post_weight, *post_bias, *pre_weight, *pre_bias;
    const void *gate;
    int64_t rows_per_gate;
    int gate_tanh;
    float residual_scale, branch_scale;
    const void *mod_scale, *mod_shift;
    int64_t rows_per_scale, rows_per_shift;
    void *x_out, *h;
    int8_t *q;
    float *scale;
    int rotate_block;
} i8f_block_norm_args;
int i8f_block_norm(const i8f_block_norm_args *args, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* I8F_BLOCKS_H */
