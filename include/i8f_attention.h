/*
 * What lies between the projections of an attention block, beside the layers of i8f.h and with its conventions (device pointers owned by
 * the caller, the caller's stream, negative i8f_status on errors, arguments checked on the host before anything is launched): the norm of
 * every head of queries and keys, the rotation by their positions, and the attention over an encoder's states.  Every pointer lies on an element of
 * its type, and no result on an input.
 */
#ifndef I8F_ATTENTION_H
#define I8F_ATTENTION_H

#include "i8f.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Heads [batch, tokens, heads, width], the last dimension contiguous, strides in elements, none negative.
 */
typedef struct i8f_heads {
    const void *x;
    int64_t batch_stride, token_stride, head_stride;
    int64_t heads;
    const void *weight;        /* [width] of weight_dtype, or NULL */
    int weight_dtype;          /* dtype or I8F_F32 */
    void *out;                 /* [batch, tokens, heads, width] of dtype, contiguous */
} i8f_heads;

/*
 * For every head x of width elements, of up to I8F_MAX_HEAD_GROUPS tensors of the same tokens:
 *   y = x / sqrt(sum x^2 / width + eps) * weight      with norm (y = x without; a weight goes with a norm)
 *   out = y with its pairs turned by the token's positions, rounded once; everything in binary32
 * Pair j of `pairs` is elements (2j, 2j + 1), or with `apart` (j, j + pairs); elements 2 pairs ... width - 1 are not turned.  Its angle is
 * rates[j] turns to a unit of position axis a, first_pair[a] <= j < first_pair[a + 1], taken in binary64: position and rate are exact in it
 * and a whole number of turns is taken off before it is rounded to binary32.
 *   rates      [pairs] binary64, turns to a unit; pairs = first_pair[axes], 2 pairs <= width
 *   positions  of positions_type, element strides position_batch, position_token, position_axis (the batch's may be 0)
 * axes 0: nothing is turned.  width up to 256, batch * tokens below 2^31.  The outputs overlap neither the inputs nor one another.
 */
#define I8F_MAX_HEAD_GROUPS 4
#define I8F_MAX_AXES 4
typedef enum i8f_position { I8F_POSITION_I32 = 0, I8F_POSITION_I64 = 1, I8F_POSITION_F32 = 2, I8F_POSITION_F64 = 3 } i8f_position;
typedef struct i8f_norm_rotate_args {
    int64_t batch, tokens, width;
    int dtype;
    int norm;
    float eps;
    int axes;
    int first_pair[I8F_MAX_AXES + 1];
    int apart;
    int positions_type;
    const double *rates;
    const void *positions;
    int64_t position_batch, position_token, position_axis;
} i8f_norm_rotate_args;
int i8f_norm_rotate(const i8f_norm_rotate_args *args, const i8f_heads *groups, int n_groups, void *stream);

/*
 * out[b, i, h] = sum_j e^s_ij v[b, j, g] / sum_j e^s_ij,   s_ij = scale q[b, i, h] . k[b, j, g] + m_bj,   g = h / (heads / kv_heads)
 * over the states j that count: j < key_lengths[b] where there are lengths, and of a mask those whose byte is not 0, or whose addend m is
 * above the lowest value of its type.  A row over which no state counts is zeros, and so is one of a finite query whose scores are all -inf;
 * what the states that do not count hold is not looked at.  Finite scores and addends of any size are the formula's; a score that passes binary32
 * upwards gives NaN.  Bfloat16 values up to 2^127 / keys cannot overflow the sums.
 * Products of dtype, sums, maximum and exponentials in binary32, e^s rounded to dtype for the second product, one rounding at the end.
 *   q, k, v      [batch, queries or keys, heads or kv_heads, width] of dtype (I8F_BF16 or I8F_F16), last dimension contiguous, strides in
 *                elements, none negative; width up to 256, heads a multiple of kv_heads
 *   out          [batch, queries, heads, width], contiguous; overlaps no input
 *   key_lengths  [batch] of int32 (lengths_type 0) or int64 (1), or NULL; values outside 0 ... keys count as the nearer of the two
 *   key_mask     NULL or element (b, j) at mask_batch b + mask_key j of mask_type
 *   scale        positive, at most 2^126
 *   workspace    any contents, 16-byte aligned, i8f_attention_workspace_bytes() of these arguments (which looks at all but workspace and
 *                key_lengths' and key_mask's contents); less, or NULL, is refused where that is not 0.  It overlaps nothing else, and calls that overlap in
 *                time do not share it.
 * batch * queries * heads is below 2^31, keys at most 2^30, batch * keys * kv_heads at most 2^49; more workgroups than a launch has (2^24 of 128 rows, of 32 where there are fewer) are
 * I8F_ERR_UNSUPPORTED.
 */
typedef enum i8f_key_mask { I8F_MASK_BYTES = 0, I8F_MASK_BF16 = 1, I8F_MASK_F16 = 2, I8F_MASK_F32 = 3 } i8f_key_mask;
typedef struct i8f_attention_args {
    const void *q, *k, *v;
    void *out;
    int64_t batch, queries, keys, heads, kv_heads, width;
    int64_t q_batch, q_token, q_head, k_batch, k_token, k_head, v_batch, v_token, v_head;
    int dtype;
    float scale;
    const void *key_lengths;
    int lengths_type;
    int mask_type;
    const void *key_mask;
    int64_t mask_batch, mask_key;
    void *workspace;
    int64_t workspace_bytes;
} i8f_attention_args;
int64_t i8f_attention_workspace_bytes(const i8f_attention_args *args);
int i8f_attention(const i8f_attention_args *args, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* I8F_ATTENTION_H */
