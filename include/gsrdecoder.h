/* gsrdecoder.h — C ABI of the decoder's operators on MI355X (gfx950),
 * libgsrdecoder.so: rotary positions with several axes, the root-mean-square
 * norm with the residual's addition, and cross attention to an encoder's
 * states, for networks that answer with Gaussians which libgsraster.so renders
 * and trains through.  No counterpart in the reference.
 *
 * Plain pointers and sizes only; tensor arguments are DEVICE pointers, strides
 * count elements and may be zero (a broadcast) or, where not said otherwise,
 * negative; the last dimension is contiguous everywhere.  `stream` is a
 * hipStream_t (NULL = the null stream); all work is enqueued on it, nothing
 * waits, and nothing allocates.
 * Pointers need only their elements' own alignment.
 *
 * Every entry point returns GSR_OK or one of gsraster.h's error codes;
 * gsd_last_error() gives the calling thread's message for the last failure.
 * Outputs are contiguous, fully written by the call and overlap no input.  Calls
 * whose launches would hold 2^32 work-items are refused.
 */
#ifndef GSRDECODER_H
#define GSRDECODER_H

#include <stddef.h>
#include <stdint.h>

#include "gsraster.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GSD_F32 0
#define GSD_BF16 1
#define GSD_F16 2

/* types of rotary positions */
#define GSD_POS_F32 0
#define GSD_POS_I32 1
#define GSD_POS_I64 2

#define GSD_MAX_AXES 8
#define GSD_MAX_NORM_WIDTH 16384
#define GSD_MAX_HEAD_DIM 128
#define GSD_MAX_ATTENTION_STRIDE 16777216 /* of one key to the next, elements */

const char* gsd_last_error(void);
const char* gsd_version(void);

/* Rotary positions with several axes.  x [batch, length, heads, dim], y the
 * same, contiguous.  P = the sum of sections[0 .. axes) pairs of channels are
 * turned, 2 P <= dim: the first sections[0] pairs by the token's position on
 * axis 0, the next sections[1] by axis 1 and so on, pair i by the angle
 * positions[token, axis] * inv_freq[i] (formed in 64 bits):
 *   u' = u cos - w sin,  w' = u sin + w cos
 * with (u, w) = channels (i, i + P), or (2 i, 2 i + 1) when interleaved.
 * Channels from 2 P on are copied.  inverse turns the other way, which is the
 * gradient with respect to x.  positions is indexed by its three strides
 * (batch, token, axis). */
typedef struct gsd_rotary {
    int dtype;
    int64_t batch, length, heads, dim;
    const void* x;
    int64_t x_stride_b, x_stride_l, x_stride_h;
    const void* positions;
    int positions_type;
    int64_t pos_stride_b, pos_stride_l, pos_stride_a;
    int axes;
    int64_t sections[GSD_MAX_AXES];
    const float* inv_freq; /* [P] */
    int interleaved;
    int inverse;
    void* y;
} gsd_rotary;
int gsd_rotary_axes(const gsd_rotary* args, void* stream);

/* The root-mean-square norm with the residual's addition, over rows of `width`
 * (1 .. GSD_MAX_NORM_WIDTH) values:
 *   h = x + residual (residual may be NULL: h = x),
 *   y = h * rstd * weight, rstd = 1 / sqrt(mean(h^2) + eps),
 * in 32 bits, h's 32-bit value entering the norm.  x and residual are rows at
 * x_stride / residual_stride; weight [width] in the same type.  h (may be NULL)
 * is the sum rounded to the type, rstd (may be NULL) [rows] the factor in 32
 * bits; both are what the backward takes.
 * gsd_rms_norm_fp8 writes y8 [rows, width] in 8-bit floats (4 exponent and 3
 * mantissa bits, largest value 448) and scale [rows]: y = y8 * scale, scale =
 * max|y| / 448 of the row (never below 2^-126), 1 for a row without a value above
 * 0. */
typedef struct gsd_norm {
    int dtype;
    int64_t rows, width;
    const void* x;
    int64_t x_stride;
    const void* residual;
    int64_t residual_stride;
    const void* weight;
    double eps;
    void* h;
    float* rstd;
} gsd_norm;
int gsd_rms_norm(const gsd_norm* args, void* y, void* stream);
int gsd_rms_norm_fp8(const gsd_norm* args, uint8_t* y8, float* scale, void* stream);

/* Its backward from h [rows, width] (contiguous, the forward's) and rstd:
 *   g = dy * weight, n = h * rstd,
 *   dx = dh + rstd (g - n mean(n g)),   dweight = sum over rows of dy * n.
 * dy, dh are rows at their strides; dh may be NULL.  dx is the gradient of x
 * and of the residual alike; dx or dweight may be NULL.  The workspace holds
 * dweight's partial sums, added in an order that depends on the sizes alone. */
size_t gsd_rms_norm_backward_workspace_bytes(int64_t rows, int64_t width);
int gsd_rms_norm_backward(int dtype, int64_t rows, int64_t width, const void* h,
                          const float* rstd, const void* weight, const void* dy,
                          int64_t dy_stride, const void* dh, int64_t dh_stride, void* dx,
                          void* dweight, void* ws, size_t ws_bytes, void* stream);

/* Cross attention from `queries` queries to `keys` encoder states.
 * q [batch, queries, heads, dim], k and v [batch, keys, kv_heads, dim], types
 * GSD_BF16 or GSD_F16, dim a multiple of 8 up to GSD_MAX_HEAD_DIM, heads a
 * multiple of kv_heads (query head h reads head h / (heads / kv_heads)).
 *   s = scale q.k over the valid keys, p = softmax(s), o = sum p v.
 * Key j of batch b is valid when j < key_lengths[b] (NULL: keys) and
 * key_mask[b, j] != 0 (NULL: all; bytes at mask_stride_b, mask_stride_s).
 * Nothing that k and v hold at other keys takes part.  A query without a valid
 * key gets o = 0 and gradients 0.  scale is positive.  k_stride_l and v_stride_l
 * lie in [0, GSD_MAX_ATTENTION_STRIDE], and keys times them below 2^30 - 1024 where
 * there is a mask (whose valid keys are listed, and only those read); for the backward, q's and do's strides of
 * queries and heads are not negative, and 65 queries and a group's heads span at
 * most 2^30 elements.
 * o [batch, queries, heads, dim] contiguous; lse (may be NULL when no backward
 * follows) [batch, kv_heads, queries, heads / kv_heads] = log2 sum 2^(s log2 e),
 * -infinity for a query without a valid key.  o_low (may be NULL), laid out as o,
 * is what the rounding of o left out, rounded to the type in its turn: with it the
 * backward forms sum do o from 32-bit values, which matters where a query has few
 * keys (a few dozen).  Sums and statistics are held in 32 bits; p is rounded to the
 * type for its product with v, and with up to 64 valid keys what that leaves out is
 * multiplied too. */
typedef struct gsd_attention {
    int dtype;
    int64_t batch, queries, keys, heads, kv_heads, dim;
    const void* q;
    int64_t q_stride_b, q_stride_l, q_stride_h;
    const void* k;
    int64_t k_stride_b, k_stride_l, k_stride_h;
    const void* v;
    int64_t v_stride_b, v_stride_l, v_stride_h;
    const int32_t* key_lengths;
    const uint8_t* key_mask;
    int64_t mask_stride_b, mask_stride_s;
    float scale;
    void* o;
    float* lse;
    void* o_low;
} gsd_attention;
size_t gsd_attention_workspace_bytes(const gsd_attention* args);
int gsd_cross_attention(const gsd_attention* args, void* ws, size_t ws_bytes, void* stream);

/* Its backward: args as in the forward, with the forward's o, lse and o_low
 * (NULL: the rounded o alone), and do [batch, queries, heads, dim] at its strides.  dq, dk, dv are contiguous;
 * dk and dv sum over the query heads that share a head, and are 0 at keys that
 * are not valid.  dq, or dk and dv together, may be NULL and are then not
 * formed.  No atomics: the result does not depend on scheduling. */
typedef struct gsd_attention_grad {
    const void* d_o;
    int64_t do_stride_b, do_stride_l, do_stride_h;
    void* dq;
    void* dk;
    void* dv;
} gsd_attention_grad;
size_t gsd_attention_backward_workspace_bytes(const gsd_attention* args);
int gsd_cross_attention_backward(const gsd_attention* args, const gsd_attention_grad* grad,
                                 void* ws, size_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GSRDECODER_H */
