/*
 * dsca_b200 — the dense gated feed-forward block and 8-bit integer products (C ABI, companion of
 * dsca_b200.h, whose conventions hold here: plain device pointers, sizes and a CUDA stream, an int
 * status, no allocation; all pointers of one call belong to the current device).
 *
 * dsca_gated_ffn            y = (act(x Wg^T) * (x Wu^T)) Wd^T
 * dsca_gated_ffn_backward   its gradients
 * dsca_quantize_rows        rows in 8-bit integers, one scale a row
 * dsca_int8_linear          y = x W^T with both in 8-bit integers, scales for each token and channel
 * dsca_gated_ffn_int8       the gated block with 8-bit integer weights
 *
 * DSCA_F32 products hold every value as three bf16 terms, 24 bits in all; magnitudes below 2^-100 keep fewer (the third
 * term becomes subnormal), which is below 2^-116 in absolute terms.  An infinite value makes its sums NaN (a term of it meets
 * zero terms of the other side).
 *
 * 16-bit sums of one sign are off by up to 2^-11 of themselves before they are rounded (the tensor cores' additions truncate;
 * every 65536 of k they are added up in rounded fp32).
 *
 * Matrices are row-major with row strides in elements (ld_*, at least the width) and a contiguous
 * last dimension; weights lie as a Linear layer holds them, [out, in].  Any sizes; rows on 16-byte
 * boundaries are taken as they lie, others are copied into the workspace first.
 */
#ifndef DSCA_B200_DENSE_H_
#define DSCA_B200_DENSE_H_

#include "dsca_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* act of the gate */
enum { DSCA_GATE_SILU = 0, DSCA_GATE_GELU = 1 /* tanh form */, DSCA_GATE_RELU = 2 };
/* Largest width (d, inter, k, n) and number of rows of these entry points. */
#define DSCA_DENSE_MAX_DIM 1048576
#define DSCA_DENSE_MAX_ROWS 16777216
/* Forward calls need no workspace for at most this many rows, whatever the sizes of their weights.  (The bytes are those up to
 * which the calls promised it before.) */
#define DSCA_DENSE_FEW_TOKENS 8
#define DSCA_DENSE_FEW_BYTES 50331648

/*
 * g = x Wg^T, u = x Wu^T, h = act(g) * u, y = h Wd^T; sums in fp32, h and y rounded to dtype.  g and u
 * are written when given (both or neither), for the backward pass: in fp32 for DSCA_F32; for DSCA_BF16 as
 * fp16 times a power of two for a few channels of a token, whose exponents gu_exp takes.  h is a work area [rows, ld_h] that the backward pass reads as well.
 */
typedef struct {
  const void* x;        /* [rows, d], dtype */
  const void* w_gate;   /* [inter, d] */
  const void* w_up;     /* [inter, d] */
  const void* w_down;   /* [d, inter] */
  void* y;              /* [rows, d] */
  void* g;              /* [rows, ld_h] fp32 or fp16, or NULL */
  void* u;
  uint8_t* gu_exp;      /* [2, rows, 4 * ceil(inter / 32)], 4-byte aligned; with DSCA_BF16 and g */
  void* h;              /* [rows, ld_h] */
  int rows, d, inter;
  int dtype;            /* DSCA_BF16, DSCA_F32 */
  int act;              /* DSCA_GATE_* */
  int64_t ld_x, ld_gate, ld_up, ld_down, ld_y;
  int64_t ld_h;         /* of g, u, h, in elements: rows of h a multiple of 16 bytes apart, at least inter; g, u, h 16-byte aligned */
  void* workspace;      /* dsca_gated_ffn_workspace(), 256-byte aligned; may be NULL when that is 0 */
  size_t workspace_bytes;
  int32_t* err;
} dsca_gated_ffn_args;

/*
 * dh = dy Wd, dg = dh * u * act'(g), du = dh * act(g), dx = dg Wg + du Wu, d_gate = dg^T x,
 * d_up = du^T x, d_down = dy^T h; sums in fp32, dg, du and the gradients rounded to dtype.  Gradients
 * that are NULL are not computed.  dg and du are work areas like h.  rows = 0 writes zeros to the
 * weights' gradients.
 */
typedef struct {
  const void* x;
  const void* w_gate;
  const void* w_up;
  const void* w_down;
  const void* dy;       /* [rows, d] */
  const void* g;        /* as dsca_gated_ffn wrote them */
  const void* u;
  const uint8_t* gu_exp;
  const void* h;
  void* dx;             /* [rows, d] contiguous, or NULL */
  void* d_gate;         /* [inter, d] contiguous, or NULL */
  void* d_up;
  void* d_down;         /* [d, inter] contiguous, or NULL */
  void* dg;             /* [rows, ld_h] */
  void* du;
  int rows, d, inter, dtype, act;
  int64_t ld_x, ld_gate, ld_up, ld_down, ld_dy, ld_h;
  void* workspace;
  size_t workspace_bytes;
  int32_t* err;
} dsca_gated_ffn_backward_args;

/*
 * Codes lie in [-127, 127].  scale[row] = max|x| / 127 (1 for a row of zeros), q = the quotient 127 x / max|x| rounded to the
 * nearest integer, ties to even, exactly.  A row with an infinity or a NaN has that as its scale and
 * codes of no meaning.  Columns [k, ld_q) of q are written as zeros.
 */
typedef struct {
  const void* x;        /* [rows, k], dtype DSCA_BF16 or DSCA_F32 */
  int rows, k, dtype;
  int64_t ld_x;
  int8_t* q;            /* [rows, ld_q], 16-byte aligned */
  int64_t ld_q;         /* a multiple of 16, at least k */
  float* scale;         /* [rows] */
} dsca_quantize_rows_args;

/*
 * y = (q w^T) * w_scale[column] * scale[row] (+ bias): the sum exact in 32-bit integers, its conversion, the products with the two
 * scales and the addition in fp32, the result rounded to dtype.  DSCA_F32: the smaller scale first; DSCA_BF16: the column's
 * first, so that a column's scale above 2^97 may make y infinite where the row's would bring it back.  With x, q and scale are work areas that dsca_quantize_rows of x fills first.
 */
typedef struct {
  const void* x;        /* [rows, k], dtype, or NULL: q and scale are given */
  int8_t* q;            /* [rows, ld_q] */
  float* scale;         /* [rows] */
  const int8_t* w;      /* [n, ld_w], 16-byte aligned; columns [k, ld_w) of w and q do not count, up to whole 16 bytes they are read */
  const float* w_scale; /* [n] */
  const void* bias;     /* [n], dtype, or NULL */
  void* y;              /* [rows, n], dtype */
  int rows, k, n, dtype;
  int64_t ld_x, ld_q, ld_w, ld_y; /* ld_q, ld_w: multiples of 16 */
  void* workspace;
  size_t workspace_bytes;
  int32_t* err;
} dsca_int8_linear_args;

/*
 * dsca_gated_ffn with its weights in 8-bit integers: x quantised by rows, h = act(g) * u in fp32 (a work area), quantised by
 * rows, then the down product.  DSCA_F32: the codes of h are those of its 64-bit value (from the exact sums and the scale
 * max|x| / 127 unrounded).  DSCA_BF16: they are those of the fp32 value, whose gate is good to 2^-18, so that a code next to a border
 * may lie on its other side.
 */
typedef struct {
  const void* x;        /* [rows, d], dtype */
  int8_t* q;            /* work area [rows, ld_q] */
  float* scale;         /* work area [rows] (DSCA_BF16: the rows' scales, DSCA_F32: their largest magnitudes) */
  const int8_t* w_gate; /* [inter, ld_gate], 16-byte aligned; columns past d do not count */
  const int8_t* w_up;
  const int8_t* w_down; /* [d, ld_down] */
  const float* gate_scale; /* [inter] */
  const float* up_scale;
  const float* down_scale; /* [d] */
  float* h;             /* work area [rows, ld_h] */
  int8_t* hq;           /* work area [rows, ld_hq] */
  float* h_scale;       /* work area [rows] */
  void* y;              /* [rows, d], dtype */
  int rows, d, inter, dtype, act;
  int64_t ld_x, ld_q, ld_gate, ld_up, ld_down, ld_h, ld_hq, ld_y; /* ld_h: a multiple of 4; 8-bit ones of 16 */
  void* workspace;
  size_t workspace_bytes;
  int32_t* err;
} dsca_gated_ffn_int8_args;

DSCA_API int dsca_gated_ffn(const dsca_gated_ffn_args* args, dsca_stream_t stream);
DSCA_API int dsca_gated_ffn_backward(const dsca_gated_ffn_backward_args* args, dsca_stream_t stream);
DSCA_API int dsca_quantize_rows(const dsca_quantize_rows_args* args, dsca_stream_t stream);
DSCA_API int dsca_int8_linear(const dsca_int8_linear_args* args, dsca_stream_t stream);
DSCA_API int dsca_gated_ffn_int8(const dsca_gated_ffn_int8_args* args, dsca_stream_t stream);

/* Bytes of workspace that a call with these arguments needs on the current device (the workspace fields
 * are not read); 0 also for arguments that the call refuses. */
DSCA_API size_t dsca_gated_ffn_workspace(const dsca_gated_ffn_args* args);
DSCA_API size_t dsca_gated_ffn_backward_workspace(const dsca_gated_ffn_backward_args* args);
DSCA_API size_t dsca_int8_linear_workspace(const dsca_int8_linear_args* args);
DSCA_API size_t dsca_gated_ffn_int8_workspace(const dsca_gated_ffn_int8_args* args);

#ifdef __cplusplus
}
#endif
#endif /* DSCA_B200_DENSE_H_ */
