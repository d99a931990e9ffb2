/*
 * dsca_b200 — operators around the MoE block of a decode step (C ABI, companion of dsca_b200.h,
 * whose conventions hold here: plain device pointers, sizes and a CUDA stream, an int status, no
 * allocation; all pointers of one call belong to the current device).
 *
 * dsca_rms_norm       the norm in front of the block, with the residual's addition and 8-bit rows
 * dsca_moe_few        the whole block for at most DSCA_FEW_TOKENS tokens in one kernel
 */
#ifndef DSCA_B200_BLOCK_H_
#define DSCA_B200_BLOCK_H_

#include "dsca_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 8-bit output of dsca_rms_norm */
enum { DSCA_NORM_Q_NONE = 0, DSCA_NORM_Q_E4M3 = 1, DSCA_NORM_Q_SPLIT = 2 };
/* Largest row the norm holds in one CTA's registers. */
#define DSCA_NORM_MAX_D 32768

/*
 * h = round(x + residual) (x itself without a residual), y = weight * h / sqrt(mean(h^2) + eps).
 * h is rounded to dtype before it is squared; the sum and y are fp32, y rounded once when stored.
 * quant:
 *   DSCA_NORM_Q_E4M3   q [rows, d] e4m3 = RN(y / s) of the unrounded y, scale[row] = s = max|y| / 448
 *                      (1 for a row of zeros; 2^-149 at least; NaN for a row with a NaN);
 *   DSCA_NORM_Q_SPLIT  q [rows, 2 * Kd] (Kd = d rounded up to 128) and scale[row] = 1 / s exactly as
 *                      dsca_split_rows writes them from the rounded y.  dtype DSCA_BF16, d % 8 == 0,
 *                      q 8-byte aligned and the rows of y and residual_out 16-byte aligned.
 * Any d from 1 to DSCA_NORM_MAX_D and any row strides (in elements, >= d); d % 8 == 0 with 16-byte
 * aligned rows takes the vector path.  y or residual_out may be the same rows as x or residual
 * (same pointer and stride); other overlaps are not supported.
 */
typedef struct {
  const void* x;              /* [rows, d], dtype */
  const void* residual;       /* [rows, d], dtype, or NULL */
  const void* weight;         /* [d], weight_dtype */
  int rows, d;
  int dtype;                  /* DSCA_BF16 or DSCA_F32 */
  int weight_dtype;           /* dtype, or DSCA_F32 */
  int64_t ld_x, ld_residual, ld_y, ld_residual_out; /* row strides in elements */
  float eps;
  int quant;                  /* DSCA_NORM_Q_* */
  void* y;                    /* [rows, d], dtype, or NULL (only the 8-bit rows are wanted) */
  void* residual_out;         /* [rows, d], dtype: h, or NULL */
  void* q;                    /* see quant */
  float* scale;               /* [rows] */
} dsca_rms_norm_args;
DSCA_API int dsca_rms_norm(const dsca_rms_norm_args* a, dsca_stream_t stream);

/* Tokens one dsca_moe_few call takes at most. */
#define DSCA_FEW_TOKENS 32
/* Bytes at the start of its workspace that are zero between calls (counters). */
#define DSCA_FEW_ZERO_BYTES 1024

/*
 * The whole MoE block for a few tokens, one kernel: router, softmax, top-k, the chosen experts'
 * FFNs, the gated shared expert and the weighted sum (dsca_router_topk, dsca_permute,
 * dsca_grouped_ffn and dsca_combine in one, for a call whose time is the reading of the weights).
 *   logits = round(x W_r^T), summed in 64 bits and rounded to fp32, then to the type; probabilities, ties and weights as dsca_router_topk
 *   out    = round(sum_j w_j down(act(up x)) + sigmoid(round(x . g)) shared(x)), summed in fp32;
 *            the activated intermediate is held to 16 significant bits (DSCA_F32: fp32; DSCA_F8E4M3: 11 bits, or 2^-16
 *            of the largest value of its token's row in that expert where that is more, for rows whose largest
 *            value is at least 2^-58 of what the scales allow: max(s_gate s_up) (448 sum|x|)^2 with SwiGLU,
 *            max(s) 448 sum|x| with ReLU)
 * Weights in the packing of dsca_ffn_args.  weights: DSCA_BF16 or DSCA_F32 (x, router and out in the
 * same type), or DSCA_F8E4M3 with the four scale arrays (x, router and out bf16).
 * d * (bytes of a weight) must be a multiple of 16 and every weight matrix 16-byte aligned.
 * workspace: dsca_few_workspace_bytes() bytes, 256-byte aligned, the first DSCA_FEW_ZERO_BYTES zero
 * before the first call; every call leaves them zero.  Calls that may overlap on the GPU must not
 * share a workspace.
 * The kernel's CTAs wait for one another, so it is launched cooperatively, one CTA per SM.  Each wait ends after
 * wait_limit_ns: the call then ends too, with DSCA_ERR_WAIT_TIMEOUT in err (dsca_check_error) and results of no
 * meaning, and the bytes above have to be zeroed again.
 */
typedef struct {
  const void* x;              /* [T, d] contiguous, 16-byte aligned */
  const void* w_router;       /* [E, d] */
  const void* w_shared_gate;  /* [d], or NULL (no shared expert) */
  int T, d, E, top_k;
  int weights;                /* DSCA_BF16, DSCA_F32 or DSCA_F8E4M3 */
  int mode;                   /* DSCA_ROUTE_* */
  int norm_topk;              /* as dsca_router_args */
  int act;                    /* DSCA_ACT_* */
  int inter, n1p, ip, dp;     /* routed experts: channels, packed rows of w1, row length and rows of w2 */
  int shared_inter, shared_n1p, shared_ip;  /* shared expert (0 without one) */
  const void* w1;             /* [E, n1p, d] */
  const void* w2;             /* [E, dp, ip] */
  const void* ws1;            /* [shared_n1p, d] */
  const void* ws2;            /* [dp, shared_ip] */
  const float* w1_scale;      /* DSCA_F8E4M3: one scale per packed row, else NULL */
  const float* w2_scale;
  const float* ws1_scale;
  const float* ws2_scale;
  float w1_max;               /* DSCA_F8E4M3: not read (0, or any finite value that is not negative) */
  void* out;                  /* [T, d] */
  void* logits;               /* [T, E] */
  int32_t* topk_ids;          /* [T, top_k] */
  float* topk_w;              /* [T, top_k] */
  int64_t* expert_index;      /* [T] first choice, or NULL */
  void* workspace;
  size_t workspace_bytes;
  int32_t* err;               /* device error word */
  uint64_t wait_limit_ns;     /* limit of each of the kernel's waits; 0: 2 s */
} dsca_few_args;
DSCA_API size_t dsca_few_workspace_bytes(int T, int d, int top_k, int inter, int shared_inter);
DSCA_API int dsca_moe_few(const dsca_few_args* a, dsca_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DSCA_B200_BLOCK_H_ */
