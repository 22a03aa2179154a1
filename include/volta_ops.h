/*
 * volta_ops.h -- operators of a feed-forward block on device tensors: the
 * linear layer, the gated layer, the RMS norm with the residual's addition,
 * and dropout whose mask is drawn from a counter, each with its gradients, in
 * float32, bfloat16 and float16.
 *
 * The training step (volta_train.h) and graph execution (volta_backend.h) run
 * whole MLPs in float32; these calls are single layers of the same kind on
 * the caller's own device buffers, for programs that put a model together
 * themselves:
 *
 *   s = x + r;  n = rms_norm(s);  h = act(n Wg + bg) * (n Wu + bu)
 *   y = s + dropout(h Wd + bd),  or  y = (h Wd + bd) + s in one call
 *
 * Conventions, all calls:
 *   - Matrices are row-major, W is [inputs x outputs] as in the training
 *     step.  ld_* is a matrix's distance between rows in elements; 0 means
 *     packed.  A matrix of rows that overlap (ld below the row's length) is
 *     refused, and so is an ld over 2^21.
 *   - Pointers are device pointers, aligned to their element.  A product's
 *     operands whose rows are 16-byte aligned (pointer and ld) and a multiple
 *     of 16 bytes long take the fast loads; operands of other lengths or ld
 *     are copied into the workspace where that pays, and else read through
 *     registers, as are misaligned pointers.
 *   - The call enqueues its kernels on `stream` (a hipStream_t; NULL: the
 *     default stream) of the current device and returns.  It allocates
 *     nothing and waits for nothing, so it can be captured into a graph.  A
 *     stream or memory of another device is refused, and so is memory that
 *     no device reads or that ends before the matrix does (what follows it
 *     directly in other allocations counts as its own).
 *   - `workspace` is device memory of at least the bytes that the operator's
 *     *_workspace call gives for the same description (0: NULL is fine),
 *     16-byte aligned.  Its contents do not matter before and after.  Calls
 *     that may run at the same time need one each; so do two graphs that may
 *     be replayed at the same time.
 *   - An output must not overlap an input or another output, except where a
 *     call names the two as allowed to be the same matrix.  Column ranges of
 *     one wider matrix (the same ld) do not overlap.
 *   - rows may be 0: nothing is read, outputs of that many rows stay as they
 *     are, and gradients of weights and biases are zero.  Elements between a
 *     row's end and the next row's start (ld > length) are neither read nor
 *     written.
 *   - Sums are held in 32 bits; every result is rounded once, to the nearest
 *     of its type.  Runs are bit-reproducible: no sum's order depends on
 *     timing.
 *   - rows is at most 2^30, every other size 2^21.  A product whose result is
 *     too large for a launch is refused: more than 2^22 of the tiles that its
 *     plan takes, so about 2^28 rows of up to 64 columns at the least.  A call
 *     looks at the products that it runs alone; *_workspace speaks for every
 *     gradient of a backward call and is refused where one of them would be
 *     (the refusal of a call that lacks workspace says how much it takes).
 *   - Returns 0, or -1 with the message in volta_rt_last_error
 *     (volta_backend.h); then nothing was enqueued, unless the message names
 *     a failed launch.
 */
#ifndef VOLTA_OPS_H
#define VOLTA_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
enum volta_op_type {
  VOLTA_OP_F32 = 0,
  VOLTA_OP_BF16 = 1,
  VOLTA_OP_F16 = 2,
  VOLTA_OP_E4M3 = 3 /* output of the norm only: 8 bits, 4 of exponent, largest value 448 */
};

/* Activations: enum volta_activation of volta_train.h without the row
 * softmax, or none. */
#define VOLTA_OP_ACT_NONE (-1)

/* Which call a workspace is for. */
enum volta_op_direction { VOLTA_OP_FORWARD = 0, VOLTA_OP_BACKWARD = 1 };

/* --- linear layer: p = x W + b;  y = act(p) + residual ------------------- */
typedef struct volta_op_linear {
  int32_t type; /* F32, BF16, F16: of every matrix */
  int32_t act;  /* enum volta_activation except softmax, or VOLTA_OP_ACT_NONE */
  int64_t rows, inputs, outputs;
  int64_t ld_x;                       /* [rows x inputs] */
  int64_t ld_w;                       /* [inputs x outputs] */
  int64_t ld_y, ld_residual, ld_pre;  /* [rows x outputs]; ld_y is dy's too */
  int64_t ld_dx, ld_dw;               /* as x and w */
} volta_op_linear;

/* Bytes of workspace of a forward or backward call; -1 for a description
 * that would be refused. */
int64_t volta_op_linear_workspace(const volta_op_linear* d, int32_t direction);

/* y = act(x W + bias) + residual.  bias [outputs], residual and pre may be
 * NULL; pre receives x W + bias, which the backward call of a layer with an
 * activation needs.  residual may be y (the same pointer and ld). */
int32_t volta_op_linear_forward(const volta_op_linear* d, const void* x, const void* w, const void* bias,
                                const void* residual, void* y, void* pre, void* workspace, int64_t workspace_bytes,
                                void* stream);

/* From dy: dp = dy act'(pre); dx = dp W^T; dw = x^T dp; db = the column sums
 * of dp.  The residual's gradient is dy itself.  pre is needed when there is
 * an activation (and not read otherwise); dx, dw, db may be NULL where not
 * wanted (at least one is); x is read for dw, w for dx.  act' is the training
 * step's: 0 at 0 for ReLU.  dp is rounded to the type before its products, as
 * matrix instructions take their operands in it (a half step of each dp, so dx
 * and dw are off by about as much again as by their own rounding), and without
 * loss of range: float16 holds dp in units of a power of two, which puts the
 * largest magnitude of dp in [2^14, 2^15); only what is under 2^-28 of that
 * loses bits.  db sums dp before its rounding. */
int32_t volta_op_linear_backward(const volta_op_linear* d, const void* dy, const void* x, const void* w,
                                 const void* pre, void* dx, void* dw, void* db, void* workspace,
                                 int64_t workspace_bytes, void* stream);

/* --- gated layer: g = x Wg + bg;  u = x Wu + bu;  h = act(g) u ----------- */
typedef struct volta_op_gated {
  int32_t type;
  int32_t act;
  int64_t rows, inputs, hidden;
  int64_t ld_x;          /* [rows x inputs] */
  int64_t ld_w;          /* Wg and Wu, [inputs x hidden] each; 2 hidden for two halves of one matrix */
  int64_t ld_h, ld_pre;  /* [rows x hidden]: h and dh; gate and up */
  int64_t ld_dx, ld_dw;
} volta_op_gated;

int64_t volta_op_gated_workspace(const volta_op_gated* d, int32_t direction);

/* Both products, the activation and the product of the two in one pass.
 * b_gate and b_up [hidden] may be NULL; gate and up, both or neither NULL,
 * receive g and u for the backward call. */
int32_t volta_op_gated_forward(const volta_op_gated* d, const void* x, const void* w_gate, const void* w_up,
                               const void* b_gate, const void* b_up, void* h, void* gate, void* up, void* workspace,
                               int64_t workspace_bytes, void* stream);

/* From dh: dg = dh u act'(g); du = dh act(g); dx = dg Wg^T + du Wu^T;
 * dw_gate = x^T dg; dw_up = x^T du; db_gate, db_up = the column sums.  dx may
 * be NULL; so may dw_gate and dw_up (both or neither), and db_gate and db_up
 * (each).  dg and du are rounded to the type before their products, as dp
 * above (float16: in units common to both). */
int32_t volta_op_gated_backward(const volta_op_gated* d, const void* dh, const void* x, const void* w_gate,
                                const void* w_up, const void* gate, const void* up, void* dx, void* dw_gate,
                                void* dw_up, void* db_gate, void* db_up, void* workspace, int64_t workspace_bytes,
                                void* stream);

/* --- RMS norm: s = x + residual;  rstd = 1 / sqrt(mean(s^2) + eps);
 *               y = s rstd weight --------------------------------------- */
typedef struct volta_op_rms_norm {
  int32_t type;     /* of x, residual, sum, weight and the gradients */
  int32_t out_type; /* of y: type, or VOLTA_OP_E4M3 */
  int64_t rows, cols;
  float eps;        /* >= 0 */
  int32_t group;    /* E4M3: columns that share a scale, 128, or 0 for the whole row */
  int64_t ld_x, ld_residual, ld_sum, ld_y; /* [rows x cols]; backward: s has ld_x, dsum ld_sum, dy ld_y */
  int64_t ld_dx;
} volta_op_rms_norm;

int64_t volta_op_rms_norm_workspace(const volta_op_rms_norm* d, int32_t direction);

/* residual, weight [cols] (NULL: ones), sum and rstd (float [rows]) may be
 * NULL.  sum receives s, and may be x or residual.  y is normalised from s
 * before its rounding to `sum`.  The squares' mean is a float too: of rows past
 * about 1e19 it is infinite, rstd 0 and y 0.  With out_type E4M3, scales receives
 * [rows x ceil(cols / group)] floats, packed (one a row for group 0): for the
 * values v of a group, scale = max(max|v| / 448, 2^-126) and y = e4m3(v * (1 /
 * scale)), so v is about y * scale; a NaN among them makes the scale NaN and
 * the group's codes NaN.  Otherwise scales is NULL. */
int32_t volta_op_rms_norm_forward(const volta_op_rms_norm* d, const void* x, const void* residual,
                                  const void* weight, void* y, void* sum, float* rstd, float* scales, void* stream);

/* From dy, the forward's s (sum, or x without a residual) and rstd:
 * dx = rstd w dy - s rstd^3 mean(w dy s) + dsum (formed without the cube, which
 * leaves 32 bits long before dx does), the gradient of x and of the
 * residual alike; dsum, the gradient that reaches s by the residual stream,
 * may be NULL, and may be dx.  dweight [cols] = the column sums of dy s rstd
 * may be NULL, and so may dx, not both.  out_type and group are not read. */
int32_t volta_op_rms_norm_backward(const volta_op_rms_norm* d, const void* dy, const void* s, const float* rstd,
                                   const void* weight, const void* dsum, void* dx, void* dweight, void* workspace,
                                   int64_t workspace_bytes, void* stream);

/* --- dropout without a stored mask --------------------------------------- */
typedef struct volta_op_dropout {
  int32_t type;
  double p; /* share of elements dropped, 0 <= p < 1 */
  int64_t rows, cols;
  int64_t ld_x, ld_residual, ld_y;
} volta_op_dropout;

/* y = residual + x keep / (1 - p).  Element i = row * cols + col is kept
 * where its 32 bits are at least floor(p 2^32): the low half (even i) or the
 * high half (odd i) of output offset + i/2 of the splitmix64 stream started
 * from `seed` (output n is the mix of seed + (n + 1) 0x9E3779B97F4A7C15, all
 * modulo 2^64).  The same seed and offset draw the same mask, whatever the
 * type and the strides: the backward pass is this call on dy without a
 * residual.  A call uses ceil(rows * cols / 2) outputs.  residual may be
 * NULL; y may be x or residual.  A dropped element of x is not multiplied:
 * an infinity or NaN there does not reach y. */
int32_t volta_op_dropout_forward(const volta_op_dropout* d, const void* x, const void* residual, void* y,
                                 uint64_t seed, uint64_t offset, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* VOLTA_OPS_H */
