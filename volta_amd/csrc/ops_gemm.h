// Matrix products of the feed-forward operators (include/volta_ops.h):
// D[m][n] = sum over k of P[m][k] Q[k][n] on the gfx950 matrix cores, with the
// layers' epilogues.  What a launch computes, and the plan that picks its
// tile; the kernels are in ops_gemm_kernels.h, instantiated once per element
// type (ops_gemm_f32.hip, ops_gemm_bf16.hip, ops_gemm_f16.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace volta {
namespace ops {

// Operand layouts: the forward product reads x with k contiguous and W with
// the columns contiguous; dx reads both with k contiguous; dW both with the
// rows or columns contiguous.
enum OpLayout { OP_NN = 0, OP_NT = 1, OP_TN = 2 };

// A blend's output as two float16 planes, the value's and its rest's: 23 bits.
constexpr int OP_PLANES = 16;

// What becomes of the sums.
enum OpKind {
  OP_LINEAR = 0,  // act(d + bias) + residual; d + bias kept on request
  OP_GATED = 1,   // two products of one P: act(d0 + b0) * (d1 + b1)
  OP_STORE = 2,   // the sums themselves
  // the loss of an output layer (ops_loss.hip); z = d + bias
  OP_STATS = 3,      // of a row's z: their largest, the sum of their exponentials, the one at the row's label
  OP_LOSS_GRAD = 4,  // (exp(z - lse) - [the label's]) dloss
  OP_ADD = 5,        // sums of several launches, in order, in 32 bits
  OP_BLEND = 6,      // alpha d + beta r + gamma w, of several matrices
  OP_MIRROR = 7      // the same of a symmetric D and r: the tiles on and over the diagonal, stored twice
};
constexpr bool op_kind_blend(int kind) { return kind == OP_BLEND || kind == OP_MIRROR; }
constexpr bool op_kind_layer(int kind) { return kind == OP_LINEAR || kind == OP_GATED; }

struct OpEpilogue {
  int32_t act;
  const void* bias[2];
  const void* residual;
  void* out[2];  // OP_STORE: one for each q (blockIdx.z)
  void* pre[2];
  int64_t ld_out, ld_residual, ld_pre;
  const float* unit;  // OP_STORE in 16 bits: one number on the device, what the sums are multiplied by; NULL: 1
};

// What the kinds from OP_STATS on and the products of codes take besides; the
// others' launches are not to carry it (0.3 us of a small one).
struct OpEpilogueMore : OpEpilogue {
  // OP_STATS, OP_LOSS_GRAD.  The launch's columns are the classes class0 ..
  // class0 + classes - 1; what D has behind them is padding: no part of the
  // statistics, a gradient of 0.
  const int32_t* labels;  // a row's class; < 0: none.  OP_STATS: NULL, none has one
  int32_t class0, classes, all_classes;
  float* stats;           // OP_STATS: [op_stats_entries][M] of {largest, sum of exp(z - largest)}
  float* at_label;        // OP_STATS: [M]
  const float *lse, *dloss;  // OP_LOSS_GRAD: [M]; unit[1] (NULL: 1) multiplies the 16-bit gradient
  int32_t rest_rows;  // and, of 16 bits: rows behind a row that what its rounding leaves goes; 0: nowhere
  // OP_ADD: d + add (NULL: d); to sum, or where it is NULL to out
  const float* add;
  float* sum;
  int64_t ld_sum;  // of both
  // products of e4m3 codes: the scale of row m and k block b at sx[m ld_sx + b
  // step_sx], of columns n and block b at sw[n / 128 ld_sw + b]
  const float *sx, *sw;
  int64_t ld_sx, step_sx, ld_sw;
  // OP_BLEND; matrix z starts z strides behind the first
  // r of the products' type, in aligned rows of whole 16-byte chunks, w of out's
  // (NULL: none)
  const void *blend, *w;
  float alpha, beta, gamma;
  float diagonal;         // OP_MIRROR with an r: added where the row is the column
  int64_t plane_blend, plane_out;  // of r and, with out_type OP_PLANES, of out: elements to the second plane; r: 0, none
  int32_t out_type;       // enum volta_op_type; also of a product of codes
  int64_t ld_blend, ld_w, stride_blend, stride_w, stride_out;
  int64_t stride_p, stride_q;  // OP_BLEND: elements from one matrix to the next
  // OP_BLEND with 3 pieces: P and Q are sums of two planes, the second (the
  // rests) so many elements behind the first: second by first, first by second,
  // then first by first, so that the small sums are rounded while they are small.
  // One piece: 0
  int64_t plane_p, plane_q;
  // OP_BLEND and OP_MIRROR of one plane: what a factor's diagonal is beyond the
  // float16 that holds it, stride_diag floats a matrix.  diag times r, the other
  // factor, joins the sum: by rows where P's (diag_rows), by columns where Q's
  // diagonal it is.  OP_MIRROR: diag2 times blend2, laid out as r is, too, each of
  // them the mean of by rows and by columns (the product turned round), times
  // diag_weight (2 for a square, which has no diag2); and r's own diagonal has
  // diag.  diag_out: the result's.
  const void* blend2;
  const float *diag, *diag2;
  float* diag_out;
  int64_t stride_diag;
  float diag_weight;
  int32_t diag_rows;
};

template <typename E>
struct OpGemmOf {
  const void* p[2];  // pieces of the sum over k (dx of the gated layer has two)
  const void* q[2];  // OP_NT: the piece's Q; OP_GATED: gate and up; OP_TN: one for each output
  int64_t ld_p, ld_q;
  int32_t M, N, K;   // K of one piece
  int32_t pieces;    // 1 or 2 pieces of the sum; OP_BLEND: 1 or 3
  int32_t outputs;   // 1 or 2 outputs (OP_STORE of OP_TN); OP_BLEND: matrices
  int32_t direct;    // rows of P and Q are 16-byte aligned and whole 16-byte chunks long
  // from the plan
  int32_t tiles_m, tiles_n;
  int32_t splits, stages_per_split;
  float* partial;    // splits > 1: [split][output or gate/up][M][N]
  E epi;
};
using OpGemm = OpGemmOf<OpEpilogue>;
using OpGemmMore = OpGemmOf<OpEpilogueMore>;

// Tiles, by rows x columns of D (gated: half the columns of each weight
// matrix).  The skinny ones take 16, 32 or 64 rows and 32 columns (of each
// weight matrix), the sum over k shared out over a block's waves.
enum OpTile {
  OP_TILE_256 = 0,
  OP_TILE_256X128 = 1,
  OP_TILE_128 = 2,
  OP_TILE_64X128 = 3,
  OP_TILE_64 = 4,
  OP_TILE_SKINNY16 = 5,
  OP_TILE_SKINNY32 = 6,
  OP_TILE_SKINNY64 = 7,
  OP_TILES = 8
};

struct OpPlan {
  int32_t tile;
  int32_t splits;
  int32_t stages_per_split;
  double us;  // what the model gives it
};

// k elements of one stage (128 bytes of every row).
inline int op_stage_k(int elem_bytes) { return 128 / elem_bytes; }

// The plan of a product.  A rule on sizes and type alone, so that the
// workspace can be asked for without a device.
OpPlan op_gemm_plan(int elem_bytes, int layout, int kind, int64_t M, int64_t N, int64_t K, int pieces, int outputs,
                    bool direct);
// Whether it pays to lay out operands of `pack_bytes` anew, in rows of whole
// 16-byte chunks, for the direct loads.
bool op_gemm_pack(int elem_bytes, int layout, int kind, int64_t M, int64_t N, int64_t K, int pieces, int outputs,
                  int64_t pack_bytes);
// Bytes of partial sums that the plan needs.
int64_t op_gemm_partial_bytes(const OpPlan& plan, int kind, int64_t M, int64_t N, int outputs);

// Tiles of D, each a block (of every split and output).
int64_t op_gemm_blocks(const OpPlan& plan, int kind, int64_t M, int64_t N);

// Enqueues the product as planned (and the launch that adds the partial sums).
hipError_t op_gemm_f32(int layout, int kind, const OpPlan& plan, OpGemm g, hipStream_t st);
hipError_t op_gemm_bf16(int layout, int kind, const OpPlan& plan, OpGemm g, hipStream_t st);
hipError_t op_gemm_f16(int layout, int kind, const OpPlan& plan, OpGemm g, hipStream_t st);
// The kinds of an output layer's loss; and OP_BLEND and OP_MIRROR, in float16.
hipError_t op_gemm_loss_f32(int layout, int kind, const OpPlan& plan, OpGemmMore g, hipStream_t st);
hipError_t op_gemm_loss_bf16(int layout, int kind, const OpPlan& plan, OpGemmMore g, hipStream_t st);
hipError_t op_gemm_loss_f16(int layout, int kind, const OpPlan& plan, OpGemmMore g, hipStream_t st);
hipError_t op_gemm_blend(int layout, int kind, const OpPlan& plan, OpGemmMore g, hipStream_t st);

// Products of e4m3 codes (OP_NT, OP_LINEAR), by the type of bias, residual and
// result.
hipError_t op_gemm8_f32(const OpPlan& plan, OpGemmMore g, hipStream_t st);
hipError_t op_gemm8_bf16(const OpPlan& plan, OpGemmMore g, hipStream_t st);
hipError_t op_gemm8_f16(const OpPlan& plan, OpGemmMore g, hipStream_t st);

// Entries of a row in OP_STATS' statistics.
int64_t op_stats_entries(const OpPlan& plan, int64_t N);

}  // namespace ops
}  // namespace volta
