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

// What becomes of the sums.
enum OpKind {
  OP_LINEAR = 0,  // act(d + bias) + residual; d + bias kept on request
  OP_GATED = 1,   // two products of one P: act(d0 + b0) * (d1 + b1)
  OP_STORE = 2    // the sums themselves
};

struct OpEpilogue {
  int32_t act;
  const void* bias[2];
  const void* residual;
  void* out[2];  // OP_STORE: one for each q (blockIdx.z)
  void* pre[2];
  int64_t ld_out, ld_residual, ld_pre;
  const float* unit;  // OP_STORE in float16: one number on the device, what the sums are multiplied by; NULL: 1
};

struct OpGemm {
  const void* p[2];  // pieces of the sum over k (dx of the gated layer has two)
  const void* q[2];  // OP_NT: the piece's Q; OP_GATED: gate and up; OP_TN: one for each output
  int64_t ld_p, ld_q;
  int32_t M, N, K;   // K of one piece
  int32_t pieces;    // 1 or 2 pieces of the sum
  int32_t outputs;   // 1 or 2 outputs (OP_STORE of OP_TN)
  int32_t direct;    // rows of P and Q are 16-byte aligned and whole 16-byte chunks long
  // from the plan
  int32_t tiles_m, tiles_n;
  int32_t splits, stages_per_split;
  float* partial;    // splits > 1: [split][output or gate/up][M][N]
  OpEpilogue epi;
};

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

}  // namespace ops
}  // namespace volta
