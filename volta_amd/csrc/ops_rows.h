// Row and element kernels of the feed-forward operators (include/volta_ops.h):
// the RMS norm, dropout, and what the layers' gradients need before their
// products (ops_rows.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/volta_ops.h"

namespace volta {
namespace ops {

struct NormArgs {
  const void *x, *residual, *weight;
  void *y, *sum;
  float *rstd, *scales;
  int64_t rows;
  int32_t cols, group;  // group: columns of a scale (cols for one a row)
  int64_t ld_x, ld_residual, ld_y, ld_sum;
  float eps;
};
hipError_t norm_forward(int type, bool e4m3, const NormArgs& a, hipStream_t st);

struct NormGradArgs {
  const void *dy, *s, *weight, *dsum;
  const float* rstd;
  void* dx;
  float* partial;  // [norm_grad_blocks][cols] where dweight is wanted, else NULL
  int64_t rows;
  int32_t cols;
  int64_t ld_dy, ld_s, ld_dsum, ld_dx;
};
// Blocks of the gradient's launch: the rows of its partial sums of dweight.
int norm_grad_blocks(int type, int64_t rows, int64_t cols);
hipError_t norm_backward(int type, const NormGradArgs& a, hipStream_t st);

// out[c] = the sum over i < n of partial[i][c], in order, rounded to the type;
// up to two such sums.
struct SumArgs {
  const float* partial[2];
  void* out[2];
  int32_t count, n;
  int64_t cols;
};
hipError_t sum_partials(int type, const SumArgs& a, hipStream_t st);

struct ActGradArgs {
  const void* dy;
  const void* pre[2];  // gated: gate and up
  void* d[2];          // dp, or dg and du, or NULL: column sums of dy alone
  void* sums[2];       // column sums of dp, or of dg and du, rounded to the type; NULL where not wanted
  float* partial[2];   // for each that is wanted, [act_grad_strips][cols] (0 of them: not read)
  float* unit;         // float16: [act_grad_units]; unit[0] receives what 1 in d stands for.  NULL: 1
  int32_t act;
  int64_t rows;
  int32_t cols;
  int64_t ld_dy, ld_pre;
  int64_t ld_d;        // whole 16-byte chunks; what a row's last chunk has behind its columns is set to 0
};
// Rows of partial sums; 0 where the sums need none.
int act_grad_strips(int type, int64_t rows, int64_t cols);
// Floats of `unit`; 0 where the type needs none.
int64_t act_grad_units(int type, int64_t rows, int64_t cols);
hipError_t act_grad(int type, bool gated, const ActGradArgs& a, hipStream_t st);

// Copies up to three matrices into rows of whole 16-byte chunks, zeros behind
// a row's columns.
struct PackArgs {
  const void* from[3];
  void* to[3];
  int64_t rows[3], ld_from[3], ld_to[3];
  int32_t cols[3];
  int32_t n;
};
hipError_t pack_rows(int type, const PackArgs& a, hipStream_t st);

struct DropoutArgs {
  const void *x, *residual;
  void* y;
  int64_t rows, cols;
  int64_t ld_x, ld_residual, ld_y;
  uint64_t seed, offset;
  uint32_t threshold;
  float scale;
};
hipError_t dropout_forward(int type, const DropoutArgs& a, hipStream_t st);

}  // namespace ops
}  // namespace volta
