// The products of an output layer's loss in f32 (ops_gemm_kernels.h).
#include "ops_gemm_kernels.h"

namespace volta {
namespace ops {
hipError_t op_gemm_loss_f32(int layout, int kind, const OpPlan& plan, OpGemmMore g, hipStream_t st) {
  return op_gemm_loss<float>(layout, kind, plan, g, st);
}
}  // namespace ops
}  // namespace volta
