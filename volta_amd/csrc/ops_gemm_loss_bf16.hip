// The products of an output layer's loss in bf16 (ops_gemm_kernels.h).
#include "ops_gemm_kernels.h"

namespace volta {
namespace ops {
hipError_t op_gemm_loss_bf16(int layout, int kind, const OpPlan& plan, OpGemmMore g, hipStream_t st) {
  return op_gemm_loss<__bf16>(layout, kind, plan, g, st);
}
}  // namespace ops
}  // namespace volta
