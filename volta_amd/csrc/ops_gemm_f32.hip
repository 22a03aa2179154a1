// The feed-forward operators' matrix products in f32 (ops_gemm_kernels.h).
#include "ops_gemm_kernels.h"

namespace volta {
namespace ops {
hipError_t op_gemm_f32(int layout, int kind, const OpPlan& plan, OpGemm g, hipStream_t st) {
  return op_gemm<float>(layout, kind, plan, g, st);
}
}  // namespace ops
}  // namespace volta
