// The feed-forward operators' matrix products in f16 (ops_gemm_kernels.h).
#include "ops_gemm_kernels.h"

namespace volta {
namespace ops {
hipError_t op_gemm_f16(int layout, int kind, const OpPlan& plan, OpGemm g, hipStream_t st) {
  return op_gemm<_Float16>(layout, kind, plan, g, st);
}
}  // namespace ops
}  // namespace volta
