// Products whose sums are blended with another matrix, for several matrices at
// once, in float16 and pairs of it (ops_gemm_kernels.h): the update's.
#include "ops_gemm_kernels.h"

namespace volta {
namespace ops {
hipError_t op_gemm_blend(int layout, int kind, const OpPlan& plan, OpGemmMore g, hipStream_t st) {
  using T = _Float16;
  if (kind == OP_MIRROR) {
    if (layout == OP_NN || g.M != g.N) return hipErrorInvalidValue;
    return layout == OP_NT ? launch<T, OP_NT, OP_MIRROR>(plan, g, st) : launch<T, OP_TN, OP_MIRROR>(plan, g, st);
  }
  if (layout == OP_NN) return launch<T, OP_NN, OP_BLEND>(plan, g, st);
  if (layout == OP_NT) return launch<T, OP_NT, OP_BLEND>(plan, g, st);
  return hipErrorInvalidValue;
}
}  // namespace ops
}  // namespace volta
