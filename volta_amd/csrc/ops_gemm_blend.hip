// Products whose sums are blended with another matrix, for several matrices at
// once, in float32 and float16 (ops_gemm_kernels.h): the update's.
#include "ops_gemm_kernels.h"

namespace volta {
namespace ops {
namespace {
template <typename T>
hipError_t blend(int layout, int kind, const OpPlan& plan, OpGemm& g, hipStream_t st) {
  if (kind == OP_MIRROR) {
    if (layout == OP_NN || g.M != g.N) return hipErrorInvalidValue;
    return layout == OP_NT ? launch<T, OP_NT, OP_MIRROR>(plan, g, st) : launch<T, OP_TN, OP_MIRROR>(plan, g, st);
  }
  if (layout == OP_NN) return launch<T, OP_NN, OP_BLEND>(plan, g, st);
  if (layout == OP_NT) return launch<T, OP_NT, OP_BLEND>(plan, g, st);
  return hipErrorInvalidValue;
}
}  // namespace
hipError_t op_gemm_blend(int type, int layout, int kind, const OpPlan& plan, OpGemm g, hipStream_t st) {
  return type == VOLTA_OP_F32 ? blend<float>(layout, kind, plan, g, st) : blend<_Float16>(layout, kind, plan, g, st);
}
}  // namespace ops
}  // namespace volta
