// Products of e4m3 codes with results in f32 (ops_gemm8_kernels.h).
#include "ops_gemm8_kernels.h"

namespace volta {
namespace ops {
hipError_t op_gemm8_f32(const OpPlan& plan, OpGemmMore g, hipStream_t st) { return launch8<float>(plan, g, st); }
}  // namespace ops
}  // namespace volta
