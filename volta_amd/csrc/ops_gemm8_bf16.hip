// Products of e4m3 codes with results in bf16 (ops_gemm8_kernels.h).
#include "ops_gemm8_kernels.h"

namespace volta {
namespace ops {
hipError_t op_gemm8_bf16(const OpPlan& plan, OpGemmMore g, hipStream_t st) { return launch8<__bf16>(plan, g, st); }
}  // namespace ops
}  // namespace volta
