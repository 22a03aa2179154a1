// Products of e4m3 codes with results in f16 (ops_gemm8_kernels.h).
#include "ops_gemm8_kernels.h"

namespace volta {
namespace ops {
hipError_t op_gemm8_f16(const OpPlan& plan, OpGemmMore g, hipStream_t st) { return launch8<_Float16>(plan, g, st); }
}  // namespace ops
}  // namespace volta
