// How the feed-forward operators launch a kernel (ops_rows.hip,
// ops_gemm_kernels.h).
#pragma once

#include <hip/hip_runtime.h>

namespace volta {
namespace ops {

template <typename P>
struct OpParam {
  typedef P type;
};

// The result is this launch's own.  hipGetLastError, which a launch in the
// triple-bracket form leaves its result in, also returns the error of any
// earlier call of the thread that nobody has read, and the thread is the
// caller's: a call would end between its launches for an error that is none of
// its own, and take that error from the caller.
template <typename... P>
hipError_t op_launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t st, typename OpParam<P>::type... args) {
  void* at[] = {static_cast<void*>(&args)...};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, at, 0, st);
  if (e != hipSuccess) (void)hipGetLastError();  // it is reported to the caller by the return value
  return e;
}

}  // namespace ops
}  // namespace volta
