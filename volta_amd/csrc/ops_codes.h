// e4m3 codes of values and the scale of a group of them, as the norm and the
// quantization leave them.
#pragma once

#include "ops_types.h"

namespace volta {
namespace ops {

typedef uint32_t chunk8_by1 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t chunk4_by1 __attribute__((aligned(1)));

// E (4 or 8) values as e4m3 codes, to the nearest.
template <int E>
__device__ __forceinline__ void store_codes(uint8_t* p, int cnt, const float (&f)[E]) {
  union { uint32_t w[E / 4]; uint8_t b[E]; } u;
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], w, true);
    u.w[i] = (uint32_t)w;
  }
  if (cnt >= E) {
    if constexpr (E == 8) *(VOLTA_GLOBAL chunk8_by1*)p = chunk8_by1{u.w[0], u.w[1]};
    else *(VOLTA_GLOBAL chunk4_by1*)p = u.w[0];
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < cnt) ((VOLTA_GLOBAL uint8_t*)p)[i] = u.b[i];
  }
}

// The larger of two magnitudes; a NaN stays.
__device__ __forceinline__ float max_or_nan(float m, float v) { return v > m || v != v ? v : m; }

constexpr float kE4m3Max = 448.0f;
constexpr float kTiny = 1.17549435e-38f;  // 2^-126
__device__ __forceinline__ float scale_of(float largest) {
  const float q = largest / kE4m3Max;
  return q < kTiny ? kTiny : q;
}

}  // namespace ops
}  // namespace volta
