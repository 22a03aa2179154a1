// Element types of the feed-forward operators (include/volta_ops.h): storage,
// conversions, vector accesses, and their matrix instruction.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/volta_ops.h"
#include "device_common.h"

namespace volta {
namespace ops {

typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

// 16 bytes of a fragment or a chunk, whatever they hold.
typedef uint32_t chunk16 __attribute__((ext_vector_type(4)));

template <typename T> __device__ __forceinline__ float to_f(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T from_f(float x) { return (T)x; }  // to the nearest, ties to even

// N consecutive elements of a row as floats, N a power of two, at any element
// address (the memory pipeline takes unaligned accesses of up to 16 bytes);
// only the first cnt are inside the row: the rest reads 0 and is not written.
#define VOLTA_GLOBAL __attribute__((address_space(1)))
template <int BYTES, int ALIGN> struct Access;
#define VOLTA_ACCESS(BYTES, ALIGN, BASE, N) \
  template <> struct Access<BYTES, ALIGN> { typedef BASE type __attribute__((ext_vector_type(N), aligned(ALIGN))); }
VOLTA_ACCESS(16, 4, uint32_t, 4);
VOLTA_ACCESS(16, 2, uint32_t, 4);
VOLTA_ACCESS(8, 4, uint32_t, 2);
VOLTA_ACCESS(8, 2, uint32_t, 2);
VOLTA_ACCESS(4, 2, uint32_t, 1);
#undef VOLTA_ACCESS
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, int cnt, float (&f)[N]) {
  constexpr int B = N * (int)sizeof(T) < 16 ? N * (int)sizeof(T) : 16, E = B / (int)sizeof(T);
  typedef typename Access<B, sizeof(T)>::type V;
  if (cnt >= N) {
#pragma unroll
    for (int c = 0; c < N / E; ++c) {
      union { V v; T e[E]; } u;
      u.v = *(const VOLTA_GLOBAL V*)(p + c * E);
#pragma unroll
      for (int i = 0; i < E; ++i) f[c * E + i] = to_f(u.e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = i < cnt ? to_f(((const VOLTA_GLOBAL T*)p)[i]) : 0.0f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, int cnt, const float (&f)[N]) {
  constexpr int B = N * (int)sizeof(T) < 16 ? N * (int)sizeof(T) : 16, E = B / (int)sizeof(T);
  typedef typename Access<B, sizeof(T)>::type V;
  if (cnt >= N) {
#pragma unroll
    for (int c = 0; c < N / E; ++c) {
      union { V v; T e[E]; } u;
#pragma unroll
      for (int i = 0; i < E; ++i) u.e[i] = from_f<T>(f[c * E + i]);
      *(VOLTA_GLOBAL V*)(p + c * E) = u.v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < cnt) ((VOLTA_GLOBAL T*)p)[i] = from_f<T>(f[i]);
  }
}

// f(x) and f'(x) of the layers' activations.  float32 results take the
// training step's own functions (device_common.h).  16-bit results need a
// relative error well under 2^-9 only: the hardware's exp2 and reciprocal (one
// unit in the last place of 32 bits each) instead of the library's functions
// and IEEE division, which would cost a gated layer's epilogue a fifth of its
// products' time.  tanh(v) = 1 - 2 / (1 + e^2v) cancels near 0, where its
// series takes over (|v| < 1/4: the next term, 17/315 v^7, is 1.3e-5 of v).
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ float fast_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-x)); }
__device__ __forceinline__ float fast_tanh(float v) {
  const float big = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + fast_exp(2.0f * v));
  const float v2 = v * v;
  const float small = v * (1.0f - v2 * (0.333333333f - 0.133333333f * v2));
  return fabsf(v) < 0.25f ? small : big;
}
constexpr float kGeluC = 0.7978845608f, kGeluK = 0.044715f;

template <typename T>
__device__ __forceinline__ float op_act(int act, float x) {
  if constexpr (sizeof(T) == 4) {
    return act_forward(act, x);
  } else {
    switch (act) {
      case VOLTA_ACT_RELU: return x > 0.0f ? x : 0.0f;
      case VOLTA_ACT_SIGMOID: return fast_sigmoid(x);
      case VOLTA_ACT_TANH: return fast_tanh(x);
      case VOLTA_ACT_LEAKY_RELU: return x > 0.0f ? x : 0.01f * x;
      case VOLTA_ACT_SILU: return x * fast_sigmoid(x);
      // 0.5 x (1 + tanh v) = x sigmoid(2v)
      case VOLTA_ACT_GELU: return x * fast_sigmoid(2.0f * kGeluC * (x + kGeluK * x * x * x));
      default: return x;
    }
  }
}

// f of N values: the activation is asked once.
template <typename T, int N>
__device__ __forceinline__ void op_act_all(int act, float (&x)[N]) {
#define VOLTA_ACT_ALL(A)                                       \
  case A:                                                   \
    _Pragma("unroll") for (int i = 0; i < N; ++i) x[i] = op_act<T>(A, x[i]); \
    break
  switch (act) {
    VOLTA_ACT_ALL(VOLTA_ACT_RELU);
    VOLTA_ACT_ALL(VOLTA_ACT_SIGMOID);
    VOLTA_ACT_ALL(VOLTA_ACT_TANH);
    VOLTA_ACT_ALL(VOLTA_ACT_LEAKY_RELU);
    VOLTA_ACT_ALL(VOLTA_ACT_SILU);
    VOLTA_ACT_ALL(VOLTA_ACT_GELU);
    default: break;
  }
#undef VOLTA_ACT_ALL
}

// Where GELU's slope is 1 or 0 to the last bit of 32: from there on x^2 has no
// say in it, and past 2^64, where x^2 is infinite, would make it 0 times that.
// A NaN stays.
__device__ __forceinline__ float gelu_slope_at(float x) { return fabsf(x) > 32.0f ? copysignf(32.0f, x) : x; }

// f and f' together (the gated layer's gradient needs both).
template <typename T>
__device__ __forceinline__ void op_act_both(int act, float x, float* f, float* slope) {
  if constexpr (sizeof(T) == 4) {
    *f = act_forward(act, x);
    *slope = act == VOLTA_ACT_RELU ? (x > 0.0f ? 1.0f : 0.0f)
                                   : act_derivative(act, act == VOLTA_ACT_GELU ? gelu_slope_at(x) : x, *f);
  } else {
    switch (act) {
      case VOLTA_ACT_RELU:
        *f = x > 0.0f ? x : 0.0f;
        *slope = x > 0.0f ? 1.0f : 0.0f;
        break;
      case VOLTA_ACT_SIGMOID: {
        const float q = fast_sigmoid(x);
        *f = q;
        *slope = q * fast_sigmoid(-x);
        break;
      }
      case VOLTA_ACT_TANH: {
        // 1 - tanh^2 = 4 q (1 - q), q = sigmoid(2x)
        *f = fast_tanh(x);
        *slope = 4.0f * fast_sigmoid(2.0f * x) * fast_sigmoid(-2.0f * x);
        break;
      }
      case VOLTA_ACT_LEAKY_RELU:
        *f = x > 0.0f ? x : 0.01f * x;
        *slope = x > 0.0f ? 1.0f : 0.01f;
        break;
      case VOLTA_ACT_SILU: {
        const float q = fast_sigmoid(x);
        *f = x * q;
        *slope = q + x * q * fast_sigmoid(-x);
        break;
      }
      case VOLTA_ACT_GELU: {
        const float s = gelu_slope_at(x);
        const float v2 = 2.0f * kGeluC * (s + kGeluK * s * s * s);
        const float q = fast_sigmoid(v2);
        *f = x * q;
        *slope = q + s * q * fast_sigmoid(-v2) * 2.0f * kGeluC * (1.0f + 3.0f * kGeluK * s * s);
        break;
      }
      default:
        *f = x;
        *slope = 1.0f;
    }
  }
}

}  // namespace ops
}  // namespace volta
