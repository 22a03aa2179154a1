// Kernels of ops_gemm.h for one element type.
//
// D is computed in blocks of 16x16 by the matrix instruction with Q as its
// first operand and P as its second, so that a lane of the result holds four
// consecutive columns of one row: rows are stored 4 elements at a time, and
// the epilogue reads bias and residual the same way.
//
// LDS.  A stage holds 128 bytes of k (64 elements of 16 bits, 32 of float) of
// every row of the operand's tile, in 16-byte chunks that one load instruction
// writes in lane order (global_load_lds, 1 KB a wave).  What is permuted is
// the global address a lane reads, so that the reads hit all banks:
//   k contiguous ("KC"): [row][8 chunks]; chunk c of row r at c ^ (r/2 & 7).
//     A fragment is one chunk of 16 rows: two rows span the 64 banks, and the
//     8 pairs read 8 different chunks.
//   row/column contiguous ("MC"): [k][C columns], in blocks of 16 columns;
//     block b of row k at b ^ f(k).  16-bit fragments are read transposed
//     (ds_read_b64_tr_b16: 16 lanes hand in 4 k-rows of 16 columns, each gets
//     its column's 4 k); 32 lanes touch k-rows {0..3, 8..11} of one block, and
//     f spreads these 8 over the banks.  Floats are read one by one, four
//     k-rows 4 apart.
// Rows that are not 16-byte aligned, or not whole chunks long, take the same
// layouts through registers (the STAGED forms): loads at any element address,
// elements past a row's end read as 0.
//
// Rows of P and columns of Q past the matrix's end read its last row or chunk
// again (their sums are not stored); k past the end reads zeros, in both
// operands, so that whatever stands behind a row's end has no say.
#pragma once

#include <algorithm>
#include <type_traits>

#include "ops_gemm.h"
#include "ops_launch.h"
#include "ops_types.h"

namespace volta {
namespace ops {

typedef __attribute__((address_space(3))) shortx4* LdsShort4;

// What a direct load reads where k is past the end.
static __device__ const __attribute__((aligned(16))) uint32_t op_zeros[4] = {0, 0, 0, 0};

template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
  static constexpr int kSteps = 1;
  static __device__ __forceinline__ floatx4 mul(int, chunk16 a, chunk16 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
};
template <> struct Mfma<_Float16> {
  static constexpr int kSteps = 1;
  static __device__ __forceinline__ floatx4 mul(int, chunk16 a, chunk16 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0,
                                                  0, 0);
  }
};
// Float fragments take four instructions: lane group g holds k = 4g .. 4g + 3
// of 16, and step j takes 4g + j.  They are issued step by step over all
// blocks, not block by block: one that adds to the sum of the one before it
// waits for it.
template <> struct Mfma<float> {
  static constexpr int kSteps = 4;
  static __device__ __forceinline__ floatx4 mul(int step, chunk16 a, chunk16 b, floatx4 c) {
    const floatx4 x = __builtin_bit_cast(floatx4, a), y = __builtin_bit_cast(floatx4, b);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(x[step], y[step], c, 0, 0, 0);
  }
};

// 16 bytes at any element address.
template <typename T>
__device__ __forceinline__ chunk16 load_unaligned(const T* p) {
  return *(const VOLTA_GLOBAL typename Access<16, sizeof(T)>::type*)p;
}
// The first `cnt` elements of a chunk, the rest 0.
template <typename T>
__device__ __forceinline__ chunk16 load_part(const T* p, int cnt) {
  constexpr int E = 16 / sizeof(T);
  union { chunk16 c; T e[E]; } u;
#pragma unroll
  for (int i = 0; i < E; ++i) u.e[i] = i < cnt ? ((const VOLTA_GLOBAL T*)p)[i] : (T)0.0f;
  return u.c;
}

// 16 bytes a lane from global memory to LDS, lane after lane from byte `lds`
// on; nothing passes through registers.  Written as asm because the compiler
// keeps apart only a few such loads: with a ring of stages it no longer knows
// which of them a read of LDS depends on, and waits for all before each read.
// The kernels wait themselves (op_wait_loads), by counting: loads return in
// order.  M0 takes a cycle to reach the load.  The compiler warns that it does
// not preserve M0 around asm; it has nothing there: it writes M0 for indexed
// registers, messages and its own loads of this kind, directly before each, and
// these kernels have none of them (their assembly has M0 in these lines alone).
__device__ __forceinline__ void op_load_lds(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds)),
               "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void op_load_lds(const char* from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(
                   __builtin_amdgcn_readfirstlane(lds)),
               "v"(from)
               : "memory", "m0");
}
__device__ __forceinline__ uint32_t op_lds_byte(const char* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// One operand's tile of one stage: R rows (KC) or R columns (MC), loaded by NW
// waves.  `off` are the byte offsets of this lane's chunks from the stage's
// base address; 32 bits hold them (ld is at most 2^21 elements and a tile has
// at most 256 rows).
template <typename T, int R, bool KC, int NW>
struct Tile {
  static constexpr int kElem = sizeof(T);
  static constexpr int kE = 16 / kElem;              // elements of a chunk
  static constexpr int kStageK = 128 / kElem;
  static constexpr int kBytes = R * 128;
  static constexpr int kLoads = kBytes / 1024 / NW;  // load instructions of a wave
  static_assert(kLoads * NW * 1024 == kBytes, "whole load instructions");
  static constexpr int kRowChunks = KC ? 8 : R / kE; // chunks of a row (KC) or a k-row (MC)
  static constexpr int kBlockChunks = 16 / kE;       // chunks of a block of 16 columns

  // MC: where block b of k-row k stands.
  static __device__ __forceinline__ int swizzle(int k) {
    if constexpr (kElem == 4) return R >= 64 ? (k >> 2) & 3 : (k >> 2) & 1;
    else if constexpr (R >= 128) return (k & 3) | ((k >> 3) & 1) << 2;
    else if constexpr (R == 64) return ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
    else return (k >> 3) & 1;
  }
  // KC: row and k-chunk, MC: k-row and column chunk, of chunk `slot` of the tile.
  static __device__ __forceinline__ void place(int slot, int* row, int* chunk) {
    const int r = slot / kRowChunks, c = slot % kRowChunks;
    *row = r;
    if constexpr (KC) *chunk = c ^ ((r >> 1) & 7);
    else *chunk = ((c / kBlockChunks) ^ swizzle(r)) * kBlockChunks + c % kBlockChunks;
  }

  uint32_t off[kLoads];

  // `left`: rows (KC) or columns (MC) of the matrix from the tile's first one on, at least 1.
  __device__ __forceinline__ void init(int64_t ld, int left, int wave, int lane) {
#pragma unroll
    for (int t = 0; t < kLoads; ++t) {
      int r, c;
      place((wave + t * NW) * 64 + lane, &r, &c);
      if constexpr (KC) r = min(r, left - 1);
      else c = min(c, (left + kE - 1) / kE - 1);
      off[t] = (uint32_t)r * (uint32_t)(ld * kElem) + (uint32_t)c * 16u;
    }
  }

  // Direct: the stage at `base`, whose k are all inside, or the first `k_left` of them.
  __device__ __forceinline__ void issue(const char* base, uint32_t lds, int wave) const {
#pragma unroll
    for (int t = 0; t < kLoads; ++t) op_load_lds(base, off[t], lds + (wave + t * NW) * 1024);
  }
  __device__ __forceinline__ void issue_tail(const char* base, uint32_t lds, int wave, int lane, int k_left) const {
#pragma unroll
    for (int t = 0; t < kLoads; ++t) {
      int r, c;
      place((wave + t * NW) * 64 + lane, &r, &c);
      const bool in = KC ? c * kE < k_left : r < k_left;
      op_load_lds(in ? base + off[t] : reinterpret_cast<const char*>(op_zeros), lds + (wave + t * NW) * 1024);
    }
  }

  // Staged: to registers, element-exact, then to LDS.
  __device__ __forceinline__ void fetch(const char* base, chunk16 (&reg)[kLoads], int wave, int lane, int left,
                                        int k_left) const {
#pragma unroll
    for (int t = 0; t < kLoads; ++t) {
      int r, c;
      place((wave + t * NW) * 64 + lane, &r, &c);
      const T* a = reinterpret_cast<const T*>(base + off[t]);
      int have;  // elements of the chunk inside the matrix (off clamps a chunk behind the last column to the last)
      if constexpr (KC) have = k_left - c * kE;
      else have = r < k_left ? left - min(c, (left + kE - 1) / kE - 1) * kE : 0;
      if (have >= kE) reg[t] = load_unaligned(a);
      else if (have <= 0) reg[t] = chunk16{0, 0, 0, 0};
      else reg[t] = load_part(a, have);
    }
  }
  __device__ __forceinline__ void put(const chunk16 (&reg)[kLoads], char* lds, int wave, int lane) const {
#pragma unroll
    for (int t = 0; t < kLoads; ++t)
      *reinterpret_cast<chunk16*>(lds + (wave + t * NW) * 1024 + lane * 16) = reg[t];
  }

  // The fragment of rows/columns x0 .. x0 + 15 and k-step kk (of two): lane l
  // gets chunk l/16 of row (column) l % 16.
  static __device__ __forceinline__ chunk16 frag(const char* tile, int x0, int kk, int lane) {
    const int l = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      return *reinterpret_cast<const chunk16*>(tile + x0 * 128 + l * 128 + (((4 * kk + g) ^ (l >> 1)) << 4));
    } else if constexpr (kElem == 2) {
      union { chunk16 c; shortx4 s[2]; } u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = 32 * kk + 8 * g + 4 * h + (l >> 2);
        const char* a = tile + k * (R * 2) + (((x0 >> 4) ^ swizzle(k)) << 5) + (l & 3) * 8;
        u.s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4)a);
      }
      return u.c;
    } else {
      union { chunk16 c; float f[4]; } u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = 16 * kk + 4 * g + j;
        u.f[j] = *reinterpret_cast<const float*>(tile + k * (R * 4) + (((x0 >> 4) ^ swizzle(k)) << 6) + l * 4);
      }
      return u.c;
    }
  }
};

template <typename T>
__device__ __forceinline__ float op_exp(float x) {
  if constexpr (sizeof(T) == 4) return expf(x);
  else return fast_exp(x);
}

// Where a blend goes: in the output's type, w of which joins it last.
template <int V>
__device__ __forceinline__ void op_blend_out(const OpEpilogueMore& e, int z, int64_t m, int n, int cnt, float (&d)[V]) {
  auto put = [&](auto like) {
    using U = decltype(like);
    if (e.w) {
      float w[V];
      load_vec(static_cast<const U*>(e.w) + z * e.stride_w + m * e.ld_w + n, cnt, w);
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] += e.gamma * w[i];
    }
    store_vec(static_cast<U*>(e.out[0]) + z * e.stride_out + m * e.ld_out + n, cnt, d);
  };
  if (e.out_type == OP_PLANES) {
    _Float16* out = static_cast<_Float16*>(e.out[0]) + z * e.stride_out + m * e.ld_out + n;
    float rest[V];
#pragma unroll
    for (int i = 0; i < V; ++i) rest[i] = d[i] - to_f(from_f<_Float16>(d[i]));  // exact
    store_vec(out, cnt, d);
    store_vec(out + e.plane_out, cnt, rest);
  } else if (e.out_type == VOLTA_OP_F32) put(0.0f);
  else if (e.out_type == VOLTA_OP_BF16) put((__bf16)0.0f);
  else put((_Float16)0.0f);
}

template <int V>
struct OpHalves {
  typedef _Float16 type __attribute__((ext_vector_type(V)));
};
// The sums, V columns n .. of row m, to what a blend makes of them.
template <int KIND, int V>
__device__ __forceinline__ void op_blend(const OpEpilogueMore& e, int z, int64_t m, int n, int cnt, float (&d)[V]) {
  if (!e.blend && !e.diag_out) {  // what follows would cost 4 us of 27 (16 matrices, 512 x 2000)
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] *= e.alpha;
    return;
  }
  using Halves = typename OpHalves<V>::type;
  const int64_t here = z * e.stride_blend + m * e.ld_blend + n;
  const _Float16* from = static_cast<const _Float16*>(e.blend);
  const _Float16* beside = e.plane_blend ? from + e.plane_blend : static_cast<const _Float16*>(e.blend2);
  Halves first{}, second{};  // r, and its second plane or the other factor
  if (from) first = *reinterpret_cast<const Halves*>(from + here);
  if (beside) second = *reinterpret_cast<const Halves*>(beside + here);
  float more = 0.0f;
  if (e.diag) {
    const bool columns = KIND == OP_MIRROR || !e.diag_rows;
    const float weight = KIND == OP_MIRROR ? 0.5f * e.diag_weight : 1.0f;
    float by[2][V];
#pragma unroll
    for (int i = 0; i < V; ++i) by[0][i] = by[1][i] = 0.0f;
    if (columns) load_vec(e.diag + z * e.stride_diag + n, cnt, by[0]);
    if (e.diag_rows) more = e.diag[z * e.stride_diag + m];
    float more2 = 0.0f;
    if (e.diag2) {
      load_vec(e.diag2 + z * e.stride_diag + n, cnt, by[1]);
      more2 = e.diag2[z * e.stride_diag + m];
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
      d[i] += weight * ((more + by[0][i]) * to_f(first[i]) + (more2 + by[1][i]) * to_f(second[i]));
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float r = to_f(first[i]);
    if (e.plane_blend) r += to_f(second[i]);
    d[i] = from ? e.alpha * d[i] + e.beta * r : e.alpha * d[i];
    if (KIND == OP_MIRROR && m == n + i) {
      d[i] += e.diagonal + e.beta * more;
      if (e.diag_out && i < cnt) e.diag_out[z * e.stride_diag + m] = d[i] - to_f(from_f<_Float16>(d[i]));  // exact
    }
  }
}

// The epilogue of V consecutive columns n .. of row m, cnt of them in the
// matrix: d0 (and, gated, d1) are the sums, b0 and b1 the columns' biases.
template <typename T, int KIND, int V, typename E>
__device__ __forceinline__ void op_epilogue(const E& e, int z, int64_t m, int n, int cnt, float (&d0)[V],
                                            float (&d1)[V], const float (&b0)[V], const float (&b1)[V]) {
  if constexpr (KIND == OP_LOSS_GRAD) {
    // (p - [label]) dloss, p = exp(z - lse) <= 1.  Rounded to the type, half a
    // step of each gradient, for the two products that take it, and with
    // `rest_rows` the rest beside it; 16 bits in units of the largest dloss.  A row
    // without a label is selected to 0, whatever z and lse are.
    const int label = e.labels[m], at = label - e.class0 - n, valid = e.classes - n;
    float g = e.dloss[m];
    if constexpr (sizeof(T) == 2) {
      if (e.unit) g *= e.unit[1];
    }
    if (label >= e.all_classes) g = __builtin_nanf("");  // no class at all: not to go unnoticed
    const float lse = e.lse[m];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float p = op_exp<T>(d0[i] + b0[i] - lse);
      d0[i] = label < 0 || i >= valid ? 0.0f : (p - (i == at ? 1.0f : 0.0f)) * g;
    }
    store_vec(static_cast<T*>(e.out[0]) + m * e.ld_out + n, cnt, d0);
    if constexpr (sizeof(T) == 2) {
      if (e.rest_rows) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float held = to_f(from_f<T>(d0[i]));
          d0[i] = fabsf(held) < __builtin_inff() ? d0[i] - held : 0.0f;  // exact
        }
        store_vec(static_cast<T*>(e.out[0]) + (m + e.rest_rows) * e.ld_out + n, cnt, d0);
      }
    }
    return;
  }
  if constexpr (KIND == OP_ADD) {
    if (e.add) {
      float r[V];
      load_vec(e.add + m * e.ld_sum + n, cnt, r);
#pragma unroll
      for (int i = 0; i < V; ++i) d0[i] += r[i];
    }
    if (e.sum) {
      store_vec(e.sum + m * e.ld_sum + n, cnt, d0);
    } else {
      if constexpr (sizeof(T) == 2) {
        const float unit = e.unit ? *e.unit : 1.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) d0[i] *= unit;
      }
      store_vec(static_cast<T*>(e.out[0]) + m * e.ld_out + n, cnt, d0);
    }
    return;
  }
  if constexpr (op_kind_blend(KIND)) {
    op_blend<KIND>(e, z, m, n, cnt, d0);
    op_blend_out(e, z, m, n, cnt, d0);
    return;
  }
  if constexpr (op_kind_layer(KIND)) {
    float r[V];
    const bool residual = KIND == OP_LINEAR && e.residual;
    if (residual) load_vec(static_cast<const T*>(e.residual) + m * e.ld_residual + n, cnt, r);
#pragma unroll
    for (int i = 0; i < V; ++i) d0[i] += b0[i];
    if constexpr (KIND == OP_GATED) {
#pragma unroll
      for (int i = 0; i < V; ++i) d1[i] += b1[i];
    }
    if (e.pre[0]) {
      store_vec(static_cast<T*>(e.pre[0]) + m * e.ld_pre + n, cnt, d0);
      if constexpr (KIND == OP_GATED) store_vec(static_cast<T*>(e.pre[1]) + m * e.ld_pre + n, cnt, d1);
    }
    op_act_all<T>(e.act, d0);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (KIND == OP_GATED) d0[i] *= d1[i];
      else if (residual) d0[i] += r[i];
    }
  }
  store_vec(static_cast<T*>(e.out[z]) + m * e.ld_out + n, cnt, d0);
}
template <typename T, int KIND, int V, typename E>
__device__ __forceinline__ void op_biases(const E& e, int n, int cnt, float (&b0)[V], float (&b1)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) b0[i] = b1[i] = 0.0f;
  if constexpr (KIND == OP_STATS || KIND == OP_LOSS_GRAD) {
    if (e.bias[0]) load_vec(static_cast<const T*>(e.bias[0]) + n, min(cnt, e.classes - n), b0);
  } else if constexpr (op_kind_layer(KIND)) {
    if (e.bias[0]) load_vec(static_cast<const T*>(e.bias[0]) + n, cnt, b0);
    if (KIND == OP_GATED && e.bias[1]) load_vec(static_cast<const T*>(e.bias[1]) + n, cnt, b1);
  }
}

// Sums alone in 16 bits may be in units of an operand's (act_grad_kernel's in
// float16; dz's).
template <typename T, int KIND>
constexpr bool kOpUnits = KIND == OP_STORE && sizeof(T) == 2;
template <typename T, int KIND>
__device__ __forceinline__ float op_unit(const OpEpilogue& e) {
  if constexpr (kOpUnits<T, KIND>)
    if (e.unit) return *e.unit;
  return 1.0f;
}
template <typename T, int KIND, int V>
__device__ __forceinline__ void op_in_units(float unit, float (&d)[V]) {
  if constexpr (kOpUnits<T, KIND>) {
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] *= unit;
  }
}

// The arguments of a kind's kernels.
template <int KIND>
constexpr bool kFlat = KIND >= OP_STATS;  // and their order of blocks (op_place)
template <int KIND>
using OpArgs = typename std::conditional<kFlat<KIND>, OpGemmMore, OpGemm>::type;

// A loop over 0 .. N - 1 whose index is a constant of its body.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void op_unroll(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    op_unroll<N, I + 1>(f);
  }
}
// Waits until at most N of the wave's loads are in flight (they return in
// order), and the block's barrier, neither moved by the compiler.
template <int N>
__device__ __forceinline__ void op_wait_loads() {
  static_assert(N < 64, "what the counter holds");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void op_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void op_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// The statistics of 16 rows' z over a wave's 16 TN columns, from the sums as the
// matrix instructions leave them: a lane has 4 TN columns of one row, its
// neighbours 16, 32 and 48 lanes on the others.  A row whose z are all -inf has
// a sum of 0.  An exponential for each sum: 2048 x 4096 x 131072 bfloat16 takes
// 1600 us with them, 1.37 PFLOP/s, the matrix instructions 70 % busy.
template <typename T, int TN>
__device__ __forceinline__ void op_row_stats(const OpGemmMore& g, const floatx4 (&d)[TN], int lane, int m0, int n0, float* top_of,
                                             float* sum_of) {
  const OpEpilogueMore& e = g.epi;
  const int m = m0 + (lane & 15), lg = lane >> 4;
  const int label = e.labels && m < g.M ? e.labels[m] : -1;
  float z[TN][4], top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + j * 16 + lg * 4, valid = e.classes - n;
    float b0[4], b1[4];
    op_biases<T, OP_STATS>(e, n, valid, b0, b1);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float v = d[j][r] + b0[r];
      if (label == n + r && r < valid) e.at_label[m] = v;
      z[j][r] = r < valid ? v : -__builtin_inff();
      top = fmaxf(top, z[j][r]);
    }
  }
  top = fmaxf(top, __shfl_xor(top, 16, kWave));
  top = fmaxf(top, __shfl_xor(top, 32, kWave));
  const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) sum += op_exp<T>(z[j][r] - base);
  sum += __shfl_xor(sum, 16, kWave);
  sum += __shfl_xor(sum, 32, kWave);
  *top_of = top;
  *sum_of = sum;
}
// Those of a block of WGM x WGN waves, whose waves side by side join theirs in
// LDS: two values a row leave the block instead of its columns.  Every wave of
// the block calls it.
template <typename T, int TM, int TN, int WGM, int WGN>
__device__ __forceinline__ void op_write_stats(const OpGemmMore& g, const floatx4 (&acc)[TM][TN], char* lds, int lane, int wm,
                                               int wn, int m0, int n0) {
  constexpr int kRows = WGM * TM * 16;
  float* all = reinterpret_cast<float*>(lds);  // [wn][top, sum][rows]
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int row = (wm * TM + i) * 16;
    float top, sum;
    op_row_stats<T, TN>(g, acc[i], lane, m0 + row, n0 + wn * (TN * 16), &top, &sum);
    if (lane < 16) {
      all[(wn * 2) * kRows + row + lane] = top;
      all[(wn * 2 + 1) * kRows + row + lane] = sum;
    }
  }
  __syncthreads();
  const int row = threadIdx.x, m = m0 + row;
  if (row >= kRows || m >= g.M) return;
  float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
  for (int w = 0; w < WGN; ++w) top = fmaxf(top, all[(w * 2) * kRows + row]);
  const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
  for (int w = 0; w < WGN; ++w) sum += all[(w * 2 + 1) * kRows + row] * op_exp<T>(all[(w * 2) * kRows + row] - base);
  float* to = g.epi.stats + 2 * ((int64_t)(n0 / (WGN * TN * 16)) * g.M + m);
  to[0] = top;
  to[1] = sum;
}

// A wave's sums (TM x TN blocks of 16x16; gated: the last half of the columns
// belongs to the second matrix) to the outputs, or to the partial sums.  They
// pass through `region`, LDS of the wave's own, 16 or 32 rows at a time, so
// that a lane then has consecutive columns of one row: accesses of 16 bytes,
// and one small loop of code for all rows
// (unrolled over the blocks, the epilogue is larger than the instruction
// cache, and its loads wait for the stores before them).  A row in LDS is 4
// floats longer than its columns, so that 16 rows' blocks meet no bank twice.
// Sums alone, and float32, have a lane for every 16 bytes of a row (8192 x 4096
// over k = 64: 61 us for 82 in float32, 21 for 25 in bf16); 16-bit epilogues
// four lanes a row with more columns each (gated, 1 row: 54.5 us for 55.5).
template <int TM, int TN>
constexpr int op_out_rows = TM % 2 == 0 ? 32 : 16;
template <int TM, int TN>
constexpr int op_region_bytes = op_out_rows<TM, TN> * (TN * 16 + 4) * 4;
// `mirror`: OP_MIRROR's tile is over the diagonal, and also stored across it, by
// lanes that take 16 bytes down a column of the region.
template <typename T, int KIND, int TM, int TN, typename G>
__device__ __forceinline__ void op_write_out(const G& g, floatx4 (&acc)[TM][TN], char* region, int lane, int m0,
                                             int n0, int z, int split, bool mirror = false) {
  constexpr bool kGated = KIND == OP_GATED;
  constexpr int kRows = op_out_rows<TM, TN>, RB = kRows / 16, kLd = TN * 16 + 4;
  constexpr int kCols = kGated ? TN * 8 : TN * 16, kE = 16 / (int)sizeof(T);  // columns of D
  constexpr bool kFew = KIND == OP_STORE || KIND == OP_ADD || op_kind_blend(KIND) || (!kGated && sizeof(T) == 4);
  constexpr int V = kFew ? kE : kCols / 4;  // of them a lane's
  constexpr int kLanes = kCols / V, kTurn = 64 / kLanes;  // lanes of a row, rows of a turn
  static_assert(kRows % kTurn == 0, "whole turns");
  float* lds = reinterpret_cast<float*>(region);
  const int row = lane / kLanes, col = lane % kLanes * V;
  const int n = n0 + col, cnt = g.N - n;
  float b0[V], b1[V], unit = 1.0f;
  if (g.splits <= 1) {
    op_biases<T, KIND>(g.epi, n, cnt, b0, b1);
    unit = op_unit<T, KIND>(g.epi);
  }
#pragma unroll 1
  for (int ph = 0; ph < TM / RB; ++ph) {
    op_unroll<TM / RB>([&](auto I) {
      int now = ph;  // opaque, or the compiler makes one indexed access of these and acc an array in memory
      asm volatile("" : "+s"(now));
      if (now == I) {
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int j = 0; j < TN; ++j)
            *reinterpret_cast<floatx4*>(lds + (b * 16 + (lane & 15)) * kLd + j * 16 + (lane >> 4) * 4) =
                acc[decltype(I)::value * RB + b][j];
      }
    });
#pragma unroll
    for (int r0 = 0; r0 < kRows; r0 += kTurn) {
      const int m = m0 + ph * kRows + r0 + row;
      const float* from = lds + (r0 + row) * kLd + col;
      float d0[V], d1[V];
#pragma unroll
      for (int c = 0; c < V; c += 4) {
        const floatx4 x = *reinterpret_cast<const floatx4*>(from + c);
        floatx4 y = {};
        if constexpr (kGated) y = *reinterpret_cast<const floatx4*>(from + kCols + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d0[c + i] = x[i];
          d1[c + i] = y[i];
        }
      }
      if (m >= g.M || cnt <= 0) continue;
      if (g.splits > 1) {
        const int64_t planes = kGated ? 2 : g.outputs;
        float* p = g.partial + ((split * planes + z) * g.M + m) * (int64_t)g.N + n;
        store_vec(p, cnt, d0);
        if constexpr (kGated) store_vec(p + (int64_t)g.M * g.N, cnt, d1);
      } else {
        op_in_units<T, KIND>(unit, d0);
        op_epilogue<T, KIND>(g.epi, z, m, n, cnt, d0, d1, b0, b1);
        if constexpr (KIND == OP_MIRROR) {  // the results, for the other side of the diagonal
#pragma unroll
          for (int c = 0; c < V && mirror; c += 4)
            *reinterpret_cast<floatx4*>(lds + (r0 + row) * kLd + col + c) = floatx4{d0[c], d0[c + 1], d0[c + 2], d0[c + 3]};
        }
      }
    }
    if constexpr (KIND == OP_MIRROR) {
      if (!mirror) continue;
      constexpr int kDown = kRows / kE, kAcross = 64 / kDown;  // lanes down a column, columns of a turn
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += kAcross) {
        const int down = lane / kAcross * kE, m = m0 + ph * kRows + down, left = g.M - m;
        const int c = c0 + lane % kAcross;
        float d[kE];
#pragma unroll
        for (int i = 0; i < kE; ++i) d[i] = lds[(down + i) * kLd + c];
        if (left <= 0 || n0 + c >= g.N) continue;
        if (g.splits > 1)
          store_vec(g.partial + ((split * (int64_t)g.outputs + z) * g.M + n0 + c) * (int64_t)g.N + m, left, d);
        else
          op_blend_out(g.epi, z, n0 + c, m, left, d);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// A wave's sums to a 16-bit output without LDS.  A lane of two blocks side by
// side has four columns of each, 8 bytes; swapping the odd quarters of the wave
// in the first with the even ones in the second (permlane16_swap) leaves eight
// columns of one of them, and the quarters hold 64 bytes of a row:
//   quarter  0: block j, columns 0..7    1: block j + 1, 0..7
//            2: block j, 8..15           3: block j + 1, 8..15
// `value(i, j, m, sums, out)` makes the four results of block i, j and row m.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ uint32_t op_pack2(float a, float b) {
  union { T e[2]; uint32_t w; } u;
  u.e[0] = from_f<T>(a);
  u.e[1] = from_f<T>(b);
  return u.w;
}
template <typename T, int TM, int TN, typename F>
__device__ __forceinline__ void op_write_swapped(T* out, int64_t ld, int M, int N, const floatx4 (&acc)[TM][TN], int lane,
                                                 int m0, int n0, F value) {
  static_assert(sizeof(T) == 2 && TN % 2 == 0, "pairs of blocks of 16 bits");
  const int quarter = lane >> 4;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + i * 16 + (lane & 15);
    uint32_t p[TN][2];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      float d[4];
      value(i, j, m, acc[i][j], d);
      p[j][0] = op_pack2<T>(d[0], d[1]);
      p[j][1] = op_pack2<T>(d[2], d[3]);
    }
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
      const auto a = __builtin_amdgcn_permlane16_swap(p[j][0], p[j + 1][0], false, false);
      const auto b = __builtin_amdgcn_permlane16_swap(p[j][1], p[j + 1][1], false, false);
      union { chunk16 v; T e[8]; } u;
      u.v = chunk16{a[0], b[0], a[1], b[1]};
      const int n = n0 + (j + (quarter & 1)) * 16 + (quarter >> 1) * 8, cnt = N - n;
      if (m >= M || cnt <= 0) continue;
      T* to = out + m * ld + n;
      if (cnt >= 8) {
        *(VOLTA_GLOBAL typename Access<16, 2>::type*)to = u.v;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < cnt) ((VOLTA_GLOBAL T*)to)[k] = u.e[k];
      }
    }
  }
}

// Where a stage of an operand starts: row or column x0, k.
template <typename T, bool KC>
__device__ __forceinline__ const char* op_stage_base(const void* p, int64_t ld, int x0, int k) {
  const int64_t e = KC ? (int64_t)x0 * ld + k : (int64_t)k * ld + x0;
  return static_cast<const char*>(p) + e * (int64_t)sizeof(T);
}

// Where the next stage to load starts, in every operand (a block's loop takes
// every `step`-th stage): advanced by additions, since a stage's address
// computed anew costs a wave more time than its loads.
template <typename T, int LAYOUT, int KIND, typename Args = OpArgs<KIND>>
struct Cursor {
  static constexpr bool GATED = KIND == OP_GATED;
  static constexpr bool P_KC = LAYOUT != OP_TN, Q_KC = LAYOUT == OP_NT;
  static constexpr int kSubs = GATED ? 2 : 1, kStageK = 128 / (int)sizeof(T);
  const char* p;
  const char* q[kSubs];
  int64_t dp, dq;  // bytes of a step
  int k, dk;       // in this piece
  int piece, m0, n0, z;

  __device__ __forceinline__ void place(const Args& g) {
    if constexpr (op_kind_blend(KIND)) {
      p = op_stage_base<T, P_KC>(static_cast<const T*>(g.p[0]) + z * g.epi.stride_p + (g.pieces == 3 && piece == 0 ? g.epi.plane_p : 0), g.ld_p,
                                 m0, k);
      q[0] = op_stage_base<T, Q_KC>(static_cast<const T*>(g.q[0]) + z * g.epi.stride_q + (piece == 1 ? g.epi.plane_q : 0), g.ld_q,
                                    n0, k);
    } else {
      p = op_stage_base<T, P_KC>(g.p[piece], g.ld_p, m0, k);
#pragma unroll
      for (int i = 0; i < kSubs; ++i)
        q[i] = op_stage_base<T, Q_KC>(g.q[GATED ? i : LAYOUT == OP_TN ? z : piece], g.ld_q, n0, k);
    }
  }
  __device__ __forceinline__ int piece_k(const Args& g) const { return (g.K + kStageK - 1) / kStageK * kStageK; }
  __device__ __forceinline__ void init(const Args& g, int m0_, int n0_, int z_, int s, int step) {
    m0 = m0_;
    n0 = n0_;
    z = z_;
    dk = step * kStageK;
    dp = (P_KC ? (int64_t)dk : dk * g.ld_p) * (int64_t)sizeof(T);
    dq = (Q_KC ? (int64_t)dk : dk * g.ld_q) * (int64_t)sizeof(T);
    k = s * kStageK;
    if constexpr (op_kind_blend(KIND)) {
      piece = min(k / piece_k(g), g.pieces - 1);
      k -= piece * piece_k(g);
    } else {
      piece = LAYOUT == OP_NT && g.pieces > 1 && k >= piece_k(g) ? 1 : 0;
      if (piece) k -= piece_k(g);
    }
    place(g);
  }
  // Inside the piece, or into the next one.
  __device__ __forceinline__ void step() {
    k += dk;
    p += dp;
#pragma unroll
    for (int i = 0; i < kSubs; ++i) q[i] += dq;
  }
  __device__ __forceinline__ void cross(const Args& g) {
    if (op_kind_blend(KIND) && piece < g.pieces - 1 && k >= piece_k(g)) {
      ++piece;
      k -= piece_k(g);
      place(g);
    }
    if (!op_kind_blend(KIND) && LAYOUT == OP_NT && g.pieces > 1 && piece == 0 && k >= piece_k(g)) {
      piece = 1;
      k -= piece_k(g);
      place(g);
    }
  }
  // Steps from here on whose stages are whole.
  __device__ __forceinline__ int whole_steps(const Args& g) const {
    const int stages = (g.K - k) / kStageK;
    return stages > 0 ? (stages - 1) / (dk / kStageK) + 1 : 0;
  }
};

// Block -> tile.  Blocks go to the 8 XCDs in turn; each XCD takes a run of
// consecutive tiles, in groups of `kGroup` rows of tiles walked column by
// column, so that the tiles an XCD works on at a time share rows of P and
// columns of Q in its L2.
__device__ __forceinline__ void op_tile_of(int b, int tiles_m, int tiles_n, int* tm, int* tn) {
  constexpr int kXcds = 8, kGroup = 8;
  const int total = tiles_m * tiles_n;
  const int per = total / kXcds, rest = total % kXcds, x = b % kXcds;
  const int id = x * per + min(x, rest) + b / kXcds;
  const int group = id / (kGroup * tiles_n);
  const int rows = min(kGroup, tiles_m - group * kGroup);
  const int in = id - group * kGroup * tiles_n;
  *tm = group * kGroup + in % rows;
  *tn = in / rows;
}

// Where a block works.  The kinds from OP_STATS on count their blocks through
// the matrices, the splits of a matrix and its tiles, and an XCD takes a run of
// that order: tiles that read the same k of the same matrix share an L2 (16
// matrices of 512 x 2000, G in float16: 28.4 us with each matrix's tiles on
// every XCD, 23.7 so).
struct OpPlace {
  int tm, tn, split, z;
};
template <bool FLAT, bool TRIANGLE, typename G>
__device__ __forceinline__ OpPlace op_place(const G& g) {
  OpPlace p;
  if constexpr (!FLAT) {
    op_tile_of(blockIdx.x, g.tiles_m, g.tiles_n, &p.tm, &p.tn);
    p.split = blockIdx.y;
    p.z = g.outputs > 1 ? blockIdx.z : 0;
    return p;
  }
  constexpr int kXcds = 8, kGroup = TRIANGLE ? 4 : 8;
  const int tiles = TRIANGLE ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
  const int total = gridDim.x, per = total / kXcds, rest = total % kXcds, x = blockIdx.x % kXcds;
  const int id = x * per + min(x, rest) + blockIdx.x / kXcds, of = id / tiles;
  int t = id - of * tiles;
  p.split = of % g.splits;
  p.z = of / g.splits;
  if constexpr (TRIANGLE) {
    // columns of squares of 4 x 4 tiles, each column's last one cut by the
    // diagonal: 8 j^2 + 2 j tiles stand before column j
    int j = (int)((sqrtf(4.0f + 32.0f * (float)t) - 2.0f) * 0.0625f);
    while (8 * j * j + 2 * j > t) --j;
    while (8 * (j + 1) * (j + 1) + 2 * (j + 1) <= t) ++j;
    t -= 8 * j * j + 2 * j;
    const int wide = min(kGroup, g.tiles_m - kGroup * j), i = t / (kGroup * wide);
    if (i < j) {
      t -= i * kGroup * wide;
      p.tm = kGroup * i + t % kGroup;
      p.tn = kGroup * j + t / kGroup;
    } else {
      t -= j * kGroup * wide;
      int n = 0;
      while ((n + 1) * (n + 2) / 2 <= t) ++n;
      p.tm = kGroup * j + t - n * (n + 1) / 2;
      p.tn = kGroup * j + n;
    }
  } else {
    const int group = t / (kGroup * g.tiles_n), rows = min(kGroup, g.tiles_m - group * kGroup);
    t -= group * kGroup * g.tiles_n;
    p.tm = group * kGroup + t % rows;
    p.tn = t / rows;
  }
  return p;
}

// ---------------------------------------------------------------------------
// Staged product, for operands whose rows direct loads cannot take: BM x BN of
// D per block, 2 x 2 waves.  A stage goes through registers into one of two
// places in LDS; the loads of the next are in flight while it is multiplied,
// one stage ahead, and their latency bounds it.  bf16 2048^3 with rows of 2049
// elements: 128x128 43 us and 64x64 51 (rows of 2048 that start one element
// off: 52 and 67; aligned, as the direct form takes them: 41 and 37), against
// 23.7 of the direct 128x128; so operands are laid out anew where that copy
// takes less.
// ---------------------------------------------------------------------------
template <typename T, int LAYOUT, int KIND, int BM, int BN>
__global__ void __launch_bounds__(256) op_gemm_staged(OpArgs<KIND> g) {
  constexpr int NW = 4, WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
  constexpr bool kGated = KIND == OP_GATED;
  constexpr int kSubs = kGated ? 2 : 1, SN = BN / kSubs;  // gated: half the columns of each weight matrix
  constexpr int TNS = TN / kSubs;
  constexpr bool P_KC = LAYOUT != OP_TN, Q_KC = LAYOUT == OP_NT;
  using PT = Tile<T, BM, P_KC, NW>;
  using QT = Tile<T, SN, Q_KC, NW>;
  constexpr int kStageK = PT::kStageK, kStageBytes = PT::kBytes + QT::kBytes * kSubs;
  __shared__ __attribute__((aligned(16))) char lds[2 * kStageBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const OpPlace place = op_place<kFlat<KIND>, KIND == OP_MIRROR>(g);
  const int tm = place.tm, tn = place.tn;
  const int m0 = tm * BM, n0 = tn * SN;
  const int z = place.z, split = place.split;
  const int p_left = g.M - m0, q_left = g.N - n0;

  PT pt;
  QT qt;
  pt.init(g.ld_p, p_left, wave, lane);
  qt.init(g.ld_q, q_left, wave, lane);
  const int per_piece = (g.K + kStageK - 1) / kStageK;
  const int s_begin = split * g.stages_per_split;
  const int s_end = min(per_piece * g.pieces, s_begin + g.stages_per_split);

  Cursor<T, LAYOUT, KIND> next;
  next.init(g, m0, n0, z, s_begin, 1);
  chunk16 rp[PT::kLoads], rq[kSubs][QT::kLoads];
  auto fetch = [&]() {  // the next stage
    const int k_left = g.K - next.k;
    pt.fetch(next.p, rp, wave, lane, p_left, k_left);
#pragma unroll
    for (int i = 0; i < kSubs; ++i) qt.fetch(next.q[i], rq[i], wave, lane, q_left, k_left);
    next.step();
    next.cross(g);
  };
  // A wave writes a place again only behind the barrier that every wave
  // reached after it had read it.
  auto put = [&](char* to) {
    pt.put(rp, to, wave, lane);
#pragma unroll
    for (int i = 0; i < kSubs; ++i) qt.put(rq[i], to + PT::kBytes + i * QT::kBytes, wave, lane);
    __syncthreads();
  };

  floatx4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  auto compute = [&](const char* from) {
    const char* lq = from + PT::kBytes;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      chunk16 fp[TM], fq[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
        fq[j] = QT::frag(lq + (j / TNS) * QT::kBytes, (wn * TNS + j % TNS) * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < TM; ++i) fp[i] = PT::frag(from, wm * WM + i * 16, kk, lane);
#pragma unroll
      for (int st = 0; st < Mfma<T>::kSteps; ++st)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = Mfma<T>::mul(st, fq[j], fp[i], acc[i][j]);
    }
  };

  if (s_begin < s_end) fetch();
  for (int s0 = s_begin; s0 < s_end; s0 += 2) {
    op_unroll<2>([&](auto i) {
      const int s = s0 + i;
      if (s >= s_end) return;
      char* at = lds + decltype(i)::value * kStageBytes;
      put(at);
      if (s + 1 < s_end) fetch();
      __builtin_amdgcn_sched_barrier(0);
      compute(at);
    });
  }

  __syncthreads();  // both places are free
  static_assert(NW * op_region_bytes<TM, TN> <= 2 * kStageBytes, "output regions fit");
  if constexpr (KIND == OP_STATS) {
    if (g.splits <= 1) return op_write_stats<T, TM, TN, 2, 2>(g, acc, lds, lane, wm, wn, m0, n0);
  }
  op_write_out<T, KIND>(g, acc, lds + wave * op_region_bytes<TM, TN>, lane, m0 + wm * WM, n0 + wn * (TNS * 16), z, split);
}

// ---------------------------------------------------------------------------
// Large product: 256x256 of D per block, eight waves (2 x 4, each
// 128x64), two stages of k in LDS in four regions each -- the halves of P's
// rows and Q's columns that a wave multiplies apart:
//
//   region P0, P1: rows 0..63 and 64..127 of each of the two wave rows
//   region Q0, Q1: columns 0..31 and 32..63 of each of the four wave columns
//                  (gated: the gate's and the up matrix's 32 columns)
//
// A stage is two phases of 32 matrix instructions; each reads what it
// multiplies, issues the loads that overwrite regions read two phases ago or
// in the one before, and multiplies:
//
//   phase   reads             loads                  multiplies
//     0     P0, Q0, Q1 of s   Q1 and P1 of s + 1     P0 by Q0, Q1
//     1     P1 of s           Q0 and P0 of s + 2     P1 by Q0, Q1
//
// The waves of the second row start half a phase later, so that of the two
// waves of a SIMD one reads LDS while the other multiplies.  Behind a region
// that is to be read, three or four more regions' loads stay in flight (48 or
// 64 KB); the wait is for the older ones alone.  (Four phases of 16
// instructions with a region each measured 4 to 12 % slower: the barrier
// between two phases costs about 90 cycles.)
//
// Bound by the matrix instructions, which are busy 70 to 76 % of the cycles,
// and by the chip's power, which lowers the clock on sums this large.  8192^3
// in bf16 from memory: x W 821 us (1339 TFLOP/s), dp W^T 746 (1475), x^T dp
// 810 (1357); 4096^3 in float32 1067 us (129).
// ---------------------------------------------------------------------------
template <typename T, bool KC, int BLK, int STRIDE>
struct Region : Tile<T, 128, KC, 8> {
  using Base = Tile<T, 128, KC, 8>;
  // Row or column j of the region is x0 + (j / BLK) STRIDE + j % BLK of the matrix.
  __device__ __forceinline__ void init(int64_t ld, int x0, int left, int wave, int lane) {
#pragma unroll
    for (int t = 0; t < Base::kLoads; ++t) {
      int r, c;
      Base::place((wave + t * 8) * 64 + lane, &r, &c);
      if constexpr (KC) {
        r = min(x0 + r / BLK * STRIDE + r % BLK, left - 1);
        this->off[t] = (uint32_t)r * (uint32_t)(ld * Base::kElem) + (uint32_t)c * 16u;
      } else {
        const int j = c * Base::kE;
        c = min(x0 + j / BLK * STRIDE + j % BLK, (left - 1) / Base::kE * Base::kE);
        this->off[t] = (uint32_t)r * (uint32_t)(ld * Base::kElem) + (uint32_t)(c * Base::kElem);
      }
    }
  }
};

template <typename T, int LAYOUT, int KIND>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) op_gemm_large(OpArgs<KIND> g) {
  constexpr bool kGated = KIND == OP_GATED, P_KC = LAYOUT != OP_TN, Q_KC = LAYOUT == OP_NT;
  constexpr int kRegion = 128 * 128, kStageK = 128 / (int)sizeof(T), SN = kGated ? 128 : 256;
  using PR = Region<T, P_KC, 64, 128>;
  using QR = Region<T, Q_KC, kGated ? 128 : 32, kGated ? 128 : 64>;
  static_assert(PR::kBytes == kRegion && PR::kLoads == 2, "two loads a wave and region");
  __shared__ __attribute__((aligned(16))) char lds[8 * kRegion];  // [stage & 1][P0, P1, Q0, Q1]

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const OpPlace place = op_place<kFlat<KIND>, KIND == OP_MIRROR>(g);
  const int tm = place.tm, tn = place.tn;
  const int m0 = tm * 256, n0 = tn * SN;
  const int z = place.z, split = place.split;
  PR pr[2];
  QR qr[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    pr[h].init(g.ld_p, h * 64, g.M - m0, wave, lane);
    qr[h].init(g.ld_q, kGated ? 0 : h * 32, g.N - n0, wave, lane);
  }
  const int per_piece = (g.K + kStageK - 1) / kStageK;
  const int s_begin = split * g.stages_per_split;
  const int S = min(per_piece * g.pieces, s_begin + g.stages_per_split) - s_begin;

  // two cursors: the halves are loaded in different phases
  Cursor<T, LAYOUT, KIND> next[2];
  next[0].init(g, m0, n0, z, s_begin, 1);
  next[1].init(g, m0, n0, z, s_begin, 1);
  // P and Q halves h of the next stage of their cursor to the stage at byte
  // `to` of LDS; `whole`: it is, and in one piece
  auto load = [&](uint32_t to, auto half, auto whole) {
    constexpr int h = decltype(half)::value;
    constexpr bool W = decltype(whole)::value;
    const uint32_t tp = to + h * kRegion, tq = to + (2 + h) * kRegion;
    const int k_left = W ? kStageK : g.K - next[h].k;
    const char* q = next[h].q[kGated ? h : 0];
    if (W || k_left >= kStageK) {
      qr[h].issue(q, tq, wave);
      pr[h].issue(next[h].p, tp, wave);
    } else {
      qr[h].issue_tail(q, tq, wave, lane, k_left);
      pr[h].issue_tail(next[h].p, tp, wave, lane, k_left);
    }
    next[h].step();
    if constexpr (!W) next[h].cross(g);
  };
  floatx4 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  chunk16 fp[4][2], fq[4][2];

  auto read_p = [&](const char* from) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i) fp[i][kk] = PR::frag(from, wm * 64 + i * 16, kk, lane);
  };
  auto read_q = [&](const char* from, int h) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int j = 0; j < 2; ++j) fq[2 * h + j][kk] = QR::frag(from, wn * 32 + j * 16, kk, lane);
  };
  auto mul = [&](int half, int h) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int st = 0; st < Mfma<T>::kSteps; ++st)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 2 * h; j < 2 * h + 2; ++j)
            acc[half * 4 + i][j] = Mfma<T>::mul(st, fq[j][kk], fp[i][kk], acc[half * 4 + i][j]);
  };
  constexpr auto H0 = std::integral_constant<int, 0>();
  constexpr auto H1 = std::integral_constant<int, 1>();
  const uint32_t lds_byte = op_lds_byte(lds);
  int from = 0;  // byte of the stage in LDS
  auto stage = [&](int s, auto whole) {
    constexpr bool W = decltype(whole)::value;
    const char* at = lds + from;
    const int left = S - 1 - s;  // stages behind this one
    read_q(at + 2 * kRegion, 0);
    read_p(at);
    __builtin_amdgcn_sched_barrier(0);
    if (W || left >= 1) {
      load(lds_byte + (from ^ 4 * kRegion), H1, whole);
      op_wait_loads<8>();  // P1 of s is there
    } else {
      op_wait_loads<0>();
    }
    op_wait_lds();
    op_barrier();
    read_q(at + 3 * kRegion, 1);  // arrives while Q0 is multiplied
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    mul(0, 0);
    __builtin_amdgcn_sched_barrier(0);
    mul(0, 1);
    __builtin_amdgcn_s_setprio(0);
    op_barrier();
    read_p(at + kRegion);
    __builtin_amdgcn_sched_barrier(0);
    if (W || left >= 2) {
      load(lds_byte + from, H0, whole);
      op_wait_loads<6>();  // P0, Q0 and Q1 of s + 1 are there
    } else {
      op_wait_loads<2>();
    }
    from ^= 4 * kRegion;
    op_wait_lds();
    op_barrier();
    __builtin_amdgcn_s_setprio(1);
    mul(1, 0);
    mul(1, 1);
    __builtin_amdgcn_s_setprio(0);
    op_barrier();
  };

  if (S > 0) {
    constexpr auto any = std::false_type();
    load(lds_byte, H0, any);
    load(lds_byte, H1, any);
    if (S > 1) {
      load(lds_byte + 4 * kRegion, H0, any);
      op_wait_loads<6>();  // P0, Q0 and Q1 of the first stage are there
    } else {
      op_wait_loads<2>();
    }
    op_barrier();
    if (wm == 1) op_barrier();
    for (int s = 0; s < S; ++s) {
      // whole stages in a loop without a branch, the others one by one
      for (int n = min(min(next[0].whole_steps(g), next[1].whole_steps(g)), S - 2 - s); n > 0; --n, ++s)
        stage(s, std::true_type());
      next[0].cross(g);
      next[1].cross(g);
      if (s < S) stage(s, any);
    }
    if (wm == 0) op_barrier();
  }
  __syncthreads();  // the regions are free
  static_assert(8 * op_region_bytes<8, 4> <= 8 * kRegion, "output regions fit");
  if constexpr (KIND == OP_STATS) {
    if (g.splits <= 1) return op_write_stats<T, 8, 4, 2, 4>(g, acc, lds, lane, wm, wn, m0, n0);
  }
  op_write_out<T, KIND>(g, acc, lds + wave * op_region_bytes<8, 4>, lane, m0 + wm * 128, n0 + wn * (kGated ? 32 : 64), z,
                        split, tm != tn);
}

// ---------------------------------------------------------------------------
// Middle-sized product: BM x BN of D per block, eight waves (WGM x WGN), a
// ring of NST stages of KS times 128 bytes of k in LDS.  As in the large form
// the waves 4 to 7 run half a stage behind the waves 0 to 3, so that of a
// SIMD's two waves one reads LDS while the other multiplies; a stage is one
// phase.
//
// Tiles for grids that 256x256 would leave CUs idle in; what bounds them is
// the time of a stage from barrier to barrier, 0.8 us (256x128), 0.45 to 0.55
// (128x128), 0.35 and 0.25, and how evenly the tiles fill the CUs.  In bf16:
//   256x128  gated, 1024 rows, 2048 to 4096   33.7 us, 1019 TFLOP/s (128x128 41.8)
//   128x128  2048^3                           22.4 us,  768 TFLOP/s (256x128 30.7)
//    64x128  gated, 1 row, 4096 to 16384      54.5 us, 4.9 TB/s of weights
//    64x64   256 rows, 4096 to 2048           18 us (128x128 33.6, 64x128 26.3)
// Tried and no faster: rings of 5 and 6 stages, two parts of k a stage at
// 64x128, and half of the waves on either half of a stage's k, which reads a
// third less of LDS and pays 1 to 2 us for adding the halves.
// ---------------------------------------------------------------------------
template <typename T, int LAYOUT, int KIND, int BM, int BN, int WGM, int WGN, int KS, int NST>
__global__ void __launch_bounds__(512) op_gemm_middle(OpArgs<KIND> g) {
  static_assert(WGM * WGN == 8, "eight waves");
  constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr bool kGated = KIND == OP_GATED, P_KC = LAYOUT != OP_TN, Q_KC = LAYOUT == OP_NT;
  constexpr int kSubs = kGated ? 2 : 1, SN = BN / kSubs, TNS = TN / kSubs;
  // 32 columns of each weight matrix are four load instructions: half of the waves load each
  constexpr bool kHalves = kGated && SN < 64;
  using PT = Tile<T, BM, P_KC, 8>;
  using QT = Tile<T, SN, Q_KC, kHalves ? 4 : 8>;
  constexpr int kStageK = PT::kStageK, kPart = PT::kBytes + QT::kBytes * kSubs, kStageBytes = KS * kPart;
  constexpr int kStageLoads = KS * (PT::kLoads + QT::kLoads * (kHalves ? 1 : kSubs));
  __shared__ __attribute__((aligned(16))) char lds[NST * kStageBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const OpPlace place = op_place<kFlat<KIND>, KIND == OP_MIRROR>(g);
  const int tm = place.tm, tn = place.tn;
  const int m0 = tm * BM, n0 = tn * SN;
  const int z = place.z, split = place.split;
  PT pt;
  QT qt;
  pt.init(g.ld_p, g.M - m0, wave, lane);
  qt.init(g.ld_q, g.N - n0, kHalves ? wave & 3 : wave, lane);
  const int s_begin = split * g.stages_per_split;
  int parts = min((g.K + kStageK - 1) / kStageK * g.pieces, s_begin + g.stages_per_split) - s_begin;
  const int S = (parts + KS - 1) / KS;
  Cursor<T, LAYOUT, KIND> next;
  next.init(g, m0, n0, z, s_begin, 1);
  // The next stage to byte `to` of LDS; `whole`: it is, and in one piece.
  auto load = [&](uint32_t to, auto whole) {
    constexpr bool W = decltype(whole)::value;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int k_left = W ? kStageK : parts > i ? g.K - next.k : 0;  // a part behind the last one is zeros
      const uint32_t lp = to + i * kPart, lq = lp + PT::kBytes;
      if constexpr (kHalves) {
        const char* q = wave < 4 ? next.q[0] : next.q[kSubs - 1];
        const uint32_t half = lq + (wave < 4 ? 0 : QT::kBytes);
        if (W || k_left >= kStageK) qt.issue(q, half, wave & 3);
        else qt.issue_tail(q, half, wave & 3, lane, k_left);
      } else {
#pragma unroll
        for (int w = 0; w < kSubs; ++w) {
          if (W || k_left >= kStageK) qt.issue(next.q[w], lq + w * QT::kBytes, wave);
          else qt.issue_tail(next.q[w], lq + w * QT::kBytes, wave, lane, k_left);
        }
      }
      if (W || k_left >= kStageK) pt.issue(next.p, lp, wave);
      else pt.issue_tail(next.p, lp, wave, lane, k_left);
      next.step();
      if constexpr (!W) next.cross(g);
    }
    parts -= KS;
  };

  floatx4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  chunk16 fp[TM][2 * KS], fq[TN][2 * KS];

  // One stage, read at byte `from` of LDS; the next loads go where the stage
  // before was, which every wave has read.
  int from = 0, to = (NST - 1) * kStageBytes;
  const uint32_t lds_byte = op_lds_byte(lds);
  auto stage = [&](int s, auto whole) {
    constexpr bool W = decltype(whole)::value;
#pragma unroll
    for (int kk = 0; kk < 2 * KS; ++kk) {
      const char* part = lds + from + (kk >> 1) * kPart;
#pragma unroll
      for (int j = 0; j < TN; ++j)
        fq[j][kk] = QT::frag(part + PT::kBytes + (j / TNS) * QT::kBytes, (wn * TNS + j % TNS) * 16, kk & 1, lane);
#pragma unroll
      for (int i = 0; i < TM; ++i) fp[i][kk] = PT::frag(part, wm * WM + i * 16, kk & 1, lane);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (W || s + NST - 1 < S) {
      load(lds_byte + to, whole);
      op_wait_loads<(NST - 2) * kStageLoads>();  // stage s + 1 is there
    } else {
      op_wait_loads<0>();
    }
    to = from;
    from = from == (NST - 1) * kStageBytes ? 0 : from + kStageBytes;
    op_wait_lds();
    op_barrier();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kk = 0; kk < 2 * KS; ++kk)
#pragma unroll
      for (int st = 0; st < Mfma<T>::kSteps; ++st)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = Mfma<T>::mul(st, fq[j][kk], fp[i][kk], acc[i][j]);
    __builtin_amdgcn_s_setprio(0);
    op_barrier();
  };

  if (S > 0) {
#pragma unroll 1
    for (int i = 0; i < NST - 1 && i < S; ++i) load(lds_byte + i * kStageBytes, std::false_type());
    if (S >= NST - 1) op_wait_loads<(NST - 2) * kStageLoads>();
    else op_wait_loads<0>();
    op_barrier();
    if (wave >= 4) op_barrier();
    for (int s = 0; s < S; ++s) {
      // whole stages in a loop without a branch, the others one by one
      for (int n = min(min(next.whole_steps(g), parts) / KS, S - (NST - 1) - s); n > 0; --n, ++s)
        stage(s, std::true_type());
      next.cross(g);
      if (s < S) stage(s, std::false_type());
    }
    if (wave < 4) op_barrier();
  }
  __syncthreads();  // the ring is free
  static_assert(8 * op_region_bytes<TM, TN> <= NST * kStageBytes, "output regions fit the ring");
  if constexpr (KIND == OP_STATS) {
    if (g.splits <= 1) return op_write_stats<T, TM, TN, WGM, WGN>(g, acc, lds, lane, wm, wn, m0, n0);
  }
  op_write_out<T, KIND>(g, acc, lds + wave * op_region_bytes<TM, TN>, lane, m0 + wm * WM, n0 + wn * (TNS * 16), z, split,
                        tm != tn);
}

// ---------------------------------------------------------------------------
// Small product of pairs of float16 numbers (OP_BLEND, OP_MIRROR): op_gemm_middle
// with both planes of both operands in a stage, so that three products are made
// of what is loaded, and read from LDS, once.  The products with a rest have a
// sum of their own, which joins the other at the end.  64x64 of D: X' of 1024 x
// 1024 13.4 us, 0.55 a stage from barrier to barrier, for 18.2 with the three
// products one after the other (float32's own matrix instruction: 26.7).
// ---------------------------------------------------------------------------
template <int LAYOUT, int KIND, int BM, int BN, int WGM, int WGN, int NST>
__global__ void __launch_bounds__(512) op_gemm_pairs(OpGemmMore g) {
  static_assert(WGM * WGN == 8, "eight waves");
  using T = _Float16;
  constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr bool P_KC = LAYOUT != OP_TN, Q_KC = LAYOUT == OP_NT;
  using PT = Tile<T, BM, P_KC, 8>;
  using QT = Tile<T, BN, Q_KC, 8>;
  constexpr int kStageK = PT::kStageK, kStageBytes = 2 * (PT::kBytes + QT::kBytes);
  constexpr int kStageLoads = 2 * (PT::kLoads + QT::kLoads);
  __shared__ __attribute__((aligned(16))) char lds[NST * kStageBytes];  // [stage][P, its rests, Q, its rests]

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const OpPlace place = op_place<true, KIND == OP_MIRROR>(g);
  const int tm = place.tm, tn = place.tn, m0 = tm * BM, n0 = tn * BN, z = place.z, split = place.split;
  PT pt;
  QT qt;
  pt.init(g.ld_p, g.M - m0, wave, lane);
  qt.init(g.ld_q, g.N - n0, wave, lane);
  const int64_t rest_p = g.epi.plane_p * (int64_t)sizeof(T), rest_q = g.epi.plane_q * (int64_t)sizeof(T);
  const int s_begin = split * g.stages_per_split;
  const int S = min((g.K + kStageK - 1) / kStageK, s_begin + g.stages_per_split) - s_begin;
  Cursor<T, LAYOUT, KIND> next;
  next.init(g, m0, n0, z, s_begin, 1);
  auto load = [&](uint32_t to, auto whole) {
    constexpr bool W = decltype(whole)::value;
    const int k_left = W ? kStageK : g.K - next.k;
    const uint32_t q = to + 2 * PT::kBytes;
    if (W || k_left >= kStageK) {
      qt.issue(next.q[0], q, wave);
      pt.issue(next.p, to, wave);
      qt.issue(next.q[0] + rest_q, q + QT::kBytes, wave);
      pt.issue(next.p + rest_p, to + PT::kBytes, wave);
    } else {
      qt.issue_tail(next.q[0], q, wave, lane, k_left);
      pt.issue_tail(next.p, to, wave, lane, k_left);
      qt.issue_tail(next.q[0] + rest_q, q + QT::kBytes, wave, lane, k_left);
      pt.issue_tail(next.p + rest_p, to + PT::kBytes, wave, lane, k_left);
    }
    next.step();
  };

  floatx4 acc[TM][TN], small[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = small[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  chunk16 fp[2][TM][2], fq[2][TN][2];  // [plane][block][half of k]

  int from = 0, to = (NST - 1) * kStageBytes;
  const uint32_t lds_byte = op_lds_byte(lds);
  auto stage = [&](int s, auto whole) {
    constexpr bool W = decltype(whole)::value;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const char* at = lds + from;
#pragma unroll
        for (int j = 0; j < TN; ++j)
          fq[plane][j][kk] = QT::frag(at + 2 * PT::kBytes + plane * QT::kBytes, wn * WN + j * 16, kk, lane);
#pragma unroll
        for (int i = 0; i < TM; ++i) fp[plane][i][kk] = PT::frag(at + plane * PT::kBytes, wm * WM + i * 16, kk, lane);
      }
    __builtin_amdgcn_sched_barrier(0);
    if (W || s + NST - 1 < S) {
      load(lds_byte + to, whole);
      op_wait_loads<(NST - 2) * kStageLoads>();  // stage s + 1 is there
    } else {
      op_wait_loads<0>();
    }
    to = from;
    from = from == (NST - 1) * kStageBytes ? 0 : from + kStageBytes;
    op_wait_lds();
    op_barrier();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          acc[i][j] = Mfma<T>::mul(0, fq[0][j][kk], fp[0][i][kk], acc[i][j]);
          small[i][j] = Mfma<T>::mul(0, fq[0][j][kk], fp[1][i][kk], small[i][j]);
          small[i][j] = Mfma<T>::mul(0, fq[1][j][kk], fp[0][i][kk], small[i][j]);
        }
    __builtin_amdgcn_s_setprio(0);
    op_barrier();
  };

  if (S > 0) {
#pragma unroll 1
    for (int i = 0; i < NST - 1 && i < S; ++i) load(lds_byte + i * kStageBytes, std::false_type());
    if (S >= NST - 1) op_wait_loads<(NST - 2) * kStageLoads>();
    else op_wait_loads<0>();
    op_barrier();
    if (wave >= 4) op_barrier();
    for (int s = 0; s < S; ++s) {
      for (int n = min(next.whole_steps(g), S - (NST - 1) - s); n > 0; --n, ++s) stage(s, std::true_type());
      if (s < S) stage(s, std::false_type());
    }
    if (wave < 4) op_barrier();
  }
  __syncthreads();  // the ring is free
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = acc[i][j] + small[i][j];
  static_assert(8 * op_region_bytes<TM, TN> <= NST * kStageBytes, "output regions fit the ring");
  op_write_out<T, KIND>(g, acc, lds + wave * op_region_bytes<TM, TN>, lane, m0 + wm * WM, n0 + wn * WN, z, split,
                        tm != tn);
}

// ---------------------------------------------------------------------------
// Skinny product, few rows: reading the weights bounds the time.  A block
// takes 16 MT rows and BN columns (of each weight matrix) and its waves take turns
// over the stages of k, each with a ring of its own in LDS for both operands
// (no barrier before the end); the waves' sums are added at the end, in wave
// order.  float32, 64 rows, 1024 to 1024: 6 us (a launch that does nothing
// takes 2); bf16, 1 row, 4096 to 4096: 11.7 us.  Columns of W in 64-byte
// pieces cost it bandwidth where W is large and comes from memory: bf16, 16
// rows, 4096 to 16384, 134 MB: 41 us, and 29 on 64x64 tiles.
// ---------------------------------------------------------------------------
template <typename T, int LAYOUT, int KIND, int MT, int BN, int NW, int NST, bool DIRECT>
__global__ void __launch_bounds__(NW * 64) op_gemm_skinny(OpArgs<KIND> g) {
  constexpr bool kGated = KIND == OP_GATED, Q_KC = LAYOUT == OP_NT;
  constexpr int kSubs = kGated ? 2 : 1, TNS = BN / 16, TN = TNS * kSubs;
  using PT = Tile<T, 16 * MT, true, 1>;
  using QT = Tile<T, BN, Q_KC, 1>;
  constexpr int kStageK = QT::kStageK;
  constexpr int kWaveBytes = PT::kBytes + QT::kBytes * kSubs;
  constexpr int kStageLoads = PT::kLoads + QT::kLoads * kSubs;
  static_assert(DIRECT ? NST >= 2 : NST == 1, "ring");
  __shared__ __attribute__((aligned(16))) char lds[NST * NW * kWaveBytes];

  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // blocks next to each other share cache lines of W: one XCD takes a run of them
  const OpPlace place = op_place<kFlat<KIND>, false>(g);
  const int m0 = place.tm * (16 * MT), n0 = place.tn * BN, split = place.split, p_left = g.M - m0, q_left = g.N - n0;
  PT pt;
  QT qt;
  pt.init(g.ld_p, p_left, 0, lane);
  qt.init(g.ld_q, q_left, 0, lane);
  const int per_piece = (g.K + kStageK - 1) / kStageK;
  const int s_begin = split * g.stages_per_split;
  const int s_end = min(per_piece * g.pieces, s_begin + g.stages_per_split);
  char* mine = lds + wave * (NST * kWaveBytes);

  chunk16 rp[DIRECT ? 1 : PT::kLoads], rq[kSubs][DIRECT ? 1 : QT::kLoads];
  Cursor<T, LAYOUT, KIND> next;
  next.init(g, m0, n0, 0, s_begin + wave, NW);
  // This wave's next stage, to byte `to` of LDS; `whole`: it is, and in one piece.
  auto load = [&](uint32_t to, auto whole) {
    constexpr bool W = decltype(whole)::value;
    const int k_left = W ? kStageK : g.K - next.k;
    if constexpr (DIRECT) {
      const uint32_t lq = to + PT::kBytes;
      if (W || k_left >= kStageK) {
#pragma unroll
        for (int i = 0; i < kSubs; ++i) qt.issue(next.q[i], lq + i * QT::kBytes, 0);
        pt.issue(next.p, to, 0);
      } else {
#pragma unroll
        for (int i = 0; i < kSubs; ++i) qt.issue_tail(next.q[i], lq + i * QT::kBytes, 0, lane, k_left);
        pt.issue_tail(next.p, to, 0, lane, k_left);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSubs; ++i) qt.fetch(next.q[i], rq[i], 0, lane, q_left, k_left);
      pt.fetch(next.p, rp, 0, lane, p_left, k_left);
    }
    next.step();
    if constexpr (!W) next.cross(g);
  };

  floatx4 acc[MT][TN];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  auto compute = [&](const char* from) {
    const char* lq = from + PT::kBytes;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      chunk16 fq[TN], fp[MT];
#pragma unroll
      for (int j = 0; j < TN; ++j) fq[j] = QT::frag(lq + (j / TNS) * QT::kBytes, (j % TNS) * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < MT; ++i) fp[i] = PT::frag(from, i * 16, kk, lane);
#pragma unroll
      for (int st = 0; st < Mfma<T>::kSteps; ++st)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = Mfma<T>::mul(st, fq[j], fp[i], acc[i][j]);
    }
  };

  // This wave's stages: s_begin + wave, + NW, ...
  const int S = s_end > s_begin + wave ? (s_end - s_begin - wave + NW - 1) / NW : 0;
  if constexpr (DIRECT) {  // NST - 1 of them in flight
    const uint32_t lds_byte = op_lds_byte(mine);
    int from = 0, to = (NST - 1) * kWaveBytes;
    auto stage = [&](int s, auto whole) {
      constexpr bool W = decltype(whole)::value;
      op_wait_lds();  // what the next loads overwrite was read one turn ago
      __builtin_amdgcn_sched_barrier(0);
      // the stage is there once only the newer stages' loads are in flight
      if (W || s + NST - 1 < S) {
        load(lds_byte + to, whole);
        op_wait_loads<(NST - 1) * kStageLoads>();
      } else {
        op_wait_loads<0>();
      }
      __builtin_amdgcn_sched_barrier(0);
      compute(mine + from);
      to = from;
      from = from == (NST - 1) * kWaveBytes ? 0 : from + kWaveBytes;
    };
#pragma unroll 1
    for (int i = 0; i < NST - 1 && i < S; ++i) load(lds_byte + i * kWaveBytes, std::false_type());
    for (int s = 0; s < S; ++s) {
      for (int n = min(next.whole_steps(g), S - (NST - 1) - s); n > 0; --n, ++s) stage(s, std::true_type());
      next.cross(g);
      if (s < S) stage(s, std::false_type());
    }
  } else {
    constexpr auto any = std::false_type();
    if (S > 0) load(0, any);
    for (int s = 0; s < S; ++s) {
      pt.put(rp, mine, 0, lane);
#pragma unroll
      for (int i = 0; i < kSubs; ++i) qt.put(rq[i], mine + PT::kBytes + i * QT::kBytes, 0, lane);
      if (s + 1 < S) load(0, any);
      __builtin_amdgcn_sched_barrier(0);
      compute(mine);
    }
  }

  // Add the waves' sums, 16 rows at a time: [wave][block][lane] of four floats.
  floatx4* sums = reinterpret_cast<floatx4*>(lds);
  // a wave adds the blocks wave, wave + NW, ... of the 16 columns each
  constexpr int kTurns = (TNS + NW - 1) / NW;
  static_assert(NW * TN * 1024 <= NST * NW * kWaveBytes, "sums fit the ring");
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < TN; ++c) sums[(wave * TN + c) * 64 + lane] = acc[i][c];
    __syncthreads();
    const int m = m0 + i * 16 + l;
    if constexpr (KIND == OP_STATS) {
      if (g.splits <= 1) {  // 16 columns an entry, whole waves
#pragma unroll
        for (int u = 0; u < kTurns; ++u) {
          const int j = wave + u * NW;
          if (j >= TNS) continue;
          floatx4 a[1] = {sums[j * 64 + lane]};
#pragma unroll
          for (int w = 1; w < NW; ++w) a[0] = a[0] + sums[(w * TN + j) * 64 + lane];
          float top, sum;
          op_row_stats<T, 1>(g, a, lane, m0 + i * 16, n0 + j * 16, &top, &sum);
          if (lane < 16 && m < g.M) {
            float* to = g.epi.stats + 2 * ((int64_t)(n0 / 16 + j) * g.M + m);
            to[0] = top;
            to[1] = sum;
          }
        }
        continue;
      }
    }
    if (m >= g.M) continue;
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int j = wave + u * NW, n = n0 + j * 16 + lg * 4, cnt = g.N - n;
      if (j >= TNS || cnt <= 0) continue;
      floatx4 a = sums[j * 64 + lane], b = {};
#pragma unroll
      for (int w = 1; w < NW; ++w) a = a + sums[(w * TN + j) * 64 + lane];
      if constexpr (kGated) {
        b = sums[(j + TNS) * 64 + lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) b = b + sums[(w * TN + j + TNS) * 64 + lane];
      }
      float d0[4], d1[4], b0[4], b1[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        d0[r] = a[r];
        d1[r] = b[r];
      }
      if (g.splits > 1) {
        float* p = g.partial + ((int64_t)(split * kSubs) * g.M + m) * g.N + n;
        store_vec(p, cnt, d0);
        if constexpr (kGated) store_vec(p + (int64_t)g.M * g.N, cnt, d1);
      } else {
        op_biases<T, KIND>(g.epi, n, cnt, b0, b1);
        op_in_units<T, KIND>(op_unit<T, KIND>(g.epi), d0);
        op_epilogue<T, KIND>(g.epi, 0, m, n, cnt, d0, d1, b0, b1);
      }
    }
  }
}

// The splits' partial sums, added in order, and the epilogue: a thread for
// four columns of a row.  Eight splits' sums are loaded at a time.  Bound by
// its launch and one latency of memory at few rows (8 splits of 16 x 4096:
// 4.7 us), by memory at many.
template <typename T, int KIND, typename Args = OpArgs<KIND>>
__global__ void __launch_bounds__(256) op_gemm_reduce(Args g) {
  const int quads = (g.N + 3) / 4, z = blockIdx.y;
  const int64_t t = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
  if (t >= (int64_t)g.M * quads) return;
  const int64_t m = t / quads;
  const int n = (int)(t - m * quads) * 4, cnt = g.N - n;
  const int64_t plane = (int64_t)g.M * g.N, planes = KIND == OP_GATED ? 2 : g.outputs;
  const float* p = g.partial + z * plane + m * g.N + n;
  float d0[4] = {}, d1[4] = {}, b0[4], b1[4];
  op_biases<T, KIND>(g.epi, n, cnt, b0, b1);
  for (int s = 0; s < g.splits; s += 8) {
    float v[8][4], w[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = s + i < g.splits;
      const float* q = p + (in ? (s + i) * (planes * plane) : 0);
      load_vec(q, cnt, v[i]);
      if constexpr (KIND == OP_GATED) load_vec(q + plane, cnt, w[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (s + i < g.splits) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          d0[c] += v[i][c];
          if constexpr (KIND == OP_GATED) d1[c] += w[i][c];
        }
      }
  }
  op_in_units<T, KIND>(op_unit<T, KIND>(g.epi), d0);
  op_epilogue<T, KIND>(g.epi, z, m, n, cnt, d0, d1, b0, b1);
}

// OP_STATS of partial sums: a wave for 256 columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) op_stats_reduce(OpGemmMore g) {
  const OpEpilogueMore& e = g.epi;
  const int lane = threadIdx.x & 63, entries = (g.N + 255) / 256;
  const int64_t id = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t m = id / entries;
  if (m >= g.M) return;
  const int entry = (int)(id - m * entries), n = entry * 256 + lane * 4, cnt = g.N - n;
  const int64_t plane = (int64_t)g.M * g.N;
  const float* p = g.partial + m * g.N + n;
  float z[4] = {}, b0[4], b1[4], top = -__builtin_inff(), sum = 0.0f;
  op_biases<T, OP_STATS>(e, n, cnt, b0, b1);
  for (int s = 0; s < g.splits; ++s) {
    float v[4];
    load_vec(p + (cnt > 0 ? s * plane : 0), cnt, v);
#pragma unroll
    for (int r = 0; r < 4; ++r) z[r] += v[r];
  }
  const int label = e.labels ? e.labels[m] : -1;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    z[r] += b0[r];
    if (r < cnt && label == n + r) e.at_label[m] = z[r];
    if (r >= cnt) z[r] = -__builtin_inff();
    top = fmaxf(top, z[r]);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
  const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
  for (int r = 0; r < 4; ++r) sum += op_exp<T>(z[r] - base);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, kWave);
  if (lane == 0) {
    e.stats[2 * (entry * (int64_t)g.M + m)] = top;
    e.stats[2 * (entry * (int64_t)g.M + m) + 1] = sum;
  }
}

// ---------------------------------------------------------------------------
template <bool FLAT, bool TRIANGLE, typename G>
dim3 op_grid(const G& g) {
  const int64_t tiles = TRIANGLE ? (int64_t)g.tiles_m * (g.tiles_m + 1) / 2 : (int64_t)g.tiles_m * g.tiles_n;
  return FLAT ? dim3((unsigned)(tiles * g.splits * g.outputs))
              : dim3((unsigned)tiles, (unsigned)g.splits, (unsigned)g.outputs);
}

template <typename T, int LAYOUT, int KIND, int BM, int BN>
hipError_t launch_staged(OpArgs<KIND>& g, hipStream_t st) {
  constexpr int SN = KIND == OP_GATED ? BN / 2 : BN;
  g.tiles_m = (g.M + BM - 1) / BM;
  g.tiles_n = (g.N + SN - 1) / SN;
  return op_launch(op_gemm_staged<T, LAYOUT, KIND, BM, BN>,
                   op_grid<kFlat<KIND>, false>(g), dim3(256), st, g);
}

template <typename T, int LAYOUT, int KIND, int BM, int BN, int WGM, int WGN, int KS, int NST>
hipError_t launch_middle(OpArgs<KIND>& g, hipStream_t st) {
  constexpr int SN = KIND == OP_GATED ? BN / 2 : BN;
  g.tiles_m = (g.M + BM - 1) / BM;
  g.tiles_n = (g.N + SN - 1) / SN;
  return op_launch(op_gemm_middle<T, LAYOUT, KIND, BM, BN, WGM, WGN, KS, NST>,
                   op_grid<kFlat<KIND>, KIND == OP_MIRROR>(g), dim3(512), st, g);
}

template <int LAYOUT, int KIND>
hipError_t launch_pairs(OpGemmMore g, hipStream_t st) {
  g.tiles_m = (g.M + 63) / 64;
  g.tiles_n = (g.N + 63) / 64;
  g.pieces = 1;
  return op_launch(op_gemm_pairs<LAYOUT, KIND, 64, 64, 2, 4, 4>, op_grid<true, KIND == OP_MIRROR>(g), dim3(512), st, g);
}

template <typename T, int LAYOUT, int KIND>
hipError_t launch_large(OpArgs<KIND>& g, hipStream_t st) {
  constexpr int SN = KIND == OP_GATED ? 128 : 256;
  g.tiles_m = (g.M + 255) / 256;
  g.tiles_n = (g.N + SN - 1) / SN;
  return op_launch(op_gemm_large<T, LAYOUT, KIND>, op_grid<kFlat<KIND>, KIND == OP_MIRROR>(g), dim3(512), st, g);
}

// Columns, waves and ring of the skinny form: what fits a CU's 160 KB of LDS.
// (64 columns, a whole cache line of 16-bit W, measured as fast as the 64x64
// tile where W comes from memory, and slower where it is small.)
template <int KIND, int MT, bool DIRECT>
struct SkinnyShape {
  static constexpr int kCols = 32;
  static constexpr int kWaves = KIND == OP_GATED || MT > 1 ? 4 : 8;
  static constexpr int kStages = !DIRECT ? 1 : KIND == OP_GATED ? (MT == 4 ? 2 : 3) : (MT == 2 ? 4 : 3);
};
template <typename T, int LAYOUT, int KIND, int MT, bool DIRECT>
hipError_t launch_skinny(OpArgs<KIND>& g, hipStream_t st) {
  using S = SkinnyShape<KIND, MT, DIRECT>;
  g.tiles_m = (g.M + 16 * MT - 1) / (16 * MT);
  g.tiles_n = (g.N + S::kCols - 1) / S::kCols;
  return op_launch(op_gemm_skinny<T, LAYOUT, KIND, MT, S::kCols, S::kWaves, S::kStages, DIRECT>,
                   op_grid<kFlat<KIND>, false>(g), dim3(S::kWaves * 64), st, g);
}

template <typename T, int LAYOUT, int KIND>
hipError_t launch(const OpPlan& plan, OpArgs<KIND>& g, hipStream_t st) {
  g.splits = plan.splits;
  g.stages_per_split = plan.stages_per_split;
  hipError_t e = hipErrorInvalidValue;
  constexpr bool kDirectOnly = op_kind_blend(KIND);
  if (kDirectOnly && !g.direct) return hipErrorInvalidValue;
  if (plan.tile >= OP_TILE_SKINNY16) {
    if constexpr (LAYOUT == OP_TN || op_kind_blend(KIND)) {
      return hipErrorInvalidValue;
    } else if (g.direct || kDirectOnly) {
      e = plan.tile == OP_TILE_SKINNY16   ? launch_skinny<T, LAYOUT, KIND, 1, true>(g, st)
          : plan.tile == OP_TILE_SKINNY32 ? launch_skinny<T, LAYOUT, KIND, 2, true>(g, st)
                                          : launch_skinny<T, LAYOUT, KIND, 4, true>(g, st);
    } else if constexpr (!kDirectOnly) {
      e = plan.tile == OP_TILE_SKINNY16   ? launch_skinny<T, LAYOUT, KIND, 1, false>(g, st)
          : plan.tile == OP_TILE_SKINNY32 ? launch_skinny<T, LAYOUT, KIND, 2, false>(g, st)
                                          : launch_skinny<T, LAYOUT, KIND, 4, false>(g, st);
    }
  } else if (plan.tile == OP_TILE_64) {
    constexpr int WGM = KIND == OP_GATED ? 4 : 2;  // a wave has columns of both weight matrices
    bool pairs = false;
    if constexpr (op_kind_blend(KIND)) pairs = g.pieces == 3;
    if (pairs) {
      if constexpr (op_kind_blend(KIND)) e = launch_pairs<LAYOUT, KIND>(g, st);
    } else if (g.direct || kDirectOnly) e = launch_middle<T, LAYOUT, KIND, 64, 64, WGM, 8 / WGM, 2, 4>(g, st);
    else if constexpr (!kDirectOnly) e = launch_staged<T, LAYOUT, KIND, 64, 64>(g, st);
  } else if (plan.tile == OP_TILE_128) {
    if (g.direct || kDirectOnly) e = launch_middle<T, LAYOUT, KIND, 128, 128, 2, 4, 1, 4>(g, st);
    else if constexpr (!kDirectOnly) e = launch_staged<T, LAYOUT, KIND, 128, 128>(g, st);
  } else if (!g.direct) {
    return hipErrorInvalidValue;  // the other tiles have no form through registers
  } else if (plan.tile == OP_TILE_256) {
    e = launch_large<T, LAYOUT, KIND>(g, st);
  } else if constexpr (KIND != OP_MIRROR) {
    e = plan.tile == OP_TILE_256X128 ? launch_middle<T, LAYOUT, KIND, 256, 128, 4, 2, 1, 3>(g, st)
                                     : launch_middle<T, LAYOUT, KIND, 64, 128, 2, 4, 1, 4>(g, st);
  }
  if (e != hipSuccess || g.splits <= 1) return e;
  if constexpr (KIND == OP_STATS) {
    const int64_t blocks = ((int64_t)g.M * ((g.N + 255) / 256) + 3) / 4, x = std::min<int64_t>(blocks, int64_t{1} << 20);
    return op_launch(op_stats_reduce<T>, dim3((unsigned)x, (unsigned)((blocks + x - 1) / x)), dim3(256), st, g);
  }
  const int64_t quads = (int64_t)g.M * ((g.N + 3) / 4);
  const int64_t blocks = (quads + 255) / 256, x = std::min<int64_t>(blocks, int64_t{1} << 20);
  return op_launch(op_gemm_reduce<T, KIND>,
                   dim3((unsigned)x, (unsigned)g.outputs, (unsigned)((blocks + x - 1) / x)), dim3(256), st, g);
}

template <typename T>
hipError_t op_gemm(int layout, int kind, const OpPlan& plan, OpGemm& g, hipStream_t st) {
  if (layout == OP_NN && kind == OP_LINEAR) return launch<T, OP_NN, OP_LINEAR>(plan, g, st);
  if (layout == OP_NN && kind == OP_GATED) return launch<T, OP_NN, OP_GATED>(plan, g, st);
  if (layout == OP_NT && kind == OP_STORE) return launch<T, OP_NT, OP_STORE>(plan, g, st);
  if (layout == OP_TN && kind == OP_STORE) return launch<T, OP_TN, OP_STORE>(plan, g, st);
  return hipErrorInvalidValue;
}

template <typename T>
hipError_t op_gemm_loss(int layout, int kind, const OpPlan& plan, OpGemmMore& g, hipStream_t st) {
  if (layout == OP_NN && kind == OP_STATS) return launch<T, OP_NN, OP_STATS>(plan, g, st);
  if (layout == OP_NN && kind == OP_LOSS_GRAD) return launch<T, OP_NN, OP_LOSS_GRAD>(plan, g, st);
  if (layout == OP_NT && kind == OP_ADD) return launch<T, OP_NT, OP_ADD>(plan, g, st);
  return hipErrorInvalidValue;
}

}  // namespace ops
}  // namespace volta
