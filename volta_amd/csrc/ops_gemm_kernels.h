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

#include "ops_gemm.h"
#include "ops_types.h"

namespace volta {
namespace ops {

typedef __attribute__((address_space(3))) void* LdsPtr;
typedef __attribute__((address_space(3))) shortx4* LdsShort4;

// What a direct load reads where k is past the end.
static __device__ const __attribute__((aligned(16))) uint32_t op_zeros[4] = {0, 0, 0, 0};

typedef uint32_t chunk16_by2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t chunk16_by4 __attribute__((ext_vector_type(4), aligned(4)));
#define VOLTA_GLOBAL __attribute__((address_space(1)))

template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
  static __device__ __forceinline__ floatx4 mul(chunk16 a, chunk16 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
};
template <> struct Mfma<_Float16> {
  static __device__ __forceinline__ floatx4 mul(chunk16 a, chunk16 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0,
                                                  0, 0);
  }
};
template <> struct Mfma<float> {  // lane group g holds k = 4g .. 4g + 3 of 16: step j takes 4g + j
  static __device__ __forceinline__ floatx4 mul(chunk16 a, chunk16 b, floatx4 c) {
    const floatx4 x = __builtin_bit_cast(floatx4, a), y = __builtin_bit_cast(floatx4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
};

// 16 bytes at any element address.
template <typename T>
__device__ __forceinline__ chunk16 load_unaligned(const T* p) {
  if constexpr (sizeof(T) == 2) return *(const VOLTA_GLOBAL chunk16_by2*)p;
  else return *(const VOLTA_GLOBAL chunk16_by4*)p;
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
  __device__ __forceinline__ void issue(const char* base, char* lds, int wave) const {
#pragma unroll
    for (int t = 0; t < kLoads; ++t)
      __builtin_amdgcn_global_load_lds((const void*)(base + off[t]), (LdsPtr)(lds + (wave + t * NW) * 1024), 16, 0, 0);
  }
  __device__ __forceinline__ void issue_tail(const char* base, char* lds, int wave, int lane, int k_left) const {
#pragma unroll
    for (int t = 0; t < kLoads; ++t) {
      int r, c;
      place((wave + t * NW) * 64 + lane, &r, &c);
      const bool in = KC ? c * kE < k_left : r < k_left;
      const char* a = in ? base + off[t] : reinterpret_cast<const char*>(op_zeros);
      __builtin_amdgcn_global_load_lds((const void*)a, (LdsPtr)(lds + (wave + t * NW) * 1024), 16, 0, 0);
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

// What a launch's epilogue has to do, in one word.
constexpr int kHasBias0 = 1, kHasBias1 = 2, kHasPre = 4, kHasResidual = 8, kVec = 16, kActShift = 8;
template <int KIND>
__device__ __forceinline__ int op_epilogue_flags(const OpEpilogue& e) {
  int f = e.vec ? kVec : 0;
  if constexpr (KIND != OP_STORE) {
    f |= (e.bias[0] ? kHasBias0 : 0) | (e.pre[0] ? kHasPre : 0) | (e.act + 1) << kActShift;
    if constexpr (KIND == OP_GATED) f |= e.bias[1] ? kHasBias1 : 0;
    else f |= e.residual ? kHasResidual : 0;
  }
  return f;
}

// The epilogue of four consecutive columns n .. of row m (cnt of them inside).
template <typename T, int KIND>
__device__ __forceinline__ void op_epilogue(const OpEpilogue& e, int flags, int z, int64_t m, int n, int cnt,
                                            float (&d0)[4], float (&d1)[4]) {
  const bool vec = (flags & kVec) && cnt == 4;
  if constexpr (KIND != OP_STORE) {
    float b[4];
    if (flags & kHasBias0) {
      load4(static_cast<const T*>(e.bias[0]) + n, vec, cnt, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) d0[i] += b[i];
    }
    if (flags & kHasPre) store4(static_cast<T*>(e.pre[0]) + m * e.ld_pre + n, vec, cnt, d0);
    const int act = (flags >> kActShift) - 1;
    if constexpr (KIND == OP_GATED) {
      if (flags & kHasBias1) {
        load4(static_cast<const T*>(e.bias[1]) + n, vec, cnt, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) d1[i] += b[i];
      }
      if (flags & kHasPre) store4(static_cast<T*>(e.pre[1]) + m * e.ld_pre + n, vec, cnt, d1);
    }
    op_act4<T>(act, d0);
    if constexpr (KIND == OP_GATED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) d0[i] *= d1[i];
    } else if (flags & kHasResidual) {
      load4(static_cast<const T*>(e.residual) + m * e.ld_residual + n, vec, cnt, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) d0[i] += b[i];
    }
  }
  store4(static_cast<T*>(e.out[z]) + m * e.ld_out + n, vec, cnt, d0);
}

__device__ __forceinline__ void store_partial(float* p, int N, int cnt, const float (&d)[4]) {
  store4<float>(p, (N & 3) == 0 && cnt == 4, cnt, d);
}

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

// ---------------------------------------------------------------------------
// Tiled product: BM x BN of D per block, WGM x WGN waves, two stages in LDS --
// the loads of stage s + 1 are issued before stage s is multiplied.
// ---------------------------------------------------------------------------
template <typename T, int LAYOUT, int KIND, int BM, int BN, int WGM, int WGN, bool DIRECT>
__global__ void __launch_bounds__(WGM* WGN * 64) op_gemm_tiled(OpGemm g) {
  constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr bool kGated = KIND == OP_GATED;
  constexpr int kSubs = kGated ? 2 : 1, SN = BN / kSubs;  // gated: half the columns of each weight matrix
  constexpr int TNS = TN / kSubs;
  constexpr bool P_KC = LAYOUT != OP_TN, Q_KC = LAYOUT == OP_NT;
  using PT = Tile<T, BM, P_KC, NW>;
  using QT = Tile<T, SN, Q_KC, NW>;
  constexpr int kStageK = PT::kStageK;
  // one array for each operand and stage: the compiler sees that the loads
  // into one do not touch what is read from the other
  __shared__ __attribute__((aligned(16))) char lds_p0[PT::kBytes];
  __shared__ __attribute__((aligned(16))) char lds_q0[QT::kBytes * kSubs];
  __shared__ __attribute__((aligned(16))) char lds_p1[PT::kBytes];
  __shared__ __attribute__((aligned(16))) char lds_q1[QT::kBytes * kSubs];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  int tm, tn;
  op_tile_of(blockIdx.x, g.tiles_m, g.tiles_n, &tm, &tn);
  const int m0 = tm * BM, n0 = tn * SN;
  const int z = g.outputs > 1 ? blockIdx.z : 0, split = blockIdx.y;
  const int p_left = g.M - m0, q_left = g.N - n0;

  PT pt;
  QT qt;
  pt.init(g.ld_p, p_left, wave, lane);
  qt.init(g.ld_q, q_left, wave, lane);
  const int per_piece = (g.K + kStageK - 1) / kStageK;
  const int s_begin = split * g.stages_per_split;
  const int s_end = min(per_piece * g.pieces, s_begin + g.stages_per_split);

  auto base_of = [&](const void* p, int64_t ld, bool kc, int x0, int k) {
    const int64_t e = kc ? (int64_t)x0 * ld + k : (int64_t)k * ld + x0;
    return static_cast<const char*>(p) + e * (int64_t)sizeof(T);
  };
  chunk16 rp[DIRECT ? 1 : PT::kLoads], rq[kSubs][DIRECT ? 1 : QT::kLoads];
  auto load = [&](int s, char* lp, char* lq) {
    const int piece = s >= per_piece ? 1 : 0;
    const int k = (s - piece * per_piece) * kStageK, k_left = g.K - k;
    const char* bp = base_of(g.p[piece], g.ld_p, P_KC, m0, k);
    const char* bq[kSubs];
#pragma unroll
    for (int i = 0; i < kSubs; ++i)
      bq[i] = base_of(g.q[kGated ? i : LAYOUT == OP_TN ? z : piece], g.ld_q, Q_KC, n0, k);
    if constexpr (DIRECT) {
      if (k_left >= kStageK) {
        pt.issue(bp, lp, wave);
#pragma unroll
        for (int i = 0; i < kSubs; ++i) qt.issue(bq[i], lq + i * QT::kBytes, wave);
      } else {
        pt.issue_tail(bp, lp, wave, lane, k_left);
#pragma unroll
        for (int i = 0; i < kSubs; ++i) qt.issue_tail(bq[i], lq + i * QT::kBytes, wave, lane, k_left);
      }
    } else {
      pt.fetch(bp, rp, wave, lane, p_left, k_left);
#pragma unroll
      for (int i = 0; i < kSubs; ++i) qt.fetch(bq[i], rq[i], wave, lane, q_left, k_left);
    }
  };
  auto put = [&](char* lp, char* lq) {
    if constexpr (!DIRECT) {
      pt.put(rp, lp, wave, lane);
#pragma unroll
      for (int i = 0; i < kSubs; ++i) qt.put(rq[i], lq + i * QT::kBytes, wave, lane);
    }
  };

  floatx4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  auto compute = [&](const char* lp, const char* lq) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      chunk16 fp[TM], fq[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
        fq[j] = QT::frag(lq + (j / TNS) * QT::kBytes, (wn * TNS + j % TNS) * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < TM; ++i) fp[i] = PT::frag(lp, wm * WM + i * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = Mfma<T>::mul(fq[j], fp[i], acc[i][j]);
    }
  };
  // Stage s has arrived (its loads, or its chunks from registers), and every
  // wave has finished reading the other pair of arrays.
  auto arrived = [&](char* lp, char* lq) {
    if constexpr (DIRECT) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
      put(lp, lq);
    }
    __syncthreads();
  };

  if (s_begin < s_end) load(s_begin, lds_p0, lds_q0);
  for (int s = s_begin; s < s_end; s += 2) {
    arrived(lds_p0, lds_q0);
    if (s + 1 < s_end) load(s + 1, lds_p1, lds_q1);
    __builtin_amdgcn_sched_barrier(0);
    compute(lds_p0, lds_q0);
    if (s + 1 < s_end) {
      arrived(lds_p1, lds_q1);
      if (s + 2 < s_end) load(s + 2, lds_p0, lds_q0);
      __builtin_amdgcn_sched_barrier(0);
      compute(lds_p1, lds_q1);
    }
  }

  // Lane: row l % 16 of its block, columns 4 (l / 16) ..
  const int all_flags = op_epilogue_flags<KIND>(g.epi);
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + i * 16 + (lane & 15);
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < TNS; ++j) {
      const int n = n0 + (wn * TNS + j) * 16 + (lane >> 4) * 4, cnt = min(4, g.N - n);
      if (cnt <= 0) continue;
      float d0[4], d1[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        d0[r] = acc[i][j][r];
        d1[r] = kGated ? acc[i][j + TNS * (kSubs - 1)][r] : 0.0f;
      }
      // asked anew for each block: the compiler would else make a copy of all
      // blocks' epilogues for each answer, and spill the sums on the way there
      int flags = all_flags;
      asm volatile("" : "+s"(flags));
      if (g.splits > 1) {
        const int64_t planes = kGated ? 2 : g.outputs;
        float* p = g.partial + ((split * planes + z) * g.M + m) * (int64_t)g.N + n;
        store_partial(p, g.N, cnt, d0);
        if constexpr (kGated) store_partial(p + (int64_t)g.M * g.N, g.N, cnt, d1);
      } else {
        op_epilogue<T, KIND>(g.epi, flags, z, m, n, cnt, d0, d1);
      }
      __builtin_amdgcn_sched_barrier(0);  // one block's values in flight
    }
  }
}

// ---------------------------------------------------------------------------
// Skinny product, M <= 16 MT: each weight is read once and bounds the time.
// A block takes 32 columns (of each weight matrix) and its waves take turns
// over the stages of k, each with stages of its own in LDS (no barrier before
// the end); the waves' sums are added at the end, in wave order.
// ---------------------------------------------------------------------------
template <typename T, int LAYOUT, int KIND, int MT, int NW, int NST, bool DIRECT>
__global__ void __launch_bounds__(NW * 64) op_gemm_skinny(OpGemm g) {
  constexpr bool kGated = KIND == OP_GATED, Q_KC = LAYOUT == OP_NT;
  constexpr int kSubs = kGated ? 2 : 1, BN = 32, TN = 2 * kSubs;
  using QT = Tile<T, BN, Q_KC, 1>;
  constexpr int kStageK = QT::kStageK, kE = QT::kE;
  constexpr int kWaveBytes = QT::kBytes * kSubs;
  constexpr int kSumBytes = NW * MT * TN * 1024;
  constexpr int kLds = NW * NST * kWaveBytes;
  __shared__ __attribute__((aligned(16))) char lds[kLds > kSumBytes ? kLds : kSumBytes];

  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // blocks next to each other share cache lines of W: one XCD takes a run of them
  int tm, tn;
  op_tile_of(blockIdx.x, 1, g.tiles_n, &tm, &tn);
  const int n0 = tn * BN, split = blockIdx.y, q_left = g.N - n0;
  QT qt;
  qt.init(g.ld_q, q_left, 0, lane);
  const int per_piece = (g.K + kStageK - 1) / kStageK;
  const int s_begin = split * g.stages_per_split;
  const int s_end = min(per_piece * g.pieces, s_begin + g.stages_per_split);
  char* mine = lds + wave * (NST * kWaveBytes);

  int64_t p_row[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) p_row[i] = (int64_t)min(i * 16 + l, g.M - 1) * g.ld_p;

  chunk16 fp[NST][MT][2];
  chunk16 rq[DIRECT ? 1 : NST][kSubs][DIRECT ? 1 : QT::kLoads];
  auto load = [&](int s, int slot) {
    const int piece = s >= per_piece ? 1 : 0;
    const int k = (s - piece * per_piece) * kStageK, k_left = g.K - k;
    char* to = mine + slot * kWaveBytes;
#pragma unroll
    for (int i = 0; i < kSubs; ++i) {
      const char* base = static_cast<const char*>(g.q[kGated ? i : piece]) +
                         (Q_KC ? (int64_t)n0 * g.ld_q + k : (int64_t)k * g.ld_q + n0) * (int64_t)sizeof(T);
      if constexpr (DIRECT) {
        if (k_left >= kStageK) qt.issue(base, to + i * QT::kBytes, 0);
        else qt.issue_tail(base, to + i * QT::kBytes, 0, lane, k_left);
      } else {
        qt.fetch(base, rq[slot][i], 0, lane, q_left, k_left);
      }
    }
    const T* p = static_cast<const T*>(g.p[piece]) + k;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int c = (4 * kk + lg) * kE, have = k_left - c;
        const T* a = p + p_row[i] + c;
        if constexpr (DIRECT) {
          // always one load, so that the loads in flight can be counted
          const void* from = have > 0 ? (const void*)a : (const void*)op_zeros;
          fp[slot][i][kk] = *(const VOLTA_GLOBAL chunk16*)from;
        } else {
          if (have >= kE) fp[slot][i][kk] = load_unaligned(a);
          else if (have <= 0) fp[slot][i][kk] = chunk16{0, 0, 0, 0};
          else fp[slot][i][kk] = load_part(a, have);
        }
      }
  };

  floatx4 acc[MT][TN];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  auto compute = [&](int slot) {
    char* from = mine + slot * kWaveBytes;
    if constexpr (!DIRECT) {
#pragma unroll
      for (int i = 0; i < kSubs; ++i) qt.put(rq[slot][i], from + i * QT::kBytes, 0, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      chunk16 fq[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) fq[j] = QT::frag(from + (j >> 1) * QT::kBytes, (j & 1) * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = Mfma<T>::mul(fq[j], fp[slot][i][kk], acc[i][j]);
    }
  };

  // This wave's stages: s_begin + wave, + NW, ...  NST - 1 of them in flight.
  int next = s_begin + wave;
#pragma unroll
  for (int i = 0; i < NST - 1; ++i, next += NW)
    if (next < s_end) load(next, i);
  for (int s = s_begin + wave; s < s_end; s += NST * NW) {
#pragma unroll
    for (int i = 0; i < NST; ++i) {
      const int cur = s + i * NW;
      if (cur < s_end) {
        // the slot this overwrites was read one turn ago
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const bool more = next < s_end;
        if (more) load(next, (i + NST - 1) % NST);
        next += NW;
        if constexpr (DIRECT) {
          // loads return in order: all but the newer stages' have to be back
          constexpr int kOps = kSubs * QT::kLoads + MT * 2;
          if (next - NW < s_end) {  // a full ring is in flight
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * kOps) : "memory");
          } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          }
        }
        compute(i);
      }
    }
  }

  // Add the waves' sums: [wave][block][lane] of four floats.
  __syncthreads();
  floatx4* sums = reinterpret_cast<floatx4*>(lds);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) sums[((wave * MT + i) * TN + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int t = tid; t < MT * 2 * 64; t += NW * 64) {
    const int ln = t & 63, j = (t >> 6) & 1, i = t >> 7;
    floatx4 a = sums[(i * TN + j) * 64 + ln], b = {};
#pragma unroll
    for (int w = 1; w < NW; ++w) a = a + sums[((w * MT + i) * TN + j) * 64 + ln];
    if constexpr (kGated) {
      b = sums[(i * TN + j + 2) * 64 + ln];
#pragma unroll
      for (int w = 1; w < NW; ++w) b = b + sums[((w * MT + i) * TN + j + 2) * 64 + ln];
    }
    const int m = i * 16 + (ln & 15), n = n0 + j * 16 + (ln >> 4) * 4, cnt = min(4, g.N - n);
    if (m >= g.M || cnt <= 0) continue;
    float d0[4], d1[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      d0[r] = a[r];
      d1[r] = b[r];
    }
    if (g.splits > 1) {
      float* p = g.partial + ((int64_t)(split * kSubs) * g.M + m) * g.N + n;
      store_partial(p, g.N, cnt, d0);
      if constexpr (kGated) store_partial(p + (int64_t)g.M * g.N, g.N, cnt, d1);
    } else {
      op_epilogue<T, KIND>(g.epi, op_epilogue_flags<KIND>(g.epi), 0, m, n, cnt, d0, d1);
    }
  }
}

// The splits' partial sums, added in order, and the epilogue: a thread for
// four columns of a row.
template <typename T, int KIND>
__global__ void __launch_bounds__(256) op_gemm_reduce(OpGemm g) {
  const int quads = (g.N + 3) / 4, z = blockIdx.y;
  const int64_t t = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
  if (t >= (int64_t)g.M * quads) return;
  const int64_t m = t / quads;
  const int n = (int)(t - m * quads) * 4, cnt = min(4, g.N - n);
  const bool vec = (g.N & 3) == 0;
  const int64_t plane = (int64_t)g.M * g.N, planes = KIND == OP_GATED ? 2 : g.outputs;
  const float* p = g.partial + z * plane + m * g.N + n;
  float d0[4], d1[4] = {}, v[4];
  load4(p, vec, cnt, d0);
  if constexpr (KIND == OP_GATED) load4(p + plane, vec, cnt, d1);
  for (int s = 1; s < g.splits; ++s) {
    p += planes * plane;
    load4(p, vec, cnt, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) d0[i] += v[i];
    if constexpr (KIND == OP_GATED) {
      load4(p + plane, vec, cnt, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) d1[i] += v[i];
    }
  }
  op_epilogue<T, KIND>(g.epi, op_epilogue_flags<KIND>(g.epi), z, m, n, cnt, d0, d1);
}

// ---------------------------------------------------------------------------
template <typename T, int LAYOUT, int KIND, int BM, int BN, int WGM, int WGN, bool DIRECT>
hipError_t launch_tiled(OpGemm& g, hipStream_t st) {
  constexpr int SN = KIND == OP_GATED ? BN / 2 : BN;
  g.tiles_m = (g.M + BM - 1) / BM;
  g.tiles_n = (g.N + SN - 1) / SN;
  hipLaunchKernelGGL((op_gemm_tiled<T, LAYOUT, KIND, BM, BN, WGM, WGN, DIRECT>),
                     dim3((unsigned)(g.tiles_m * g.tiles_n), (unsigned)g.splits, (unsigned)g.outputs),
                     dim3(WGM * WGN * 64), 0, st, g);
  return hipGetLastError();
}

template <typename T, int LAYOUT, int KIND, int MT, bool DIRECT>
hipError_t launch_skinny(OpGemm& g, hipStream_t st) {
  g.tiles_m = 1;
  g.tiles_n = (g.N + 31) / 32;
  constexpr int NW = KIND == OP_GATED ? 4 : 8, NST = KIND == OP_GATED || !DIRECT ? 2 : 4;
  hipLaunchKernelGGL((op_gemm_skinny<T, LAYOUT, KIND, MT, NW, NST, DIRECT>),
                     dim3((unsigned)g.tiles_n, (unsigned)g.splits), dim3(NW * 64), 0, st, g);
  return hipGetLastError();
}

template <typename T, int LAYOUT, int KIND>
hipError_t launch(const OpPlan& plan, OpGemm& g, hipStream_t st) {
  g.splits = plan.splits;
  g.stages_per_split = plan.stages_per_split;
  hipError_t e;
  if (plan.tile == OP_TILE_SKINNY) {
    if constexpr (LAYOUT == OP_TN) {
      return hipErrorInvalidValue;
    } else {
      const int mt = (g.M + 15) / 16;
      if (g.direct)
        e = mt <= 1   ? launch_skinny<T, LAYOUT, KIND, 1, true>(g, st)
            : mt == 2 ? launch_skinny<T, LAYOUT, KIND, 2, true>(g, st)
                      : launch_skinny<T, LAYOUT, KIND, 4, true>(g, st);
      else
        e = mt <= 1   ? launch_skinny<T, LAYOUT, KIND, 1, false>(g, st)
            : mt == 2 ? launch_skinny<T, LAYOUT, KIND, 2, false>(g, st)
                      : launch_skinny<T, LAYOUT, KIND, 4, false>(g, st);
    }
  } else if (plan.tile == OP_TILE_256 && g.direct) {
    if constexpr (sizeof(T) == 2) e = launch_tiled<T, LAYOUT, KIND, 256, 256, 2, 4, true>(g, st);
    else return hipErrorInvalidValue;
  } else if (plan.tile == OP_TILE_64) {
    e = g.direct ? launch_tiled<T, LAYOUT, KIND, 64, 64, 2, 2, true>(g, st)
                 : launch_tiled<T, LAYOUT, KIND, 64, 64, 2, 2, false>(g, st);
  } else {
    e = g.direct ? launch_tiled<T, LAYOUT, KIND, 128, 128, 2, 2, true>(g, st)
                 : launch_tiled<T, LAYOUT, KIND, 128, 128, 2, 2, false>(g, st);
  }
  if (e != hipSuccess || g.splits <= 1) return e;
  const int64_t quads = (int64_t)g.M * ((g.N + 3) / 4);
  const int64_t blocks = (quads + 255) / 256, x = std::min<int64_t>(blocks, int64_t{1} << 20);
  hipLaunchKernelGGL((op_gemm_reduce<T, KIND>),
                     dim3((unsigned)x, (unsigned)g.outputs, (unsigned)((blocks + x - 1) / x)), dim3(256), 0, st, g);
  return hipGetLastError();
}

template <typename T>
hipError_t op_gemm(int layout, int kind, const OpPlan& plan, OpGemm& g, hipStream_t st) {
  if (layout == OP_NN && kind == OP_LINEAR) return launch<T, OP_NN, OP_LINEAR>(plan, g, st);
  if (layout == OP_NN && kind == OP_GATED) return launch<T, OP_NN, OP_GATED>(plan, g, st);
  if (layout == OP_NT && kind == OP_STORE) return launch<T, OP_NT, OP_STORE>(plan, g, st);
  if (layout == OP_TN && kind == OP_STORE) return launch<T, OP_TN, OP_STORE>(plan, g, st);
  return hipErrorInvalidValue;
}

}  // namespace ops
}  // namespace volta
