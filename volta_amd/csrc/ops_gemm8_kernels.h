// Products of e4m3 codes with scales, for one type of the result:
//   D[m][n] = sum over k blocks of 128, b, of sx[m][b] sw[n / 128][b] *
//             (sum over the block's k of x[m][k] w[n][k])
// Both operands have k contiguous, and a stage of 128 bytes of a row is one
// block, so the tiles, their order in LDS, the rings and the epilogues are
// those of ops_gemm_kernels.h.
//
// v_mfma_f32_16x16x128 takes 32 codes of a row a lane and sums a whole block
// for 16x16 of D, exactly scaled by nothing; which k a lane holds does not
// matter as long as both operands agree, so a lane's two chunks are g and g + 4
// of the row's eight.  Its four sums a lane are then added to the running ones,
// times the row's and the columns' scale: 4 FMAs for the 32 cycles that the
// instruction takes, which the vector unit has to spare (scales as powers of
// two in the instruction itself would be free, but ours are floats).
//
// The rows' scales go to LDS with the stage, four bytes a lane, by one load
// more; the columns' one (a wave's columns share their 128) is a scalar load a
// stage ahead.
#pragma once

#include "ops_gemm_kernels.h"

namespace volta {
namespace ops {

typedef int32_t intx8 __attribute__((ext_vector_type(8)));

// 32 codes of a row: chunks g and g + 4.
struct Frag8 {
  chunk16 c[2];
};
__device__ __forceinline__ floatx4 mfma8(const Frag8& a, const Frag8& b) {
  // scale operands of 0 select the instruction without scales
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(intx8, a), __builtin_bit_cast(intx8, b),
                                                          floatx4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
}
template <typename Tile8>
__device__ __forceinline__ Frag8 frag8(const char* tile, int x0, int lane) {
  return Frag8{{Tile8::frag(tile, x0, 0, lane), Tile8::frag(tile, x0, 1, lane)}};
}

// 4 bytes a lane to LDS, lane after lane (op_load_lds).
__device__ __forceinline__ void op_load_lds4(const float* from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)),
               "v"(from)
               : "memory", "m0");
}

// A scalar load whatever the compiler thinks of the asm around it.
__device__ __forceinline__ float scalar_load(const float* p) {
  return *(const __attribute__((address_space(4))) float*)p;
}

// The instruction adds eight products at a time, of which it keeps what is not
// under about 2^-17 of the largest: normal values' sums are 1.2e-5 of their norm
// off, which 16-bit results do not see and float32 ones do.  Those take the
// codes as float16 (exactly) on its instructions, at half the rate or less.
struct Frag16 {
  chunk16 c[4];
};
__device__ __forceinline__ Frag16 widen(const Frag8& f) {
  typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
  Frag16 w;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const half2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(f.c[h][i], 1.0f, false);
      const half2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(f.c[h][i], 1.0f, true);
      w.c[h * 2 + (i >> 1)][(i & 1) * 2] = __builtin_bit_cast(uint32_t, lo);
      w.c[h * 2 + (i >> 1)][(i & 1) * 2 + 1] = __builtin_bit_cast(uint32_t, hi);
    }
  return w;
}

// acc += s t, of blocks TM x TN of 16x16.
template <typename T, int TM, int TN>
__device__ __forceinline__ void mul8(const Frag8 (&fp)[TM], const Frag8 (&fq)[TN], const float (&s)[TM],
                                     floatx4 (&acc)[TM][TN]) {
  if constexpr (sizeof(T) == 4) {
    Frag16 q[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) q[j] = widen(fq[j]);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const Frag16 p = widen(fp[i]);
      floatx4 t[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) t[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < TN; ++j) t[j] = Mfma<_Float16>::mul(0, q[j].c[k], p.c[k], t[j]);
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(t[j][r], s[i], acc[i][j][r]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const floatx4 t = mfma8(fq[j], fp[i]);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(t[r], s[i], acc[i][j][r]);
      }
  }
}

// The rows' scales of a block's tile: row m0 + r of k block b.
struct RowScales {
  const float* at;  // this lane's row, block 0
  int64_t step;     // from a block to the next
  int last;         // the last block
  __device__ __forceinline__ void init(const OpGemmMore& g, int m0, int row) {
    at = g.epi.sx + (int64_t)min(m0 + row, g.M - 1) * g.epi.ld_sx;
    step = g.epi.step_sx;
    last = (g.K + 127) / 128 - 1;
  }
  __device__ __forceinline__ const float* of(int b) const { return at + min(b, last) * step; }
};
// The columns' scales of a wave's columns from n on.
struct ColumnScales {
  const float* at;
  int last;
  __device__ __forceinline__ void init(const OpGemmMore& g, int n) {
    at = g.epi.sw + (int64_t)(min(n, g.N - 1) / 128) * g.epi.ld_sw;
    last = (g.K + 127) / 128 - 1;
  }
  __device__ __forceinline__ float of(int b) const { return scalar_load(at + min(b, last)); }
};

using Cursor8 = Cursor<uint8_t, OP_NT, OP_STORE, OpGemmMore>;

// The linear layer's epilogue by op_write_swapped, one copy of the code for
// each activation.
template <typename T, int TM, int TN>
__device__ __forceinline__ void write_linear8(const OpGemmMore& g, const floatx4 (&acc)[TM][TN], int lane, int m0, int n0) {
  const OpEpilogueMore& e = g.epi;
  float bias[TN][4], none[4];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + j * 16 + (lane >> 4) * 4;
    op_biases<T, OP_LINEAR>(e, n, g.N - n, bias[j], none);
  }
  const T* residual = static_cast<const T*>(e.residual);
  auto run = [&](auto act) {
    op_write_swapped<T>(static_cast<T*>(e.out[0]), e.ld_out, g.M, g.N, acc, lane, m0, n0,
                        [&](int, int j, int m, const floatx4& d, float (&v)[4]) {
                          float r[4] = {};
                          const int n = n0 + j * 16 + (lane >> 4) * 4, cnt = m < g.M ? g.N - n : 0;
                          if (residual) load_vec(residual + (cnt > 0 ? m * e.ld_residual + n : 0), cnt, r);
#pragma unroll
                          for (int k = 0; k < 4; ++k) v[k] = op_act<T>(decltype(act)::value, d[k] + bias[j][k]) + r[k];
                        });
  };
#define VOLTA_ACT_CASE(A) \
  case A: return run(std::integral_constant<int, A>())
  switch (e.act) {
    VOLTA_ACT_CASE(VOLTA_ACT_RELU);
    VOLTA_ACT_CASE(VOLTA_ACT_SIGMOID);
    VOLTA_ACT_CASE(VOLTA_ACT_TANH);
    VOLTA_ACT_CASE(VOLTA_ACT_LEAKY_RELU);
    VOLTA_ACT_CASE(VOLTA_ACT_SILU);
    VOLTA_ACT_CASE(VOLTA_ACT_GELU);
    default: return run(std::integral_constant<int, VOLTA_OP_ACT_NONE>());
  }
#undef VOLTA_ACT_CASE
}

// ---------------------------------------------------------------------------
// BM x BN of D per block, eight waves, a ring of NST stages of KS blocks of k
// (op_gemm_middle).  512 x 4096 x 4096 to bfloat16 20.8 us, 0.83 PFLOP/s, to
// float32 28.6: a block's 32 stages, each as long as its loads take to arrive.
// ---------------------------------------------------------------------------
template <typename T, int BM, int BN, int WGM, int WGN, int KS, int NST>
__global__ void __launch_bounds__(512) op_gemm8_middle(OpGemmMore g) {
  constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  using PT = Tile<uint8_t, BM, true, 8>;
  using QT = Tile<uint8_t, BN, true, 8>;
  constexpr int kPart = PT::kBytes + QT::kBytes + BM * 4, kStageBytes = KS * kPart;
  constexpr int kStageLoads = KS * (PT::kLoads + QT::kLoads + 1);
  __shared__ __attribute__((aligned(16))) char lds[NST * kStageBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const OpPlace place = op_place<true, false>(g);
  const int m0 = place.tm * BM, n0 = place.tn * BN, split = place.split;
  PT pt;
  QT qt;
  pt.init(g.ld_p, g.M - m0, wave, lane);
  qt.init(g.ld_q, g.N - n0, wave, lane);
  // every wave loads 64 rows' scales, so that all count the same loads; waves
  // that load the same rows write the same values
  const int scales_at = wave % (BM / 64) * 64;
  RowScales sx;
  sx.init(g, m0, scales_at + lane);
  ColumnScales sw;
  sw.init(g, n0 + wn * WN);
  const int s_begin = split * g.stages_per_split;
  const int blocks = (g.K + 127) / 128;
  int parts = min(blocks, s_begin + g.stages_per_split) - s_begin;
  const int S = (parts + KS - 1) / KS;
  Cursor8 next;
  next.init(g, m0, n0, 0, s_begin, 1);
  auto load = [&](uint32_t to, auto whole) {
    constexpr bool W = decltype(whole)::value;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int k_left = W ? 128 : parts > i ? g.K - next.k : 0;  // a part behind the last one is zeros
      const uint32_t lp = to + i * kPart, lq = lp + PT::kBytes;
      op_load_lds4(sx.of(next.k >> 7), lq + QT::kBytes + scales_at * 4);
      if (W || k_left >= 128) {
        qt.issue(next.q[0], lq, wave);
        pt.issue(next.p, lp, wave);
      } else {
        qt.issue_tail(next.q[0], lq, wave, lane, k_left);
        pt.issue_tail(next.p, lp, wave, lane, k_left);
      }
      next.step();
    }
    parts -= KS;
  };

  floatx4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  int from = 0, to = (NST - 1) * kStageBytes;
  const uint32_t lds_byte = op_lds_byte(lds);
  float w_scale[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) w_scale[i] = sw.of(s_begin + i);
  auto stage = [&](int s, auto whole) {
    constexpr bool W = decltype(whole)::value;
    Frag8 fp[KS][TM], fq[KS][TN];
    float sc[KS][TM], w_next[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) w_next[i] = sw.of(s_begin + (s + 1) * KS + i);
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const char* part = lds + from + kk * kPart;
      const float* scales = reinterpret_cast<const float*>(part + PT::kBytes + QT::kBytes);
#pragma unroll
      for (int j = 0; j < TN; ++j) fq[kk][j] = frag8<QT>(part + PT::kBytes, wn * WN + j * 16, lane);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        fp[kk][i] = frag8<PT>(part, wm * WM + i * 16, lane);
        sc[kk][i] = scales[wm * WM + i * 16 + (lane & 15)];
      }
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
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
#pragma unroll
      for (int i = 0; i < TM; ++i) sc[kk][i] *= w_scale[kk];
      mul8<T, TM, TN>(fp[kk], fq[kk], sc[kk], acc);
      w_scale[kk] = w_next[kk];
    }
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
      for (int n = min(min(next.whole_steps(g), parts) / KS, S - (NST - 1) - s); n > 0; --n, ++s)
        stage(s, std::true_type());
      if (s < S) stage(s, std::false_type());
    }
    if (wave < 4) op_barrier();
  }
  __syncthreads();  // the ring is free
  static_assert(8 * op_region_bytes<TM, TN> <= NST * kStageBytes, "output regions fit the ring");
  op_write_out<T, OP_LINEAR>(g, acc, lds + wave * op_region_bytes<TM, TN>, lane, m0 + wm * WM, n0 + wn * WN, 0, split);
}

// ---------------------------------------------------------------------------
// Large product of codes: 256x256 of D per block, in the regions, phases and
// order of loads of op_gemm_large.  A stage is one block of k: two phases of 16
// matrix instructions of 32 cycles, and the 64 FMAs that scale a phase's sums.
// K is whole blocks: the code for a last part of one takes registers that the
// loop then spills.  The rows' 256 scales are a fifth load of
// the stage's first half, read with P0 before that half's place is loaded
// again.  8192 x 4096 x 16384 to bfloat16 with SiLU 555 us, 1.98 PFLOP/s, matrix
// instructions 46 % busy: of a tile's 70 us 25 are the epilogue and the next one's
// start (K = 16384 reaches 2.6).
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) op_gemm8_large(OpGemmMore g) {
  constexpr int kRegion = 128 * 128, kScales = 8 * kRegion;
  using PR = Region<uint8_t, true, 64, 128>;
  using QR = Region<uint8_t, true, 32, 64>;
  static_assert(PR::kBytes == kRegion && PR::kLoads == 2, "two loads a wave and region");
  __shared__ __attribute__((aligned(16))) char lds[kScales + 2 * 1024];  // [stage & 1][P0, P1, Q0, Q1], [stage & 1][256]

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const OpPlace place = op_place<true, false>(g);
  const int m0 = place.tm * 256, n0 = place.tn * 256, split = place.split;
  PR pr[2];
  QR qr[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    pr[h].init(g.ld_p, h * 64, g.M - m0, wave, lane);
    qr[h].init(g.ld_q, h * 32, g.N - n0, wave, lane);
    // opaque, or each is kept with the upper half of the product it comes from
#pragma unroll
    for (int i = 0; i < 2; ++i) asm volatile("" : "+v"(pr[h].off[i]), "+v"(qr[h].off[i]));
  }
  // every wave loads 64 rows' scales; the two that load the same rows write the same values
  RowScales sx;
  sx.init(g, m0, (wave & 3) * 64 + lane);
  ColumnScales sw;
  sw.init(g, n0 + wn * 64);
  const int s_begin = split * g.stages_per_split;
  const int S = min((g.K + 127) / 128, s_begin + g.stages_per_split) - s_begin;
  Cursor8 next[2];  // the halves are loaded in different phases
  next[0].init(g, m0, n0, 0, s_begin, 1);
  next[1].init(g, m0, n0, 0, s_begin, 1);
  const uint32_t lds_byte = op_lds_byte(lds);
  auto load = [&](int to, auto half) {
    constexpr int h = decltype(half)::value;
    if constexpr (h == 0) op_load_lds4(sx.of(next[0].k >> 7), lds_byte + kScales + (to ? 1024 : 0) + (wave & 3) * 256);
    qr[h].issue(next[h].q[0], lds_byte + to + (2 + h) * kRegion, wave);
    pr[h].issue(next[h].p, lds_byte + to + h * kRegion, wave);
    next[h].step();
  };
  floatx4 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  Frag8 fp[4], fq[4];
  float sc[8];
  auto read_p = [&](const char* from) {
#pragma unroll
    for (int i = 0; i < 4; ++i) fp[i] = frag8<PR>(from, wm * 64 + i * 16, lane);
  };
  auto read_q = [&](const char* from, int h) {
#pragma unroll
    for (int j = 0; j < 2; ++j) fq[2 * h + j] = frag8<QR>(from, wn * 32 + j * 16, lane);
  };
  // Blocks (half 4 + i, j) of the phase, j in twos so that Q1 is not needed at
  // once.  A block's sums are scaled kLate instructions behind its own, in an
  // order that the compiler keeps: its own would wait for each of them.  The
  // last ones' are left for the next phase, where this wave reads LDS and the
  // other one multiplies.
  constexpr int kLate = 3;
  floatx4 t[kLate + 1];
  float late[2];  // the scales of the rows of the blocks left
  auto scale = [&](int half, int o, float by) {
    const int i = half * 4 + ((o >> 1) & 3), j = (o & 1) + (o >> 3) * 2;
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(t[o % (kLate + 1)][r], by, acc[i][j][r]);
  };
  auto mul = [&](int half) {
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      t[n % (kLate + 1)] = mfma8(fq[(n & 1) + (n >> 3) * 2], fp[(n >> 1) & 3]);
      if (n >= kLate) scale(half, n - kLate, sc[half * 4 + (((n - kLate) >> 1) & 3)]);
      __builtin_amdgcn_sched_barrier(0);
    }
    late[0] = sc[half * 4 + 2];
    late[1] = sc[half * 4 + 3];
  };
  auto scale_late = [&](int half) {
#pragma unroll
    for (int o = 16 - kLate; o < 16; ++o) scale(half, o, late[((o >> 1) & 3) - 2]);
  };
  constexpr auto H0 = std::integral_constant<int, 0>();
  constexpr auto H1 = std::integral_constant<int, 1>();
  int from = 0;  // byte of the stage in LDS
  float w_scale = sw.of(s_begin);
  auto stage = [&](int s, auto behind) {
    constexpr int left = decltype(behind)::value;  // stages behind this one: 0, 1, or more
    const char* at = lds + from;
    const float w_next = sw.of(s_begin + s + 1);
    read_q(at + 2 * kRegion, 0);
    read_p(at);
    const float* scales = reinterpret_cast<const float*>(lds + kScales + (from ? 1024 : 0));
#pragma unroll
    for (int i = 0; i < 8; ++i) sc[i] = scales[wm * 128 + i * 16 + (lane & 15)];
    __builtin_amdgcn_sched_barrier(0);
    scale_late(1);  // of the stage before, while LDS is read
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (left >= 1) {
      load(from ^ 4 * kRegion, H1);
      op_wait_loads<9>();  // P1 of s is there
    } else {
      op_wait_loads<0>();
    }
    op_wait_lds();
    op_barrier();
#pragma unroll
    for (int i = 0; i < 8; ++i) sc[i] *= w_scale;
    w_scale = w_next;
    read_q(at + 3 * kRegion, 1);  // arrives while Q0 is multiplied
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    mul(0);
    __builtin_amdgcn_s_setprio(0);
    op_barrier();
    read_p(at + kRegion);
    __builtin_amdgcn_sched_barrier(0);
    scale_late(0);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (left >= 2) {
      load(from, H0);
      op_wait_loads<7>();  // P0, Q0, Q1 and the scales of s + 1 are there
    } else {
      op_wait_loads<2>();
    }
    from ^= 4 * kRegion;
    op_wait_lds();
    op_barrier();
    __builtin_amdgcn_s_setprio(1);
    mul(1);
    __builtin_amdgcn_s_setprio(0);
    op_barrier();
  };
#pragma unroll
  for (int i = 0; i <= kLate; ++i) t[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  late[0] = late[1] = 0.0f;
  load(0, H0);
  load(0, H1);
  if (S > 1) {
    load(4 * kRegion, H0);
    op_wait_loads<7>();  // P0, Q0, Q1 and the scales of the first stage are there
  } else {
    op_wait_loads<2>();
  }
  op_barrier();
  if (wm == 1) op_barrier();
  int s = 0;
  for (; s < S - 2; ++s) stage(s, std::integral_constant<int, 2>());
  if (s < S - 1) stage(s++, std::integral_constant<int, 1>());
  stage(s, std::integral_constant<int, 0>());
  scale_late(1);
  if (wm == 0) op_barrier();
  if (g.splits <= 1) return write_linear8<T>(g, acc, lane, m0 + wm * 128, n0 + wn * 64);
  __syncthreads();  // the regions are free
  static_assert(8 * op_region_bytes<8, 4> <= 8 * kRegion, "output regions fit");
  op_write_out<T, OP_LINEAR>(g, acc, lds + wave * op_region_bytes<8, 4>, lane, m0 + wm * 128, n0 + wn * 64, 0, split);
}

// ---------------------------------------------------------------------------
// The same through registers, for rows that direct loads cannot take
// (op_gemm_staged).  300 x 1000 x 2500: 11.4 us, eight stages whose loads are
// waited for one after another.
// ---------------------------------------------------------------------------
template <typename T, int BM, int BN>
__global__ void __launch_bounds__(256) op_gemm8_staged(OpGemmMore g) {
  constexpr int NW = 4, WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
  using PT = Tile<uint8_t, BM, true, NW>;
  using QT = Tile<uint8_t, BN, true, NW>;
  constexpr int kStageBytes = PT::kBytes + QT::kBytes;
  __shared__ __attribute__((aligned(16))) char lds[2 * kStageBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const OpPlace place = op_place<true, false>(g);
  const int m0 = place.tm * BM, n0 = place.tn * BN, split = place.split;
  const int p_left = g.M - m0, q_left = g.N - n0;
  PT pt;
  QT qt;
  pt.init(g.ld_p, p_left, wave, lane);
  qt.init(g.ld_q, q_left, wave, lane);
  RowScales sx[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) sx[i].init(g, m0, wm * WM + i * 16 + (lane & 15));
  ColumnScales sw;
  sw.init(g, n0 + wn * WN);
  const int s_begin = split * g.stages_per_split, s_end = min((g.K + 127) / 128, s_begin + g.stages_per_split);
  Cursor8 next;
  next.init(g, m0, n0, 0, s_begin, 1);
  chunk16 rp[PT::kLoads], rq[QT::kLoads];
  float scale[TM], now[TM];
  int block = s_begin;
  auto fetch = [&]() {
    const int k_left = g.K - next.k;
    pt.fetch(next.p, rp, wave, lane, p_left, k_left);
    qt.fetch(next.q[0], rq, wave, lane, q_left, k_left);
    const float w = sw.of(block);
#pragma unroll
    for (int i = 0; i < TM; ++i) scale[i] = *sx[i].of(block) * w;
    ++block;
    next.step();
  };
  auto put = [&](char* to) {
    pt.put(rp, to, wave, lane);
    qt.put(rq, to + PT::kBytes, wave, lane);
#pragma unroll
    for (int i = 0; i < TM; ++i) now[i] = scale[i];
    __syncthreads();
  };
  floatx4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  if (s_begin < s_end) fetch();
  for (int s0 = s_begin; s0 < s_end; s0 += 2) {
    op_unroll<2>([&](auto i) {
      const int s = s0 + i;
      if (s >= s_end) return;
      char* at = lds + decltype(i)::value * kStageBytes;
      put(at);
      if (s + 1 < s_end) fetch();
      __builtin_amdgcn_sched_barrier(0);
      Frag8 fp[TM], fq[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) fq[j] = frag8<QT>(at + PT::kBytes, wn * WN + j * 16, lane);
#pragma unroll
      for (int j = 0; j < TM; ++j) fp[j] = frag8<PT>(at, wm * WM + j * 16, lane);
      mul8<T, TM, TN>(fp, fq, now, acc);
    });
  }
  __syncthreads();  // both places are free
  static_assert(NW * op_region_bytes<TM, TN> <= 2 * kStageBytes, "output regions fit");
  op_write_out<T, OP_LINEAR>(g, acc, lds + wave * op_region_bytes<TM, TN>, lane, m0 + wm * WM, n0 + wn * WN, 0, split);
}

// ---------------------------------------------------------------------------
// Few rows: 16 MT rows and 32 columns a block, whose waves take turns over the
// blocks of k (op_gemm_skinny).  Bound by memory: one row, 16384 x 4096, 12.6 us,
// 5.3 TB/s.
// ---------------------------------------------------------------------------
template <typename T, int MT, int NW, int NST, bool DIRECT>
__global__ void __launch_bounds__(NW * 64) op_gemm8_skinny(OpGemmMore g) {
  constexpr int BN = 32, TN = BN / 16;
  using PT = Tile<uint8_t, 16 * MT, true, 1>;
  using QT = Tile<uint8_t, BN, true, 1>;
  constexpr int kWaveBytes = PT::kBytes + QT::kBytes + (DIRECT ? 256 : 0);
  constexpr int kStageLoads = PT::kLoads + QT::kLoads + 1;
  static_assert(DIRECT ? NST >= 2 : NST == 1, "ring");
  __shared__ __attribute__((aligned(16))) char lds[NST * NW * kWaveBytes];

  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const OpPlace place = op_place<true, false>(g);
  const int m0 = place.tm * (16 * MT), n0 = place.tn * BN, split = place.split, p_left = g.M - m0, q_left = g.N - n0;
  PT pt;
  QT qt;
  pt.init(g.ld_p, p_left, 0, lane);
  qt.init(g.ld_q, q_left, 0, lane);
  RowScales sx;
  sx.init(g, m0, lane % (16 * MT));
  ColumnScales sw;
  sw.init(g, n0);
  const int s_begin = split * g.stages_per_split, s_end = min((g.K + 127) / 128, s_begin + g.stages_per_split);
  char* mine = lds + wave * (NST * kWaveBytes);
  chunk16 rp[DIRECT ? 1 : PT::kLoads], rq[DIRECT ? 1 : QT::kLoads];
  float held = 0.0f;  // staged: the scale of this lane's row
  Cursor8 next;
  next.init(g, m0, n0, 0, s_begin + wave, NW);
  auto load = [&](uint32_t to, auto whole) {
    constexpr bool W = decltype(whole)::value;
    const int k_left = W ? 128 : g.K - next.k;
    if constexpr (DIRECT) {
      const uint32_t lq = to + PT::kBytes;
      op_load_lds4(sx.of(next.k >> 7), lq + QT::kBytes);
      if (W || k_left >= 128) {
        qt.issue(next.q[0], lq, 0);
        pt.issue(next.p, to, 0);
      } else {
        qt.issue_tail(next.q[0], lq, 0, lane, k_left);
        pt.issue_tail(next.p, to, 0, lane, k_left);
      }
    } else {
      held = *sx.of(next.k >> 7);
      qt.fetch(next.q[0], rq, 0, lane, q_left, k_left);
      pt.fetch(next.p, rp, 0, lane, p_left, k_left);
    }
    next.step();
  };
  floatx4 acc[MT][TN];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  auto compute = [&](const char* from, const float (&s)[MT]) {
    Frag8 fq[TN], fp[MT];
#pragma unroll
    for (int j = 0; j < TN; ++j) fq[j] = frag8<QT>(from + PT::kBytes, j * 16, lane);
#pragma unroll
    for (int i = 0; i < MT; ++i) fp[i] = frag8<PT>(from, i * 16, lane);
    mul8<T, MT, TN>(fp, fq, s, acc);
  };
  const int S = s_end > s_begin + wave ? (s_end - s_begin - wave + NW - 1) / NW : 0;
  float w_scale = sw.of(s_begin + wave);
  if constexpr (DIRECT) {  // NST - 1 stages in flight
    const uint32_t lds_byte = op_lds_byte(mine);
    int from = 0, to = (NST - 1) * kWaveBytes;
    auto stage = [&](int s, auto whole) {
      constexpr bool W = decltype(whole)::value;
      op_wait_lds();  // what the next loads overwrite was read one turn ago
      __builtin_amdgcn_sched_barrier(0);
      const float w_next = sw.of(s_begin + wave + (s + 1) * NW);
      if (W || s + NST - 1 < S) {
        load(lds_byte + to, whole);
        op_wait_loads<(NST - 1) * kStageLoads>();
      } else {
        op_wait_loads<0>();
      }
      __builtin_amdgcn_sched_barrier(0);
      const float* scales = reinterpret_cast<const float*>(mine + from + PT::kBytes + QT::kBytes);
      float sc[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) sc[i] = scales[i * 16 + l] * w_scale;
      compute(mine + from, sc);
      w_scale = w_next;
      to = from;
      from = from == (NST - 1) * kWaveBytes ? 0 : from + kWaveBytes;
    };
#pragma unroll 1
    for (int i = 0; i < NST - 1 && i < S; ++i) load(lds_byte + i * kWaveBytes, std::false_type());
    for (int s = 0; s < S; ++s) {
      for (int n = min(next.whole_steps(g), S - (NST - 1) - s); n > 0; --n, ++s) stage(s, std::true_type());
      if (s < S) stage(s, std::false_type());
    }
  } else {
    constexpr auto any = std::false_type();
    if (S > 0) load(0, any);
    for (int s = 0; s < S; ++s) {
      pt.put(rp, mine, 0, lane);
      qt.put(rq, mine + PT::kBytes, 0, lane);
      float sc[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) sc[i] = __shfl(held, i * 16 + l, kWave) * w_scale;
      w_scale = sw.of(s_begin + wave + (s + 1) * NW);
      if (s + 1 < S) load(0, any);
      __builtin_amdgcn_sched_barrier(0);
      compute(mine, sc);
    }
  }

  // The waves' sums, in wave order, 16 rows at a time.
  floatx4* sums = reinterpret_cast<floatx4*>(lds);
  static_assert(NW * TN * 1024 <= NST * NW * kWaveBytes, "sums fit the ring");
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < TN; ++c) sums[(wave * TN + c) * 64 + lane] = acc[i][c];
    __syncthreads();
    const int m = m0 + i * 16 + l, j = wave, n = n0 + j * 16 + lg * 4, cnt = g.N - n;
    if (m >= g.M || j >= TN || cnt <= 0) continue;
    floatx4 a = sums[j * 64 + lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) a = a + sums[(w * TN + j) * 64 + lane];
    float d0[4], d1[4] = {}, b0[4], b1[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) d0[r] = a[r];
    if (g.splits > 1) {
      store_vec(g.partial + ((int64_t)split * g.M + m) * g.N + n, cnt, d0);
    } else {
      op_biases<T, OP_LINEAR>(g.epi, n, cnt, b0, b1);
      op_epilogue<T, OP_LINEAR>(g.epi, 0, m, n, cnt, d0, d1, b0, b1);
    }
  }
}

// ---------------------------------------------------------------------------
template <typename T, int BM, int BN, int WGM, int WGN, int KS, int NST>
hipError_t launch8_middle(OpGemmMore& g, hipStream_t st) {
  g.tiles_m = (g.M + BM - 1) / BM;
  g.tiles_n = (g.N + BN - 1) / BN;
  return op_launch(op_gemm8_middle<T, BM, BN, WGM, WGN, KS, NST>,
                   op_grid<true, false>(g), dim3(512), st, g);
}
template <typename T>
hipError_t launch8_large(OpGemmMore& g, hipStream_t st) {
  g.tiles_m = (g.M + 255) / 256;
  g.tiles_n = (g.N + 255) / 256;
  return op_launch(op_gemm8_large<T>, op_grid<true, false>(g), dim3(512), st, g);
}
template <typename T, int BM, int BN>
hipError_t launch8_staged(OpGemmMore& g, hipStream_t st) {
  g.tiles_m = (g.M + BM - 1) / BM;
  g.tiles_n = (g.N + BN - 1) / BN;
  return op_launch(op_gemm8_staged<T, BM, BN>, op_grid<true, false>(g), dim3(256),
                   st, g);
}
template <typename T, int MT, bool DIRECT>
hipError_t launch8_skinny(OpGemmMore& g, hipStream_t st) {
  using S = SkinnyShape<OP_LINEAR, MT, DIRECT>;
  g.tiles_m = (g.M + 16 * MT - 1) / (16 * MT);
  g.tiles_n = (g.N + S::kCols - 1) / S::kCols;
  return op_launch(op_gemm8_skinny<T, MT, S::kWaves, S::kStages, DIRECT>,
                   op_grid<true, false>(g), dim3(S::kWaves * 64), st, g);
}

template <typename T>
hipError_t launch8(const OpPlan& plan, OpGemmMore& g, hipStream_t st) {
  g.splits = plan.splits;
  g.stages_per_split = plan.stages_per_split;
  hipError_t e = hipErrorInvalidValue;
  switch (plan.tile) {
    case OP_TILE_SKINNY16: e = g.direct ? launch8_skinny<T, 1, true>(g, st) : launch8_skinny<T, 1, false>(g, st); break;
    case OP_TILE_SKINNY32: e = g.direct ? launch8_skinny<T, 2, true>(g, st) : launch8_skinny<T, 2, false>(g, st); break;
    case OP_TILE_SKINNY64: e = g.direct ? launch8_skinny<T, 4, true>(g, st) : launch8_skinny<T, 4, false>(g, st); break;
    case OP_TILE_64:
      e = g.direct ? launch8_middle<T, 64, 64, 2, 4, 2, 4>(g, st) : launch8_staged<T, 64, 64>(g, st);
      break;
    case OP_TILE_128:
      e = g.direct ? launch8_middle<T, 128, 128, 2, 4, 1, 4>(g, st) : launch8_staged<T, 128, 128>(g, st);
      break;
    case OP_TILE_64X128:
      if (g.direct) e = launch8_middle<T, 64, 128, 2, 4, 1, 4>(g, st);
      break;
    case OP_TILE_256X128:
      if (g.direct) e = launch8_middle<T, 256, 128, 4, 2, 1, 3>(g, st);
      break;
    default:
      // 256x256 of float32 results, whose fragments take more registers than that
      // tile has, and of a last part of a block of k run on 256x128, in the same
      // splits; what the plan weighed is the larger tile's time
      if constexpr (sizeof(T) < 4) {
        if (g.direct && g.K % 128 == 0) {
          e = launch8_large<T>(g, st);
          break;
        }
      }
      if (g.direct) e = launch8_middle<T, 256, 128, 4, 2, 1, 3>(g, st);
  }
  if (e != hipSuccess || g.splits <= 1) return e;
  const int64_t quads = (int64_t)g.M * ((g.N + 3) / 4);
  const int64_t blocks = (quads + 255) / 256, x = std::min<int64_t>(blocks, int64_t{1} << 20);
  return op_launch(op_gemm_reduce<T, OP_LINEAR, OpGemmMore>, dim3((unsigned)x, 1, (unsigned)((blocks + x - 1) / x)), dim3(256), st, g);
}

}  // namespace ops
}  // namespace volta
