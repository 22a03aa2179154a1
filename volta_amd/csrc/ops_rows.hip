// Row and element kernels of the feed-forward operators: ops_rows.h.  All are
// bound by memory: each matrix is read or written once, 16 bytes a lane, at
// any element alignment (the memory pipeline takes unaligned 16-byte
// accesses); a row's last elements, less than 16 bytes, go one by one.
#include "ops_rows.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ops_codes.h"
#include "ops_launch.h"
#include "ops_types.h"

namespace volta {
namespace ops {
namespace {

// A grid of n blocks and the block's number in it: a dimension of a grid has
// fewer than 2^32 threads, so many blocks take two.
dim3 grid_of(int64_t n) {
  const int64_t x = std::min<int64_t>(n, int64_t{1} << 20);
  return dim3((unsigned)x, (unsigned)((n + x - 1) / x));
}
__device__ __forceinline__ int64_t block_id() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// The elements of one 16-byte access.
template <typename T> constexpr int kChunk = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ void load_row(const T* p, int cnt, float (&f)[kChunk<T>]) {
  load_vec(p, cnt, f);
}
template <typename T>
__device__ __forceinline__ void store_row(T* p, int cnt, const float (&f)[kChunk<T>]) {
  store_vec(p, cnt, f);
}
// Sum (or maximum) over the TPR threads of a row: over a wave by a butterfly,
// over a block's waves through LDS, always in the same order.  `red` holds a
// float for each wave; uses of it alternate between two arrays.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) v += red[w];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ float row_max(float v, float* red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = max_or_nan(v, __shfl_xor(v, off, kWave));
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) v = max_or_nan(v, red[w]);
  }
  return v;
}

// ---------------------------------------------------------------------------
// RMS norm.  TPR threads a row (a wave, or a block), which hold the row in
// registers between the sum and the output: chunk t + i TPR for i < NCH.
// NCH = 0: rows too long for that, read again for each pass (from L2).
// 8192 x 4096 bf16 with a residual and its sum, 268 MB: 51 us, 5.25 TB/s, a
// large copy's rate; the same to e4m3, 235 MB, 49 us with a scale for each 128
// columns or for the row; 512 x 65536 (NCH = 0) 30 us, 4.5 TB/s.
// ---------------------------------------------------------------------------
template <typename T, bool E4M3, int TPR, int NCH>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) norm_kernel(NormArgs a) {
  constexpr int E = kChunk<T>, RPB = (TPR < 256 ? 256 : TPR) / TPR, kHeld = NCH > 0 ? NCH : 1;
  __shared__ float red[2][TPR / 64];
  const int t = threadIdx.x % TPR;
  const int64_t row = block_id() * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;  // whole waves, and whole blocks where the row has a block to itself
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.ld_residual : nullptr;
  T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.ld_sum : nullptr;
  const T* w = static_cast<const T*>(a.weight);
  const int chunks = (a.cols + E - 1) / E;
  const int turns = NCH > 0 ? NCH : (chunks + TPR - 1) / TPR;

  auto load_s = [&](int ch, float (&s)[E]) {
    const int c = ch * E, cnt = a.cols - c;
    load_row(x + c, cnt, s);
    if (res) {
      float r[E];
      load_row(res + c, cnt, r);
#pragma unroll
      for (int i = 0; i < E; ++i) s[i] += r[i];
    }
  };
  float held[kHeld][E];
  float ss = 0.0f;
  if constexpr (NCH > 0) {
    // every load of the row before the first use
    float r[NCH][E];
#pragma unroll
    for (int k = 0; k < NCH; ++k) load_row(x + (t + k * TPR) * E, a.cols - (t + k * TPR) * E, held[k]);
    if (res) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) load_row(res + (t + k * TPR) * E, a.cols - (t + k * TPR) * E, r[k]);
#pragma unroll
      for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int i = 0; i < E; ++i) held[k][i] += r[k][i];
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int i = 0; i < E; ++i) ss = fmaf(held[k][i], held[k][i], ss);
  } else {
    for (int k = 0; k < turns; ++k) {
      load_s(t + k * TPR, held[0]);
#pragma unroll
      for (int i = 0; i < E; ++i) ss = fmaf(held[0][i], held[0][i], ss);
    }
  }
  ss = row_sum<TPR>(ss, red[0]);
  const float rstd = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
  if (a.rstd && t == 0) a.rstd[row] = rstd;

  // y of chunk k from s in `v`
  auto finish = [&](int k, float (&v)[E]) {
    const int c = (t + k * TPR) * E, cnt = a.cols - c;
    float wv[E];
    if (w) load_row(w + c, cnt, wv);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      v[i] *= rstd;
      if (w) v[i] *= wv[i];
    }
  };
  auto largest = [&](const float (&v)[E]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) m = max_or_nan(m, fabsf(v[i]));
    return m;
  };
  if constexpr (!E4M3) {
    T* y = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      for (int kk = k; kk < turns; kk += kHeld) {  // NCH > 0: once
        if constexpr (NCH == 0) load_s(t + kk * TPR, held[0]);
        const int c = (t + kk * TPR) * E, cnt = a.cols - c;
        if (sum) store_row(sum + c, cnt, held[k]);
        finish(kk, held[k]);
        store_row(y + c, cnt, held[k]);
      }
    }
  } else {
    uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.ld_y;
    if (a.group == a.cols) {  // one scale for the row
      float m = 0.0f;
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        for (int kk = k; kk < turns; kk += kHeld) {
          if constexpr (NCH == 0) load_s(t + kk * TPR, held[0]);
          const int c = (t + kk * TPR) * E;
          if constexpr (NCH > 0)
            if (sum) store_row(sum + c, a.cols - c, held[k]);
          finish(kk, held[k]);
          m = max_or_nan(m, largest(held[k]));
        }
      const float scale = scale_of(row_max<TPR>(m, red[1])), inv = 1.0f / scale;
      if (t == 0) a.scales[row] = scale;
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        for (int kk = k; kk < turns; kk += kHeld) {
          const int c = (t + kk * TPR) * E, cnt = a.cols - c;
          if constexpr (NCH == 0) {
            load_s(t + kk * TPR, held[0]);
            if (sum) store_row(sum + c, cnt, held[0]);
            finish(kk, held[0]);
          }
#pragma unroll
          for (int i = 0; i < E; ++i) held[k][i] *= inv;
          store_codes<E>(y + c, cnt, held[k]);
        }
    } else {  // one for each 128 columns: 128 / E neighbouring lanes
      const int groups = (a.cols + 127) / 128;
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        for (int kk = k; kk < turns; kk += kHeld) {
          if constexpr (NCH == 0) load_s(t + kk * TPR, held[0]);
          const int c = (t + kk * TPR) * E, cnt = a.cols - c;
          if (sum) store_row(sum + c, cnt, held[k]);
          finish(kk, held[k]);
          float m = largest(held[k]);
#pragma unroll
          for (int off = 64 / E; off >= 1; off >>= 1) m = max_or_nan(m, __shfl_xor(m, off, kWave));
          const float scale = scale_of(m), inv = 1.0f / scale;
          if (c % 128 == 0 && cnt > 0) a.scales[row * groups + c / 128] = scale;
#pragma unroll
          for (int i = 0; i < E; ++i) held[k][i] *= inv;
          store_codes<E>(y + c, cnt, held[k]);
        }
    }
  }
}

template <typename T, bool E4M3>
hipError_t norm_launch(const NormArgs& a, hipStream_t st) {
  if (a.rows == 0) return hipSuccess;
  constexpr int E = kChunk<T>;
  const int chunks = (a.cols + E - 1) / E;
#define VOLTA_NORM(TPR, NCH)                                                                             \
  return op_launch(norm_kernel<T, E4M3, TPR, NCH>, grid_of(TPR == 64 ? (a.rows + 3) / 4 : a.rows), \
                   dim3(TPR < 256 ? 256 : TPR), st, a)
  if (chunks <= 64) VOLTA_NORM(64, 1);
  if (chunks <= 128) VOLTA_NORM(64, 2);
  if (chunks <= 256) VOLTA_NORM(256, 1);
  if (chunks <= 512) VOLTA_NORM(256, 2);
  if (chunks <= 1024) VOLTA_NORM(256, 4);
  if (chunks <= 2048) VOLTA_NORM(1024, 2);
  if (chunks <= 4096) VOLTA_NORM(1024, 4);
  VOLTA_NORM(1024, 0);
#undef VOLTA_NORM
}

// ---------------------------------------------------------------------------
// Gradients of the norm.  With hat = s rstd, dx = rstd (w dy - hat mean(w dy
// hat)): the same as the formula with rstd^3, whose cube leaves 32 bits from
// rows of 1e13 or 1e-13 on, where dx is an ordinary number.  Block b takes rows
// b, b + blocks, ... and keeps the sums of dweight of its rows in registers, a
// partial sum for each block.
// 8192 x 4096 bf16 with dsum, 268 MB and 17 MB of partial sums: 55 us, 5.2
// TB/s, and 5 us for the launch that adds the partial sums.
// ---------------------------------------------------------------------------
template <typename T, int TPR, int NCH>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) norm_grad_kernel(NormGradArgs a) {
  constexpr int E = kChunk<T>, RPB = (TPR < 256 ? 256 : TPR) / TPR;
  __shared__ float red[2][TPR / 64];
  const int t = threadIdx.x % TPR;
  const T* w = static_cast<const T*>(a.weight);
  float wv[NCH][E], dw[NCH][E];
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int c = (t + k * TPR) * E;
    if (w) load_row(w + c, a.cols - c, wv[k]);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      dw[k][i] = 0.0f;
      if (!w) wv[k][i] = 1.0f;
    }
  }
  const int64_t step = (int64_t)gridDim.x * RPB;
  int parity = 0;
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += step) {
    const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
    const T* s = static_cast<const T*>(a.s) + row * a.ld_s;
    const float rstd = a.rstd[row];
    float dv[NCH][E], sv[NCH][E], add[NCH][E];
#pragma unroll
    for (int k = 0; k < NCH; ++k) load_row(dy + (t + k * TPR) * E, a.cols - (t + k * TPR) * E, dv[k]);
#pragma unroll
    for (int k = 0; k < NCH; ++k) load_row(s + (t + k * TPR) * E, a.cols - (t + k * TPR) * E, sv[k]);
    if (a.dx && a.dsum) {
      const T* ds = static_cast<const T*>(a.dsum) + row * a.ld_dsum;
#pragma unroll
      for (int k = 0; k < NCH; ++k) load_row(ds + (t + k * TPR) * E, a.cols - (t + k * TPR) * E, add[k]);
    }
    float dot = 0.0f;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int i = 0; i < E; ++i) {
        sv[k][i] *= rstd;  // hat
        dw[k][i] = fmaf(dv[k][i], sv[k][i], dw[k][i]);
        dv[k][i] *= wv[k][i];
        dot = fmaf(dv[k][i], sv[k][i], dot);
      }
    if (!a.dx) continue;
    dot = row_sum<TPR>(dot, red[parity]);
    parity ^= 1;
    const float f = dot / (float)a.cols;
    T* dx = static_cast<T*>(a.dx) + row * a.ld_dx;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        dv[k][i] = rstd * (dv[k][i] - sv[k][i] * f);
        if (a.dsum) dv[k][i] += add[k][i];
      }
      store_row(dx + (t + k * TPR) * E, a.cols - (t + k * TPR) * E, dv[k]);
    }
  }
  if (!a.partial) return;
  float* p = a.partial + (int64_t)blockIdx.x * a.cols;
  if constexpr (RPB > 1) {  // the block's waves' sums, in wave order
    __shared__ float sums[RPB - 1][NCH][E][TPR];
    const int w = threadIdx.x / TPR;
    if (w > 0) {
#pragma unroll
      for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int i = 0; i < E; ++i) sums[w - 1][k][i][t] = dw[k][i];
    }
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int u = 0; u < RPB - 1; ++u)
#pragma unroll
      for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int i = 0; i < E; ++i) dw[k][i] += sums[u][k][i][t];
  }
#pragma unroll
  for (int k = 0; k < NCH; ++k) store_vec(p + (t + k * TPR) * E, a.cols - (t + k * TPR) * E, dw[k]);
}

// Rows too long for registers: dx row by row, read twice, and dweight column
// by column.  512 x 65536 bf16: 48 + 24 us.
template <typename T>
__global__ void __launch_bounds__(1024) norm_grad_wide_dx(NormGradArgs a) {
  constexpr int E = kChunk<T>;
  __shared__ float red[16];
  const int64_t row = block_id();
  if (row >= a.rows) return;
  const int chunks = (a.cols + E - 1) / E;
  const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
  const T* s = static_cast<const T*>(a.s) + row * a.ld_s;
  const T* w = static_cast<const T*>(a.weight);
  const T* ds = a.dsum ? static_cast<const T*>(a.dsum) + row * a.ld_dsum : nullptr;
  T* dx = static_cast<T*>(a.dx) + row * a.ld_dx;
  const float rstd = a.rstd[row];
  float dv[E], sv[E], o[E], dot = 0.0f;
  auto load = [&](int c, int cnt) {
    load_row(dy + c, cnt, dv);
    load_row(s + c, cnt, sv);
#pragma unroll
    for (int i = 0; i < E; ++i) sv[i] *= rstd;  // hat
    if (w) {
      load_row(w + c, cnt, o);
#pragma unroll
      for (int i = 0; i < E; ++i) dv[i] *= o[i];
    }
  };
  for (int ch = threadIdx.x; ch < chunks; ch += 1024) {
    load(ch * E, a.cols - ch * E);
#pragma unroll
    for (int i = 0; i < E; ++i) dot = fmaf(dv[i], sv[i], dot);
  }
  dot = row_sum<1024>(dot, red);
  const float f = dot / (float)a.cols;
  for (int ch = threadIdx.x; ch < chunks; ch += 1024) {
    const int c = ch * E, cnt = a.cols - c;
    load(c, cnt);
    if (ds) load_row(ds + c, cnt, o);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      dv[i] = rstd * (dv[i] - sv[i] * f);
      if (ds) dv[i] += o[i];
    }
    store_row(dx + c, cnt, dv);
  }
}

// Column strips: a block takes 64 chunks of columns of `per` rows, its waves
// the rows r0 + wave, + kStripWaves, ..., and adds the waves' sums in wave
// order, to a row of partial sums or (one strip) to the output.
// Sixteen, because a row's loads and activation take a wave 1.7 us one after
// another: gradients of 256 rows of 1024 with biases took 11.3 us with 4 waves
// of 4 rows, and take 8.5.
constexpr int kStripWaves = 16;
template <typename T>
__device__ __forceinline__ void strip_store(float (*lds)[64][kChunk<T>], const float (&acc)[kChunk<T>], float* partial,
                                            T* out, int cols, int c, int lane, int wave) {
  constexpr int E = kChunk<T>;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < E; ++i) lds[wave][lane][i] = acc[i];
  __syncthreads();
  if (wave == 0 && c < cols) {
    float v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      v[i] = lds[0][lane][i];
#pragma unroll
      for (int w = 1; w < kStripWaves; ++w) v[i] += lds[w][lane][i];
    }
    if (out) store_vec(out + c, cols - c, v);
    else store_vec(partial + (int64_t)blockIdx.y * cols + c, cols - c, v);
  }
}

template <typename T>
__global__ void __launch_bounds__(kStripWaves * 64) norm_grad_wide_dw(NormGradArgs a, int per) {
  constexpr int E = kChunk<T>;
  __shared__ float lds[kStripWaves][64][E];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (blockIdx.x * 64 + lane) * E, cnt = a.cols - c;
  const int64_t r0 = (int64_t)blockIdx.y * per, r1 = min(a.rows, r0 + per);
  float acc[E] = {};
  for (int64_t r = r0 + wave; r < r1; r += kStripWaves) {
    float dv[E], sv[E];
    load_row(static_cast<const T*>(a.dy) + r * a.ld_dy + c, cnt, dv);
    load_row(static_cast<const T*>(a.s) + r * a.ld_s + c, cnt, sv);
    const float rstd = a.rstd[r];
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = fmaf(dv[i], sv[i] * rstd, acc[i]);
  }
  strip_store<T>(lds, acc, a.partial, nullptr, a.cols, c, lane, wave);
}

// ---------------------------------------------------------------------------
// What a layer's gradients need before their products, with the columns'
// sums, from 32 bits: linear, dp = dy f'(pre); gated, dg = dh u f'(g) and
// du = dh f(g).  dp, dg and du are rounded to the type, once: the matrix
// instructions take no wider operands, and the two products read half the
// bytes.  Kept apart from the products, which read each element many times
// and would form it anew each time.  Gated, 8192 x 16384 bf16, 1.34 GB: 254
// us, 5.3 TB/s.
//
// float16 ends at 65504 and has all of its bits from 2^-14 on, and dh u f'(g)
// leaves that range where dx and dW do not.  So its d are held in a common
// unit, the power of two that puts the largest magnitude of d between 2^14 and
// 2^15 (found by a pass of its own, act_grad_largest), and the products'
// epilogues multiply their sums by it: exact but for what is under 2^-28 of
// the largest.  That pass is 5 us of a linear layer's gradients of 16 rows of
// 1024 (12.0 without it, 17.4 with it), and 167 of a gated layer's of 8192 rows
// of 4096 and 16384 (3433 and 3600).
// ---------------------------------------------------------------------------
// Chunk c of row r: dp in d, or dg in u and du in d.  What is behind the
// columns comes out as 0.
template <typename T, bool GATED>
__device__ __forceinline__ void act_grad_chunk(const ActGradArgs& a, int64_t r, int c, int cnt, float (&d)[kChunk<T>],
                                               float (&u)[kChunk<T>]) {
  constexpr int E = kChunk<T>;
  float g[E];
  load_row(static_cast<const T*>(a.dy) + r * a.ld_dy + c, cnt, d);
  if (a.pre[0]) load_row(static_cast<const T*>(a.pre[0]) + r * a.ld_pre + c, cnt, g);
  if constexpr (GATED) load_row(static_cast<const T*>(a.pre[1]) + r * a.ld_pre + c, cnt, u);
  if (!a.pre[0]) return;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    float f, slope;
    op_act_both<T>(a.act, g[i], &f, &slope);
    if constexpr (GATED) {
      u[i] = d[i] * u[i] * slope;  // dg
      d[i] = d[i] * f;             // du
    } else {
      d[i] = d[i] * slope;
    }
  }
}

// The largest of a block's values, on every thread.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* lds) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, kWave));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < kStripWaves; ++w) v = max(v, lds[w]);
  return v;
}

// unit[1 + block]: the bits of the largest magnitude among the d that the
// block of act_grad_kernel's grid forms (an infinity or a NaN is larger than
// any number).  Reads what that kernel reads again, from the memory-side
// cache where it fits.
template <bool GATED>
__global__ void __launch_bounds__(kStripWaves * 64) act_grad_largest(ActGradArgs a, int per) {
  using T = _Float16;
  constexpr int E = kChunk<T>;
  __shared__ uint32_t lds[kStripWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (blockIdx.x * 64 + lane) * E, cnt = a.cols - c;
  const int64_t r0 = (int64_t)blockIdx.y * per, r1 = min(a.rows, r0 + per);
  uint32_t m = 0;
  for (int64_t r = r0 + wave; r < r1; r += kStripWaves) {
    float d[E], u[E];
    act_grad_chunk<T, GATED>(a, r, c, cnt, d, u);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      m = max(m, __float_as_uint(fabsf(d[i])));
      if constexpr (GATED) m = max(m, __float_as_uint(fabsf(u[i])));
    }
  }
  m = block_max(m, lds);
  if (threadIdx.x == 0) a.unit[1 + (int64_t)blockIdx.y * gridDim.x + blockIdx.x] = __uint_as_float(m);
}

// What 1 / unit multiplies d by, from the blocks' largest magnitudes; the
// first block leaves unit[0].  All zeros, and an infinity or a NaN among them:
// 1.  The exponents stay inside those of normal numbers.
__device__ __forceinline__ float per_unit(const ActGradArgs& a, uint32_t* lds) {
  const int n = (int)(gridDim.x * gridDim.y);
  uint32_t m = 0;
  for (int i = threadIdx.x; i < n; i += kStripWaves * 64) m = max(m, __float_as_uint(a.unit[1 + i]));
  m = block_max(m, lds);
  int up = 0;
  if (m != 0 && m < 0x7f800000u) up = min(14 - (max((int)(m >> 23), 1) - 127), 126);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.unit[0] = __uint_as_float((uint32_t)(127 - up) << 23);
  return __uint_as_float((uint32_t)(127 + up) << 23);
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(kStripWaves * 64) act_grad_kernel(ActGradArgs a, int per) {
  constexpr int E = kChunk<T>;
  __shared__ float lds[kStripWaves][64][E];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (blockIdx.x * 64 + lane) * E, cnt = a.cols - c;
  const int64_t r0 = (int64_t)blockIdx.y * per, r1 = min(a.rows, r0 + per);
  float s0[E] = {}, s1[E] = {}, up = 1.0f;
  constexpr bool kUnits = std::is_same<T, _Float16>::value;
  if constexpr (kUnits) {
    __shared__ uint32_t top[kStripWaves];
    if (a.unit) up = per_unit(a, top);
  }
  for (int64_t r = r0 + wave; r < r1; r += kStripWaves) {
    float d[E], u[E];
    act_grad_chunk<T, GATED>(a, r, c, cnt, d, u);
    if constexpr (GATED) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        s0[i] += u[i];
        s1[i] += d[i];
        if constexpr (kUnits) {
          u[i] *= up;
          d[i] *= up;
        }
      }
      if (cnt > 0) {
        store_row(static_cast<T*>(a.d[0]) + r * a.ld_d + c, E, u);
        store_row(static_cast<T*>(a.d[1]) + r * a.ld_d + c, E, d);
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        s0[i] += d[i];
        if constexpr (kUnits) d[i] *= up;
      }
      if (a.d[0] && cnt > 0) store_row(static_cast<T*>(a.d[0]) + r * a.ld_d + c, E, d);
    }
  }
  const bool one = gridDim.y == 1;
  if (a.sums[0])
    strip_store<T>(lds, s0, a.partial[0], one ? static_cast<T*>(a.sums[0]) : nullptr, a.cols, c, lane, wave);
  if (GATED && a.sums[1])
    strip_store<T>(lds, s1, a.partial[1], one ? static_cast<T*>(a.sums[1]) : nullptr, a.cols, c, lane, wave);
}

// Partial sums of 64 columns: 16 waves take a sixteenth of the rows each, in
// order, and their sums are added in wave order.  1024 rows of 4096: 5 us, a
// launch and the latency of eight loads after another.
template <typename T>
__global__ void __launch_bounds__(1024) sum_partials_kernel(SumArgs a) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  const int per = (a.n + 15) / 16, i0 = wave * per, i1 = min(a.n, i0 + per);
  float s = 0.0f;
  if (c < a.cols) {
    const float* p = a.partial[blockIdx.y] + c;
#pragma unroll 8
    for (int i = i0; i < i1; ++i) s += p[(int64_t)i * a.cols];
  }
  lds[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < a.cols) {
    s = lds[0][lane];
#pragma unroll
    for (int w = 1; w < 16; ++w) s += lds[w][lane];
    static_cast<T*>(a.out[blockIdx.y])[c] = from_f<T>(s);
  }
}

// A thread for 16 bytes of a row of the copy.  10 MB: 5 to 6 us, of which a
// launch is 2.
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(PackArgs a) {
  constexpr int E = kChunk<T>;
  const int i = blockIdx.z;
  const int64_t chunks = a.ld_to[i] / E, id = block_id() * 256 + threadIdx.x, row = id / chunks;
  if (row >= a.rows[i]) return;
  const int c = (int)(id - row * chunks) * E;
  float f[E];
  load_row(static_cast<const T*>(a.from[i]) + row * a.ld_from[i] + c, a.cols[i] - c, f);
  store_row(static_cast<T*>(a.to[i]) + row * a.ld_to[i] + c, E, f);
}

// The same of codes, whose rows start at any byte.
__global__ void __launch_bounds__(256) pack_codes_kernel(PackArgs a) {
  const int i = blockIdx.z;
  const int64_t chunks = a.ld_to[i] / 16, id = block_id() * 256 + threadIdx.x, row = id / chunks;
  if (row >= a.rows[i]) return;
  const int c = (int)(id - row * chunks) * 16, cnt = a.cols[i] - c;
  const uint8_t* from = static_cast<const uint8_t*>(a.from[i]) + row * a.ld_from[i] + c;
  union { chunk16 v; uint8_t b[16]; } u;
  if (cnt >= 16) {
    u.v = *(const VOLTA_GLOBAL Access<16, 1>::type*)from;
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) u.b[k] = k < cnt ? ((const VOLTA_GLOBAL uint8_t*)from)[k] : 0;
  }
  *reinterpret_cast<chunk16*>(static_cast<uint8_t*>(a.to[i]) + row * a.ld_to[i] + c) = u.v;
}

// ---------------------------------------------------------------------------
// Dropout: a thread for 16 bytes of a row.  Element i's 32 bits are half of
// output i/2 of the stream: E/2 outputs for a chunk that starts at an even i,
// one more for an odd one.  The counter replaces a stored mask's bytes; its
// arithmetic, two 64-bit products for two elements, stays below the memory's
// time: 8192 x 4096 bf16 with a residual, 201 MB, 38 us, 5.3 TB/s.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint64_t stream_output(uint64_t seed, uint64_t n) {
  uint64_t z = seed + (n + 1) * 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}

template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs a, int64_t chunks_per_row) {
  constexpr int E = kChunk<T>;
  const int64_t id = block_id() * 256 + threadIdx.x;
  const int64_t row = a.rows == 1 ? 0 : id / chunks_per_row;
  const int64_t c = (id - row * chunks_per_row) * E;
  if (row >= a.rows || c >= a.cols) return;
  const int cnt = (int)min((int64_t)E, a.cols - c);
  float v[E], r[E];
  load_row(static_cast<const T*>(a.x) + row * a.ld_x + c, cnt, v);
  if (a.residual) load_row(static_cast<const T*>(a.residual) + row * a.ld_residual + c, cnt, r);
  const uint64_t i0 = (uint64_t)row * (uint64_t)a.cols + (uint64_t)c, first = a.offset + (i0 >> 1);
  const bool odd = i0 & 1;
  uint32_t bits[E + 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const uint64_t z = stream_output(a.seed, first + i);
    bits[2 * i] = (uint32_t)z;
    bits[2 * i + 1] = (uint32_t)(z >> 32);
  }
  if (odd) {
    bits[E] = (uint32_t)stream_output(a.seed, first + E / 2);
#pragma unroll
    for (int i = 0; i < E; ++i) bits[i] = bits[i + 1];
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    v[i] = bits[i] >= a.threshold ? v[i] * a.scale : 0.0f;
    if (a.residual) v[i] += r[i];
  }
  store_row(static_cast<T*>(a.y) + row * a.ld_y + c, cnt, v);
}

// Calls f with a value of the element type.
template <typename F>
auto with_type(int type, F f) {
  if (type == VOLTA_OP_BF16) return f((__bf16)0.0f);
  if (type == VOLTA_OP_F16) return f((_Float16)0.0f);
  return f(0.0f);
}
int chunks_of(int type, int64_t cols) {
  const int e = type == VOLTA_OP_F32 ? 4 : 8;
  return (int)((cols + e - 1) / e);
}

constexpr int kNormGradHeld = 2048;  // chunks of a row that the gradient's kernel holds at most

template <typename T, int TPR, int NCH>
hipError_t norm_grad_launch(const NormGradArgs& a, int blocks, hipStream_t st) {
  return op_launch(norm_grad_kernel<T, TPR, NCH>, dim3((unsigned)blocks), dim3(TPR < 256 ? 256 : TPR), st, a);
}

// Rows of a column strip and strips, for about 512 blocks (gradients of 2000
// rows of 2 x 3000: 21.6 us, and 23.8 for about 1024).
int strip_rows(int chunks, int64_t rows) {
  const int64_t across = (chunks + 63) / 64;
  const int64_t strips = std::max<int64_t>(1, std::min<int64_t>((rows + 15) / 16, 512 / across));
  return (int)std::max<int64_t>(1, (rows + strips - 1) / strips);
}
int strips_of(int chunks, int64_t rows) {
  const int per = strip_rows(chunks, rows);
  return (int)std::max<int64_t>(1, (rows + per - 1) / per);
}

}  // namespace

hipError_t norm_forward(int type, bool e4m3, const NormArgs& a, hipStream_t st) {
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    return e4m3 ? norm_launch<T, true>(a, st) : norm_launch<T, false>(a, st);
  });
}

int norm_grad_blocks(int type, int64_t rows, int64_t cols) {
  const int chunks = chunks_of(type, cols);
  if (chunks > kNormGradHeld) return strips_of(chunks, rows);
  // as many blocks as the chip holds: 8192 x 4096 bf16 took 84 us with 512 blocks, 57 with 1024 (55 since the cube
  // of rstd went), 61 with 2048 (and 4 us more for the sum of their partial sums)
  const int rpb = chunks <= 128 ? 4 : 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + rpb - 1) / rpb, chunks <= 512 ? 1024 : 512));
}

hipError_t norm_backward(int type, const NormGradArgs& a, hipStream_t st) {
  const int chunks = chunks_of(type, a.cols);
  const int rows = norm_grad_blocks(type, a.rows, a.cols);
  return with_type(type, [&](auto t) -> hipError_t {
    using T = decltype(t);
    if (chunks <= 64) return norm_grad_launch<T, 64, 1>(a, rows, st);
    if (chunks <= 128) return norm_grad_launch<T, 64, 2>(a, rows, st);
    if (chunks <= 256) return norm_grad_launch<T, 256, 1>(a, rows, st);
    if (chunks <= 512) return norm_grad_launch<T, 256, 2>(a, rows, st);
    if (chunks <= 1024) return norm_grad_launch<T, 256, 4>(a, rows, st);
    if (chunks <= kNormGradHeld) return norm_grad_launch<T, 1024, 2>(a, rows, st);
    hipError_t e = hipSuccess;
    if (a.dx && a.rows > 0) e = op_launch(norm_grad_wide_dx<T>, grid_of(a.rows), dim3(1024), st, a);
    if (e == hipSuccess && a.partial)
      e = op_launch(norm_grad_wide_dw<T>, dim3((unsigned)((chunks + 63) / 64), (unsigned)rows), dim3(kStripWaves * 64),
                    st, a, strip_rows(chunks, a.rows));
    return e;
  });
}

hipError_t sum_partials(int type, const SumArgs& a, hipStream_t st) {
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    return op_launch(sum_partials_kernel<T>, dim3((unsigned)((a.cols + 63) / 64), (unsigned)a.count), dim3(1024), st, a);
  });
}

// Up to 32 rows are one strip, which stores the sums themselves: 7.5 us for 32
// rows of 1024 with biases, 8.5 with a launch that adds two strips' (64 rows:
// 11.1 and 8.5).
int act_grad_rows(int chunks, int64_t rows) { return rows <= 32 ? 32 : strip_rows(chunks, rows); }

int act_grad_strips(int type, int64_t rows, int64_t cols) {
  const int per = act_grad_rows(chunks_of(type, cols), rows);
  return rows <= per ? 0 : (int)((rows + per - 1) / per);
}

int64_t act_grad_units(int type, int64_t rows, int64_t cols) {
  if (type != VOLTA_OP_F16 || rows == 0) return 0;
  return 1 + (chunks_of(type, cols) + 63) / 64 * (int64_t)std::max(1, act_grad_strips(type, rows, cols));
}

hipError_t act_grad(int type, bool gated, const ActGradArgs& a, hipStream_t st) {
  const int chunks = chunks_of(type, a.cols), per = act_grad_rows(chunks, a.rows);
  const int strips = act_grad_strips(type, a.rows, a.cols);
  const dim3 grid((unsigned)((chunks + 63) / 64), (unsigned)std::max(1, strips));
  if (a.unit) {
    const hipError_t e =
        op_launch(gated ? act_grad_largest<true> : act_grad_largest<false>, grid, dim3(kStripWaves * 64), st, a, per);
    if (e != hipSuccess) return e;
  }
  const hipError_t e = with_type(type, [&](auto t) {
    using T = decltype(t);
    return op_launch(gated ? act_grad_kernel<T, true> : act_grad_kernel<T, false>, grid, dim3(kStripWaves * 64), st, a,
                     per);
  });
  if (e != hipSuccess || strips == 0) return e;
  SumArgs s{};
  for (int i = 0; i < 2; ++i) {
    if (!a.sums[i]) continue;
    s.partial[s.count] = a.partial[i];
    s.out[s.count++] = a.sums[i];
  }
  s.n = strips;
  s.cols = a.cols;
  return s.count ? sum_partials(type, s, st) : hipSuccess;
}

hipError_t pack_rows(int type, const PackArgs& a, hipStream_t st) {
  if (type == VOLTA_OP_E4M3) {
    int64_t blocks = 1;
    for (int i = 0; i < a.n; ++i) blocks = std::max(blocks, (a.rows[i] * (a.ld_to[i] / 16) + 255) / 256);
    dim3 grid = grid_of(blocks);
    grid.z = (unsigned)a.n;
    return op_launch(pack_codes_kernel, grid, dim3(256), st, a);
  }
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    int64_t blocks = 1;
    for (int i = 0; i < a.n; ++i) blocks = std::max(blocks, (a.rows[i] * (a.ld_to[i] / kChunk<T>) + 255) / 256);
    dim3 grid = grid_of(blocks);
    grid.z = (unsigned)a.n;
    return op_launch(pack_kernel<T>, grid, dim3(256), st, a);
  });
}

hipError_t dropout_forward(int type, const DropoutArgs& in, hipStream_t st) {
  DropoutArgs a = in;
  if (a.ld_x == a.cols && a.ld_y == a.cols && (!a.residual || a.ld_residual == a.cols)) {  // packed: one long row
    a.cols *= a.rows;
    a.rows = a.cols > 0 ? 1 : 0;
  }
  if (a.rows == 0) return hipSuccess;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    const int64_t per_row = (a.cols + kChunk<T> - 1) / kChunk<T>;
    return op_launch(dropout_kernel<T>, grid_of((per_row * a.rows + 255) / 256), dim3(256), st, a, per_row);
  });
}

}  // namespace ops
}  // namespace volta
