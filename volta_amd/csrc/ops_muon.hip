// The update by orthogonalised momentum (include/volta_ops.h): entry points,
// and the passes before the products, which are ops_gemm_kernels.h's OP_BLEND.
//
// A step is three dependent products of all matrices of the batch at once: G of
// X with itself (the smaller side), B = b G + c G^2, and X' = a X + B X (or X B
// where the matrix is tall); the last one's epilogue writes the result, or the
// weights.
//
// Two steps at once.  With P = a + b G + c G^2 a step is X' = P X, and G of X'
// is P G P; P and G are polynomials of the first G, so they commute and all
// their products are symmetric:
//   P0 of G,  T = P0 G,  G1 = P0 T,  P1 of G1,  Q = P1 P0,  X'' = Q X
// take 3 + 5 small / large products of small^2 large for two steps instead of 6
// + 2, and read and write X once.  Rounded where the kernels round, two steps
// at once leave the same error as one by one (0.9 to 1.6 times over shapes from
// 16 x 3000 to 512 x 512 and gradients of few and many directions); three or
// five at once lose small singular directions.  Which of the two forms is taken
// follows from the planned products' times.
//
// G and the polynomials are symmetric: the tiles on and over the diagonal are
// computed and stored twice, and the products that take them read their rows
// where they would need columns.
//
// The products are float16's.  X's singular values stay in a range that follows
// from the coefficients, so X, G and the polynomials have fixed units that put
// them under 2^15: all 11 bits, and no element lost that is not 2^-29 of the
// largest.
//
// float32, float16, bfloat16 with `exact` and all sides of up to 96 hold each
// matrix as two such numbers, 23 bits, and take three products, of all but the two
// rests: the product left out is 2^-24 of the result, and the sums are chains of
// half as many additions (of eight products) as those of float32's own matrix
// instruction, which does a sixteenth of the work in the same time.
//
// bfloat16 else holds them as one.  A rounding of X is noise in all
// directions, 2^-12 / sqrt(3) of X's norm, and the steps enlarge small directions by
// 3.4445 each.  Where u fills its directions evenly the result is 0.04 to 0.21 % of
// its norm off, its rounding being 0.17 % (bfloat16's 8 bits in the products: 1.2 %).
// Where it does not, the noise is what fills the others: 512 x 1024 of rank 1 9.6 %,
// of rank 16 4.3, of rank 64 2.2, of 256 0.7; the whole of it goes by the second
// number (0.002 % at rank 16).  That takes 4096 x 16384 from 3200 to 8900 us, 16 x
// 512 x 2000 from 313 to 580, 1024 x 1024 from 156 to 195, so it is the caller's
// choice; of sides of up to 96, whose small products are one launch in pairs, 64 x
// 64 from 62 to 63, 96 x 16384 from 102 to 113, 24 x 64 x 4096 from 119 to 136, and
// it is none.
//
// With one number the diagonals of G and the polynomials, nearly multiples of the
// unit matrix, are all rounded one way, and where they are far larger than what is
// beside them that is most of the error (noise of 136 x 2200: 0.22 %, 0.06 without
// it).  At sides of up to 256 and of one to more than four
// what a diagonal is beyond its float16 is kept as a float32 and multiplied in the
// epilogues, which read X and G once more for it.  Percent of the norm off before
// the result's rounding, and us, with it and without:
//   104 x 2000   0.04 0.12   126 110       512 x 2000       0.06 0.14   156 149
//   256 x 256    0.09 0.14   108 101       16 x 512 x 2000  0.06 0.15   362 305
//   256 x 1000   0.07 0.14   124 115       1024 x 4096      0.05 0.10   238 219
//   512 x 5000   0.05 0.18   186 168       2048 x 8192      0.06 0.13   697 642
//   1024 x 8192  0.04 0.10   306 282       4096 x 16384                3370 3140
// The left ones have it, the right ones do not: no edge in the figures asks for the
// rule, which keeps the error without it under the result's rounding, 0.17 %, and
// the time of large and batched matrices.
#include "ops_call.h"
#include "ops_launch.h"
#include "ops_types.h"

namespace volta {
namespace ops {
namespace {

constexpr int kMaxSteps = 64;
constexpr int64_t kMaxBatch = 65535;  // a grid's third dimension

// ---------------------------------------------------------------------------
// u and its norm.  Two passes: momentum and the sum of squares (in 64 bits:
// gradients may be of 1e-25 or 1e25), and X = u / (norm + eps) in its unit, with
// zeros in what pads it to whole chunks.  Bound by memory; the second pass finds
// a few ten MB in the memory-side cache (16 x 512 x 2000 bfloat16 with momentum:
// 30 and 22 us for 164 and 131 MB).
// ---------------------------------------------------------------------------
__device__ __forceinline__ floatx4 mul16(chunk16 a, chunk16 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}
// Four numbers at an address of 8 bytes.
__device__ __forceinline__ void store4(_Float16* to, const float (&d)[4]) {
  union { _Float16 e[4]; uint64_t w; } u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u.e[i] = from_f<_Float16>(d[i]);
  *reinterpret_cast<uint64_t*>(to) = u.w;
}

struct MuonArgs {
  const void* g;       // u, or the gradient
  const float* m;      // momentum, or NULL
  float* m_out;
  _Float16* x;         // [batch][rows_p][ld_x]
  int64_t plane;       // elements to a second plane of it; 0: there is none
  double* partial;     // [batch][gridDim.x]
  int64_t rows, cols;  // of a matrix
  int64_t rows_p, cols_p, ld_x, ld_g, ld_m;
  float beta, eps, unit;
  int32_t nesterov;
};

// The sum over the block's 256 threads, on every thread, in a fixed order.
__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, kWave);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return ((lds[0] + lds[1]) + lds[2]) + lds[3];
}

// Chunks of E elements are dealt to the blocks of a matrix in turn.
template <typename T>
__global__ void __launch_bounds__(256) muon_norm(MuonArgs a) {
  constexpr int E = 16 / (int)sizeof(T);
  __shared__ double lds[4];
  const int64_t per_row = (a.cols + E - 1) / E, chunks = per_row * a.rows, z = blockIdx.y;
  double ss = 0.0;
#pragma unroll 2
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row, row = z * a.rows + r;
    const int c = (int)(i - r * per_row) * E, cnt = (int)min((int64_t)E, a.cols - c);
    float u[E];
    load_vec(static_cast<const T*>(a.g) + row * a.ld_g + c, cnt, u);
    if (a.m) {
      float m[E];
      load_vec(a.m + row * a.ld_m + c, cnt, m);
#pragma unroll
      for (int k = 0; k < E; ++k) {
        m[k] = a.beta * m[k] + u[k];
        u[k] = a.nesterov ? u[k] + a.beta * m[k] : m[k];
      }
      store_vec(a.m_out + row * a.ld_m + c, cnt, m);
    }
#pragma unroll
    for (int k = 0; k < E; ++k) ss += (double)u[k] * (double)u[k];
  }
  ss = block_sum(ss, lds);
  if (threadIdx.x == 0) a.partial[z * gridDim.x + blockIdx.x] = ss;
}

template <typename T>
__global__ void __launch_bounds__(256) muon_scale(MuonArgs a, int parts) {
  constexpr int E = 8;
  __shared__ double lds[4];
  const int64_t z = blockIdx.y, per_row = a.cols_p / E, chunks = per_row * a.rows_p;
  double ss = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) ss += a.partial[z * parts + i];
  ss = block_sum(ss, lds);
  const double norm = sqrt(ss) + (double)a.eps;
  const double per = norm == 0.0 ? 0.0 : (double)a.unit / norm;  // zeros stay zeros, without an eps too
#pragma unroll 2
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row, row = z * a.rows + r;
    const int c = (int)(i - r * per_row) * E;
    const int cnt = r < a.rows ? (int)min((int64_t)E, a.cols - c) : 0;
    float u[E];
    load_vec(static_cast<const T*>(a.g) + (cnt > 0 ? row * a.ld_g + c : 0), cnt, u);
    if (a.m) {
      float m[E];
      load_vec(static_cast<const float*>(a.m_out) + (cnt > 0 ? row * a.ld_m + c : 0), cnt, m);
#pragma unroll
      for (int k = 0; k < E; ++k) u[k] = a.nesterov ? u[k] + a.beta * m[k] : m[k];
    }
    // what is behind a row's end was read as 0; no norm makes anything else of it
#pragma unroll
    for (int k = 0; k < E; ++k) u[k] = k < cnt ? (float)((double)u[k] * per) : 0.0f;
    _Float16* to = a.x + (z * a.rows_p + r) * a.ld_x + c;
    store_vec(to, E, u);
    if (a.plane) {
#pragma unroll
      for (int k = 0; k < E; ++k) u[k] -= to_f(from_f<_Float16>(u[k]));  // exact
      store_vec(to + a.plane, E, u);
    }
  }
}

// Blocks of a matrix in the two passes: about as many as the chip holds.
int norm_blocks(int64_t batch, int64_t chunks) {
  const int64_t want = std::max<int64_t>(1, 2048 / batch);
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, (chunks + 511) / 512));
}

// ---------------------------------------------------------------------------
// The small products of a step, or of two at once, in one launch: a block for a
// matrix whose smaller side is at most S, with G and the polynomials in LDS, as
// pairs of float16 numbers.  Each
// product is S x S x S, one row of 16x16 blocks a wave; what bounds it is one
// latency after another (LDS, matrix instructions, barrier): the five products
// of two steps take 13.7 us at S = 96, 6.6 at 64 and 4.2 at 32, one step's 5.0, 2.8
// and 2.0; a launch for each takes 4 to 6.
//
// Rows of S + 8 numbers: 16 rows' chunks of a fragment meet every bank once.  A
// matrix's rows and columns from its side on are zeros (the diagonal's a times
// zeros in G).
// ---------------------------------------------------------------------------
struct ChainArgs {
  const _Float16* g;
  _Float16* out;
  int64_t plane, stride, ld;
  int32_t side, pairs;
  // a product's sums times alpha, the sum's other matrix times beta, the diagonal:
  // the polynomial; T, G of the next step, its polynomial, and both together
  float alpha[5], beta[5], diagonal[5];
};
template <int S>
__global__ void __launch_bounds__(512) muon_chain(ChainArgs a) {
  constexpr int PLANES = 2, LD = S + 8, kBlocks = S / 16, kRows = (kBlocks + 7) / 8;
  __shared__ __attribute__((aligned(16))) _Float16 lds[3][PLANES][S * LD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, lg = lane >> 4;
  const _Float16* g = a.g + blockIdx.x * a.stride;
  _Float16* out = a.out + blockIdx.x * a.stride;
  // rows of whole chunks: the side is a multiple of 8
  for (int i = threadIdx.x; i < S * (S / 8); i += 512) {
    const int r = i / (S / 8), c = i % (S / 8) * 8;
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
      chunk16 v{0, 0, 0, 0};
      if (r < a.side && c < a.side) v = *reinterpret_cast<const chunk16*>(g + p * a.plane + r * a.ld + c);
      *reinterpret_cast<chunk16*>(&lds[0][p][r * LD + c]) = v;
    }
  }
  __syncthreads();
  // alpha x y + beta r (r < 0: none), to a matrix in LDS or (to < 0) to the output
  auto product = [&](int x, int y, int which, int r, int to) {
    const float alpha = a.alpha[which], beta = a.beta[which], diagonal = a.diagonal[which];
#pragma unroll
    for (int row = 0; row < kRows; ++row) {
      const int m0 = (row * 8 + wave) * 16;
      if (m0 >= S) continue;
      floatx4 acc[kBlocks], small[kBlocks];
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) acc[j] = small[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < S; k += 32) {
        chunk16 f[PLANES];
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
          f[p] = *reinterpret_cast<const chunk16*>(&lds[x][p][(m0 + l) * LD + k + lg * 8]);
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
          chunk16 q[PLANES];
#pragma unroll
          for (int p = 0; p < PLANES; ++p)
            q[p] = *reinterpret_cast<const chunk16*>(&lds[y][p][(j * 16 + l) * LD + k + lg * 8]);
          acc[j] = mul16(q[0], f[0], acc[j]);
          small[j] = mul16(q[0], f[1], small[j]);
          small[j] = mul16(q[1], f[0], small[j]);
        }
      }
      const int m = m0 + l;
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        const int n = j * 16 + lg * 4;
        acc[j] = acc[j] + small[j];
        float d[4], rest[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d[i] = alpha * acc[j][i];
          if (r >= 0) d[i] += beta * (to_f(lds[r][0][m * LD + n + i]) + to_f(lds[r][1][m * LD + n + i]));
          if (m == n + i) d[i] += diagonal;
          rest[i] = d[i] - to_f(from_f<_Float16>(d[i]));  // exact
        }
        if (to >= 0) {
          store4(&lds[to][0][m * LD + n], d);
          store4(&lds[to][1][m * LD + n], rest);
        } else if (m < a.side && n < a.side) {
          store4(out + m * a.ld + n, d);
          store4(out + a.plane + m * a.ld + n, rest);
        }
      }
    }
    __syncthreads();
  };
  if (!a.pairs) {
    product(0, 0, 0, 0, -1);
    return;
  }
  product(0, 0, 0, 0, 1);     // P0
  product(1, 0, 1, -1, 2);    // T = P0 G
  product(1, 2, 2, -1, 0);    // G1 = P0 T
  product(0, 0, 3, 0, 2);     // P1
  product(2, 1, 4, -1, -1);   // Q = P1 P0
}
// The largest side that the chain takes: what three matrices leave of a CU's LDS.
constexpr int64_t kChainSide = 96;
hipError_t chain(const ChainArgs& a, int64_t batch, hipStream_t st) {
  const dim3 grid((unsigned)batch), block(512);
  if (a.side <= 32) return op_launch(muon_chain<32>, grid, block, st, a);
  if (a.side <= 64) return op_launch(muon_chain<64>, grid, block, st, a);
  return op_launch(muon_chain<96>, grid, block, st, a);
}

// ---------------------------------------------------------------------------
// Units of what a step takes: 1 in each stands for 1 / unit.
struct Units {
  double x, g, b, p, t;
};
struct Muon {
  volta_op_muon d;
  bool tall, pairs;        // pairs: two steps at once
  bool chain;              // the small products in one launch
  bool diag;               // the diagonals' rests are kept
  int planes;              // of X and the products; of larger bfloat16 that is not to be exact: 1
  int64_t rows_p, cols_p;  // padded to whole chunks: the products run over zeros there
  int64_t small, large;
  int64_t ld_x, ld_small;
  int parts;
  Units unit[kMaxSteps];
  int layout[3];           // of G, the small products and X'
  OpPlan plan[3];
  int64_t x_bytes, g_bytes, diag_bytes, sum_bytes, partial_bytes;
  int64_t bytes() const { return 2 * x_bytes + smalls() * (g_bytes + diag_bytes) + sum_bytes + partial_bytes; }
  int smalls() const { return pairs && !chain ? 3 : 2; }  // matrices of the smaller side
};

// The largest power of two that keeps `bound` at 2^15 or under.
double unit_of(double bound) { return std::exp2(15.0 - std::ceil(std::log2(bound))); }

Muon muon_of(const volta_op_muon* in) {
  need(in, "the description");
  Muon l{};
  volta_op_muon& d = l.d;
  d = *in;
  check_type(d.type);
  check_dims("steps", d.steps, 1, kMaxSteps);
  check_dims("batch", d.batch, 1, kMaxBatch);
  check_dims("rows", d.rows, 1, kMaxLd);
  check_dims("cols", d.cols, 1, kMaxLd);
  if (d.batch * d.rows > kMaxRows) refuse("batch times rows is over 2^30");
  if (!(d.eps >= 0.0f) || !std::isfinite(d.eps)) refuse("eps is negative or not finite");
  const double a = d.a, b = d.b, c = d.c;
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) refuse("a coefficient is not finite");
  d.ld_u = ld_of("ld_u", d.ld_u, d.cols);
  d.ld_m = ld_of("ld_m", d.ld_m, d.cols);
  d.ld_o = ld_of("ld_o", d.ld_o, d.cols);
  if (d.exact != 0 && d.exact != 1) refuse("exact is " + std::to_string(d.exact) + ", must be 0 or 1");
  l.rows_p = packed_ld(VOLTA_OP_F16, d.rows);
  l.cols_p = packed_ld(VOLTA_OP_F16, d.cols);
  l.tall = d.rows > d.cols;
  l.small = l.tall ? l.cols_p : l.rows_p;
  l.large = l.tall ? l.rows_p : l.cols_p;
  l.chain = l.small <= kChainSide;
  l.planes = d.type == VOLTA_OP_BF16 && !d.exact && !l.chain ? 1 : 2;
  // Singular values before each step are at most r: 1 at first (the sum of
  // squares of X is at most 1), then the largest |a s + b s^3 + c s^5| on [0, r]
  // (at the ends and between, by 4096 samples and a margin for what lies
  // between two).  An element is at most the largest singular value.
  double r = 1.0;
  for (int i = 0; i < d.steps; ++i) {
    double next = 0.0, poly = 0.0, whole = 0.0, times = 0.0;
    for (int k = 0; k <= 4096; ++k) {
      const double s = r * k / 4096, q = s * s, p = a + b * q + c * q * q;
      next = std::max(next, std::fabs(s * p));
      poly = std::max(poly, std::fabs(b * q + c * q * q));
      whole = std::max(whole, std::fabs(p));
      times = std::max(times, std::fabs(q * p));
    }
    if (!(std::max({r, next, whole}) <= 1024.0 && std::max(poly, times) <= 1e6))
      refuse("the coefficients let singular values grow past 1024");
    l.unit[i] = Units{unit_of(r), unit_of(r * r), unit_of(std::max(poly, 1e-6)), unit_of(std::max(whole, 1e-6)),
                      unit_of(std::max(times, 1e-6))};
    r = std::max(next * 1.001, 1e-6);
  }
  l.layout[0] = l.tall ? OP_TN : OP_NT;
  l.layout[1] = OP_NT;
  l.layout[2] = l.tall ? OP_NT : OP_NN;
  const int64_t M[3] = {l.small, l.small, l.tall ? l.large : l.small};
  const int64_t N[3] = {l.small, l.small, l.tall ? l.small : l.large};
  const int64_t K[3] = {l.large, l.small, l.small};
  for (int i = 0; i < 3; ++i) {
    l.plan[i] = op_gemm_plan(2, l.layout[i], i < 2 ? OP_MIRROR : OP_BLEND, M[i], N[i], K[i], l.planes == 2 ? 3 : 1,
                             (int)d.batch, true);
    l.partial_bytes = std::max(l.partial_bytes, align256(op_gemm_partial_bytes(l.plan[i], OP_BLEND, M[i], N[i], (int)d.batch)));
    if (op_gemm_blocks(l.plan[i], OP_BLEND, M[i], N[i]) * d.batch > kMaxBlocks) refuse("the rows and columns of a product are too many");
  }
  l.diag = l.planes == 1 && (l.small <= 256 || l.large > 4 * l.small);
  const double one = l.plan[0].us + l.plan[1].us + l.plan[2].us;
  const double two = l.plan[0].us + 5.0 * l.plan[1].us + l.plan[2].us;
  l.pairs = d.steps >= 2 && (l.chain || two < 2.0 * one);
  l.ld_x = line_ld(2, l.cols_p);
  l.ld_small = line_ld(2, l.small);
  l.x_bytes = align256(d.batch * l.rows_p * l.ld_x * 2 * l.planes);
  l.g_bytes = align256(d.batch * l.small * l.ld_small * 2 * l.planes);
  l.diag_bytes = l.diag ? align256(d.batch * l.small * 4) : 0;
  l.parts = norm_blocks(d.batch, d.rows * ((d.cols + 3) / 4));
  l.sum_bytes = align256(8 * d.batch * l.parts);
  return l;
}

hipError_t passes(const Muon& l, MuonArgs a, hipStream_t st) {
  const dim3 grid((unsigned)l.parts, (unsigned)l.d.batch);
  auto run = [&](auto like) {
    using T = decltype(like);
    const hipError_t e = op_launch(muon_norm<T>, grid, dim3(256), st, a);
    return e != hipSuccess ? e : op_launch(muon_scale<T>, grid, dim3(256), st, a, l.parts);
  };
  return l.d.type == VOLTA_OP_F32    ? run(0.0f)
         : l.d.type == VOLTA_OP_BF16 ? run((__bf16)0.0f)
                                     : run((_Float16)0.0f);
}

// The passes and products of a call; `last` says what becomes of the last X:
// out, w, gamma, and in alpha what it is multiplied by.
void run(const Muon& l, MuonArgs a, const OpEpilogueMore& last, char* workspace, hipStream_t st) {
  const volta_op_muon& d = l.d;
  char* x[2] = {workspace, workspace + l.x_bytes};
  char* small[3];  // matrices of the smaller side
  for (int i = 0; i < 3; ++i) small[i] = workspace + 2 * l.x_bytes + i * l.g_bytes;
  char* rest = small[l.smalls() - 1] + l.g_bytes;
  auto diag_of = [&](const char* p) -> float* {  // of one of them
    return !l.diag ? nullptr : reinterpret_cast<float*>(rest + (p - small[0]) / l.g_bytes * l.diag_bytes);
  };
  char* sums = rest + l.smalls() * l.diag_bytes;
  a.partial = reinterpret_cast<double*>(sums);
  float* partial = reinterpret_cast<float*>(sums + l.sum_bytes);
  const int64_t x_size = l.rows_p * l.ld_x, g_size = l.small * l.ld_small;
  const int64_t x_plane = l.planes == 2 ? d.batch * x_size : 0, g_plane = d.batch * g_size;
  const int out_type = l.planes == 2 ? OP_PLANES : VOLTA_OP_F16;
  a.x = reinterpret_cast<_Float16*>(x[0]);
  a.plane = x_plane;
  a.rows = d.rows;
  a.cols = d.cols;
  a.rows_p = l.rows_p;
  a.cols_p = l.cols_p;
  a.ld_x = l.ld_x;
  a.ld_g = d.ld_u;
  a.ld_m = d.ld_m;
  a.eps = d.eps;
  a.unit = (float)l.unit[0].x;
  check_hip(passes(l, a, st), "norm");
  struct Of {  // a matrix of each of the batch
    const char* p;
    int64_t ld, stride, plane;
  };
  auto of_x = [&](const char* p) { return Of{p, l.ld_x, x_size, x_plane}; };
  auto of_small = [&](const char* p) { return Of{p, l.ld_small, g_size, l.planes == 2 ? g_plane : 0}; };
  auto product = [&](int which, const Of& p, const Of& q, int64_t M, int64_t N, int64_t K, const OpEpilogueMore& epi,
                     const char* what) {
    OpGemmMore m{};
    m.epi = epi;
    m.p[0] = m.p[1] = p.p;
    m.q[0] = m.q[1] = q.p;
    m.ld_p = p.ld;
    m.ld_q = q.ld;
    m.epi.stride_p = p.stride;
    m.epi.stride_q = q.stride;
    m.epi.plane_p = p.plane;
    m.epi.plane_q = q.plane;
    m.M = (int32_t)M;
    m.N = (int32_t)N;
    m.K = (int32_t)K;
    m.pieces = l.planes == 2 ? 3 : 1;
    m.outputs = (int32_t)d.batch;
    m.direct = 1;
    m.partial = partial;
    check_hip(op_gemm_blend(l.layout[which], which < 2 ? OP_MIRROR : OP_BLEND, l.plan[which], m, st), what);
  };
  auto blend_with = [&](OpEpilogueMore& o, const Of& r, double beta) {
    o.beta = (float)beta;
    o.blend = r.p;
    o.ld_blend = r.ld;
    o.stride_blend = r.stride;
    o.plane_blend = r.plane;
  };
  // out = alpha d: matrices of the smaller side
  auto to_small = [&](char* out, double alpha) {
    OpEpilogueMore o{};
    o.out[0] = out;
    o.out_type = out_type;
    o.diag_out = diag_of(out);
    o.stride_diag = l.small;
    o.ld_out = l.ld_small;
    o.stride_out = g_size;
    o.plane_out = g_plane;
    o.alpha = (float)alpha;
    return o;
  };
  auto gram = [&](const char* from, char* out, const Units& u) {
    product(0, of_x(from), of_x(from), l.small, l.small, l.large, to_small(out, u.g / (u.x * u.x)), "gram");
  };
  auto multiply = [&](const char* p, const char* q, OpEpilogueMore o) {
    o.ld_blend = l.ld_small;
    o.stride_blend = g_size;
    o.diag_weight = p == q ? 2.0f : 1.0f;
    o.diag = diag_of(p);
    o.diag_rows = 1;
    if (o.diag) o.blend = q;
    if (o.diag && p != q) {
      o.diag2 = diag_of(q);
      o.blend2 = p;
    }
    product(1, of_small(p), of_small(q), l.small, l.small, l.small, o, "polynomial");
  };
  // b G + c G^2 in `unit`, and a on the diagonal
  auto polynomial = [&](const char* g, char* out, const Units& u, double unit, double diagonal) {
    OpEpilogueMore o = to_small(out, d.c * unit / (u.g * u.g));
    blend_with(o, of_small(g), d.b * unit / u.g);
    o.diagonal = (float)(diagonal * unit);
    multiply(g, g, o);
  };
  int at = 0;
  for (int i = 0; i < d.steps;) {
    const int n = l.pairs && i + 1 < d.steps ? 2 : 1;
    const char *from = x[at], *by;
    const Units &u = l.unit[i], &v = l.unit[i + n - 1];
    double by_unit;
    gram(from, small[0], u);
    if (l.chain) {
      ChainArgs c{};
      c.g = reinterpret_cast<const _Float16*>(small[0]);
      c.out = reinterpret_cast<_Float16*>(small[1]);
      c.plane = g_plane;
      c.stride = g_size;
      c.ld = l.ld_small;
      c.side = (int32_t)l.small;
      c.pairs = n == 2;
      auto set = [&](int i, double alpha, double beta, double diagonal) {
        c.alpha[i] = (float)alpha;
        c.beta[i] = (float)beta;
        c.diagonal[i] = (float)diagonal;
      };
      const double p = n == 2 ? u.p : u.b;
      set(0, d.c * p / (u.g * u.g), d.b * p / u.g, n == 2 ? d.a * p : 0.0);
      by_unit = n == 2 ? u.p * v.p * 0x1p-15 : u.b;
      if (n == 2) {
        set(1, u.t / (u.p * u.g), 0.0, 0.0);
        set(2, v.g / (u.p * u.t), 0.0, 0.0);
        set(3, d.c * v.p / (v.g * v.g), d.b * v.p / v.g, d.a * v.p);
        set(4, by_unit / (u.p * v.p), 0.0, 0.0);
      }
      check_hip(chain(c, d.batch, st), "polynomials");
      by = small[1];
    } else if (n == 2) {
      polynomial(small[0], small[1], u, u.p, d.a);
      multiply(small[1], small[0], to_small(small[2], u.t / (u.p * u.g)));
      multiply(small[1], small[2], to_small(small[0], v.g / (u.p * u.t)));
      polynomial(small[0], small[2], v, v.p, d.a);
      // at most the product of both largest values, each at most 2^15 in its unit
      by_unit = u.p * v.p * 0x1p-15;
      multiply(small[2], small[1], to_small(small[0], by_unit / (u.p * v.p)));
      by = small[0];
    } else {
      by_unit = u.b;
      polynomial(small[0], small[1], u, u.b, 0.0);
      by = small[1];
    }
    i += n;
    // X' in the next step's unit, or the result
    const bool end = i == d.steps;
    const double to = end ? (double)last.alpha : l.unit[i].x;
    OpEpilogueMore o{};
    if (end) {
      o = last;
    } else {
      o.out[0] = x[at ^ 1];
      o.out_type = out_type;
      o.ld_out = l.ld_x;
      o.stride_out = x_size;
      o.plane_out = x_plane;
    }
    o.alpha = (float)(to / (by_unit * u.x));
    if (n == 1) blend_with(o, of_x(from), to * d.a / u.x);
    o.ld_blend = l.ld_x;
    o.stride_blend = x_size;
    o.stride_diag = l.small;
    o.diag = diag_of(by);
    o.diag_rows = !l.tall;
    if (o.diag) o.blend = from;
    const int64_t M = end ? d.rows : l.rows_p, N = end ? d.cols : l.cols_p;
    if (l.tall) product(2, of_x(from), of_small(by), M, N, l.small, o, "step");
    else product(2, of_small(by), of_x(from), M, N, l.small, o, "step");
    at ^= 1;
  }
}

}  // namespace
}  // namespace ops
}  // namespace volta

using namespace volta;
using namespace volta::ops;

extern "C" {

int64_t volta_op_muon_workspace(const volta_op_muon* d) {
  return bytes_of("volta_op_muon_workspace", VOLTA_OP_FORWARD, [&](bool) { return muon_of(d).bytes(); });
}

int32_t volta_op_muon_orthogonalize(const volta_op_muon* in, const void* u, void* o, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  return guarded("volta_op_muon_orthogonalize", [&] {
    const Muon l = muon_of(in);
    const volta_op_muon& d = l.d;
    const int e = elem_bytes(d.type);
    need(u, "u");
    need(o, "o");
    check_workspace(workspace, workspace_bytes, l.bytes());
    const hipStream_t st = check_call({{"u", u, d.batch * d.rows, d.cols, d.ld_u, e, false},
                                       {"o", o, d.batch * d.rows, d.cols, d.ld_o, e, true}},
                                      {{"u", "o"}}, workspace, l.bytes(), stream);
    MuonArgs a{};
    a.g = u;
    OpEpilogueMore last{};
    last.out[0] = o;
    last.out_type = d.type;
    last.ld_out = d.ld_o;
    last.stride_out = d.rows * d.ld_o;
    last.alpha = 1.0f;
    run(l, a, last, static_cast<char*>(workspace), st);
  });
}

int32_t volta_op_muon_step(const volta_op_muon* in, const void* g, const float* m, const void* w, float* m_out,
                           void* w_out, float lr, float beta, int32_t nesterov, float decay, float scale,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded("volta_op_muon_step", [&] {
    const Muon l = muon_of(in);
    const volta_op_muon& d = l.d;
    const int e = elem_bytes(d.type);
    need(g, "g");
    need(m, "m");
    need(w, "w");
    need(m_out, "m_out");
    need(w_out, "w_out");
    for (float v : {lr, beta, decay, scale})
      if (!std::isfinite(v)) refuse("lr, beta, decay or scale is not finite");
    check_workspace(workspace, workspace_bytes, l.bytes());
    const int64_t rows = d.batch * d.rows;
    const hipStream_t st = check_call({{"g", g, rows, d.cols, d.ld_u, e, false},
                                       {"m", m, rows, d.cols, d.ld_m, 4, false},
                                       {"w", w, rows, d.cols, d.ld_o, e, false},
                                       {"m_out", m_out, rows, d.cols, d.ld_m, 4, true},
                                       {"w_out", w_out, rows, d.cols, d.ld_o, e, true}},
                                      {{"m", "m_out"}, {"w", "w_out"}}, workspace, l.bytes(), stream);
    MuonArgs a{};
    a.g = g;
    a.m = m;
    a.m_out = m_out;
    a.beta = beta;
    a.nesterov = nesterov != 0;
    OpEpilogueMore last{};
    last.out[0] = w_out;
    last.out_type = d.type;
    last.ld_out = last.ld_w = d.ld_o;
    last.stride_out = last.stride_w = d.rows * d.ld_o;
    last.w = w;
    last.alpha = -(lr * scale);
    last.gamma = 1.0f - lr * decay;
    run(l, a, last, static_cast<char*>(workspace), st);
  });
}

}  // extern "C"
