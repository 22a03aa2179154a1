// The loss of an output layer over many classes (include/volta_ops.h): entry
// points and what surrounds their products (ops_gemm_kernels.h).
//
// Forward.  The product's blocks leave {largest, sum of exponentials} of each
// row over its columns, and a second launch joins them:
//   lse = t + log(sum over i of s_i exp(t_i - t)),  t = the largest t_i.
//
// Backward.  The classes in pieces.  For each: z anew, its epilogue forms dz
// (in the type, as the products take it); dx adds dz W^T of the pieces in 32
// bits; dw's columns are the piece's own.  A piece is as many classes as 256
// MiB of dz hold, what the memory-side cache holds: larger ones are read from
// memory, smaller ones add dx more often.
//
// The roundings of dz to 16 bits average out over many rows: they add as much to
// the gradients' error as the gradients' own rounding does (bfloat16 0.17 % each,
// 0.22 % together).  The label's element is about -dloss in every row where its p
// is small, so dz is in units of the largest |dloss|, which the sums are multiplied
// by in 32 bits: of a mean's equal dloss it is -1 then and exact, where 1 / 1020
// itself would be rounded the same way in every row (0.40 % of dx, dW and db, 0.17
// in units).  Rows of a few other dloss still round their labels' elements alike,
// by half a step at most.
//
// Over few rows less averages out (bfloat16, 1 to 32 rows: gradients up to 0.28 %
// off with their own rounding, 0.17 of it), and the products take the time that W
// and dw take to move.  There dz is held as two numbers of its type, the second in rows
// behind the first: dw's product runs over both, x laid out twice; dx's halves
// are added by a launch of their own.
#include "ops_call.h"
#include "ops_launch.h"
#include "ops_types.h"

namespace volta {
namespace ops {
namespace {

constexpr unsigned RUN_DZ = 8;  // beside those of ops_call.h
constexpr int64_t kPieceBytes = int64_t{256} << 20;
constexpr int64_t kTwiceRows = 128;  // dz of up to so many rows is held as two numbers

// ---------------------------------------------------------------------------
// Joins a row's entries.  A block takes 16 rows, which lie side by side in an
// entry, and 64 lanes share out the entries, in a fixed order.  Bound by memory
// (2048 rows of 512 entries 9.5 us) and, at few rows, by the launch (4.7).
// ---------------------------------------------------------------------------
struct JoinArgs {
  const float* stats;  // [entries][rows] of {largest, sum}
  const float* at_label;
  const int32_t* labels;
  float *loss, *lse;
  int64_t rows, entries;
  int32_t classes;
};

__device__ __forceinline__ void join(float& t, float& s, float t2, float s2) {
  const float top = fmaxf(t, t2), base = top == -__builtin_inff() ? 0.0f : top;
  s = s * expf(t - base) + s2 * expf(t2 - base);
  t = top;
}

template <int ROWS>
__global__ void __launch_bounds__(1024) join_kernel(JoinArgs a) {
  constexpr int LANES = 1024 / ROWS;
  __shared__ float lds[2][LANES][ROWS];
  const int r = threadIdx.x % ROWS, l = threadIdx.x / ROWS;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * ROWS + r;
  float t = -__builtin_inff(), s = 0.0f;
  if (row < a.rows) {
    for (int64_t i = l; i < a.entries; i += LANES) {
      const float* p = a.stats + 2 * (i * a.rows + row);
      join(t, s, p[0], p[1]);
    }
  }
  lds[0][l][r] = t;
  lds[1][l][r] = s;
  for (int half = LANES / 2; half >= 1; half /= 2) {
    __syncthreads();
    if (l < half) {
      join(t, s, lds[0][l + half][r], lds[1][l + half][r]);
      lds[0][l][r] = t;
      lds[1][l][r] = s;
    }
  }
  if (l != 0 || row >= a.rows) return;
  const float lse = t + logf(s);
  if (a.lse) a.lse[row] = lse;
  if (!a.loss) return;
  const int label = a.labels[row];
  a.loss[row] = label < 0 ? 0.0f : label >= a.classes ? __builtin_nanf("") : lse - a.at_label[row];
}

hipError_t join_rows(const JoinArgs& a, hipStream_t st) {
  // few rows: more lanes for each
  const int per = a.rows >= 16 ? 16 : a.rows >= 4 ? 4 : 1;
  const int64_t n = (a.rows + per - 1) / per, x = std::min<int64_t>(n, int64_t{1} << 20);
  const dim3 grid((unsigned)x, (unsigned)((n + x - 1) / x));
  return op_launch(per == 16 ? join_kernel<16> : per == 4 ? join_kernel<4> : join_kernel<1>, grid, dim3(1024), st, a);
}

// The units of dz in 16 bits, from m, the largest |dloss| of a row with a label
// (|dz| is at most |dloss|): unit[1], 2^14 / m, and unit[0], m / 2^14.  `whole`, for
// dz held as two numbers, which need no exact m: the powers of two next to them,
// which put m in [2^14, 2^15).  No such row, and zeros alone: 1.  Infinities and NaN
// are left out.  An m under 2^-100 counts as that, so that no unit leaves the normal
// numbers (float16's gradients are 0 long before).  One block for each 65536 rows and
// at most 64; of more than one a second launch joins theirs.  4.2 us at 1000 rows:
// the launch.
constexpr int64_t kUnitRows = 65536;
constexpr int kUnitBlocks = 64;
__device__ __forceinline__ void units_of(uint32_t m, bool whole, float* unit) {
  float u0 = 1.0f, u1 = 1.0f;
  if (m != 0) {
    float top = fmaxf(__uint_as_float(m), 0x1p-100f);
    if (whole) top = __uint_as_float(__float_as_uint(top) & 0x7f800000u);
    u0 = top * 0x1p-14f;
    u1 = 0x1p14f / top;
  }
  unit[0] = u0;
  unit[1] = u1;
}
// `partial` NULL: one block, to `unit`; else each block's m.
__global__ void __launch_bounds__(1024) unit_kernel(const float* dloss, const int32_t* labels, int64_t rows, bool whole,
                                                    uint32_t* partial, float* unit) {
  __shared__ uint32_t lds[16];
  uint32_t m = 0;
#pragma unroll 8
  for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < rows; i += (int64_t)gridDim.x * 1024) {
    const uint32_t v = __float_as_uint(fabsf(dloss[i]));
    m = max(m, labels[i] >= 0 && v < 0x7f800000u ? v : 0u);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, kWave));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 0; w < 16; ++w) m = max(m, lds[w]);
  if (partial) partial[blockIdx.x] = m;
  else units_of(m, whole, unit);
}
__global__ void __launch_bounds__(64) unit_join(const uint32_t* partial, int n, bool whole, float* unit) {
  uint32_t m = (int)threadIdx.x < n ? partial[threadIdx.x] : 0u;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, kWave));
  if (threadIdx.x == 0) units_of(m, whole, unit);
}
// `unit`: 64 floats, then the blocks' maxima.
hipError_t units(const float* dloss, const int32_t* labels, int64_t rows, bool whole, float* unit, hipStream_t st) {
  const int blocks = (int)std::min<int64_t>(kUnitBlocks, std::max<int64_t>(1, (rows + kUnitRows - 1) / kUnitRows));
  uint32_t* partial = blocks > 1 ? reinterpret_cast<uint32_t*>(unit + 64) : nullptr;
  const hipError_t e = op_launch(unit_kernel, dim3(blocks), dim3(1024), st, dloss, labels, rows, whole, partial, unit);
  return e != hipSuccess || !partial ? e : op_launch(unit_join, dim3(1), dim3(64), st, partial, blocks, whole, unit);
}

// dx of dz held as two numbers: the sums of the first's rows and the second's
// (16 rows of 4096 inputs: 4.6 us, the launch).
template <typename T>
__global__ void __launch_bounds__(256) add_halves(const float* sum, int64_t rows, int64_t cols, const float* unit, T* dx,
                                                  int64_t ld) {
  const int64_t per_row = (cols + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * per_row) return;
  const int64_t r = i / per_row, c = i % per_row * 4;
  const int cnt = (int)min((int64_t)4, cols - c);
  float a[4], b[4];
  load_vec(sum + r * cols + c, cnt, a);
  load_vec(sum + (rows + r) * cols + c, cnt, b);
  const float u = unit ? *unit : 1.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] = (a[k] + b[k]) * u;
  store_vec(dx + r * ld + c, cnt, a);
}

// Column sums of dz: 64 lanes of 16 bytes, eight waves on the rows of a strip
// each, in order; the strips' sums are added by sum_partials.  Whole chunks are
// read: what a row has behind its columns is dz's own memory, and its sums are
// not stored.  Bound by memory: 1000 rows of 10000 float16 5.5 us, 3.6 TB/s.
constexpr int kSumWaves = 8;
template <typename T>
__global__ void __launch_bounds__(kSumWaves * 64) column_sums(const T* dz, int64_t ld, int64_t rows, int cols, int64_t per,
                                                              const float* unit, float* partial) {
  constexpr int E = 16 / (int)sizeof(T);
  __shared__ float lds[kSumWaves][64][E];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (blockIdx.x * 64 + lane) * E, cnt = cols - c;
  const int64_t r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
  float acc[E] = {};
  const T* from = dz + (cnt > 0 ? c : 0);
#pragma unroll 8
  for (int64_t r = r0 + wave; r < r1; r += kSumWaves) {
    union { chunk16 v; T e[E]; } u;
    u.v = *reinterpret_cast<const chunk16*>(from + r * ld);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] += to_f(u.e[i]);
  }
#pragma unroll
  for (int i = 0; i < E; ++i) lds[wave][lane][i] = acc[i];
  __syncthreads();
  if (wave != 0 || cnt <= 0) return;
  const float u = unit ? *unit : 1.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
#pragma unroll
    for (int w = 1; w < kSumWaves; ++w) acc[i] += lds[w][lane][i];
    acc[i] *= u;
  }
  store_vec(partial + (int64_t)blockIdx.y * cols + c, cnt, acc);
}
// Rows of a strip: 64 or more, so that its sums are few beside what it reads.
int64_t strip_rows(int64_t rows) { return std::max<int64_t>(64, (rows + 63) / 64); }
int64_t strips_of(int64_t rows) { return std::max<int64_t>(1, (rows + strip_rows(rows) - 1) / strip_rows(rows)); }

hipError_t sum_columns(int type, const void* dz, int64_t ld, int64_t rows, int64_t cols, const float* unit, float* partial,
                       void* db, hipStream_t st) {
  const int64_t per = strip_rows(rows), strips = strips_of(rows);
  const int across = 64 * 16 / elem_bytes(type);
  const dim3 grid((unsigned)((cols + across - 1) / across), (unsigned)strips);
  auto run = [&](auto like) {
    using T = decltype(like);
    return op_launch(column_sums<T>, grid, dim3(kSumWaves * 64), st, static_cast<const T*>(dz), ld, rows, (int)cols, per, unit,
                     partial);
  };
  const hipError_t e = type == VOLTA_OP_F32    ? run(0.0f)
                       : type == VOLTA_OP_BF16 ? run((__bf16)0.0f)
                                               : run((_Float16)0.0f);
  if (e != hipSuccess) return e;
  const SumArgs s{{partial, nullptr}, {db, nullptr}, 1, (int32_t)strips, cols};
  return sum_partials(type, s, st);
}

// ---------------------------------------------------------------------------
// The three products of a piece of `count` classes.
struct Piece {
  int64_t count, columns;  // columns: of dz, with padding where W is laid out anew
  Shape z, dx, dw;
  int64_t bytes() const { return std::max(z.bytes(), std::max(dx.bytes(), dw.bytes())); }
};

struct Loss {
  volta_op_cross_entropy d;
  int e;
  // forward
  Shape fwd;
  int64_t stats_bytes, at_bytes;
  // backward
  bool pack_x, pack_w;
  int64_t held;  // rows of dz: `rows`, or twice as many
  int64_t pieces, piece, ld_dz;
  Piece whole, last;
  int64_t dz_bytes, x_bytes, w_bytes, sum_bytes, partial_bytes, unit_bytes;
  int64_t forward_bytes() const { return stats_bytes + at_bytes + fwd.bytes(); }
  int64_t backward_bytes() const {
    return dz_bytes + x_bytes + w_bytes + sum_bytes + partial_bytes + unit_bytes + std::max(whole.bytes(), last.bytes());
  }
};

Piece piece_of(const Loss& l, int64_t count, unsigned run) {
  const volta_op_cross_entropy& d = l.d;
  Piece p{};
  p.count = count;
  p.columns = l.pack_w ? packed_ld(d.type, count) : count;
  const int64_t x_ld = l.pack_x ? line_ld(l.e, d.inputs) : d.ld_x, x_len = l.pack_x ? packed_ld(d.type, d.inputs) : d.inputs;
  const int64_t w_ld = l.pack_w ? line_ld(l.e, count) : d.ld_w;
  const Operand x{d.rows, x_len, x_ld, 1}, w{d.inputs, p.columns, w_ld, 1}, dz{l.held, p.columns, l.ld_dz, 1};
  p.z = shape_of(d.type, OP_NN, OP_LOSS_GRAD, d.rows, p.columns, d.inputs, 1, 1, x, w);
  if (run & RUN_DX) p.dx = shape_of(d.type, OP_NT, OP_ADD, l.held, d.inputs, count, 1, 1, dz, w);
  if (run & RUN_DW) {
    const Operand again{l.held, x_len, x_ld, 1};
    p.dw = shape_of(d.type, OP_TN, OP_STORE, d.inputs, count, l.held, 1, 1, again, dz);
  }
  return p;
}

Loss loss_of(const volta_op_cross_entropy* in, unsigned run) {
  need(in, "the description");
  Loss l{};
  volta_op_cross_entropy& d = l.d;
  d = *in;
  check_type(d.type);
  check_dims("rows", d.rows, 0, kMaxRows);
  check_dims("inputs", d.inputs, 1, kMaxLd);
  check_dims("classes", d.classes, 1, kMaxLd);
  d.ld_x = ld_of("ld_x", d.ld_x, d.inputs);
  d.ld_w = ld_of("ld_w", d.ld_w, d.classes);
  d.ld_dx = ld_of("ld_dx", d.ld_dx, d.inputs);
  d.ld_dw = ld_of("ld_dw", d.ld_dw, d.classes);
  l.e = elem_bytes(d.type);
  const Operand x{d.rows, d.inputs, d.ld_x, 1}, w{d.inputs, d.classes, d.ld_w, 1};
  if (run & RUN_FORWARD) {
    l.fwd = shape_of(d.type, OP_NN, OP_STATS, d.rows, d.classes, d.inputs, 1, 1, x, w);
    for (bool direct : {false, true}) {
      const int64_t n = d.rows > 0 ? op_stats_entries(plan_of(d.type, l.fwd, direct), d.classes) : 0;
      l.stats_bytes = std::max(l.stats_bytes, align256(8 * n * d.rows));
    }
    l.at_bytes = align256(4 * d.rows);
  }
  if (run & RUN_DZ) {
    const bool twice = d.type != VOLTA_OP_F32 && d.rows <= kTwiceRows;
    l.held = twice ? 2 * d.rows : d.rows;
    // Operands whose rows are not whole chunks are laid out anew once a piece,
    // for the two or three products that take them.  Few rows of dz read them once
    // and a half as it is, and so do a few more where W and its copy are more than
    // the memory-side cache, 256 MiB.  In us, W laid out anew and not, bfloat16:
    //   32 x 1000 x 10007   53  64      60 x 4096 x 32769   384 302
    //   60 x 1000 x 10007   58  71      80 x 4096 x 32769   391 391
    //   60 x 256 x 50001    66  70      100 x 4096 x 32769  415 501
    //   64 x 4096 x 16385  178 173      1000 x 1000 x 10007 115 147
    // Over 21 sizes of 32 to 1000 rows in three types this rule takes the faster way
    // or one within 4 % of it, but for float32, 64 x 1000 x 10007: 88 for 82.  (The
    // plans' own times, summed over the products, take the slower one by 16 to 24 %
    // at 32 to 60 rows of 1000 inputs.)
    l.pack_x = (twice && (run & RUN_DW)) || (l.held >= 64 && !whole_chunks(d.type, x));
    l.pack_w = l.held >= 64 && !whole_chunks(d.type, w) &&
               (d.rows > 64 || d.inputs * d.classes * l.e <= int64_t{128} << 20);
    const int64_t most = std::max<int64_t>(256, kPieceBytes / (l.e * std::max<int64_t>(1, l.held)) / 256 * 256);
    l.pieces = (d.classes + most - 1) / most;
    l.piece = l.pieces == 1 ? d.classes : ((d.classes + l.pieces - 1) / l.pieces + 255) / 256 * 256;
    l.pieces = (d.classes + l.piece - 1) / l.piece;
    l.ld_dz = line_ld(l.e, l.piece);
    l.whole = piece_of(l, l.piece, run);
    l.last = piece_of(l, d.classes - (l.pieces - 1) * l.piece, run);
    l.dz_bytes = align256(l.held * l.ld_dz * l.e);
    l.x_bytes = l.pack_x ? align256(l.held * line_ld(l.e, d.inputs) * l.e) : 0;
    l.w_bytes = l.pack_w ? align256(d.inputs * line_ld(l.e, l.piece) * l.e) : 0;
    l.sum_bytes = (twice || l.pieces > 1) && (run & RUN_DX) ? align256(4 * l.held * d.inputs) : 0;
    l.partial_bytes = align256(4 * strips_of(l.held) * l.piece);
    // two numbers of bfloat16 hold dz to 2^-16 in its own range: no unit
    l.unit_bytes = d.type == VOLTA_OP_F16 || (d.type == VOLTA_OP_BF16 && !twice) ? 512 : 0;
  }
  return l;
}

}  // namespace
}  // namespace ops
}  // namespace volta

using namespace volta;
using namespace volta::ops;

extern "C" {

int64_t volta_op_cross_entropy_workspace(const volta_op_cross_entropy* d, int32_t direction) {
  return bytes_of("volta_op_cross_entropy_workspace", direction, [&](bool backward) {
    const Loss l = loss_of(d, backward ? RUN_DZ | RUN_DX | RUN_DW : RUN_FORWARD);
    return backward ? l.backward_bytes() : l.forward_bytes();
  });
}

int32_t volta_op_cross_entropy_forward(const volta_op_cross_entropy* in, const void* x, const void* w,
                                       const void* bias, const int32_t* labels, float* loss, float* lse,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded("volta_op_cross_entropy_forward", [&] {
    const Loss l = loss_of(in, RUN_FORWARD);
    const volta_op_cross_entropy& d = l.d;
    if (d.rows > 0) {
      if (!loss && !lse) refuse("loss and lse are both NULL");
      need(x, "x");
      if (loss) need(labels, "labels");
    }
    need(w, "w");
    check_workspace(workspace, workspace_bytes, l.forward_bytes());
    const hipStream_t st = check_call({{"x", x, d.rows, d.inputs, d.ld_x, l.e, false},
                                       {"w", w, d.inputs, d.classes, d.ld_w, l.e, false},
                                       {"bias", bias, 1, d.classes, d.classes, l.e, false},
                                       {"labels", labels, d.rows, 1, 1, 4, false},
                                       {"loss", loss, d.rows, 1, 1, 4, true},
                                       {"lse", lse, d.rows, 1, 1, 4, true}},
                                      {}, workspace, l.forward_bytes(), stream);
    if (d.rows == 0) return;
    char* ws = static_cast<char*>(workspace);
    OpEpilogueMore epi{};
    epi.bias[0] = bias;
    epi.labels = loss ? labels : nullptr;
    epi.classes = epi.all_classes = (int32_t)d.classes;
    epi.stats = reinterpret_cast<float*>(ws);
    epi.at_label = reinterpret_cast<float*>(ws + l.stats_bytes);
    const bool direct =
        product(d.type, l.fwd, &x, &w, epi, ws + l.stats_bytes + l.at_bytes, st, "product");
    JoinArgs a{};
    a.stats = epi.stats;
    a.at_label = epi.at_label;
    a.labels = labels;
    a.loss = loss;
    a.lse = lse;
    a.rows = d.rows;
    a.entries = op_stats_entries(plan_of(d.type, l.fwd, direct), d.classes);
    a.classes = (int32_t)d.classes;
    check_hip(join_rows(a, st), "join");
  });
}

int32_t volta_op_cross_entropy_backward(const volta_op_cross_entropy* in, const void* x, const void* w,
                                        const void* bias, const int32_t* labels, const float* lse,
                                        const float* dloss, void* dx, void* dw, void* db, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
  return guarded("volta_op_cross_entropy_backward", [&] {
    const Loss l = loss_of(in, RUN_DZ | (dx ? RUN_DX : 0) | (dw ? RUN_DW : 0));
    const volta_op_cross_entropy& d = l.d;
    if (!dx && !dw && !db && d.rows > 0) refuse("dx, dw and db are all NULL");
    if (d.rows > 0) {
      need(x, "x");
      need(w, "w");
      need(labels, "labels");
      need(lse, "lse");
      need(dloss, "dloss");
    }
    check_workspace(workspace, workspace_bytes, l.backward_bytes());
    const hipStream_t st = check_call({{"x", x, d.rows, d.inputs, d.ld_x, l.e, false},
                                       {"w", w, d.inputs, d.classes, d.ld_w, l.e, false},
                                       {"bias", bias, 1, d.classes, d.classes, l.e, false},
                                       {"labels", labels, d.rows, 1, 1, 4, false},
                                       {"lse", lse, d.rows, 1, 1, 4, false},
                                       {"dloss", dloss, d.rows, 1, 1, 4, false},
                                       {"dx", dx, d.rows, d.inputs, d.ld_dx, l.e, true},
                                       {"dw", dw, d.inputs, d.classes, d.ld_dw, l.e, true},
                                       {"db", db, 1, d.classes, d.classes, l.e, true}},
                                      {}, workspace, l.backward_bytes(), stream);
    char* at = static_cast<char*>(workspace);
    auto take = [&](int64_t n) {
      char* p = at;
      at += n;
      return p;
    };
    char* dz = take(l.dz_bytes);
    char* x_new = take(l.x_bytes);
    char* w_new = take(l.w_bytes);
    float* sum = reinterpret_cast<float*>(take(l.sum_bytes));
    float* partial = reinterpret_cast<float*>(take(l.partial_bytes));
    float* unit = l.unit_bytes ? reinterpret_cast<float*>(take(l.unit_bytes)) : nullptr;
    auto pack = [&](const void* from, int64_t rows, int64_t cols, int64_t ld, char* to, int64_t ld_to, int times) {
      PackArgs a{};
      a.n = times;
      for (int i = 0; i < times; ++i) {
        a.from[i] = from;
        a.to[i] = to + i * rows * ld_to * l.e;
        a.rows[i] = rows;
        a.cols[i] = (int32_t)cols;
        a.ld_from[i] = ld;
        a.ld_to[i] = ld_to;
      }
      check_hip(pack_rows(d.type, a, st), "layout");
    };
    const bool twice = l.held > d.rows;
    if (unit) check_hip(units(dloss, labels, d.rows, twice, unit, st), "unit");
    const int64_t ld_new = line_ld(l.e, d.inputs);
    if (l.pack_x) pack(x, d.rows, d.inputs, d.ld_x, x_new, ld_new, twice && dw ? 2 : 1);
    const void* px = l.pack_x ? x_new : x;
    for (int64_t i = 0; i < l.pieces; ++i) {
      const bool end = i == l.pieces - 1;
      const Piece& p = end ? l.last : l.whole;
      const int64_t first = i * l.piece;
      auto classes_from = [&](void* v) { return v ? static_cast<char*>(v) + first * l.e : nullptr; };
      const void* pw = classes_from(const_cast<void*>(w));
      if (l.pack_w) {
        pack(pw, d.inputs, p.count, d.ld_w, w_new, line_ld(l.e, p.count), 1);
        pw = w_new;
      }
      OpEpilogueMore epi{};
      epi.bias[0] = classes_from(const_cast<void*>(bias));
      epi.labels = labels;
      epi.lse = lse;
      epi.dloss = dloss;
      epi.unit = unit;
      epi.class0 = (int32_t)first;
      epi.classes = (int32_t)p.count;
      epi.all_classes = (int32_t)d.classes;
      epi.out[0] = dz;
      epi.ld_out = l.ld_dz;
      epi.rest_rows = twice ? (int32_t)d.rows : 0;
      product(d.type, p.z, &px, &pw, epi, at, st, "dz");
      if (db) check_hip(sum_columns(d.type, dz, l.ld_dz, l.held, p.count, unit, partial, classes_from(db), st), "db");
      const void* pz = dz;
      if (dx) {
        OpEpilogueMore o{};
        o.unit = unit;
        o.out[0] = dx;
        o.ld_out = d.ld_dx;
        o.add = i > 0 ? sum : nullptr;
        o.sum = end && !twice ? nullptr : sum;
        o.ld_sum = d.inputs;
        product(d.type, p.dx, &pz, &pw, o, at, st, "dx");
        if (end && twice) {
          const dim3 grid((unsigned)((d.rows * ((d.inputs + 3) / 4) + 255) / 256));
          check_hip(d.type == VOLTA_OP_BF16
                        ? op_launch(add_halves<__bf16>, grid, dim3(256), st, static_cast<const float*>(sum), d.rows,
                                    d.inputs, static_cast<const float*>(unit), static_cast<__bf16*>(dx), d.ld_dx)
                        : op_launch(add_halves<_Float16>, grid, dim3(256), st, static_cast<const float*>(sum), d.rows,
                                    d.inputs, static_cast<const float*>(unit), static_cast<_Float16*>(dx), d.ld_dx),
                    "dx");
        }
      }
      if (dw) {
        OpEpilogue o{};
        o.unit = unit;
        o.out[0] = classes_from(dw);
        o.ld_out = d.ld_dw;
        product(d.type, p.dw, &px, &pz, o, at, st, "dw");
      }
    }
  });
}

}  // extern "C"
