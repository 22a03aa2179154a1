// e4m3 codes of matrices, and the linear layer of such codes
// (include/volta_ops.h): entry points and the quantization's kernels.  The
// product's are in ops_gemm8_kernels.h.
#include "ops_call.h"
#include "ops_codes.h"
#include "ops_launch.h"

namespace volta {
namespace ops {
namespace {

struct QuantizeArgs {
  const void* x;
  uint8_t* y;
  float* scales;
  int64_t rows, ld_x, ld_y;
  int32_t cols, groups;  // groups of 128: of a row's columns (ROWS), of rows (BLOCKS)
};

// ROWS: a thread for 16 bytes of a row, a group's 16 or 32 lanes side by side.
// Bound by memory, each element read and each code written once: 8192 x 4096
// bfloat16 20.9 us, 4.9 TB/s, and float32 29.0, 5.8.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows(QuantizeArgs a) {
  constexpr int E = 16 / (int)sizeof(T), LANES = 128 / E;
  const int64_t id = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
  const int64_t row = id / a.groups;
  if (row >= a.rows) return;  // all lanes of a group
  const int group = (int)(id - row * a.groups), c = group * 128 + threadIdx.x % LANES * E, cnt = a.cols - c;
  float v[E], m = 0.0f;
  load_vec(static_cast<const T*>(a.x) + row * a.ld_x + c, cnt, v);
#pragma unroll
  for (int i = 0; i < E; ++i) m = max_or_nan(m, fabsf(v[i]));
#pragma unroll
  for (int off = LANES / 2; off >= 1; off >>= 1) m = max_or_nan(m, __shfl_xor(m, off, kWave));
  const float scale = scale_of(m), inv = 1.0f / scale;
  if (threadIdx.x % LANES == 0) a.scales[id] = scale;
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] *= inv;
  store_codes<E>(a.y + row * a.ld_y + c, cnt, v);
}

// BLOCKS: a block of threads for 128 rows (k) and 128 columns (n) of x.  A
// thread has eight columns of eight rows, four after another twice, so that
// the codes of four k of a column are one word of the transposed tile in LDS
// (rows of 33 words: the reads of 16 bytes of a row meet every bank), from where
// a thread writes 16 bytes of a row of y.  Bound by memory: 4096 x 16384 bfloat16
// 43.5 us, 4.6 TB/s, and float32 63.3, 5.3.
template <typename T>
__global__ void __launch_bounds__(256) quantize_blocks(QuantizeArgs a) {
  __shared__ uint32_t codes[128][33];
  __shared__ float largest[4];
  const int tid = threadIdx.x, nc = tid & 15, kq = tid >> 4;
  const int64_t id = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int nb = (int)(id / a.groups);
  if (nb * 128 >= a.cols) return;  // the whole block
  const int64_t k0 = (id - (int64_t)nb * a.groups) * 128;
  const int n = nb * 128 + nc * 8, cnt = a.cols - n;
  const T* x = static_cast<const T*>(a.x);
  float v[2][4][8], m = 0.0f;
  if (k0 + 128 <= a.rows && nb * 128 + 128 <= a.cols) {  // no branch between the loads
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) load_vec(x + (k0 + (h * 16 + kq) * 4 + r) * a.ld_x + n, 8, v[h][r]);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t k = k0 + (h * 16 + kq) * 4 + r;
        load_vec(x + (k < a.rows ? k * a.ld_x + n : 0), k < a.rows ? cnt : 0, v[h][r]);
      }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_or_nan(m, fabsf(v[h][r][i]));
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = max_or_nan(m, __shfl_xor(m, off, kWave));
  if ((tid & 63) == 0) largest[tid >> 6] = m;
  __syncthreads();
  m = largest[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) m = max_or_nan(m, largest[w]);
  const float scale = scale_of(m), inv = 1.0f / scale;
  if (tid == 0) a.scales[id] = scale;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[h][0][i] * inv, v[h][1][i] * inv, 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(v[h][2][i] * inv, v[h][3][i] * inv, w, true);
      codes[nc * 8 + i][h * 16 + kq] = (uint32_t)w;
    }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int row = t * 32 + (tid >> 3), c = tid & 7;
    const int64_t k = k0 + c * 16;
    if (nb * 128 + row >= a.cols || k >= a.rows) continue;
    uint8_t* to = a.y + (int64_t)(nb * 128 + row) * a.ld_y + k;
    union { chunk16 v; uint8_t b[16]; } u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u.v[i] = codes[row][c * 4 + i];
    if (k + 16 <= a.rows) {
      *(VOLTA_GLOBAL Access<16, 1>::type*)to = u.v;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k + i < a.rows) ((VOLTA_GLOBAL uint8_t*)to)[i] = u.b[i];
    }
  }
}

hipError_t quantize(int type, bool blocks, const QuantizeArgs& a, hipStream_t st) {
  const int per = blocks ? 1 : type == VOLTA_OP_F32 ? 8 : 16;  // groups of a block of threads
  const int64_t groups = blocks ? (int64_t)a.groups * ((a.cols + 127) / 128) : a.rows * a.groups;
  const int64_t n = (groups + per - 1) / per, x = std::min<int64_t>(n, int64_t{1} << 20);
  if (n == 0) return hipSuccess;
  const dim3 grid((unsigned)x, (unsigned)((n + x - 1) / x));
  auto run = [&](auto like) {
    using T = decltype(like);
    return op_launch(blocks ? quantize_blocks<T> : quantize_rows<T>, grid, dim3(256), st, a);
  };
  return type == VOLTA_OP_F32    ? run(0.0f)
         : type == VOLTA_OP_BF16 ? run((__bf16)0.0f)
                                 : run((_Float16)0.0f);
}

// The rows' scales by blocks of k: [blocks][rows] of [rows][blocks].  A stage of a
// product loads one block's for its rows, side by side so, and else each from a
// cache line of its own, which costs the large tile as much as a sixth of its
// operands.  8192 rows of 32: 5 us, the launch.
__global__ void __launch_bounds__(256) turn_scales(const float* from, float* to, int64_t rows, int64_t rows_p, int blocks) {
  __shared__ float lds[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, b0 = blockIdx.y * 32;
  for (int64_t r0 = (int64_t)blockIdx.x * 32; r0 < rows; r0 += (int64_t)gridDim.x * 32) {
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      const int64_t r = r0 + y + i;
      if (r < rows && b0 + x < blocks) lds[y + i][x] = from[r * blocks + b0 + x];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32; i += 8)
      if (b0 + y + i < blocks && r0 + x < rows) to[(b0 + y + i) * rows_p + r0 + x] = lds[x][y + i];
    __syncthreads();
  }
}

struct Linear8 {
  volta_op_linear8 d;
  int64_t blocks, x_groups;  // of 128 inputs; scales of a row of x
  Shape fwd;
  int64_t turned_bytes;  // of the rows' scales by blocks, where that pays
  int64_t rows_p;
  int64_t bytes() const { return turned_bytes + fwd.bytes(); }
};
Linear8 linear8_of(const volta_op_linear8* in) {
  need(in, "the description");
  Linear8 l{};
  volta_op_linear8& d = l.d;
  d = *in;
  check_type(d.type);
  check_act(d.act);
  check_dims("rows", d.rows, 0, kMaxRows);
  check_dims("inputs", d.inputs, 1, kMaxLd);
  check_dims("outputs", d.outputs, 1, kMaxLd);
  if (d.group != 0 && d.group != 128) refuse("group is " + std::to_string(d.group) + ", must be 0 or 128");
  d.ld_x = ld_of("ld_x", d.ld_x, d.inputs);
  d.ld_w = ld_of("ld_w", d.ld_w, d.inputs);
  d.ld_y = ld_of("ld_y", d.ld_y, d.outputs);
  d.ld_residual = ld_of("ld_residual", d.ld_residual, d.outputs);
  l.blocks = (d.inputs + 127) / 128;
  l.x_groups = d.group ? l.blocks : 1;
  const Operand x{d.rows, d.inputs, d.ld_x, 1}, w{d.outputs, d.inputs, d.ld_w, 1};
  l.fwd = shape_of(VOLTA_OP_E4M3, OP_NT, OP_LINEAR, d.rows, d.outputs, d.inputs, 1, 1, x, w);
  // A launch of 3 us and two passes over the scales, for less time of every stage:
  // for products of some size and many blocks of k.  (The plan's times are made of
  // constants of 16-bit products; those of codes take 1.1 to 2.2 times them.)  In
  // us, turned and not, rows x inputs x outputs to bfloat16 and to float32:
  //   2048 x 4096 x 4096     41  44    64  64      8192 x 512 x 4096    50  48    65  62
  //   4096 x 4096 x 4096     70  70   120 124      4096 x 512 x 16384   92  90   122 118
  //   1024 x 16384 x 4096    81  87   131 133      8192 x 1024 x 8192  117 115   168 165
  //   8192 x 4096 x 16384   533 589   930 987      1024 x 4096 x 4096   28  28    42  39
  const OpPlan plan = plan_of(VOLTA_OP_E4M3, l.fwd, true);
  l.rows_p = (d.rows + 31) / 32 * 32;
  if (l.x_groups >= 16 && plan.tile <= OP_TILE_128 && plan.us >= 30.0) l.turned_bytes = align256(4 * l.rows_p * l.blocks);
  return l;
}

}  // namespace
}  // namespace ops
}  // namespace volta

using namespace volta;
using namespace volta::ops;

extern "C" {

int32_t volta_op_quantize_forward(const volta_op_quantize* in, const void* x, void* y, float* scales, void* stream) {
  return guarded("volta_op_quantize_forward", [&] {
    need(in, "the description");
    volta_op_quantize d = *in;
    check_type(d.type);
    if (d.groups != VOLTA_OP_ROWS && d.groups != VOLTA_OP_BLOCKS)
      refuse("groups is " + std::to_string(d.groups) + ", must be rows (0) or blocks (1)");
    const bool blocks = d.groups == VOLTA_OP_BLOCKS;
    check_dims("rows", d.rows, 0, blocks ? kMaxLd : kMaxRows);
    check_dims("cols", d.cols, 1, kMaxLd);
    d.ld_x = ld_of("ld_x", d.ld_x, d.cols);
    d.ld_y = ld_of("ld_y", d.ld_y, blocks ? d.rows : d.cols);
    const int64_t across = (d.cols + 127) / 128, down = (d.rows + 127) / 128;
    if (d.rows > 0) {
      need(x, "x");
      need(y, "y");
      need(scales, "scales");
    }
    const Mat my = blocks ? Mat{"y", y, d.rows > 0 ? d.cols : 0, d.rows, d.ld_y, 1, true}
                          : Mat{"y", y, d.rows, d.cols, d.ld_y, 1, true};
    const Mat ms = blocks ? Mat{"scales", scales, d.rows > 0 ? across : 0, down, down, 4, true}
                          : Mat{"scales", scales, d.rows, across, across, 4, true};
    const hipStream_t st = check_call({{"x", x, d.rows, d.cols, d.ld_x, elem_bytes(d.type), false}, my, ms}, {}, nullptr,
                                      0, stream);
    QuantizeArgs a{};
    a.x = x;
    a.y = static_cast<uint8_t*>(y);
    a.scales = scales;
    a.rows = d.rows;
    a.cols = (int32_t)d.cols;
    a.groups = (int32_t)(blocks ? down : across);
    a.ld_x = d.ld_x;
    a.ld_y = d.ld_y;
    check_hip(quantize(d.type, blocks, a, st), "quantization");
  });
}

int64_t volta_op_linear8_workspace(const volta_op_linear8* d) {
  return bytes_of("volta_op_linear8_workspace", VOLTA_OP_FORWARD, [&](bool) { return linear8_of(d).bytes(); });
}

int32_t volta_op_linear8_forward(const volta_op_linear8* in, const void* x, const float* x_scales, const void* w,
                                 const float* w_scales, const void* bias, const void* residual, void* y,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded("volta_op_linear8_forward", [&] {
    const Linear8 l = linear8_of(in);
    const volta_op_linear8& d = l.d;
    const int e = elem_bytes(d.type);
    if (d.rows > 0) {
      need(x, "x");
      need(x_scales, "x_scales");
      need(y, "y");
    }
    need(w, "w");
    need(w_scales, "w_scales");
    const int64_t bytes = l.bytes();
    check_workspace(workspace, workspace_bytes, bytes);
    const hipStream_t st = check_call({{"x", x, d.rows, d.inputs, d.ld_x, 1, false},
                                       {"x_scales", x_scales, d.rows, l.x_groups, l.x_groups, 4, false},
                                       {"w", w, d.outputs, d.inputs, d.ld_w, 1, false},
                                       {"w_scales", w_scales, (d.outputs + 127) / 128, l.blocks, l.blocks, 4, false},
                                       {"bias", bias, 1, d.outputs, d.outputs, e, false},
                                       {"residual", residual, d.rows, d.outputs, d.ld_residual, e, false},
                                       {"y", y, d.rows, d.outputs, d.ld_y, e, true}},
                                      {{"residual", "y"}}, workspace, bytes, stream);
    OpEpilogueMore epi{};
    epi.act = d.act;
    epi.out_type = d.type;
    epi.bias[0] = bias;
    epi.residual = residual;
    epi.out[0] = y;
    epi.ld_out = d.ld_y;
    epi.ld_residual = d.ld_residual;
    epi.sx = x_scales;
    epi.sw = w_scales;
    epi.ld_sx = l.x_groups;
    epi.step_sx = d.group ? 1 : 0;
    epi.ld_sw = l.blocks;
    char* ws = static_cast<char*>(workspace);
    if (l.turned_bytes && d.rows > 0) {
      float* to = reinterpret_cast<float*>(ws);
      const dim3 grid((unsigned)std::min<int64_t>(l.rows_p / 32, 1 << 16), (unsigned)((l.blocks + 31) / 32));
      check_hip(op_launch(turn_scales, grid, dim3(256), st, x_scales, to, d.rows, l.rows_p, (int)l.blocks), "scales");
      epi.sx = to;
      epi.ld_sx = 1;
      epi.step_sx = l.rows_p;
    }
    product(VOLTA_OP_E4M3, l.fwd, &x, &w, epi, ws + l.turned_bytes, st, "product");
  });
}

}  // extern "C"
