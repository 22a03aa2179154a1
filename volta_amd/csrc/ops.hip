// Entry points of the feed-forward operators (include/volta_ops.h): argument
// checks, workspaces, and the launches of a call in order (ops_call.h).
#include "ops_call.h"

namespace volta {
namespace ops {
namespace {

// ---------------------------------------------------------------------------
struct Linear {
  volta_op_linear d;
  Shape fwd, dx, dw;
  int64_t ld_dp, dp_bytes, sums_bytes, unit_bytes;
  int64_t forward_bytes() const { return fwd.bytes(); }
  int64_t backward_bytes() const { return dp_bytes + sums_bytes + unit_bytes + std::max(dx.bytes(), dw.bytes()); }
};

Linear linear_of(const volta_op_linear* in, unsigned run) {
  need(in, "the description");
  Linear l{};
  volta_op_linear& d = l.d;
  d = *in;
  check_type(d.type);
  check_act(d.act);
  check_dims("rows", d.rows, 0, kMaxRows);
  check_dims("inputs", d.inputs, 1, kMaxLd);
  check_dims("outputs", d.outputs, 1, kMaxLd);
  d.ld_x = ld_of("ld_x", d.ld_x, d.inputs);
  d.ld_w = ld_of("ld_w", d.ld_w, d.outputs);
  d.ld_y = ld_of("ld_y", d.ld_y, d.outputs);
  d.ld_residual = ld_of("ld_residual", d.ld_residual, d.outputs);
  d.ld_pre = ld_of("ld_pre", d.ld_pre, d.outputs);
  d.ld_dx = ld_of("ld_dx", d.ld_dx, d.inputs);
  d.ld_dw = ld_of("ld_dw", d.ld_dw, d.outputs);
  // without an activation dp is dy itself
  l.ld_dp = d.act == VOLTA_OP_ACT_NONE ? d.ld_y : packed_ld(d.type, d.outputs);
  l.dp_bytes = d.act == VOLTA_OP_ACT_NONE ? 0 : packed_bytes(d.type, {d.rows, d.outputs, 0, 1});
  const int64_t dp_len = d.act == VOLTA_OP_ACT_NONE ? d.outputs : l.ld_dp;
  const Operand x{d.rows, d.inputs, d.ld_x, 1}, w{d.inputs, d.outputs, d.ld_w, 1}, dp{d.rows, dp_len, l.ld_dp, 1};
  if (run & RUN_FORWARD) l.fwd = shape_of(d.type, OP_NN, OP_LINEAR, d.rows, d.outputs, d.inputs, 1, 1, x, w);
  if (run & RUN_DX) l.dx = shape_of(d.type, OP_NT, OP_STORE, d.rows, d.inputs, d.outputs, 1, 1, dp, w);
  if (run & RUN_DW) l.dw = shape_of(d.type, OP_TN, OP_STORE, d.inputs, d.outputs, d.rows, 1, 1, x, dp);
  l.sums_bytes = align256(4 * act_grad_strips(d.type, d.rows, d.outputs) * d.outputs);
  l.unit_bytes = d.act == VOLTA_OP_ACT_NONE ? 0 : align256(4 * act_grad_units(d.type, d.rows, d.outputs));
  return l;
}

struct Gated {
  volta_op_gated d;
  Shape fwd, dx, dw;
  int64_t ld_d, d_bytes, sums_bytes, unit_bytes;
  int64_t forward_bytes() const { return fwd.bytes(); }
  int64_t backward_bytes() const { return 2 * (d_bytes + sums_bytes) + unit_bytes + std::max(dx.bytes(), dw.bytes()); }
};

Gated gated_of(const volta_op_gated* in, unsigned run) {
  need(in, "the description");
  Gated l{};
  volta_op_gated& d = l.d;
  d = *in;
  check_type(d.type);
  check_act(d.act);
  check_dims("rows", d.rows, 0, kMaxRows);
  check_dims("inputs", d.inputs, 1, kMaxLd);
  check_dims("hidden", d.hidden, 1, kMaxLd);
  d.ld_x = ld_of("ld_x", d.ld_x, d.inputs);
  d.ld_w = ld_of("ld_w", d.ld_w, d.hidden);
  d.ld_h = ld_of("ld_h", d.ld_h, d.hidden);
  d.ld_pre = ld_of("ld_pre", d.ld_pre, d.hidden);
  d.ld_dx = ld_of("ld_dx", d.ld_dx, d.inputs);
  d.ld_dw = ld_of("ld_dw", d.ld_dw, d.hidden);
  l.ld_d = packed_ld(d.type, d.hidden);
  l.d_bytes = packed_bytes(d.type, {d.rows, d.hidden, 0, 1});
  const Operand x{d.rows, d.inputs, d.ld_x, 1}, w{d.inputs, d.hidden, d.ld_w, 2}, dg{d.rows, l.ld_d, l.ld_d, 2};
  if (run & RUN_FORWARD) l.fwd = shape_of(d.type, OP_NN, OP_GATED, d.rows, d.hidden, d.inputs, 1, 1, x, w);
  if (run & RUN_DX) l.dx = shape_of(d.type, OP_NT, OP_STORE, d.rows, d.inputs, d.hidden, 2, 1, dg, w);
  if (run & RUN_DW) l.dw = shape_of(d.type, OP_TN, OP_STORE, d.inputs, d.hidden, d.rows, 1, 2, x, dg);
  l.sums_bytes = align256(4 * act_grad_strips(d.type, d.rows, d.hidden) * d.hidden);
  l.unit_bytes = align256(4 * act_grad_units(d.type, d.rows, d.hidden));
  return l;
}

struct Norm {
  volta_op_rms_norm d;
  int partial_rows;
  int64_t backward_bytes() const { return align256(4 * partial_rows * d.cols); }
};

Norm norm_of(const volta_op_rms_norm* in, bool backward) {
  need(in, "the description");
  Norm n{};
  volta_op_rms_norm& d = n.d;
  d = *in;
  check_type(d.type);
  check_dims("rows", d.rows, 0, kMaxRows);
  check_dims("cols", d.cols, 1, kMaxLd);
  if (!(d.eps >= 0.0f) || !std::isfinite(d.eps)) refuse("eps is negative or not finite");
  if (!backward) {
    if (d.out_type != d.type && d.out_type != VOLTA_OP_E4M3) refuse("out_type must be type or E4M3");
    if (d.group != 0 && (d.out_type != VOLTA_OP_E4M3 || d.group != 128))
      refuse("group is " + std::to_string(d.group) + ", must be 0, or 128 with out_type E4M3");
  }
  d.ld_x = ld_of("ld_x", d.ld_x, d.cols);
  d.ld_residual = ld_of("ld_residual", d.ld_residual, d.cols);
  d.ld_sum = ld_of("ld_sum", d.ld_sum, d.cols);
  d.ld_y = ld_of("ld_y", d.ld_y, d.cols);
  d.ld_dx = ld_of("ld_dx", d.ld_dx, d.cols);
  n.partial_rows = norm_grad_blocks(d.type, d.rows, d.cols);
  return n;
}

}  // namespace
}  // namespace ops
}  // namespace volta

using namespace volta;
using namespace volta::ops;

extern "C" {

int64_t volta_op_linear_workspace(const volta_op_linear* d, int32_t direction) {
  return bytes_of("volta_op_linear_workspace", direction, [&](bool backward) {
    const Linear l = linear_of(d, backward ? RUN_DX | RUN_DW : RUN_FORWARD);
    return backward ? l.backward_bytes() : l.forward_bytes();
  });
}

int32_t volta_op_linear_forward(const volta_op_linear* in, const void* x, const void* w, const void* bias,
                                const void* residual, void* y, void* pre, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  return guarded("volta_op_linear_forward", [&] {
    const Linear l = linear_of(in, RUN_FORWARD);
    const volta_op_linear& d = l.d;
    const int e = elem_bytes(d.type);
    if (d.rows > 0) {
      need(x, "x");
      need(y, "y");
    }
    need(w, "w");
    const Mat mx{"x", x, d.rows, d.inputs, d.ld_x, e, false}, mw{"w", w, d.inputs, d.outputs, d.ld_w, e, false};
    const Mat mb{"bias", bias, 1, d.outputs, d.outputs, e, false};
    const Mat mr{"residual", residual, d.rows, d.outputs, d.ld_residual, e, false};
    const Mat my{"y", y, d.rows, d.outputs, d.ld_y, e, true}, mp{"pre", pre, d.rows, d.outputs, d.ld_pre, e, true};
    check_workspace(workspace, workspace_bytes, l.forward_bytes());
    const hipStream_t st = check_call({mx, mw, mb, mr, my, mp}, {{"residual", "y"}}, workspace, l.forward_bytes(), stream);
    OpEpilogue epi{};
    epi.act = d.act;
    epi.bias[0] = bias;
    epi.residual = residual;
    epi.out[0] = y;
    epi.pre[0] = pre;
    epi.ld_out = d.ld_y;
    epi.ld_residual = d.ld_residual;
    epi.ld_pre = d.ld_pre;
    product(d.type, l.fwd, &x, &w, epi, static_cast<char*>(workspace), st, "product");
  });
}

int32_t volta_op_linear_backward(const volta_op_linear* in, const void* dy, const void* x, const void* w,
                                 const void* pre, void* dx, void* dw, void* db, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  return guarded("volta_op_linear_backward", [&] {
    const Linear l = linear_of(in, (dx ? RUN_DX : 0) | (dw ? RUN_DW : 0));
    const volta_op_linear& d = l.d;
    const int e = elem_bytes(d.type);
    const bool act = d.act != VOLTA_OP_ACT_NONE;
    if (!dx && !dw && !db && d.rows > 0) refuse("dx, dw and db are all NULL");
    if (d.rows > 0) {
      need(dy, "dy");
      if (act) need(pre, "pre");
      if (dw) need(x, "x");
    }
    if (dx) need(w, "w");
    const Mat mdy{"dy", dy, d.rows, d.outputs, d.ld_y, e, false}, mx{"x", x, d.rows, d.inputs, d.ld_x, e, false};
    const Mat mw{"w", w, d.inputs, d.outputs, d.ld_w, e, false};
    const Mat mp{"pre", act ? pre : nullptr, d.rows, d.outputs, d.ld_pre, e, false};
    const Mat mdx{"dx", dx, d.rows, d.inputs, d.ld_dx, e, true}, mdw{"dw", dw, d.inputs, d.outputs, d.ld_dw, e, true};
    const Mat mdb{"db", db, 1, d.outputs, d.outputs, e, true};
    check_workspace(workspace, workspace_bytes, l.backward_bytes());
    const hipStream_t st = check_call({mdy, mx, mw, mp, mdx, mdw, mdb}, {}, workspace, l.backward_bytes(), stream);
    char* ws = static_cast<char*>(workspace);
    float* sums = reinterpret_cast<float*>(ws + l.dp_bytes);
    float* unit = l.unit_bytes && (dx || dw) ? reinterpret_cast<float*>(ws + l.dp_bytes + l.sums_bytes) : nullptr;
    char* rest = ws + l.dp_bytes + l.sums_bytes + l.unit_bytes;
    const void* dp = act ? ws : dy;
    if ((act && (dx || dw) && d.rows > 0) || db) {
      ActGradArgs a{};
      a.dy = dy;
      a.pre[0] = act ? pre : nullptr;
      a.d[0] = act && (dx || dw) ? ws : nullptr;
      a.sums[0] = db;
      a.partial[0] = sums;
      a.unit = unit;
      a.act = d.act;
      a.rows = d.rows;
      a.cols = (int32_t)d.outputs;
      a.ld_dy = d.ld_y;
      a.ld_pre = d.ld_pre;
      a.ld_d = l.ld_dp;
      check_hip(act_grad(d.type, false, a, st), "activation gradient");
    }
    OpEpilogue epi{};
    epi.unit = unit;
    if (dx) {
      epi.out[0] = dx;
      epi.ld_out = d.ld_dx;
      product(d.type, l.dx, &dp, &w, epi, rest, st, "dx");
    }
    if (dw) {
      epi.out[0] = dw;
      epi.ld_out = d.ld_dw;
      product(d.type, l.dw, &x, &dp, epi, rest, st, "dw");
    }
  });
}

int64_t volta_op_gated_workspace(const volta_op_gated* d, int32_t direction) {
  return bytes_of("volta_op_gated_workspace", direction, [&](bool backward) {
    const Gated l = gated_of(d, backward ? RUN_DX | RUN_DW : RUN_FORWARD);
    return backward ? l.backward_bytes() : l.forward_bytes();
  });
}

int32_t volta_op_gated_forward(const volta_op_gated* in, const void* x, const void* w_gate, const void* w_up,
                               const void* b_gate, const void* b_up, void* h, void* gate, void* up, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  return guarded("volta_op_gated_forward", [&] {
    const Gated l = gated_of(in, RUN_FORWARD);
    const volta_op_gated& d = l.d;
    const int e = elem_bytes(d.type);
    if (d.rows > 0) {
      need(x, "x");
      need(h, "h");
    }
    need(w_gate, "w_gate");
    need(w_up, "w_up");
    if (!gate != !up) refuse("gate and up are kept both or neither");
    const Mat mx{"x", x, d.rows, d.inputs, d.ld_x, e, false};
    const Mat mg{"w_gate", w_gate, d.inputs, d.hidden, d.ld_w, e, false};
    const Mat mu{"w_up", w_up, d.inputs, d.hidden, d.ld_w, e, false};
    const Mat bg{"b_gate", b_gate, 1, d.hidden, d.hidden, e, false}, bu{"b_up", b_up, 1, d.hidden, d.hidden, e, false};
    const Mat mh{"h", h, d.rows, d.hidden, d.ld_h, e, true};
    const Mat pg{"gate", gate, d.rows, d.hidden, d.ld_pre, e, true}, pu{"up", up, d.rows, d.hidden, d.ld_pre, e, true};
    check_workspace(workspace, workspace_bytes, l.forward_bytes());
    const hipStream_t st = check_call({mx, mg, mu, bg, bu, mh, pg, pu}, {}, workspace, l.forward_bytes(), stream);
    OpEpilogue epi{};
    epi.act = d.act;
    epi.bias[0] = b_gate;
    epi.bias[1] = b_up;
    epi.out[0] = h;
    epi.pre[0] = gate;
    epi.pre[1] = up;
    epi.ld_out = d.ld_h;
    epi.ld_pre = d.ld_pre;
    const void* w[2] = {w_gate, w_up};
    product(d.type, l.fwd, &x, w, epi, static_cast<char*>(workspace), st, "product");
  });
}

int32_t volta_op_gated_backward(const volta_op_gated* in, const void* dh, const void* x, const void* w_gate,
                                const void* w_up, const void* gate, const void* up, void* dx, void* dw_gate,
                                void* dw_up, void* db_gate, void* db_up, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  return guarded("volta_op_gated_backward", [&] {
    const Gated l = gated_of(in, (dx ? RUN_DX : 0) | (dw_gate ? RUN_DW : 0));
    const volta_op_gated& d = l.d;
    const int e = elem_bytes(d.type);
    if (!dw_gate != !dw_up) refuse("dw_gate and dw_up are wanted both or neither");
    if (!dx && !dw_gate && !db_gate && !db_up && d.rows > 0) refuse("every gradient is NULL");
    if (d.rows > 0) {
      need(dh, "dh");
      need(gate, "gate");
      need(up, "up");
      if (dw_gate) need(x, "x");
    }
    if (dx) {
      need(w_gate, "w_gate");
      need(w_up, "w_up");
    }
    const Mat mdh{"dh", dh, d.rows, d.hidden, d.ld_h, e, false}, mx{"x", x, d.rows, d.inputs, d.ld_x, e, false};
    const Mat mg{"w_gate", w_gate, d.inputs, d.hidden, d.ld_w, e, false};
    const Mat mu{"w_up", w_up, d.inputs, d.hidden, d.ld_w, e, false};
    const Mat pg{"gate", gate, d.rows, d.hidden, d.ld_pre, e, false}, pu{"up", up, d.rows, d.hidden, d.ld_pre, e, false};
    const Mat mdx{"dx", dx, d.rows, d.inputs, d.ld_dx, e, true};
    const Mat wg{"dw_gate", dw_gate, d.inputs, d.hidden, d.ld_dw, e, true};
    const Mat wu{"dw_up", dw_up, d.inputs, d.hidden, d.ld_dw, e, true};
    const Mat bg{"db_gate", db_gate, 1, d.hidden, d.hidden, e, true}, bu{"db_up", db_up, 1, d.hidden, d.hidden, e, true};
    check_workspace(workspace, workspace_bytes, l.backward_bytes());
    const hipStream_t st = check_call({mdh, mx, mg, mu, pg, pu, mdx, wg, wu, bg, bu}, {}, workspace,
                                      l.backward_bytes(), stream);
    char* ws = static_cast<char*>(workspace);
    float* sums[2] = {reinterpret_cast<float*>(ws + 2 * l.d_bytes),
                      reinterpret_cast<float*>(ws + 2 * l.d_bytes + l.sums_bytes)};
    float* unit =
        l.unit_bytes && (dx || dw_gate) ? reinterpret_cast<float*>(ws + 2 * (l.d_bytes + l.sums_bytes)) : nullptr;
    char* rest = ws + 2 * (l.d_bytes + l.sums_bytes) + l.unit_bytes;
    if (d.rows > 0 || db_gate || db_up) {
      ActGradArgs a{};
      a.dy = dh;
      a.pre[0] = gate;
      a.pre[1] = up;
      a.d[0] = ws;
      a.d[1] = ws + l.d_bytes;
      a.sums[0] = db_gate;
      a.sums[1] = db_up;
      a.partial[0] = sums[0];
      a.partial[1] = sums[1];
      a.unit = unit;
      a.act = d.act;
      a.rows = d.rows;
      a.cols = (int32_t)d.hidden;
      a.ld_dy = d.ld_h;
      a.ld_pre = d.ld_pre;
      a.ld_d = l.ld_d;
      check_hip(act_grad(d.type, true, a, st), "activation gradient");
    }
    const void *dgu[2] = {ws, ws + l.d_bytes}, *w[2] = {w_gate, w_up};
    OpEpilogue epi{};
    epi.unit = unit;
    if (dx) {
      epi.out[0] = dx;
      epi.ld_out = d.ld_dx;
      product(d.type, l.dx, dgu, w, epi, rest, st, "dx");
    }
    if (dw_gate) {
      epi.out[0] = dw_gate;
      epi.out[1] = dw_up;
      epi.ld_out = d.ld_dw;
      product(d.type, l.dw, &x, dgu, epi, rest, st, "dw");
    }
  });
}

int64_t volta_op_rms_norm_workspace(const volta_op_rms_norm* d, int32_t direction) {
  return bytes_of("volta_op_rms_norm_workspace", direction, [&](bool backward) {
    const Norm n = norm_of(d, backward);
    return backward ? n.backward_bytes() : (int64_t)0;
  });
}

int32_t volta_op_rms_norm_forward(const volta_op_rms_norm* in, const void* x, const void* residual,
                                  const void* weight, void* y, void* sum, float* rstd, float* scales, void* stream) {
  return guarded("volta_op_rms_norm_forward", [&] {
    const Norm n = norm_of(in, false);
    const volta_op_rms_norm& d = n.d;
    const int e = elem_bytes(d.type);
    const bool e4m3 = d.out_type == VOLTA_OP_E4M3;
    if (d.rows > 0) {
      need(x, "x");
      need(y, "y");
      if (e4m3) need(scales, "scales");
    }
    if (!e4m3 && scales) refuse("scales are of out_type E4M3 alone");
    const int64_t groups = d.group ? (d.cols + d.group - 1) / d.group : 1;
    const hipStream_t st = check_call(
        {{"x", x, d.rows, d.cols, d.ld_x, e, false},
         {"residual", residual, d.rows, d.cols, d.ld_residual, e, false},
         {"weight", weight, 1, d.cols, d.cols, e, false},
         {"y", y, d.rows, d.cols, d.ld_y, elem_bytes(d.out_type), true},
         {"sum", sum, d.rows, d.cols, d.ld_sum, e, true},
         {"rstd", rstd, d.rows, 1, 1, 4, true},
         {"scales", scales, d.rows, groups, groups, 4, true}},
        {{"sum", "x"}, {"sum", "residual"}}, nullptr, 0, stream);
    NormArgs a{};
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.y = y;
    a.sum = sum;
    a.rstd = rstd;
    a.scales = scales;
    a.rows = d.rows;
    a.cols = (int32_t)d.cols;
    a.group = d.group ? d.group : (int32_t)d.cols;
    a.ld_x = d.ld_x;
    a.ld_residual = d.ld_residual;
    a.ld_y = d.ld_y;
    a.ld_sum = d.ld_sum;
    a.eps = d.eps;
    check_hip(norm_forward(d.type, e4m3, a, st), "norm");
  });
}

int32_t volta_op_rms_norm_backward(const volta_op_rms_norm* in, const void* dy, const void* s, const float* rstd,
                                   const void* weight, const void* dsum, void* dx, void* dweight, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  return guarded("volta_op_rms_norm_backward", [&] {
    const Norm n = norm_of(in, true);
    const volta_op_rms_norm& d = n.d;
    const int e = elem_bytes(d.type);
    if (!dx && !dweight && d.rows > 0) refuse("dx and dweight are both NULL");
    if (d.rows > 0) {
      need(dy, "dy");
      need(s, "s");
      need(rstd, "rstd");
    }
    if (dweight) check_workspace(workspace, workspace_bytes, n.backward_bytes());
    const hipStream_t st = check_call(
        {{"dy", dy, d.rows, d.cols, d.ld_y, e, false},
         {"s", s, d.rows, d.cols, d.ld_x, e, false},
         {"rstd", rstd, d.rows, 1, 1, 4, false},
         {"weight", weight, 1, d.cols, d.cols, e, false},
         {"dsum", dsum, d.rows, d.cols, d.ld_sum, e, false},
         {"dx", dx, d.rows, d.cols, d.ld_dx, e, true},
         {"dweight", dweight, 1, d.cols, d.cols, e, true}},
        {{"dsum", "dx"}}, workspace, dweight ? n.backward_bytes() : 0, stream);
    NormGradArgs a{};
    a.dy = dy;
    a.s = s;
    a.weight = weight;
    a.dsum = dsum;
    a.rstd = rstd;
    a.dx = dx;
    a.partial = dweight ? static_cast<float*>(workspace) : nullptr;
    a.rows = d.rows;
    a.cols = (int32_t)d.cols;
    a.ld_dy = d.ld_y;
    a.ld_s = d.ld_x;
    a.ld_dsum = d.ld_sum;
    a.ld_dx = d.ld_dx;
    check_hip(norm_backward(d.type, a, st), "norm gradient");
    if (dweight) {
      const SumArgs s{{a.partial, nullptr}, {dweight, nullptr}, 1, n.partial_rows, d.cols};
      check_hip(sum_partials(d.type, s, st), "weight gradient");
    }
  });
}

int32_t volta_op_dropout_forward(const volta_op_dropout* in, const void* x, const void* residual, void* y,
                                 uint64_t seed, uint64_t offset, void* stream) {
  return guarded("volta_op_dropout_forward", [&] {
    need(in, "the description");
    volta_op_dropout d = *in;
    check_type(d.type);
    check_dims("rows", d.rows, 0, kMaxRows);
    check_dims("cols", d.cols, 1, kMaxLd);
    if (!(d.p >= 0.0 && d.p < 1.0)) refuse("p must be at least 0 and below 1");
    d.ld_x = ld_of("ld_x", d.ld_x, d.cols);
    d.ld_residual = ld_of("ld_residual", d.ld_residual, d.cols);
    d.ld_y = ld_of("ld_y", d.ld_y, d.cols);
    const int e = elem_bytes(d.type);
    if (d.rows > 0) {
      need(x, "x");
      need(y, "y");
    }
    const hipStream_t st = check_call(
        {{"x", x, d.rows, d.cols, d.ld_x, e, false},
         {"residual", residual, d.rows, d.cols, d.ld_residual, e, false},
         {"y", y, d.rows, d.cols, d.ld_y, e, true}},
        {{"x", "y"}, {"residual", "y"}}, nullptr, 0, stream);
    DropoutArgs a{};
    a.x = x;
    a.residual = residual;
    a.y = y;
    a.rows = d.rows;
    a.cols = d.cols;
    a.ld_x = d.ld_x;
    a.ld_residual = d.ld_residual;
    a.ld_y = d.ld_y;
    a.seed = seed;
    a.offset = offset;
    a.threshold = (uint32_t)(d.p * 4294967296.0);
    a.scale = (float)(1.0 / (1.0 - d.p));
    check_hip(dropout_forward(d.type, a, st), "dropout");
  });
}

}  // extern "C"
