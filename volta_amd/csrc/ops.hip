// Entry points of the feed-forward operators (include/volta_ops.h): argument
// checks, workspaces, and the launches of a call in order.  Nothing here
// keeps state between calls.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <initializer_list>
#include <string>

#include "../../include/volta_ops.h"
#include "../../include/volta_train.h"
#include "ops_gemm.h"
#include "ops_rows.h"
#include "rt_lower.h"

namespace volta {
namespace ops {
namespace {

constexpr int64_t kMaxLd = int64_t{1} << 21;
constexpr int64_t kMaxRows = int64_t{1} << 30;
constexpr int64_t kMaxBlocks = int64_t{1} << 22;  // a dimension of a grid has fewer than 2^32 threads

struct Refused {
  std::string what;
};
[[noreturn]] void refuse(const std::string& m) { throw Refused{m}; }

int elem_bytes(int type) { return type == VOLTA_OP_F32 ? 4 : type == VOLTA_OP_E4M3 ? 1 : 2; }
int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// Runs a call's body; every way it can end becomes the entry point's return.
template <typename F>
int32_t guarded(const char* call, F body) {
  try {
    body();
    return 0;
  } catch (const Refused& r) {
    try { rt_set_error(std::string(call) + ": " + r.what); } catch (...) {}
  } catch (const std::exception& e) {
    try { rt_set_error(std::string(call) + ": " + e.what()); } catch (...) {}
  } catch (...) {
  }
  return -1;
}

void check_hip(hipError_t e, const char* what) {
  if (e != hipSuccess) refuse(std::string(what) + " launch failed: " + hipGetErrorString(e));
}

// A matrix of a call: `rows` x `cols` elements of `bytes`, `ld` apart.
struct Mat {
  const char* name;
  const void* p;
  int64_t rows, cols, ld;
  int bytes;
  bool out;
  int64_t span() const { return p && rows > 0 ? ((rows - 1) * ld + cols) * bytes : 0; }
};

void check_dims(const char* what, int64_t n, int64_t lo, int64_t hi) {
  if (n < lo || n > hi)
    refuse(std::string(what) + " is " + std::to_string(n) + ", must be " + std::to_string(lo) + " to " +
           std::to_string(hi));
}
int64_t ld_of(const char* what, int64_t ld, int64_t cols) {
  if (ld == 0) ld = cols;
  if (ld < cols || ld > kMaxLd)
    refuse(std::string(what) + " is " + std::to_string(ld) + ", must be " + std::to_string(cols) + " to " +
           std::to_string(kMaxLd) + " (0: packed)");
  return ld;
}
void check_type(int type) {
  if (type != VOLTA_OP_F32 && type != VOLTA_OP_BF16 && type != VOLTA_OP_F16)
    refuse("type is " + std::to_string(type) + ", must be F32, BF16 or F16");
}
void check_act(int act) {
  if (act != VOLTA_OP_ACT_NONE && (act < VOLTA_ACT_RELU || act > VOLTA_ACT_GELU))
    refuse("act is " + std::to_string(act) + ", must be none (-1) or relu .. gelu (0 .. 5)");
}

struct Shared {  // two matrices of a call that may be the same one
  const void *a, *b;
};

// Alignment of every pointer, and no output over anything else but where
// `same` allows the two to be one matrix.
void check_mats(std::initializer_list<Mat> list, std::initializer_list<Shared> same, const void* workspace,
                int64_t workspace_bytes) {
  const Mat* mats = list.begin();
  for (const Mat& m : list)
    if (m.p && (uintptr_t)m.p % m.bytes != 0) refuse(std::string(m.name) + " is not aligned to its element");
  auto meet = [](const void* p, int64_t n, const void* q, int64_t k) {
    const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
    return n > 0 && k > 0 && a < b + (uintptr_t)k && b < a + (uintptr_t)n;
  };
  // Column ranges of one wider matrix: the later one starts behind the
  // earlier one's columns and ends before its next row.
  auto beside = [](const Mat& a, const Mat& b) {
    const Mat &lo = (uintptr_t)a.p <= (uintptr_t)b.p ? a : b, &hi = &lo == &a ? b : a;
    const int64_t apart = (int64_t)((uintptr_t)hi.p - (uintptr_t)lo.p);
    if (a.ld != b.ld || a.bytes != b.bytes || apart % a.bytes != 0) return false;
    const int64_t col = apart / a.bytes % a.ld;
    return col >= lo.cols && col + hi.cols <= a.ld;
  };
  for (size_t i = 0; i < list.size(); ++i) {
    for (size_t j = i + 1; j < list.size(); ++j) {
      const Mat &a = mats[i], &b = mats[j];
      if (!a.out && !b.out) continue;
      if (!meet(a.p, a.span(), b.p, b.span()) || beside(a, b)) continue;
      bool ok = false;
      for (const Shared& s : same)
        if (((s.a == a.p && s.b == b.p) || (s.a == b.p && s.b == a.p)) && a.p == b.p && a.ld == b.ld &&
            a.cols == b.cols && a.bytes == b.bytes)
          ok = true;
      if (!ok) refuse(std::string(a.name) + " and " + b.name + " overlap");
    }
    if (meet(mats[i].p, mats[i].span(), workspace, workspace_bytes))
      refuse(std::string(mats[i].name) + " overlaps the workspace");
  }
}
// Memory of another device or of the host's own, and addresses behind the end
// of all memory, would be a fault of the GPU.  A lookup takes 70 ns, so what an
// allocation covers that this call has looked up already is not looked up again
// (small tensors of one pool often share one).
struct Allocation {
  uintptr_t from, to;
};
struct Known {
  Allocation seen[8];
  int n = 0;
  bool covers(uintptr_t from, uintptr_t to) const {
    for (int i = 0; i < n; ++i)
      if (seen[i].from <= from && to <= seen[i].to) return true;
    return false;
  }
  void add(const Allocation& a) {
    if (n < 8) seen[n++] = a;
  }
};
// The allocation at `at`, or false where the runtime does not say.
bool allocation_of(uintptr_t at, Allocation* a) {
  hipDeviceptr_t base = nullptr;
  size_t bytes = 0;
  if (hipMemGetAddressRange(&base, &bytes, reinterpret_cast<hipDeviceptr_t>(at)) != hipSuccess) {
    (void)hipGetLastError();
    return false;
  }
  *a = {(uintptr_t)base, (uintptr_t)base + bytes};
  return a->from <= at && at < a->to;
}
void check_memory(const char* name, const void* p, int64_t bytes, int device, Known* known) {
  uintptr_t at = (uintptr_t)p;
  const uintptr_t end = at + (uintptr_t)bytes;
  if (known->covers(at, end)) return;
  // one allocation after another: memory that was mapped piece by piece lies side by side
  for (bool first = true; at < end; first = false) {
    hipPointerAttribute_t attr{};
    if (hipPointerGetAttributes(&attr, reinterpret_cast<const void*>(at)) != hipSuccess ||
        attr.type == hipMemoryTypeUnregistered) {
      (void)hipGetLastError();
      if (first) refuse(std::string(name) + " is not memory that the device reads");
      refuse(std::string(name) + " ends " + std::to_string(end - at) + " bytes behind the end of its memory");
    }
    if (attr.type == hipMemoryTypeDevice && attr.device != device)
      refuse(std::string(name) + " is of device " + std::to_string(attr.device) + ", the current device is " +
             std::to_string(device));
    // the ends of other kinds of memory (pinned, managed) are not looked up
    Allocation a;
    if (attr.type != hipMemoryTypeDevice || !allocation_of(at, &a)) return;
    known->add(a);
    at = a.to;
  }
}

// A lookup that has to succeed; its error is in the message, and not left for
// the caller's next hipGetLastError.
void look_up(hipError_t e, const char* what) {
  if (e == hipSuccess) return;
  (void)hipGetLastError();
  refuse(std::string(what) + ": " + hipGetErrorString(e));
}

// What every call checks of its matrices, workspace and stream.
hipStream_t check_call(std::initializer_list<Mat> mats, std::initializer_list<Shared> same, const void* workspace,
                       int64_t workspace_bytes, void* stream) {
  check_mats(mats, same, workspace, workspace_bytes);
  int device = 0;
  look_up(hipGetDevice(&device), "the current device");
  // NULL and the runtime's two named streams are the current device's
  if ((uintptr_t)stream > 2) {
    hipDevice_t of = 0;
    look_up(hipStreamGetDevice(static_cast<hipStream_t>(stream), &of), "the stream's device");
    if (of != device)
      refuse("the stream is of device " + std::to_string(of) + ", the current device is " + std::to_string(device));
  }
  Known known;
  for (const Mat& m : mats)
    if (m.span() > 0) check_memory(m.name, m.p, m.span(), device, &known);
  if (workspace_bytes > 0) check_memory("the workspace", workspace, workspace_bytes, device, &known);
  return static_cast<hipStream_t>(stream);
}
void need(const void* p, const char* name) {
  if (!p) refuse(std::string(name) + " is NULL");
}
void check_workspace(const void* p, int64_t have, int64_t want) {
  if (want == 0) return;
  if (!p || have < want)
    refuse("the workspace holds " + std::to_string(p ? have : 0) + " bytes, needed are " + std::to_string(want));
  if ((uintptr_t)p % 16 != 0) refuse("the workspace is not 16-byte aligned");
}

hipError_t gemm(int type, int layout, int kind, const OpPlan& plan, const OpGemm& g, hipStream_t st) {
  return type == VOLTA_OP_F32    ? op_gemm_f32(layout, kind, plan, g, st)
         : type == VOLTA_OP_BF16 ? op_gemm_bf16(layout, kind, plan, g, st)
                                 : op_gemm_f16(layout, kind, plan, g, st);
}

// An operand of a product as its description gives it: rows of `len`
// contiguous elements, `ld` apart.
struct Operand {
  int64_t rows, len, ld;
  int count;  // matrices of it
};
bool whole_chunks(int type, const Operand& o) {
  const int64_t e = 16 / elem_bytes(type);
  return o.len % e == 0 && o.ld % e == 0;
}
int64_t packed_ld(int type, int64_t len) {
  const int64_t e = 16 / elem_bytes(type);
  return (len + e - 1) / e * e;
}
int64_t packed_bytes(int type, const Operand& o) {
  return align256(o.rows * packed_ld(type, o.len) * elem_bytes(type));
}

// Which of a layer's products a call runs; the others are not planned, and
// what they would be refused for does not matter.
enum : unsigned { RUN_FORWARD = 1, RUN_DX = 2, RUN_DW = 4 };

// The shape of a product, and what follows for it from the description alone:
// whether operands are laid out anew in rows of whole chunks, and the
// workspace.  (Where a pointer turns out not to be 16-byte aligned, the
// product takes the loads through registers.)
struct Shape {
  int layout, kind;
  int64_t M, N, K;
  int pieces, outputs;
  Operand p, q;
  bool pack_p, pack_q;
  int64_t partial_bytes, pack_bytes;  // partial sums, then the copies
  int64_t blocks;                     // of D's tiles, at most
  // The workspace of a call with this product.
  int64_t bytes() const {
    if (blocks > kMaxBlocks) refuse("the rows and columns of a product are too many");
    return partial_bytes + pack_bytes;
  }
};
OpPlan plan_of(int type, const Shape& s, bool direct) {
  return op_gemm_plan(elem_bytes(type), s.layout, s.kind, s.M, s.N, s.K, s.pieces, s.outputs, direct);
}
Shape shape_of(int type, int layout, int kind, int64_t M, int64_t N, int64_t K, int pieces, int outputs, Operand p,
               Operand q) {
  Shape s{layout, kind, M, N, K, pieces, outputs, p, q, !whole_chunks(type, p), !whole_chunks(type, q), 0, 0, 0};
  if (s.pack_p || s.pack_q) {
    s.pack_bytes = (s.pack_p ? p.count * packed_bytes(type, p) : 0) + (s.pack_q ? q.count * packed_bytes(type, q) : 0);
    if (!op_gemm_pack(elem_bytes(type), layout, kind, M, N, K, pieces, outputs, s.pack_bytes)) {
      s.pack_p = s.pack_q = false;
      s.pack_bytes = 0;
    }
  }
  for (bool direct : {false, true}) {
    const OpPlan plan = plan_of(type, s, direct);
    s.partial_bytes = std::max(s.partial_bytes, align256(op_gemm_partial_bytes(plan, kind, M, N, outputs)));
    s.blocks = std::max(s.blocks, op_gemm_blocks(plan, kind, M, N));
  }
  return s;
}

// One product of a call: its operands' matrices (one, or p.count / q.count
// different ones), epilogue and workspace.
void product(int type, const Shape& s, const void* const* ps, const void* const* qs, const OpEpilogue& epi,
             char* workspace, hipStream_t st, const char* what) {
  if (s.M == 0 || s.N == 0) return;
  OpGemm g{};
  PackArgs pack{};
  char* at = workspace + s.partial_bytes;
  bool direct = true;
  auto operand = [&](const Operand& o, const void* const* from, bool packs, const void** to, int64_t* ld) {
    *ld = packs ? packed_ld(type, o.len) : o.ld;
    for (int i = 0; i < 2; ++i) {
      if (i >= o.count) {
        to[i] = to[0];
        continue;
      }
      to[i] = from[i];
      if (packs) {
        pack.from[pack.n] = from[i];
        pack.to[pack.n] = at;
        pack.rows[pack.n] = o.rows;
        pack.cols[pack.n] = (int32_t)o.len;
        pack.ld_from[pack.n] = o.ld;
        pack.ld_to[pack.n] = *ld;
        ++pack.n;
        to[i] = at;
        at += packed_bytes(type, o);
      }
      direct = direct && (uintptr_t)to[i] % 16 == 0 && (packs || whole_chunks(type, o));
    }
  };
  operand(s.p, ps, s.pack_p, g.p, &g.ld_p);
  operand(s.q, qs, s.pack_q, g.q, &g.ld_q);
  if (pack.n && !direct) {  // one operand would still not do: none is laid out anew
    pack.n = 0;
    for (int i = 0; i < 2; ++i) {
      g.p[i] = ps[std::min(i, s.p.count - 1)];
      g.q[i] = qs[std::min(i, s.q.count - 1)];
    }
    g.ld_p = s.p.ld;
    g.ld_q = s.q.ld;
  }
  g.M = (int32_t)s.M;
  g.N = (int32_t)s.N;
  g.K = (int32_t)s.K;
  g.pieces = s.pieces;
  g.outputs = s.outputs;
  g.direct = direct;
  g.partial = reinterpret_cast<float*>(workspace);
  g.epi = epi;
  const OpPlan plan = plan_of(type, s, direct);
  if (pack.n) check_hip(pack_rows(type, pack, st), "layout");
  check_hip(gemm(type, s.layout, s.kind, plan, g, st), what);
}

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

template <typename F>
int64_t bytes_of(const char* call, int32_t direction, F f) {
  int64_t n = -1;
  guarded(call, [&] {
    if (direction != VOLTA_OP_FORWARD && direction != VOLTA_OP_BACKWARD)
      refuse("direction is " + std::to_string(direction) + ", must be forward (0) or backward (1)");
    n = f(direction == VOLTA_OP_BACKWARD);
  });
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
    const hipStream_t st = check_call({mx, mw, mb, mr, my, mp}, {{residual, y}}, workspace, l.forward_bytes(), stream);
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
    if (!dx && !dw && !db) refuse("dx, dw and db are all NULL");
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
    if (!dx && !dw_gate && !db_gate && !db_up) refuse("every gradient is NULL");
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
        {{sum, x}, {sum, residual}}, nullptr, 0, stream);
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
    if (!dx && !dweight) refuse("dx and dweight are both NULL");
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
        {{dsum, dx}}, workspace, dweight ? n.backward_bytes() : 0, stream);
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
        {{x, y}, {residual, y}}, nullptr, 0, stream);
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
