// What every entry point of the operators on device tensors shares: argument
// checks, workspaces, and a product with its operands laid out anew where that
// pays.  Included by the files that define entry points (ops.hip, ops_loss.hip,
// ops_muon.hip, ops_eight.hip); nothing here keeps state between calls.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
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

struct Shared {  // the names of two matrices of a call that may be the same one
  const char *a, *b;
  bool is(const Mat& x, const Mat& y) const { return std::strcmp(a, x.name) == 0 && std::strcmp(b, y.name) == 0; }
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
        if ((s.is(a, b) || s.is(b, a)) && a.p == b.p && a.ld == b.ld && a.cols == b.cols && a.bytes == b.bytes)
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
hipError_t gemm(int type, int layout, int kind, const OpPlan& plan, const OpGemmMore& g, hipStream_t st) {
  if (type == VOLTA_OP_E4M3)
    return g.epi.out_type == VOLTA_OP_F32    ? op_gemm8_f32(plan, g, st)
           : g.epi.out_type == VOLTA_OP_BF16 ? op_gemm8_bf16(plan, g, st)
                                             : op_gemm8_f16(plan, g, st);
  return type == VOLTA_OP_F32    ? op_gemm_loss_f32(layout, kind, plan, g, st)
         : type == VOLTA_OP_BF16 ? op_gemm_loss_bf16(layout, kind, plan, g, st)
                                 : op_gemm_loss_f16(layout, kind, plan, g, st);
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
// Rows of a matrix of our own: whole cache lines, so that a stage's 128 bytes of
// a row are one (dx of 1000 rows of 10007 classes in float16, with rows of 20016
// bytes: 34.1 us, and 30.0 so).
int64_t line_ld(int elem, int64_t len) {
  const int64_t e = 128 / elem;
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
// different ones), epilogue and workspace.  Returns whether it took the direct
// loads.
template <typename E>
bool product(int type, const Shape& s, const void* const* ps, const void* const* qs, const E& epi,
             char* workspace, hipStream_t st, const char* what) {
  if (s.M == 0 || s.N == 0) return true;
  OpGemmOf<E> g{};
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
  return direct;
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
