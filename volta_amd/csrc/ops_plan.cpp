// Which tile a product of the feed-forward operators takes (ops_gemm.h), and
// over how many blocks its sum over k is split.  Host code without a device.
#include <algorithm>
#include <cstdint>

#include "ops_gemm.h"

namespace volta {
namespace ops {
namespace {

constexpr int64_t kCus = 256;  // of an MI355X

struct TileCost {
  int bm, bn;        // rows and columns of D
  int resident;      // blocks a CU holds
  double rate16, rate32;  // share of the matrix rate that a full CU reaches
};
// Measured on large products (bf16, float32).
constexpr TileCost kTiles[5] = {
    {256, 256, 1, 0.50, 0.85}, {128, 128, 2, 0.40, 0.85}, {64, 64, 4, 0.22, 0.75}, {64, 32, 1, 1, 1}, {64, 128, 1, .3, .8}};
constexpr double kCuFlops16 = 9.8e6, kCuFlops32 = 0.61e6;  // of one CU in a microsecond
constexpr double kStageUs = 0.6;                           // a stage's loads, when nothing else hides them
constexpr double kReduceUs = 4.0, kReduceBytesPerUs = 3e6; // the launch that adds the partial sums

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

OpPlan op_gemm_plan(int elem_bytes, int layout, int kind, int64_t M, int64_t N, int64_t K, int pieces, int outputs,
                    bool direct) {
  const int64_t stages = pieces * ceil_div(K, op_stage_k(elem_bytes));
  const int planes = kind == OP_GATED ? 2 : outputs;
  OpPlan best{OP_TILE_128, 1, (int32_t)stages};
  if (stages == 0 || M == 0) return best;
  auto split_plan = [&](int tile, int64_t splits) {
    const int64_t per = ceil_div(stages, splits);
    return OpPlan{tile, (int32_t)ceil_div(stages, per), (int32_t)per};
  };
  if (M <= 64 && layout != OP_TN) {
    // A block's waves share its stages out; with few column blocks the sum is
    // split over blocks too, as long as every wave keeps four stages.
    const int64_t blocks = ceil_div(N, 32), waves = kind == OP_GATED || M > 16 ? 4 : 8;
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(128 / blocks, stages / (4 * waves)));
    return split_plan(OP_TILE_SKINNY, splits);
  }
  const double cu = elem_bytes == 4 ? kCuFlops32 : kCuFlops16;
  double best_us = 1e30;
  for (int t = 0; t < 3; ++t) {
    const TileCost& c = kTiles[t];
    if (c.bm == 256 && (!direct || elem_bytes == 4)) continue;
    const int64_t sn = kind == OP_GATED ? c.bn / 2 : c.bn;
    const int64_t tiles = ceil_div(M, c.bm) * ceil_div(N, sn) * outputs;
    const double stage_us = 2.0 * c.bm * c.bn * op_stage_k(elem_bytes) / (cu * (elem_bytes == 4 ? c.rate32 : c.rate16));
    for (int64_t splits = 1; splits <= 64 && splits <= std::max<int64_t>(1, stages / 2); splits *= 2) {
      const OpPlan p = split_plan(t, splits);
      const int64_t blocks = tiles * p.splits, room = kCus * c.resident;
      const int64_t rounds = blocks / room, rest = ceil_div(blocks - rounds * room, kCus);
      // a full CU works at its rate; a part-full one at least as fast as its loads come
      const double full = std::max(c.resident * stage_us, kStageUs);
      const double part = rest == 0 ? 0.0 : std::max(rest * stage_us, kStageUs);
      double us = p.stages_per_split * (rounds * full + part) + (rounds + (rest > 0)) * 1.5;
      if (p.splits > 1) us += kReduceUs + 8.0 * p.splits * planes * (double)M * (double)N / kReduceBytesPerUs;
      if (us < best_us) {
        best_us = us;
        best = p;
      }
    }
  }
  return best;
}

int64_t op_gemm_partial_bytes(const OpPlan& plan, int kind, int64_t M, int64_t N, int outputs) {
  if (plan.splits <= 1) return 0;
  const int64_t planes = kind == OP_GATED ? 2 : outputs;
  return 4 * plan.splits * planes * M * N;
}

int64_t op_gemm_blocks(const OpPlan& plan, int kind, int64_t M, int64_t N) {
  if (plan.tile == OP_TILE_SKINNY) return ceil_div(N, 32);
  const TileCost& c = kTiles[plan.tile];
  return ceil_div(M, c.bm) * ceil_div(N, kind == OP_GATED ? c.bn / 2 : c.bn);
}

}  // namespace ops
}  // namespace volta
