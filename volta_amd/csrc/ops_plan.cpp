// Which tile a product of the feed-forward operators takes (ops_gemm.h), and
// over how many blocks its sum over k is split: the one of least time by a
// model of a block's time, measured tile by tile.  Host code without a device.
#include <algorithm>
#include <cstdint>

#include "ops_gemm.h"

namespace volta {
namespace ops {
namespace {

constexpr int64_t kCus = 256;  // of an MI355X

// A block's time in microseconds: `fixed` for its start, its first loads and
// its epilogue, and `stage` for 128 bytes of k, or more where the matrix
// instructions of float32 take longer.
struct TileCost {
  int bm, bn;      // rows and columns of D (gated: half the columns of each weight matrix)
  double fixed, stage;
  double flops32;  // float32 flops of a CU in a microsecond
};
// Measured on an MI355X.
constexpr TileCost kTiles[OP_TILES] = {
    {256, 256, 6.0, 0.95, 0.55e6}, {256, 128, 4.4, 0.80, 0.52e6}, {128, 128, 3.2, 0.43, 0.47e6}, {64, 128, 2.4, 0.33, 0.42e6}, {64, 64, 2.2, 0.23, 0.38e6},
    {16, 32, 1.0, 0.0, 0.45e6},    {32, 32, 1.0, 0.0, 0.45e6},    {64, 32, 1.2, 0.0, 0.45e6},
};
constexpr double kPairStage = 0.55;                        // of op_gemm_pairs: a stage of all three products
constexpr double kSkinnyBytes = 80e3;                      // what a CU's waves load in a microsecond
constexpr double kReadBytes = 5.5e6;                       // what the chip reads in a microsecond
constexpr double kLaunchUs = 2.2;                          // of a launch, whatever it does
constexpr double kReduceUs = 5.0, kReduceBytes = 4e6;      // the launch that adds the partial sums
constexpr double kPackUs = 3.0;                            // the launch that lays operands out again, at the same rate

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

OpPlan op_gemm_plan(int elem_bytes, int layout, int kind, int64_t M, int64_t N, int64_t K, int pieces, int outputs,
                    bool direct) {
  const int64_t all_stages = pieces * ceil_div(K, op_stage_k(elem_bytes));
  const int planes = kind == OP_GATED ? 2 : outputs, subs = kind == OP_GATED ? 2 : 1;
  OpPlan best{OP_TILE_128, 1, (int32_t)all_stages, 0.0};
  if (all_stages == 0 || M == 0) return best;
  // every product reads both operands, from memory at the rate of memory
  const double read_us = (double)elem_bytes * pieces * K * ((double)M + (double)subs * N * outputs) / kReadBytes;
  double best_us = 1e30;
  for (int t = 0; t < OP_TILES; ++t) {
    const TileCost& c = kTiles[t];
    const bool skinny = t >= OP_TILE_SKINNY16;
    if (skinny && (layout == OP_TN || op_kind_blend(kind) || M > 512)) continue;
    if (kind == OP_MIRROR && c.bm != c.bn) continue;
    if (!direct && (t == OP_TILE_256 || t == OP_TILE_256X128 || t == OP_TILE_64X128)) continue;
    const int64_t sn = skinny ? c.bn : kind == OP_GATED ? c.bn / 2 : c.bn;
    const int64_t side = ceil_div(M, c.bm);
    const int64_t tiles = (kind == OP_MIRROR ? side * (side + 1) / 2 : side * ceil_div(N, sn)) * outputs;
    const int waves = !skinny ? 1 : kind == OP_GATED || c.bm > 16 ? 4 : 8;
    const bool pairs = pieces == 3 && t == OP_TILE_64;  // three products a stage
    const int64_t stages = pairs ? all_stages / 3 : all_stages;
    double stage_us = pairs ? kPairStage : c.stage, tile_read_us = read_us;
    // half cache lines of W: whole ones are fetched (134 MB of W from memory: 40 us in 64-byte pieces, 29 in 128)
    const bool halves = layout == OP_NN && sn * elem_bytes < 128;
    if (halves) tile_read_us *= 1.45;
    if (skinny) stage_us = waves * 128.0 * ((double)sn * subs * (halves ? 1.6 : 1.0) + c.bm) / kSkinnyBytes;  // a turn
    if (elem_bytes == 4)
      stage_us = std::max(stage_us, 2.0 * c.bm * sn * subs * op_stage_k(4) * waves / c.flops32);
    // through registers, one stage ahead
    if (!direct) stage_us = skinny ? 1.1 * stage_us + 0.5 : stage_us * (t == OP_TILE_64 ? 2.0 : 4.0);
    for (int64_t splits = 1; splits <= 32 && (splits == 1 || stages / splits >= 2 * waves); splits *= 2) {
      const int64_t per = ceil_div(stages, splits), used = ceil_div(stages, per);
      const double rounds = (double)ceil_div(tiles * used, kCus);
      double us = kLaunchUs + rounds * c.fixed + std::max(rounds * ceil_div(per, waves) * stage_us, tile_read_us);
      if (used > 1) us += kReduceUs + 8.0 * used * planes * (double)M * (double)N / kReduceBytes;
      if (us < best_us * (splits > 1 ? 0.93 : 1.0)) {
        best_us = us;
        best = OpPlan{t, (int32_t)used, (int32_t)per, us};
      }
    }
  }
  return best;
}

bool op_gemm_pack(int elem_bytes, int layout, int kind, int64_t M, int64_t N, int64_t K, int pieces, int outputs,
                  int64_t pack_bytes) {
  const double staged = op_gemm_plan(elem_bytes, layout, kind, M, N, K, pieces, outputs, false).us;
  const double direct = op_gemm_plan(elem_bytes, layout, kind, M, N, K, pieces, outputs, true).us;
  return direct + kPackUs + 2.0 * (double)pack_bytes / kReduceBytes < staged;
}

int64_t op_gemm_partial_bytes(const OpPlan& plan, int kind, int64_t M, int64_t N, int outputs) {
  if (plan.splits <= 1) return 0;
  const int64_t planes = kind == OP_GATED ? 2 : outputs;
  return 4 * plan.splits * planes * M * N;
}

int64_t op_stats_entries(const OpPlan& plan, int64_t N) {
  // a block's columns; 16 in the skinny tiles, a wave's in the launch that adds the splits
  if (plan.splits > 1) return ceil_div(N, 256);
  const int bn = kTiles[plan.tile].bn;
  return plan.tile >= OP_TILE_SKINNY16 ? ceil_div(N, bn) * (bn / 16) : ceil_div(N, bn);
}

int64_t op_gemm_blocks(const OpPlan& plan, int kind, int64_t M, int64_t N) {
  const TileCost& c = kTiles[plan.tile];
  const int64_t sn = plan.tile >= OP_TILE_SKINNY16 ? c.bn : kind == OP_GATED ? c.bn / 2 : c.bn;
  return ceil_div(M, c.bm) * ceil_div(N, sn);
}

}  // namespace ops
}  // namespace volta
