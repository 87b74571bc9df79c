// Host side of the matrix products: which kernel runs one, and how its tiles
// are dealt out.
#pragma once

#include <cmath>

#include "gemm_kernel.hpp"
#include "mhc_launch.hpp"

namespace mhc {

// Operands as a product's plan sees them: the block's products differ in
// which index of A and B is contiguous, in the epilogue and in the batch.
struct GemmShape {
  int la, lb, epi, batch, segments;
  int64_t M, N, K, lda, ldb, ldo;
};

// The kernels: tile, blocks a CU, and microseconds for one step (128 bytes of
// k) of one tile, for operands of 16 bits and 4 bytes: what a CU with all its
// blocks takes, and what a block alone on its CU takes (measured; `reg`: through
// registers).
enum { kTile16, kTile64x128, kTile64, kTile128, kWide128, kWide256, kKinds };
struct StepCost {
  double full, alone;
};
struct KernelCost {
  int bm, bn, per_cu;
  StepCost dma16, dma32, reg16, reg32;
};
constexpr KernelCost kCosts[kKinds] = {
    {16, 128, 1, {0.8, 0.8}, {0.8, 0.8}, {1.2, 1.2}, {1.2, 1.2}},
    {64, 128, 1, {0.9, 0.9}, {1.8, 1.8}, {1.2, 1.2}, {2.0, 2.0}},
    {64, 64, 4, {0.23, 0.6}, {0.6, 0.8}, {0.4, 0.76}, {0.65, 1.0}},
    {128, 128, 2, {0.49, 0.8}, {2.3, 3.2}, {0.8, 1.28}, {2.5, 3.5}},
    {128, 256, 1, {0.87, 0.75}, {4.4, 4.4}, {}, {}},
    {256, 256, 1, {1.46, 1.25}, {8.5, 8.5}, {}, {}}};
// both operands kCol: twice the LDS reads, which the large tiles feel
constexpr double kColCol = 1.16;
constexpr int kFewRows = 4;
constexpr double kJoinUs = 5., kJoinBytesPerUs = 3.5e6, kLaunchUs = 3.;

struct GemmPlan {
  bool dma;   // operands' lines are whole 16-byte chunks
  int kind;
  int whole_tiles, run_tiles, run_blocks;
  double us;
};

inline int64_t tiles_of(const GemmShape& s, int64_t bm, int64_t bn) {
  const int64_t cols = s.epi == kEpiGated ? bn / 2 : bn;
  return ((s.M + bm - 1) / bm) * ((s.ldo + cols - 1) / cols) * s.batch;
}

// Whole tiles go out in rounds of all blocks that fit the card at once; the
// last round's tiles are cut into equal runs of steps if that, with the
// partial sums' way through memory, is less than the round.
inline GemmPlan deal_tiles(const GemmShape& s, size_t es, int kind, bool dma) {
  const KernelCost& c = kCosts[kind];
  const StepCost& cost = dma ? (es == 4 ? c.dma32 : c.dma16) : (es == 4 ? c.reg32 : c.reg16);
  const int64_t cus = device_cu_count(), slots = cus * c.per_cu;
  const int64_t tiles = tiles_of(s, c.bm, c.bn), steps = (s.K * (int64_t)es + 127) / 128 * s.segments;
  // n steps of `blocks` blocks side by side: on a part of the CUs each runs
  // faster, as the card's power then allows a higher clock
  const auto side_by_side = [&](double blocks, double n) {
    const double part = blocks < cus ? blocks / cus : 1.;
    const double few = c.per_cu > 1 ? cost.alone : cost.alone + (cost.full - cost.alone) * part;
    const double full = blocks < cus ? 0. : std::ceil(blocks / cus) * cost.full;
    return n * (full > few ? full : few) * (s.la == kCol && kind >= kWide128 ? kColCol : 1.);
  };
  const int64_t rest = tiles % slots, rounds = tiles / slots;
  const double rounds_us = kLaunchUs + rounds * side_by_side((double)slots, (double)steps);
  GemmPlan p = {dma, kind, (int)tiles, 0, 0, rounds_us};
  if (rest == 0) return p;
  p.us += side_by_side((double)rest, (double)steps);
  // Runs of six steps or more.  The large tiles' blocks that work side by side
  // have to be at the same k of neighbouring tiles, or every one of them
  // fetches its operands for itself: a tile is cut into as many equal runs as
  // there is room for.
  int64_t blocks = rest * steps / 6;
  if (blocks > slots) blocks = slots;
  if (kind >= kWide128) blocks = blocks / rest * rest;
  if (blocks > rest) {
    const double bytes = (double)(blocks + rest) * (s.M < c.bm ? s.M : c.bm) * c.bn * 4 * 2;
    const double us = rounds_us + side_by_side((double)blocks, (double)rest * steps / blocks) + kJoinUs + bytes / kJoinBytesPerUs;
    if (us < p.us) p = {dma, kind, (int)(tiles - rest), (int)rest, (int)blocks, us};
  }
  return p;
}

inline GemmPlan plan_rows(const GemmShape& s, size_t es) {
  const int64_t line_a = s.lda * (int64_t)es, line_b = s.ldb * (int64_t)es;
  // 32-bit offsets within a tile's lines
  const bool dma = line_a % 16 == 0 && line_b % 16 == 0 && line_a < (1 << 23) && line_b < (1 << 23);
  GemmPlan p = {};
  for (int kind = 0; kind < kKinds; ++kind) {
    if (kind >= kWide128 && !dma) break;
    const bool few = kind <= kTile64x128;  // rows: the tile that holds them all; kCol tiles have 64 rows or more
    if (few && (s.la == kCol || s.M > kCosts[kind].bm)) continue;
    const GemmPlan q = deal_tiles(s, es, kind, dma);
    if (p.us == 0. || q.us < p.us) p = q;
    if (few) break;
  }
  return p;
}

// A product is one launch, or two: the rows past the last whole 256 go apart
// where they are few and would take a row of large tiles.
struct GemmPlans {
  GemmPlan main, tail;
  int64_t main_rows;  // M: no tail
};
inline GemmPlans plan_gemm(const GemmShape& s, size_t es) {
  GemmPlans p = {};
  if (s.la == kRow && s.lb == kRow && s.M <= kFewRows) return p;  // a kernel of its own
  p = {plan_rows(s, es), {}, s.M};
  const int64_t over = s.M % 256;
  if (s.la == kRow && s.M > 256 && over > 0 && over <= 64) {
    GemmShape m = s, t = s;
    m.M = s.M - over;
    t.M = over;
    const GemmPlan a = plan_rows(m, es), b = plan_rows(t, es);
    if (a.us + b.us < p.main.us) p = {a, b, m.M};
  }
  return p;
}

inline size_t part_bytes(const GemmPlans& p) {
  size_t n = 0;
  for (const GemmPlan* q : {&p.main, &p.tail}) {
    const size_t b = (size_t)2 * q->run_blocks * kCosts[q->kind].bm * kCosts[q->kind].bn * sizeof(float);
    n = b > n ? b : n;
  }
  return n;
}

}  // namespace mhc
