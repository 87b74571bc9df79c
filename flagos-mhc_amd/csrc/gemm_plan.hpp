// Host side of the matrix products: which kernel runs one, and how its tiles
// are dealt out.  Plain C++ with no HIP in it: a test compiles it alone and
// walks the plans of many shapes on the CPU.
#pragma once

#include <math.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define MHC_HOST_DEVICE __host__ __device__
#else
#define MHC_HOST_DEVICE
#endif

namespace mhc {

enum { kRow = 0, kCol = 1 };  // an operand's contiguous index: k, or m or n

// What becomes of a product C (gemm_kernel.hpp).
enum { kEpiStore = 0, kEpiGated = 1, kEpiGatedGrad = 2 };

// ---- runs of steps ------------------------------------------------------------
// run_tiles tiles of `steps` steps each, dealt to run_blocks blocks in runs of
// equal length (to one step).

// Where block b's run starts, in steps from the first tile's first.
MHC_HOST_DEVICE inline int64_t run_start(int64_t b, int tiles, int steps, int blocks) { return b * tiles * steps / blocks; }

// The i-th piece of block b's run (a run is no longer than a tile, so it has
// one or two): its tile, steps and slot of the partial sums (-1: the whole tile).
struct RunPiece {
  int64_t tile, s0, s1, slot;
};
MHC_HOST_DEVICE inline bool run_piece(int64_t b, int i, int tiles, int steps, int blocks, RunPiece* p) {
  const int64_t lo = run_start(b, tiles, steps, blocks), hi = run_start(b + 1, tiles, steps, blocks);
  const int64_t t = lo / steps + i, first = t * steps;
  p->tile = t;
  p->s0 = lo > first ? lo - first : 0;
  p->s1 = hi - first < steps ? hi - first : steps;
  p->slot = p->s0 == 0 && p->s1 == steps ? -1 : 2 * b + i;
  return p->s0 < p->s1;
}

// The blocks with a piece of tile t: [first, last).  Only `first` can have
// begun before the tile (its piece is then its second); none if one block has
// the whole tile.
struct RunBlocks {
  int64_t first, last;
  bool begun_before;
};
MHC_HOST_DEVICE inline RunBlocks run_blocks_of(int64_t t, int tiles, int steps, int blocks) {
  const int64_t begin = t * steps, end = begin + steps, total = (int64_t)tiles * steps;
  RunBlocks r;
  r.first = begin * blocks / total;
  while (r.first > 0 && run_start(r.first, tiles, steps, blocks) > begin) --r.first;
  while (run_start(r.first + 1, tiles, steps, blocks) <= begin) ++r.first;
  r.last = end * blocks / total;
  while (r.last < blocks && run_start(r.last, tiles, steps, blocks) < end) ++r.last;
  while (run_start(r.last - 1, tiles, steps, blocks) >= end) --r.last;
  r.begun_before = run_start(r.first, tiles, steps, blocks) < begin;
  if (r.last - r.first == 1 && !r.begun_before && run_start(r.last, tiles, steps, blocks) >= end) r.last = r.first;
  return r;
}

// ---- plans ---------------------------------------------------------------------

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
    {16, 128, 1, {0.72, 0.4}, {0.72, 0.4}, {1.2, 1.2}, {1.2, 1.2}},
    {64, 128, 1, {0.72, 0.4}, {1.8, 1.8}, {1.2, 1.2}, {2.0, 2.0}},
    {64, 64, 4, {0.23, 0.6}, {0.6, 0.8}, {0.4, 1.2}, {0.65, 1.4}},
    {128, 128, 2, {0.49, 0.8}, {2.3, 3.2}, {0.8, 1.5}, {2.5, 3.5}},
    {128, 256, 1, {0.87, 0.75}, {4.4, 4.4}, {}, {}},
    {256, 256, 1, {1.46, 1.25}, {8.5, 8.5}, {}, {}}};
// both operands kCol: twice the LDS reads, which the large tiles feel; B's
// lines of k through registers: a wait for memory every step
constexpr double kColCol = 1.16, kColRegs = 1.7;
constexpr int kFewRows = 4;
// a launch, and the join's (the kernel takes 5 us for few bytes)
constexpr double kLaunchUs = 3., kJoinUs = kLaunchUs + 5., kJoinBytesPerUs = 3.5e6;
constexpr double kCuBytesPerUs = 16e3;  // of a tile's results, with every CU at it

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
inline GemmPlan deal_tiles(const GemmShape& s, size_t es, int kind, bool dma, int64_t cus) {
  const KernelCost& c = kCosts[kind];
  const StepCost& cost = dma ? (es == 4 ? c.dma32 : c.dma16) : (es == 4 ? c.reg32 : c.reg16);
  const int64_t slots = cus * c.per_cu;
  const int64_t tiles = tiles_of(s, c.bm, c.bn), steps = (s.K * (int64_t)es + 127) / 128 * s.segments;
  // n steps of `blocks` blocks side by side: on a part of the CUs each runs
  // faster, as the card's power then allows a higher clock, and each has more
  // of the memory's rate (forwards with the gated product in whole tiles, and in
  // 256 runs with a join, weights out of HBM: T = 64, D = 4096, F = 11008 bf16,
  // 172 tiles, 75 and 77 us; D = 1024, F = 2816, 44 tiles, 28 and 31; D = 7168, F =
  // 18432, 288 tiles, whose last round is nearly empty, 207 and 174)
  const auto side_by_side = [&](double blocks, double n) {
    const double part = blocks < cus ? blocks / cus : 1.;
    const double few = c.per_cu > 1 ? cost.alone : cost.alone + (cost.full - cost.alone) * part;
    const double full = blocks < cus ? 0. : ceil(blocks / cus) * cost.full;
    return n * (full > few ? full : few) * (s.la == kCol && kind >= kWide128 ? kColCol : (s.lb == kCol && !dma ? kColRegs : 1.));
  };
  const int64_t rest = tiles % slots, rounds = tiles / slots;
  // what a column of a tile's row reads and writes at the end, which only
  // another block of the CU can overlap
  const double ends = s.epi == kEpiStore ? es : (s.epi == kEpiGated ? (8. + es) / 2 : 8. + 2 * es);
  const double end_us = c.bm * c.bn * ends / kCuBytesPerUs / (c.per_cu > 1 ? 2 : 1);
  const double rounds_us = kLaunchUs + rounds * (side_by_side((double)slots, (double)steps) + c.per_cu * end_us);
  GemmPlan p = {dma, kind, (int)tiles, 0, 0, rounds_us};
  if (rest == 0) return p;
  p.us += side_by_side((double)rest, (double)steps) + ceil((double)rest / cus) * end_us;
  // Runs of six steps or more.  The large tiles' blocks that work side by side
  // have to be at the same k of neighbouring tiles, or every one of them
  // fetches its operands for itself: a tile is cut into as many equal runs as
  // there is room for.
  int64_t blocks = rest * steps / 6;
  if (blocks > slots) blocks = slots;
  if (kind >= kWide128) blocks = blocks / rest * rest;
  if (blocks > rest) {
    const double bytes = (double)(blocks + rest) * (s.M < c.bm ? s.M : c.bm) * c.bn * 4 * 2;
    const double us = rounds_us + end_us + side_by_side((double)blocks, (double)rest * steps / blocks) + kJoinUs + bytes / kJoinBytesPerUs;
    if (us < p.us) p = {dma, kind, (int)(tiles - rest), (int)rest, (int)blocks, us};
  }
  return p;
}

inline GemmPlan plan_rows(const GemmShape& s, size_t es, int64_t cus) {
  const int64_t line_a = s.lda * (int64_t)es, line_b = s.ldb * (int64_t)es;
  // 32-bit offsets within a tile's lines
  const bool dma = line_a % 16 == 0 && line_b % 16 == 0 && line_a < (1 << 23) && line_b < (1 << 23);
  GemmPlan p = {};
  for (int kind = 0; kind < kKinds; ++kind) {
    if (kind >= kWide128 && !dma) break;
    const bool few = kind <= kTile64x128;  // rows: the tile that holds them all; kCol tiles have 64 rows or more
    if (few && (s.la == kCol || s.M > kCosts[kind].bm)) continue;
    const GemmPlan q = deal_tiles(s, es, kind, dma, cus);
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
inline GemmPlans plan_gemm(const GemmShape& s, size_t es, int64_t cus) {
  GemmPlans p = {};
  if (s.la == kRow && s.lb == kRow && s.M <= kFewRows) return p;  // a kernel of its own
  p = {plan_rows(s, es, cus), {}, s.M};
  const int64_t over = s.M % 256;
  if (s.la == kRow && s.M > 256 && over > 0 && over <= 64) {
    GemmShape m = s, t = s;
    m.M = s.M - over;
    t.M = over;
    const GemmPlan a = plan_rows(m, es, cus), b = plan_rows(t, es, cus);
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
