// Gated feed-forward block, forward and backward.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, out = h Wd^T      (x (T,D), Wg, Wu (F,D), Wd (O,F))
//   dh = dout Wd, du = dh act(g), dg = dh u act'(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dout^T h
#include <cmath>
#include <initializer_list>

#include "gemm_kernel.hpp"
#include "mhc_launch.hpp"

namespace mhc {
namespace {

struct FfnDims {
  int64_t T;
  int D, F, O;
};

size_t elem_bytes(int32_t dtype) { return dtype == MHC_DTYPE_F32 ? 4 : 2; }
int64_t hidden_ld(int64_t F) { return (F + 7) / 8 * 8; }

// ---- which kernel runs a product ---------------------------------------------

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
constexpr double kColCol = 1.13;
constexpr int kFewRows = 4;
constexpr double kJoinUs = 5., kJoinBytesPerUs = 3.5e6, kLaunchUs = 3.;

struct GemmPlan {
  bool dma;   // operands' lines are whole 16-byte chunks
  int kind;
  int whole_tiles, run_tiles, run_blocks;
  double us;
};

int64_t tiles_of(const GemmShape& s, int64_t bm, int64_t bn) {
  const int64_t cols = s.epi == kEpiGated ? bn / 2 : bn;
  return ((s.M + bm - 1) / bm) * ((s.ldo + cols - 1) / cols) * s.batch;
}

// Whole tiles go out in rounds of all blocks that fit the card at once; the
// last round's tiles are cut into equal runs of steps if that, with the
// partial sums' way through memory, is less than the round.
GemmPlan deal_tiles(const GemmShape& s, size_t es, int kind, bool dma) {
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

GemmPlan plan_rows(const GemmShape& s, size_t es) {
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
GemmPlans plan_gemm(const GemmShape& s, size_t es) {
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

size_t part_bytes(const GemmPlans& p) {
  size_t n = 0;
  for (const GemmPlan* q : {&p.main, &p.tail}) {
    const size_t b = (size_t)2 * q->run_blocks * kCosts[q->kind].bm * kCosts[q->kind].bn * sizeof(float);
    n = b > n ? b : n;
  }
  return n;
}

template <typename C>
int launch_join(const GemmArgs& a, hipStream_t st) {
  if (a.run_tiles == 0) return MHC_OK;
  const dim3 g((unsigned)a.run_tiles * (C::BM * (C::kCols / 4) / 256)), b(256);
  if (const int rc = check_grid(g, b, "gated_ffn")) return rc;
  hipLaunchKernelGGL((gemm_join_kernel<C>), g, b, 0, st, a);
  return check_launch("gated_ffn");
}

template <typename C>
int launch_tile(const GemmArgs& a, hipStream_t st) {
  const dim3 g((unsigned)a.whole_tiles + (unsigned)a.run_blocks), b(256);
  if (const int rc = check_grid(g, b, "gated_ffn")) return rc;
  hipLaunchKernelGGL((gemm_tile_kernel<C>), g, b, 0, st, a);
  if (const int rc = check_launch("gated_ffn")) return rc;
  return launch_join<C>(a, st);
}

template <typename C>
int launch_wide(const GemmArgs& a, hipStream_t st) {
  const dim3 g((unsigned)a.whole_tiles + (unsigned)a.run_blocks), b(512);
  if (const int rc = check_grid(g, b, "gated_ffn")) return rc;
  hipLaunchKernelGGL((gemm_wide_kernel<C>), g, b, 0, st, a);
  if (const int rc = check_launch("gated_ffn")) return rc;
  return launch_join<C>(a, st);
}

template <typename S, int LA, int LB, int EPI>
int launch_plan(GemmArgs a, const GemmPlan& p, float* part, hipStream_t st) {
  a.whole_tiles = p.whole_tiles, a.run_tiles = p.run_tiles, a.run_blocks = p.run_blocks;
  a.part = part;
  if (p.kind == kWide256) return launch_wide<WideCfg<S, LA, LB, 256, EPI>>(a, st);
  if (p.kind == kWide128) return launch_wide<WideCfg<S, LA, LB, 128, EPI>>(a, st);
  if constexpr (LA == kRow) {
    if (p.kind == kTile64x128)
      return p.dma ? launch_tile<TileCfg<S, LA, LB, 64, 128, 1, 6, 1, EPI, true>>(a, st)
                   : launch_tile<TileCfg<S, LA, LB, 64, 128, 1, 2, 1, EPI, false>>(a, st);
    if (p.kind == kTile16)
      return p.dma ? launch_tile<TileCfg<S, LA, LB, 16, 128, 1, 8, 1, EPI, true>>(a, st)
                   : launch_tile<TileCfg<S, LA, LB, 16, 128, 1, 2, 1, EPI, false>>(a, st);
  }
  if (p.kind == kTile64)
    return p.dma ? launch_tile<TileCfg<S, LA, LB, 64, 64, 2, 2, 4, EPI, true>>(a, st)
                 : launch_tile<TileCfg<S, LA, LB, 64, 64, 2, 2, 4, EPI, false>>(a, st);
  return p.dma ? launch_tile<TileCfg<S, LA, LB, 128, 128, 2, 2, 2, EPI, true>>(a, st)
               : launch_tile<TileCfg<S, LA, LB, 128, 128, 2, 2, 2, EPI, false>>(a, st);
}

template <typename S, int EPI>
int launch_few_rows(const GemmArgs& a, hipStream_t st) {
  constexpr int kCols = EPI == kEpiGated ? 2 : 4;
  const dim3 g((unsigned)((a.ldo + kCols - 1) / kCols)), b(256);
  if (const int rc = check_grid(g, b, "gated_ffn")) return rc;
  if (a.M == 1)
    hipLaunchKernelGGL((few_rows_kernel<S, 1, EPI>), g, b, 0, st, a);
  else if (a.M == 2)
    hipLaunchKernelGGL((few_rows_kernel<S, 2, EPI>), g, b, 0, st, a);
  else
    hipLaunchKernelGGL((few_rows_kernel<S, 4, EPI>), g, b, 0, st, a);
  return check_launch("gated_ffn");
}

template <typename S, int LA, int LB, int EPI>
int launch_gemm(GemmArgs a, const GemmShape& s, float* part, hipStream_t st) {
  if constexpr (LA == kRow && LB == kRow)
    if (s.M <= kFewRows) return launch_few_rows<S, EPI>(a, st);
  const GemmPlans p = plan_gemm(s, sizeof(S));
  a.M = (int)p.main_rows;
  if (const int rc = launch_plan<S, LA, LB, EPI>(a, p.main, part, st)) return rc;
  if (p.main_rows == s.M) return MHC_OK;
  const int64_t r = p.main_rows;
  a.M = (int)(s.M - r);
  for (const void*& q : a.A) q = static_cast<const S*>(q) + r * s.lda;
  a.out0 = static_cast<S*>(a.out0) + r * s.ldo;
  if (a.out1) a.out1 = static_cast<S*>(a.out1) + r * s.ldo;
  if (a.gate) a.gate += r * s.N, a.up += r * s.N;
  return launch_plan<S, LA, LB, EPI>(a, p.tail, part, st);
}

// ---- the block's products ------------------------------------------------------

GemmShape fwd_hidden(const FfnDims& d) { return {kRow, kRow, kEpiGated, 1, 1, d.T, d.F, d.D, d.D, d.D, hidden_ld(d.F)}; }
GemmShape fwd_out(const FfnDims& d) { return {kRow, kRow, kEpiStore, 1, 1, d.T, d.O, d.F, hidden_ld(d.F), d.F, d.O}; }
GemmShape bwd_hidden(const FfnDims& d) { return {kRow, kCol, kEpiGatedGrad, 1, 1, d.T, d.F, d.O, d.O, d.F, hidden_ld(d.F)}; }
GemmShape bwd_x(const FfnDims& d) { return {kRow, kCol, kEpiStore, 1, 2, d.T, d.D, d.F, hidden_ld(d.F), d.D, d.D}; }
GemmShape bwd_down(const FfnDims& d) { return {kCol, kCol, kEpiStore, 1, 1, d.O, d.F, d.T, d.O, hidden_ld(d.F), d.F}; }
GemmShape bwd_gate_up(const FfnDims& d) { return {kCol, kCol, kEpiStore, 2, 1, d.F, d.D, d.T, hidden_ld(d.F), d.D, d.D}; }

size_t round_up(size_t n) { return (n + 255) / 256 * 256; }
size_t most(size_t a, size_t b) { return a > b ? a : b; }
size_t hidden_bytes(const FfnDims& d, size_t es) { return round_up((size_t)d.T * hidden_ld(d.F) * es); }
size_t fwd_part_bytes(const FfnDims& d, size_t es) {
  size_t n = 0;
  for (const GemmShape& s : {fwd_hidden(d), fwd_out(d)}) n = most(n, part_bytes(plan_gemm(s, es)));
  return n;
}
size_t bwd_part_bytes(const FfnDims& d, size_t es) {
  size_t n = 0;
  for (const GemmShape& s : {bwd_hidden(d), bwd_x(d), bwd_down(d), bwd_gate_up(d)}) n = most(n, part_bytes(plan_gemm(s, es)));
  return n;
}

GemmArgs gemm_args(const GemmShape& s, const void* a0, const void* a1, const void* b0, const void* b1, void* out0, void* out1) {
  GemmArgs a = {};
  a.A[0] = a0, a.A[1] = a1, a.B[0] = b0, a.B[1] = b1;
  a.lda = s.lda, a.ldb = s.ldb, a.ldo = s.ldo;
  a.M = (int)s.M, a.N = (int)s.N, a.K = (int)s.K;
  a.segments = s.segments, a.batch = s.batch;
  a.out0 = out0, a.out1 = out1;
  return a;
}

template <typename S>
int ffn_fwd(const void* x, const void* wg, const void* wu, const void* wd, int act, void* out, float* gate, float* up,
            void* h, float* part, const FfnDims& d, hipStream_t st) {
  GemmArgs a = gemm_args(fwd_hidden(d), x, x, wg, wu, h, nullptr);
  a.act = act, a.gate = gate, a.up = up;
  if (const int rc = launch_gemm<S, kRow, kRow, kEpiGated>(a, fwd_hidden(d), part, st)) return rc;
  return launch_gemm<S, kRow, kRow, kEpiStore>(gemm_args(fwd_out(d), h, h, wd, wd, out, nullptr), fwd_out(d), part, st);
}

template <typename S>
int ffn_bwd(const void* gout, const void* x, const void* wg, const void* wu, const void* wd, const float* gate,
            const float* up, const void* h, int act, void* gx, void* gwg, void* gwu, void* gwd, void* dg, void* du,
            float* part, const FfnDims& d, hipStream_t st) {
  GemmArgs a = gemm_args(bwd_hidden(d), gout, gout, wd, wd, dg, du);
  a.act = act, a.gate = const_cast<float*>(gate), a.up = const_cast<float*>(up);
  if (const int rc = launch_gemm<S, kRow, kCol, kEpiGatedGrad>(a, bwd_hidden(d), part, st)) return rc;
  if (const int rc = launch_gemm<S, kRow, kCol, kEpiStore>(gemm_args(bwd_x(d), dg, du, wg, wu, gx, nullptr), bwd_x(d), part, st))
    return rc;
  if (const int rc = launch_gemm<S, kCol, kCol, kEpiStore>(gemm_args(bwd_down(d), gout, gout, h, h, gwd, nullptr), bwd_down(d), part, st))
    return rc;
  return launch_gemm<S, kCol, kCol, kEpiStore>(gemm_args(bwd_gate_up(d), dg, du, x, x, gwg, gwu), bwd_gate_up(d), part, st);
}

int check_ffn(const char* who, const FfnDims& d, int32_t dtype, int32_t act) {
  if (d.T < 0 || d.D < 1 || d.F < 1 || d.O < 1)
    return set_error(MHC_ERR_INVALID, "%s: T=%lld D=%d F=%d O=%d", who, (long long)d.T, d.D, d.F, d.O);
  if (d.T > kMaxTokens) return check_tokens(d.T, who);
  if (dtype != MHC_DTYPE_F32 && dtype != MHC_DTYPE_BF16 && dtype != MHC_DTYPE_F16)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: dtype %d not supported", who, dtype);
  // tiles are counted in 32 bits
  if (((d.T + 15) / 16) * (((int64_t)(d.F > d.O ? d.F : d.O) + 63) / 64) > 0x3fffffff ||
      (((int64_t)d.F + 63) / 64) * (((int64_t)(d.D > d.O ? d.D : d.O) + 63) / 64) > 0x3fffffff ||
      ((d.T + 15) / 16) * (((int64_t)d.D + 63) / 64) > 0x3fffffff)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: T=%lld D=%d F=%d O=%d are too many tiles", who, (long long)d.T, d.D, d.F, d.O);
  if (act < 0 || act > kActRelu) return set_error(MHC_ERR_INVALID, "%s: activation %d", who, act);
  return MHC_OK;
}

int check_buffers(const char* who, const void* const* p, int n, const void* ws, size_t ws_bytes, size_t need) {
  for (int i = 0; i < n; ++i) {
    if (!p[i]) return set_error(MHC_ERR_INVALID, "%s: null pointer", who);
    if (!aligned16(p[i])) return set_error(MHC_ERR_INVALID, "%s: a tensor is not 16-byte aligned", who);
  }
  if (need && (!ws || ws_bytes < need || !aligned16(ws)))
    return set_error(MHC_ERR_INVALID, "%s: workspace too small or not 16-byte aligned (%zu < %zu bytes)", who,
                     ws ? ws_bytes : (size_t)0, need);
  return MHC_OK;
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" size_t mhc_gated_ffn_fwd_workspace_size(int64_t T, int32_t D, int32_t F, int32_t O, int32_t dtype) {
  if (check_ffn("", {T, D, F, O}, dtype, 0)) return 0;
  const FfnDims d = {T, D, F, O};
  return T ? hidden_bytes(d, elem_bytes(dtype)) + fwd_part_bytes(d, elem_bytes(dtype)) : 0;
}

extern "C" int mhc_gated_ffn_fwd(const void* x, const void* w_gate, const void* w_up, const void* w_down,
                                 int32_t dtype, int32_t activation, void* out, float* gate, float* up, void* hidden,
                                 void* workspace, size_t workspace_bytes, int64_t T, int32_t D, int32_t F, int32_t O,
                                 void* stream) {
  clear_error();
  const FfnDims d = {T, D, F, O};
  if (const int rc = check_ffn("gated_ffn", d, dtype, activation)) return rc;
  if (T == 0) return MHC_OK;
  if (!gate != !up || !gate != !hidden)
    return set_error(MHC_ERR_INVALID, "gated_ffn: gate, up and hidden go together");
  const void* bufs[] = {x, w_gate, w_up, w_down, out};
  if (const int rc = check_buffers("gated_ffn", bufs, 5, workspace, workspace_bytes,
                                   mhc_gated_ffn_fwd_workspace_size(T, D, F, O, dtype)))
    return rc;
  void* h = hidden ? hidden : workspace;
  float* part = reinterpret_cast<float*>(static_cast<char*>(workspace) + hidden_bytes(d, elem_bytes(dtype)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MHC_DTYPE_F32) return ffn_fwd<float>(x, w_gate, w_up, w_down, activation, out, gate, up, h, part, d, st);
  if (dtype == MHC_DTYPE_BF16) return ffn_fwd<bf16_t>(x, w_gate, w_up, w_down, activation, out, gate, up, h, part, d, st);
  return ffn_fwd<f16_t>(x, w_gate, w_up, w_down, activation, out, gate, up, h, part, d, st);
}

extern "C" size_t mhc_gated_ffn_bwd_workspace_size(int64_t T, int32_t D, int32_t F, int32_t O, int32_t dtype) {
  if (check_ffn("", {T, D, F, O}, dtype, 0)) return 0;
  const FfnDims d = {T, D, F, O};
  return T ? 2 * hidden_bytes(d, elem_bytes(dtype)) + bwd_part_bytes(d, elem_bytes(dtype)) : 0;
}

extern "C" int mhc_gated_ffn_bwd(const void* grad_out, const void* x, const void* w_gate, const void* w_up,
                                 const void* w_down, const float* gate, const float* up, const void* hidden,
                                 int32_t dtype, int32_t activation, void* grad_x, void* grad_w_gate, void* grad_w_up,
                                 void* grad_w_down, void* workspace, size_t workspace_bytes, int64_t T, int32_t D,
                                 int32_t F, int32_t O, void* stream) {
  clear_error();
  const FfnDims d = {T, D, F, O};
  if (const int rc = check_ffn("gated_ffn_backward", d, dtype, activation)) return rc;
  if (T == 0) return MHC_OK;
  const void* bufs[] = {grad_out, x, w_gate, w_up, w_down, gate, up, hidden, grad_x, grad_w_gate, grad_w_up, grad_w_down};
  if (const int rc = check_buffers("gated_ffn_backward", bufs, 12, workspace, workspace_bytes,
                                   mhc_gated_ffn_bwd_workspace_size(T, D, F, O, dtype)))
    return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t hb = hidden_bytes(d, elem_bytes(dtype));
  char* ws = static_cast<char*>(workspace);
  const auto run = [&](auto s) {
    using S = decltype(s);
    return ffn_bwd<S>(grad_out, x, w_gate, w_up, w_down, gate, up, hidden, activation, grad_x, grad_w_gate, grad_w_up,
                      grad_w_down, ws, ws + hb, reinterpret_cast<float*>(ws + 2 * hb), d, st);
  };
  if (dtype == MHC_DTYPE_F32) return run(float{});
  if (dtype == MHC_DTYPE_BF16) return run(bf16_t{});
  return run(f16_t{});
}
