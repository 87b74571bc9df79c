// Gated feed-forward block, forward and backward.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, out = h Wd^T      (x (T,D), Wg, Wu (F,D), Wd (O,F))
//   dh = dout Wd, du = dh act(g), dg = dh u act'(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dout^T h
#include <math.h>

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

struct GemmPlan {
  bool dma;    // operands' lines are whole 16-byte chunks
  bool wide;   // the large tile's kernel
  int bm;      // rows of a tile of the tile kernel
  int splits;  // of k
};

// Operands as a product's plan sees them: the block's products differ in
// which index of A and B is contiguous, in the epilogue and in the batch.
struct GemmShape {
  int la, lb, epi, batch, segments;
  int64_t M, N, K, lda, ldb, ldo;
};

// Time of a 256 x 256 tile on a CU against two 128 x 128 tiles.
constexpr int kWideWorth = 3;

GemmPlan plan_gemm(const GemmShape& s, size_t es) {
  GemmPlan p;
  const int64_t line_a = s.lda * (int64_t)es, line_b = s.ldb * (int64_t)es;
  // 32-bit offsets within a tile's lines
  p.dma = line_a % 16 == 0 && line_b % 16 == 0 && line_a < (1 << 23) && line_b < (1 << 23);
  const int64_t steps = ((s.K * (int64_t)es + 127) / 128) * s.segments;
  const int64_t cus = device_cu_count();
  const auto tiles = [&](int64_t bm, int64_t bn) {
    const int64_t cols = s.epi == kEpiGated ? bn / 2 : bn;
    return ((s.M + bm - 1) / bm) * ((s.ldo + cols - 1) / cols) * s.batch;
  };
  const auto rounds = [](int64_t n, int64_t slots) { return (n + slots - 1) / slots; };
  p.bm = s.la == kCol || s.M > 64 ? 128 : (s.M > 16 ? 64 : 16);
  p.wide = p.dma && p.bm == 128 && kWideWorth * rounds(tiles(256, 256), cus) <= 2 * rounds(tiles(128, 128), 2 * cus);
  // too few tiles to fill the card: split k, in pieces of eight steps or more
  const int64_t n = p.wide ? tiles(256, 256) : tiles(p.bm, 128), slots = p.wide ? cus : 2 * cus;
  int64_t splits = n >= slots ? 1 : slots / n;
  if (splits > steps / 8) splits = steps / 8;
  p.splits = (int)(splits < 1 ? 1 : (splits > 64 ? 64 : splits));
  return p;
}

int64_t part_ld(const GemmShape& s) { return (s.ldo + 3) / 4 * 4; }
size_t part_bytes(const GemmShape& s, const GemmPlan& p) {
  if (p.splits == 1) return 0;
  return (size_t)p.splits * s.batch * (s.epi == kEpiGated ? 2 : 1) * s.M * part_ld(s) * sizeof(float);
}

template <typename C>
int launch_tile(const GemmArgs& a, hipStream_t st) {
  const int64_t tiles = (int64_t)((a.M + C::BM - 1) / C::BM) * ((a.ldo + C::kCols - 1) / C::kCols);
  const dim3 g((unsigned)tiles, (unsigned)a.splits, (unsigned)a.batch), b(256);
  if (tiles > 0x7fffffff) return set_error(MHC_ERR_UNSUPPORTED, "gated_ffn: %lld tiles", (long long)tiles);
  if (const int rc = check_grid(g, b, "gated_ffn")) return rc;
  hipLaunchKernelGGL((gemm_tile_kernel<C>), g, b, 0, st, a);
  return check_launch("gated_ffn");
}

template <typename C>
int launch_wide(const GemmArgs& a, hipStream_t st) {
  const int64_t tiles = (int64_t)((a.M + C::BM - 1) / C::BM) * ((a.ldo + C::kCols - 1) / C::kCols);
  const dim3 g((unsigned)tiles, (unsigned)a.splits, (unsigned)a.batch), b(512);
  if (tiles > 0x7fffffff) return set_error(MHC_ERR_UNSUPPORTED, "gated_ffn: %lld tiles", (long long)tiles);
  if (const int rc = check_grid(g, b, "gated_ffn")) return rc;
  hipLaunchKernelGGL((gemm_wide_kernel<C>), g, b, 0, st, a);
  return check_launch("gated_ffn");
}

template <typename S, int EPI>
int launch_join(const GemmArgs& a, hipStream_t st) {
  const int64_t n = a.ldp / 4 * a.M;
  const dim3 g((unsigned)((n + 255) / 256), 1, (unsigned)a.batch), b(256);
  if (const int rc = check_grid(g, b, "gated_ffn")) return rc;
  hipLaunchKernelGGL((gemm_join_kernel<S, EPI>), g, b, 0, st, a);
  return check_launch("gated_ffn");
}

template <typename S, int LA, int LB, int EPI>
int launch_gemm(GemmArgs a, const GemmShape& s, float* part, hipStream_t st) {
  const GemmPlan p = plan_gemm(s, sizeof(S));
  a.splits = p.splits;
  a.part = part;
  a.ldp = part_ld(s);
  int rc = MHC_OK;
  if (p.wide) {
    rc = launch_wide<WideCfg<S, LA, LB, EPI>>(a, st);
  } else if (p.bm == 128) {
    rc = p.dma ? launch_tile<TileCfg<S, LA, LB, 128, 128, 2, 2, EPI, true>>(a, st)
               : launch_tile<TileCfg<S, LA, LB, 128, 128, 2, 2, EPI, false>>(a, st);
  } else if constexpr (LA == kRow) {
    if (p.bm == 64)
      rc = p.dma ? launch_tile<TileCfg<S, LA, LB, 64, 128, 1, 3, EPI, true>>(a, st)
                 : launch_tile<TileCfg<S, LA, LB, 64, 128, 1, 2, EPI, false>>(a, st);
    else
      rc = p.dma ? launch_tile<TileCfg<S, LA, LB, 16, 128, 1, 4, EPI, true>>(a, st)
                 : launch_tile<TileCfg<S, LA, LB, 16, 128, 1, 2, EPI, false>>(a, st);
  }
  if (rc || p.splits == 1) return rc;
  return launch_join<S, EPI>(a, st);
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
  for (const GemmShape& s : {fwd_hidden(d), fwd_out(d)}) n = most(n, part_bytes(s, plan_gemm(s, es)));
  return n;
}
size_t bwd_part_bytes(const FfnDims& d, size_t es) {
  size_t n = 0;
  for (const GemmShape& s : {bwd_hidden(d), bwd_x(d), bwd_down(d), bwd_gate_up(d)}) n = most(n, part_bytes(s, plan_gemm(s, es)));
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
