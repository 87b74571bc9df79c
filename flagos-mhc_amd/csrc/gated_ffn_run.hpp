// The gated feed-forward block's kernels and launches of one type.
#pragma once

#include "gated_ffn.hpp"
#include "gemm_kernel.hpp"

namespace mhc {

// ---- padded copies -------------------------------------------------------------

struct PadArgs {
  const void* src[4];
  void* dst[4];
  int64_t rows[4];
  int cols[4];
  int64_t ld[4];  // of dst: a multiple of 16 bytes; columns from `cols` on become zero
};

// A wave a row at a time; blockIdx.y is the tensor.
template <typename S>
__global__ __launch_bounds__(256) void pad_rows_kernel(PadArgs a) {
  constexpr int V = kVec<S>;
  const int k = blockIdx.y, lane = threadIdx.x & 63;
  const int cols = a.cols[k];
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.rows[k]; r += (int64_t)gridDim.x * 4) {
    const S* s = static_cast<const S*>(a.src[k]) + r * cols;
    S* d = static_cast<S*>(a.dst[k]) + r * a.ld[k];
    for (int e = lane * V; e < a.ld[k]; e += kWave * V) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (e + V <= cols)
        v = *reinterpret_cast<const u32x4_a2*>(s + e);
      else if (e < cols)
        v = ld16_elems<S>(s + e, cols - e);
      st16(d + e, v);
    }
  }
}

// Collects the tensors to copy and where they go, and launches the copies.
template <typename S>
struct Padder {
  PadArgs a = {};
  int n = 0;
  char* at;
  explicit Padder(char* ws) : at(ws) {}
  const void* copy(const void* src, int64_t rows, int cols, int64_t ld) {
    a.src[n] = src, a.dst[n] = at, a.rows[n] = rows, a.cols[n] = cols, a.ld[n] = ld;
    ++n;
    const void* dst = at;
    at += ffn_round_up((size_t)rows * ld * sizeof(S));
    return dst;
  }
  int launch(hipStream_t st) {
    if (n == 0) return MHC_OK;
    int64_t rows = 0;
    for (int i = 0; i < n; ++i) rows = a.rows[i] > rows ? a.rows[i] : rows;
    const int64_t blocks = (rows + 3) / 4, most = (int64_t)device_cu_count() * 16;
    hipLaunchKernelGGL((pad_rows_kernel<S>), dim3((unsigned)(blocks < most ? blocks : most), (unsigned)n), dim3(256), 0, st, a);
    n = 0;
    return check_launch("gated_ffn");
  }
};

// ---- products ----------------------------------------------------------------------

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
  const GemmPlans p = plan_gemm(s, sizeof(S), device_cu_count());
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

// ---- the block ------------------------------------------------------------------------

inline GemmArgs gemm_args(const GemmShape& s, const void* a0, const void* a1, const void* b0, const void* b1, void* out0,
                          void* out1) {
  GemmArgs a = {};
  a.A[0] = a0, a.A[1] = a1, a.B[0] = b0, a.B[1] = b1;
  a.lda = s.lda, a.ldb = s.ldb, a.ldo = s.ldo;
  a.M = (int)s.M, a.N = (int)s.N, a.K = (int)s.K;
  a.segments = s.segments, a.batch = s.batch;
  a.out0 = out0, a.out1 = out1;
  return a;
}

template <typename S>
int ffn_fwd(const FfnFwd& f, const FfnDims& d, char* ws, hipStream_t st) {
  const FfnLines l(d, sizeof(S), false, device_cu_count());
  const FfnWorkspace w(d, sizeof(S), false, device_cu_count());
  void* h = f.hidden ? f.hidden : ws;
  Padder<S> pad(f.hidden ? ws : ws + w.hidden);
  const void *x = f.x, *wg = f.w_gate, *wu = f.w_up, *wd = f.w_down;
  if (l.copy_D) x = pad.copy(x, d.T, d.D, l.D), wg = pad.copy(wg, d.F, d.D, l.D), wu = pad.copy(wu, d.F, d.D, l.D);
  if (l.copy_F) wd = pad.copy(wd, d.O, d.F, l.F);
  if (const int rc = pad.launch(st)) return rc;
  float* part = reinterpret_cast<float*>(pad.at);
  GemmArgs a = gemm_args(fwd_hidden(d, l), x, x, wg, wu, h, nullptr);
  a.act = f.act, a.gate = f.gate, a.up = f.up;
  if (const int rc = launch_gemm<S, kRow, kRow, kEpiGated>(a, fwd_hidden(d, l), part, st)) return rc;
  a = gemm_args(fwd_out(d, l), h, h, wd, wd, f.out, nullptr);
  return launch_gemm<S, kRow, kRow, kEpiStore>(a, fwd_out(d, l), part, st);
}

template <typename S>
int ffn_bwd(const FfnBwd& f, const FfnDims& d, char* ws, hipStream_t st) {
  const FfnLines l(d, sizeof(S), true, device_cu_count());
  const FfnWorkspace w(d, sizeof(S), true, device_cu_count());
  void *dg = ws, *du = ws + w.hidden;
  Padder<S> pad(ws + 2 * w.hidden);
  const void *go = f.grad_out, *x = f.x, *wg = f.w_gate, *wu = f.w_up, *wd = f.w_down;
  if (l.copy_D) x = pad.copy(x, d.T, d.D, l.D), wg = pad.copy(wg, d.F, d.D, l.D), wu = pad.copy(wu, d.F, d.D, l.D);
  if (const int rc = pad.launch(st)) return rc;
  if (l.copy_F) wd = pad.copy(wd, d.O, d.F, l.F);
  if (l.copy_O) go = pad.copy(go, d.T, d.O, l.O);
  if (const int rc = pad.launch(st)) return rc;
  float* part = reinterpret_cast<float*>(pad.at);
  GemmArgs a = gemm_args(bwd_hidden(d, l), go, go, wd, wd, dg, du);
  a.act = f.act, a.gate = const_cast<float*>(f.gate), a.up = const_cast<float*>(f.up);
  if (const int rc = launch_gemm<S, kRow, kCol, kEpiGatedGrad>(a, bwd_hidden(d, l), part, st)) return rc;
  a = gemm_args(bwd_x(d, l), dg, du, wg, wu, f.grad_x, nullptr);
  if (const int rc = launch_gemm<S, kRow, kCol, kEpiStore>(a, bwd_x(d, l), part, st)) return rc;
  if (!f.grad_w_down) return MHC_OK;
  a = gemm_args(bwd_down(d, l), go, go, f.hidden, f.hidden, f.grad_w_down, nullptr);
  if (const int rc = launch_gemm<S, kCol, kCol, kEpiStore>(a, bwd_down(d, l), part, st)) return rc;
  a = gemm_args(bwd_gate_up(d, l), dg, du, x, x, f.grad_w_gate, f.grad_w_up);
  return launch_gemm<S, kCol, kCol, kEpiStore>(a, bwd_gate_up(d, l), part, st);
}

}  // namespace mhc
