// The gated feed-forward block's products and workspaces.  Plain C++ with no
// HIP in it, as gemm_plan.hpp.
#pragma once

#include <initializer_list>

#include "gemm_plan.hpp"

namespace mhc {

struct FfnDims {
  int64_t T;
  int D, F, O;
};

inline int64_t hidden_ld(int64_t F) { return (F + 7) / 8 * 8; }
inline size_t ffn_round_up(size_t n) { return (n + 255) / 256 * 256; }

// Rows that are no multiples of 16 bytes cannot go straight to LDS, and a
// product through registers runs at a third of the rate (16 bits; fp32 is
// bound by its matrix instructions either way).  With enough tokens the
// operands are first copied to padded rows: measured at D = 1003, F = 2677 the
// copies pay from some 200 tokens on.
struct FfnLines {
  int64_t D, F, O;  // elements from row to row of x, w_gate and w_up; of w_down; of grad_out
  bool copy_D, copy_F, copy_O;
  FfnLines(const FfnDims& d, size_t es) {
    const bool many = d.T > (es == 4 ? 1024 : 256);
    const auto odd = [&](int64_t n) { return many && n * (int64_t)es % 16 != 0; };
    const auto pad = [](int64_t n) { return (n + 63) / 64 * 64; };
    copy_D = odd(d.D), copy_F = odd(d.F), copy_O = odd(d.O);
    D = copy_D ? pad(d.D) : d.D;
    F = copy_F ? pad(d.F) : d.F;
    O = copy_O ? pad(d.O) : d.O;
  }
};

inline GemmShape fwd_hidden(const FfnDims& d, const FfnLines& l) {
  return {kRow, kRow, kEpiGated, 1, 1, d.T, d.F, d.D, l.D, l.D, hidden_ld(d.F)};
}
inline GemmShape fwd_out(const FfnDims& d, const FfnLines& l) {
  return {kRow, kRow, kEpiStore, 1, 1, d.T, d.O, d.F, hidden_ld(d.F), l.F, d.O};
}
inline GemmShape bwd_hidden(const FfnDims& d, const FfnLines& l) {
  return {kRow, kCol, kEpiGatedGrad, 1, 1, d.T, d.F, d.O, l.O, l.F, hidden_ld(d.F)};
}
inline GemmShape bwd_x(const FfnDims& d, const FfnLines& l) {
  return {kRow, kCol, kEpiStore, 1, 2, d.T, d.D, d.F, hidden_ld(d.F), l.D, d.D};
}
inline GemmShape bwd_down(const FfnDims& d, const FfnLines& l) {
  return {kCol, kCol, kEpiStore, 1, 1, d.O, d.F, d.T, l.O, hidden_ld(d.F), d.F};
}
inline GemmShape bwd_gate_up(const FfnDims& d, const FfnLines& l) {
  return {kCol, kCol, kEpiStore, 2, 1, d.F, d.D, d.T, hidden_ld(d.F), l.D, d.D};
}

// Parts of a workspace, from its start on.
struct FfnWorkspace {
  size_t hidden = 0;       // bytes of one (T, F) intermediate
  size_t x = 0, w = 0, w_down = 0, grad_out = 0;  // of the padded copies: x, w_gate (and w_up), w_down, grad_out
  size_t part = 0;         // of the partial sums
  FfnWorkspace(const FfnDims& d, size_t es, bool backward, int64_t cus) {
    const FfnLines l(d, es);
    hidden = ffn_round_up((size_t)d.T * hidden_ld(d.F) * es);
    if (l.copy_D) x = ffn_round_up((size_t)d.T * l.D * es), w = ffn_round_up((size_t)d.F * l.D * es);
    if (l.copy_F) w_down = ffn_round_up((size_t)d.O * l.F * es);
    if (l.copy_O && backward) grad_out = ffn_round_up((size_t)d.T * l.O * es);
    const auto add = [&](const GemmShape& s) {
      const size_t n = part_bytes(plan_gemm(s, es, cus));
      part = n > part ? n : part;
    };
    if (backward)
      for (const GemmShape& s : {bwd_hidden(d, l), bwd_x(d, l), bwd_down(d, l), bwd_gate_up(d, l)}) add(s);
    else
      for (const GemmShape& s : {fwd_hidden(d, l), fwd_out(d, l)}) add(s);
  }
  size_t bytes(bool backward) const { return (backward ? 2 : 1) * hidden + x + 2 * w + w_down + grad_out + part; }
};

}  // namespace mhc
