// The gated feed-forward block's products and workspaces.  Plain C++ with no
// HIP in it, as gemm_plan.hpp.
#pragma once

#include "gemm_plan.hpp"

namespace mhc {

struct FfnDims {
  int64_t T;
  int D, F, O;
};

inline int64_t hidden_ld(int64_t F) { return (F + 7) / 8 * 8; }
inline size_t ffn_round_up(size_t n) { return (n + 255) / 256 * 256; }

// Rows that are no multiples of 16 bytes cannot go straight to LDS, and a
// product through registers has a third of the rate.  Where it pays, by the
// plans' times, the operands are first copied to padded rows.
struct FfnLines {
  int64_t D, F, O;  // elements from row to row of x, w_gate and w_up; of w_down; of grad_out
  bool copy_D = false, copy_F = false, copy_O = false;
  inline FfnLines(const FfnDims& d, size_t es, bool backward, int64_t cus);
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

// The products of a pass.
struct FfnShapes {
  GemmShape s[4];
  int n;
  FfnShapes(const FfnDims& d, const FfnLines& l, bool backward) {
    if (backward)
      s[0] = bwd_hidden(d, l), s[1] = bwd_x(d, l), s[2] = bwd_down(d, l), s[3] = bwd_gate_up(d, l), n = 4;
    else
      s[0] = fwd_hidden(d, l), s[1] = fwd_out(d, l), n = 2;
  }
};

constexpr double kCopyBytesPerUs = 4.5e6;
constexpr int kCopyTokens = 64;  // below, the weights' copies cost more than they are read for

inline FfnLines::FfnLines(const FfnDims& d, size_t es, bool backward, int64_t cus) : D(d.D), F(d.F), O(d.O) {
  const auto odd = [&](int64_t n) { return n * (int64_t)es % 16 != 0; };
  if (d.T <= kCopyTokens || !(odd(D) || odd(F) || (backward && odd(O)))) return;
  const auto us = [&] {
    double t = 0.;
    const FfnShapes f(d, *this, backward);
    for (int i = 0; i < f.n; ++i) {
      const GemmPlans p = plan_gemm(f.s[i], es, cus);
      t += p.main.us + p.tail.us;
    }
    return t;
  };
  const double plain = us();
  const auto pad = [](int64_t n) { return (n + 63) / 64 * 64; };
  copy_D = odd(D), copy_F = odd(F), copy_O = backward && odd(O);
  int64_t copied = 0;  // elements
  if (copy_D) copied += ((int64_t)d.T + 2 * (int64_t)d.F) * D, D = pad(D);
  if (copy_F) copied += (int64_t)d.O * F, F = pad(F);
  if (copy_O) copied += d.T * O, O = pad(O);
  if (us() + kLaunchUs + 2 * copied * es / kCopyBytesPerUs < plain) return;
  D = d.D, F = d.F, O = d.O;
  copy_D = copy_F = copy_O = false;
}

// Parts of a workspace, from its start on.
struct FfnWorkspace {
  size_t hidden = 0;       // bytes of one (T, F) intermediate
  size_t x = 0, w = 0, w_down = 0, grad_out = 0;  // of the padded copies: x, w_gate (and w_up), w_down, grad_out
  size_t part = 0;         // of the partial sums
  FfnWorkspace(const FfnDims& d, size_t es, bool backward, int64_t cus) {
    const FfnLines l(d, es, backward, cus);
    hidden = ffn_round_up((size_t)d.T * hidden_ld(d.F) * es);
    if (l.copy_D) x = ffn_round_up((size_t)d.T * l.D * es), w = ffn_round_up((size_t)d.F * l.D * es);
    if (l.copy_F) w_down = ffn_round_up((size_t)d.O * l.F * es);
    if (l.copy_O) grad_out = ffn_round_up((size_t)d.T * l.O * es);
    const FfnShapes f(d, l, backward);
    for (int i = 0; i < f.n; ++i) {
      const size_t n = part_bytes(plan_gemm(f.s[i], es, cus));
      part = n > part ? n : part;
    }
  }
  size_t bytes(bool backward) const { return (backward ? 2 : 1) * hidden + x + 2 * w + w_down + grad_out + part; }
  // of a forward whose hidden is the caller's
  size_t bytes_saving() const { return bytes(false) - hidden; }
};

}  // namespace mhc
