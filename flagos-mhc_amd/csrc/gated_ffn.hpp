// The gated feed-forward block's products, as its entry points and the files
// that hold its kernels (one for each type) share them.
#pragma once

#include "common.hpp"
#include "gated_ffn_plan.hpp"
#include "mhc_launch.hpp"

namespace mhc {

struct FfnFwd {
  const void *x, *w_gate, *w_up, *w_down;
  void *out, *hidden;  // hidden null: in the workspace
  float *gate, *up;
  int act;
};
struct FfnBwd {
  const void *grad_out, *x, *w_gate, *w_up, *w_down;
  const float *gate, *up;
  const void* hidden;
  void *grad_x, *grad_w_gate, *grad_w_up, *grad_w_down;  // the weights' may be null
  int act;
};
template <typename S>
int ffn_fwd(const FfnFwd& f, const FfnDims& d, char* ws, hipStream_t st);
template <typename S>
int ffn_bwd(const FfnBwd& f, const FfnDims& d, char* ws, hipStream_t st);

}  // namespace mhc
