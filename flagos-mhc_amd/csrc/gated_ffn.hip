// Gated feed-forward block, forward and backward.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, out = h Wd^T      (x (T,D), Wg, Wu (F,D), Wd (O,F))
//   dh = dout Wd, du = dh act(g), dg = dh u act'(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dout^T h
//
// Three products forward, five backward, each on the matrix instructions in
// fp32 sums (gemm_kernel.hpp); hidden and the gradients of gate and up are
// rounded to the operands' type between them, gate and up are kept in fp32.
#include "gated_ffn.hpp"

namespace mhc {

extern template int ffn_fwd<float>(const FfnFwd&, const FfnDims&, char*, hipStream_t);
extern template int ffn_fwd<bf16_t>(const FfnFwd&, const FfnDims&, char*, hipStream_t);
extern template int ffn_fwd<f16_t>(const FfnFwd&, const FfnDims&, char*, hipStream_t);
extern template int ffn_bwd<float>(const FfnBwd&, const FfnDims&, char*, hipStream_t);
extern template int ffn_bwd<bf16_t>(const FfnBwd&, const FfnDims&, char*, hipStream_t);
extern template int ffn_bwd<f16_t>(const FfnBwd&, const FfnDims&, char*, hipStream_t);

namespace {

// The kernels round a size up to a tile's rows, or a step's k, in 32 bits.
constexpr int64_t kMaxSize = (1ll << 31) - 256;

size_t elem_bytes(int32_t dtype) { return dtype == MHC_DTYPE_F32 ? 4 : 2; }

int check_ffn(const char* who, const FfnDims& d, int32_t dtype, int32_t act) {
  if (d.T < 0 || d.D < 1 || d.F < 1 || d.O < 1)
    return set_error(MHC_ERR_INVALID, "%s: T=%lld D=%d F=%d O=%d", who, (long long)d.T, d.D, d.F, d.O);
  if (dtype != MHC_DTYPE_F32 && dtype != MHC_DTYPE_BF16 && dtype != MHC_DTYPE_F16)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: dtype %d not supported", who, dtype);
  if (d.T > kMaxSize || d.D > kMaxSize || d.F > kMaxSize || d.O > kMaxSize)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: T=%lld D=%d F=%d O=%d, above the supported %lld", who, (long long)d.T, d.D,
                     d.F, d.O, (long long)kMaxSize);
  // tiles are counted in 32 bits
  if (((d.T + 15) / 16) * (((int64_t)(d.F > d.O ? d.F : d.O) + 63) / 64) > 0x3fffffff ||
      (((int64_t)d.F + 63) / 64) * (((int64_t)(d.D > d.O ? d.D : d.O) + 63) / 64) > 0x3fffffff ||
      ((d.T + 15) / 16) * (((int64_t)d.D + 63) / 64) > 0x3fffffff)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: T=%lld D=%d F=%d O=%d are too many tiles", who, (long long)d.T, d.D, d.F, d.O);
  if (act < 0 || act > MHC_ACT_RELU) return set_error(MHC_ERR_INVALID, "%s: activation %d", who, act);
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
  if (check_ffn("", {T, D, F, O}, dtype, 0) || T == 0) return 0;
  return FfnWorkspace({T, D, F, O}, elem_bytes(dtype), false, device_cu_count()).bytes(false);
}

extern "C" size_t mhc_gated_ffn_fwd_save_workspace_size(int64_t T, int32_t D, int32_t F, int32_t O, int32_t dtype) {
  if (check_ffn("", {T, D, F, O}, dtype, 0) || T == 0) return 0;
  return FfnWorkspace({T, D, F, O}, elem_bytes(dtype), false, device_cu_count()).bytes_saving();
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
                                   hidden ? mhc_gated_ffn_fwd_save_workspace_size(T, D, F, O, dtype)
                                          : mhc_gated_ffn_fwd_workspace_size(T, D, F, O, dtype)))
    return rc;
  if (gate && !(aligned16(gate) && aligned16(up) && aligned16(hidden)))
    return set_error(MHC_ERR_INVALID, "gated_ffn: gate, up or hidden is not 16-byte aligned");
  const FfnFwd f = {x, w_gate, w_up, w_down, out, hidden, gate, up, activation};
  char* ws = static_cast<char*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MHC_DTYPE_F32) return ffn_fwd<float>(f, d, ws, st);
  if (dtype == MHC_DTYPE_BF16) return ffn_fwd<bf16_t>(f, d, ws, st);
  return ffn_fwd<f16_t>(f, d, ws, st);
}

extern "C" size_t mhc_gated_ffn_bwd_workspace_size(int64_t T, int32_t D, int32_t F, int32_t O, int32_t dtype) {
  if (check_ffn("", {T, D, F, O}, dtype, 0) || T == 0) return 0;
  return FfnWorkspace({T, D, F, O}, elem_bytes(dtype), true, device_cu_count()).bytes(true);
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
  if (!grad_w_gate != !grad_w_up || !grad_w_gate != !grad_w_down)
    return set_error(MHC_ERR_INVALID, "gated_ffn_backward: the weights' gradients go together");
  const void* bufs[] = {grad_out, x, w_gate, w_up, w_down, gate, up, hidden, grad_x, grad_w_gate, grad_w_up, grad_w_down};
  if (const int rc = check_buffers("gated_ffn_backward", bufs, grad_w_gate ? 12 : 9, workspace, workspace_bytes,
                                   mhc_gated_ffn_bwd_workspace_size(T, D, F, O, dtype)))
    return rc;
  const FfnBwd f = {grad_out, x, w_gate, w_up, w_down, gate, up, hidden, grad_x, grad_w_gate, grad_w_up, grad_w_down, activation};
  char* ws = static_cast<char*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MHC_DTYPE_F32) return ffn_bwd<float>(f, d, ws, st);
  if (dtype == MHC_DTYPE_BF16) return ffn_bwd<bf16_t>(f, d, ws, st);
  return ffn_bwd<f16_t>(f, d, ws, st);
}
