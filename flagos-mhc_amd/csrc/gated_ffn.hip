// Gated feed-forward block, forward and backward.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, out = h Wd^T      (x (T,D), Wg, Wu (F,D), Wd (O,F))
//   dh = dout Wd, du = dh act(g), dg = dh u act'(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dout^T h
#include <math.h>

#include "common.hpp"
#include "mhc_launch.hpp"

namespace mhc {
namespace {

enum { kSilu = 0, kGelu = 1, kGeluTanh = 2, kRelu = 3 };

// act(g) and act'(g) in fp32.
__device__ __forceinline__ void act_both(int kind, float g, float* a, float* d) {
  if (kind == kSilu) {
    const float s = 1.f / (1.f + expf(-g));
    *a = g * s;
    *d = s * (1.f + g * (1.f - s));
  } else if (kind == kGelu) {
    const float p = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    *a = g * p;
    *d = p + g * 0.39894228040143268f * expf(-0.5f * g * g);
  } else if (kind == kGeluTanh) {
    // 0.5 (1 + tanh v) = 1 / (1 + exp(-2 v))
    const float v = 0.79788456080286536f * (g + 0.044715f * g * g * g);
    const float s = 1.f / (1.f + expf(-2.f * v));
    *a = g * s;
    *d = s + g * 2.f * s * (1.f - s) * 0.79788456080286536f * (1.f + 0.134145f * fminf(g * g, 1e30f));
  } else {
    *a = g > 0.f ? g : (g != g ? g : 0.f);
    *d = g > 0.f ? 1.f : 0.f;
  }
}

enum { kStore = 0, kGated = 1, kGatedGrad = 2 };

// C[m][n] = sum over segments and k of A(m, k) B(n, k), elements addressed by
// strides; EPI decides what becomes of C.
struct MmArgs {
  const void* A[2];
  const void* B[2];
  int nseg;  // segments of k (kStore); kGated has one k range and two B
  int64_t am, ak, bn, bk;
  int M, N, K;
  int64_t ldo;  // row stride of out0 and out1; gate and up: N
  int act;
  void* out0;  // C, h or dg
  void* out1;  // du
  float* gate;
  float* up;
};

template <typename S, int EPI>
__global__ __launch_bounds__(256) void mm_simple_kernel(MmArgs a) {
  constexpr int NB = EPI == kGated ? 2 : 1;
  __shared__ float As[16][65], Bs[NB][16][65];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  float acc[NB][4][4] = {};
  for (int seg = 0; seg < a.nseg; ++seg)
    for (int k0 = 0; k0 < a.K; k0 += 16) {
      for (int i = threadIdx.x; i < 1024; i += 256) {
        // the fast index along whichever stride is 1
        const int r = a.ak == 1 ? i >> 4 : i & 63, k = a.ak == 1 ? i & 15 : i >> 6;
        As[k][r] = m0 + r < a.M && k0 + k < a.K
                       ? load_elem<S>(static_cast<const S*>(a.A[seg]), (m0 + r) * a.am + (k0 + k) * a.ak)
                       : 0.f;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
        for (int i = threadIdx.x; i < 1024; i += 256) {
          const int r = a.bk == 1 ? i >> 4 : i & 63, k = a.bk == 1 ? i & 15 : i >> 6;
          Bs[b][k][r] = n0 + r < a.N && k0 + k < a.K
                            ? load_elem<S>(static_cast<const S*>(a.B[EPI == kGated ? b : seg]),
                                           (n0 + r) * a.bn + (k0 + k) * a.bk)
                            : 0.f;
        }
      __syncthreads();
      // 16 products are added before they meet the running sum: its rounding
      // error grows with K / 16 additions instead of K
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < 16; ++k) s += As[k][ty + 16 * i] * Bs[b][k][tx + 16 * j];
            acc[b][i][j] += s;
          }
      __syncthreads();
    }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m >= a.M || n >= a.ldo) continue;
      const int64_t e = m * a.N + n, o = m * a.ldo + n;
      if (n >= a.N) {  // the rest of a row of h, dg or du
        store_elem<S>(static_cast<S*>(a.out0), o, 0.f);
        if (EPI == kGatedGrad) store_elem<S>(static_cast<S*>(a.out1), o, 0.f);
        continue;
      }
      if constexpr (EPI == kStore) {
        store_elem<S>(static_cast<S*>(a.out0), o, acc[0][i][j]);
      } else if constexpr (EPI == kGated) {
        const float g = acc[0][i][j], u = acc[1][i][j];
        float v, d;
        act_both(a.act, g, &v, &d);
        store_elem<S>(static_cast<S*>(a.out0), o, v * u);
        if (a.gate) {
          a.gate[e] = g;
          a.up[e] = u;
        }
      } else {
        const float dh = acc[0][i][j], u = a.up[e];
        float v, d;
        act_both(a.act, a.gate[e], &v, &d);
        store_elem<S>(static_cast<S*>(a.out0), o, dh * u * d);
        store_elem<S>(static_cast<S*>(a.out1), o, dh * v);
      }
    }
}

template <typename S, int EPI>
int launch_mm(const MmArgs& a, hipStream_t st) {
  const dim3 g((unsigned)((a.ldo + 63) / 64), (unsigned)((a.M + 63) / 64)), b(256);
  if (g.y > 65535u) return set_error(MHC_ERR_UNSUPPORTED, "gated_ffn: M=%d too large", a.M);
  hipLaunchKernelGGL((mm_simple_kernel<S, EPI>), g, b, 0, st, a);
  return check_launch("gated_ffn");
}

struct FfnDims {
  int64_t T;
  int D, F, O;
};

size_t elem_bytes(int32_t dtype) { return dtype == MHC_DTYPE_F32 ? 4 : 2; }
int64_t hidden_ld(int64_t F) { return (F + 7) / 8 * 8; }

template <typename S>
int ffn_fwd(const void* x, const void* wg, const void* wu, const void* wd, int act, void* out, float* gate, float* up,
            void* h, const FfnDims& d, hipStream_t st) {
  const int T = (int)d.T;
  const int64_t ld = hidden_ld(d.F);
  MmArgs a = {{x, x}, {wg, wu}, 1, d.D, 1, d.D, 1, T, d.F, d.D, ld, act, h, nullptr, gate, up};
  if (const int rc = launch_mm<S, kGated>(a, st)) return rc;
  MmArgs b = {{h, h}, {wd, wd}, 1, ld, 1, d.F, 1, T, d.O, d.F, d.O, act, out, nullptr, nullptr, nullptr};
  return launch_mm<S, kStore>(b, st);
}

template <typename S>
int ffn_bwd(const void* gout, const void* x, const void* wg, const void* wu, const void* wd, const float* gate,
            const float* up, const void* h, int act, void* gx, void* gwg, void* gwu, void* gwd, S* dg, S* du,
            const FfnDims& d, hipStream_t st) {
  const int T = (int)d.T;
  const int64_t ld = hidden_ld(d.F);
  MmArgs a = {{gout, gout}, {wd, wd}, 1, d.O, 1, 1, d.F, T, d.F, d.O, ld, act, dg, du, const_cast<float*>(gate),
              const_cast<float*>(up)};
  if (const int rc = launch_mm<S, kGatedGrad>(a, st)) return rc;
  MmArgs b = {{dg, du}, {wg, wu}, 2, ld, 1, 1, d.D, T, d.D, d.F, d.D, act, gx, nullptr, nullptr, nullptr};
  if (const int rc = launch_mm<S, kStore>(b, st)) return rc;
  MmArgs c = {{gout, gout}, {h, h}, 1, 1, d.O, 1, ld, d.O, d.F, T, d.F, act, gwd, nullptr, nullptr, nullptr};
  if (const int rc = launch_mm<S, kStore>(c, st)) return rc;
  MmArgs e = {{dg, dg}, {x, x}, 1, 1, ld, 1, d.D, d.F, d.D, T, d.D, act, gwg, nullptr, nullptr, nullptr};
  if (const int rc = launch_mm<S, kStore>(e, st)) return rc;
  MmArgs f = {{du, du}, {x, x}, 1, 1, ld, 1, d.D, d.F, d.D, T, d.D, act, gwu, nullptr, nullptr, nullptr};
  return launch_mm<S, kStore>(f, st);
}

int check_ffn(const char* who, const FfnDims& d, int32_t dtype, int32_t act) {
  if (d.T < 0 || d.D < 1 || d.F < 1 || d.O < 1)
    return set_error(MHC_ERR_INVALID, "%s: T=%lld D=%d F=%d O=%d", who, (long long)d.T, d.D, d.F, d.O);
  if (d.T > kMaxTokens) return check_tokens(d.T, who);
  if (dtype != MHC_DTYPE_F32 && dtype != MHC_DTYPE_BF16 && dtype != MHC_DTYPE_F16)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: dtype %d not supported", who, dtype);
  if (act < 0 || act > kRelu) return set_error(MHC_ERR_INVALID, "%s: activation %d", who, act);
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
  return (size_t)T * hidden_ld(F) * elem_bytes(dtype);
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
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MHC_DTYPE_F32) return ffn_fwd<float>(x, w_gate, w_up, w_down, activation, out, gate, up, h, d, st);
  if (dtype == MHC_DTYPE_BF16) return ffn_fwd<bf16_t>(x, w_gate, w_up, w_down, activation, out, gate, up, h, d, st);
  return ffn_fwd<f16_t>(x, w_gate, w_up, w_down, activation, out, gate, up, h, d, st);
}

extern "C" size_t mhc_gated_ffn_bwd_workspace_size(int64_t T, int32_t D, int32_t F, int32_t O, int32_t dtype) {
  if (check_ffn("", {T, D, F, O}, dtype, 0)) return 0;
  return 2 * (size_t)T * hidden_ld(F) * elem_bytes(dtype);
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
  const auto run = [&](auto s) {
    using S = decltype(s);
    S* dg = static_cast<S*>(workspace);
    return ffn_bwd<S>(grad_out, x, w_gate, w_up, w_down, gate, up, hidden, activation, grad_x, grad_w_gate, grad_w_up,
                      grad_w_down, dg, dg + (size_t)T * hidden_ld(F), d, st);
  };
  if (dtype == MHC_DTYPE_F32) return run(float{});
  if (dtype == MHC_DTYPE_BF16) return run(bf16_t{});
  return run(f16_t{});
}
