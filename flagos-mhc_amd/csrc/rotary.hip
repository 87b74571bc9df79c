// Rotary positions of the queries and keys, forward and inverse.
//
//   (a, b) -> amplitude (a cos w - b sin w, a sin w + b cos w),  w = position * freq_i
//
// for the r / 2 pairs of a head's first r elements: (i, i + r / 2) or
// (2 i, 2 i + 1); elements past r are copied.  The backward is the rotation by
// -w.  A position's angles are the same for every head: a block takes a few
// tokens, computes their sines and cosines once, into LDS, and rotates every
// head of both tensors with them, so that nothing but q and k is read and
// written.  Angles are reduced in 64 bits (turns = position * freq / 2 pi, less
// their nearest integer): in 32 a position of 10^6 would be off by 0.06.  HBM
// bounds it: 65536 tokens, 64 heads of 128 bf16 in 433 us (median), 5.0 TB/s.
#include "attention.hpp"
#include "mhc_launch.hpp"

namespace mhc {
namespace {

struct RotArgs {
  const void* x[2];         // q, k
  void* y[2];               // contiguous
  int64_t ts[2], hs[2];     // elements
  int heads[2];
  const double* freqs;      // radians a position
  const void* positions;    // (T,) int32 or int64, or null: from cu or t % S
  const int32_t* cu;
  int64_t T, S;
  int wide, B;              // wide: positions are int64
  int d, r;
  float amplitude;
  int sign;
};

// Tokens before t of t's own sequence: 64 candidates a step, one a lane.
__device__ __forceinline__ int64_t packed_position(const int32_t* cu, int B, int64_t T, int64_t t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = B + 1;
  while (n > 1) {
    const int step = (n + 63) / 64, c = lane * step;
    int hit = __popcll(__ballot(c < n && cu_at(cu, lo + c, T) <= t));
    hit = hit < 1 ? 1 : hit;
    const int skip = (hit - 1) * step;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  return t - cu_at(cu, lo, T);
}

constexpr int kThreads = 256, kTrig = 2048;  // float2 of LDS: tokens * r / 2 at most

// VEC elements at any alignment: 16 bytes, or 8.
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
template <typename S, bool WHOLE> struct Piece;
template <typename S> struct Piece<S, true> {
  using T = u32x4;
  static __device__ __forceinline__ T load(const S* p) { return ld16nt_u(p); }
  static __device__ __forceinline__ void store(S* p, T w) { st16nt_u(p, w); }
  static __device__ __forceinline__ void unpack(T w, float (&v)[Store<S>::VEC]) { Store<S>::unpack(w, v); }
  static __device__ __forceinline__ T pack(const float (&v)[Store<S>::VEC]) { return Store<S>::pack(v); }
};
template <typename S> struct Piece<S, false> {
  static constexpr int N = Store<S>::VEC / 2;
  using T = u32x2;
  static __device__ __forceinline__ T load(const S* p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x2_a2*>(p)); }
  static __device__ __forceinline__ void store(S* p, T w) { __builtin_nontemporal_store(w, reinterpret_cast<u32x2_a2*>(p)); }
  static __device__ __forceinline__ void unpack(T w, float (&v)[N]) {
    float all[2 * N];
    Store<S>::unpack(u32x4{w[0], w[1], 0u, 0u}, all);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = all[j];
  }
  static __device__ __forceinline__ T pack(const float (&v)[N]) {
    float all[2 * N] = {};
#pragma unroll
    for (int j = 0; j < N; ++j) all[j] = v[j];
    const u32x4 w = Store<S>::pack(all);
    return u32x2{w[0], w[1]};
  }
};

// VEC: elements of an access; 1: any sizes.
template <typename S, int VEC, bool HALF>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotArgs a, int tokens) {
  __shared__ float2 trig[kTrig];
  const int64_t t0 = xcd_contig(blockIdx.x, gridDim.x) * tokens;
  const int n = (int)(a.T - t0 < tokens ? a.T - t0 : tokens), half = a.r / 2, wave = threadIdx.x >> 6;
  // a head's items: pairs of vectors (HALF), vectors of pairs, or single pairs;
  // then what is copied, as many elements an item
  const int rot = VEC > 1 && !HALF ? a.r / VEC : half / VEC;
  const int wide = VEC > 1 && !HALF ? VEC : 2 * VEC;  // elements of an item
  const int per = rot + (a.d - a.r + wide - 1) / wide, heads = a.heads[0] + a.heads[1];
  // item `at` of head `th` of token `tok`; the next one is kThreads items on
  const int step_th = kThreads / per, step_at = kThreads % per, step_i = step_th / heads, step_h = step_th % heads;
  int at = threadIdx.x % per, th = threadIdx.x / per % heads, tok = threadIdx.x / per / heads;
  for (int i = wave; i < n; i += kThreads / 64) {
    const int64_t t = t0 + i;
    int64_t p;
    if (a.positions) p = a.wide ? static_cast<const int64_t*>(a.positions)[t] : static_cast<const int32_t*>(a.positions)[t];
    else if (a.cu) p = packed_position(a.cu, a.B, a.T, t);
    else p = t % a.S;
    for (int j = threadIdx.x & 63; j < half; j += 64) {
      const double turns = (double)p * (a.freqs[j] * 0.15915494309189533577);
      const float f = (float)(turns - rint(turns));
      float sn, cs;
      sincospif(2.f * f, &sn, &cs);
      trig[i * half + j] = make_float2(cs * a.amplitude, a.sign < 0 ? -sn * a.amplitude : sn * a.amplitude);
    }
  }
  __syncthreads();
  while (tok < n) {
    const int w = th >= a.heads[0], h = th - (w ? a.heads[0] : 0);
    const int64_t t = t0 + tok;
    const S* x = static_cast<const S*>(a.x[w]) + t * a.ts[w] + (int64_t)h * a.hs[w];
    S* y = static_cast<S*>(a.y[w]) + (t * a.heads[w] + h) * (int64_t)a.d;
    // Turned or copied, an item is loaded and stored by the same instructions:
    // apart, a wave with both waits for memory twice (16384 x 64 heads of 80, 40
    // turned, bf16: 155 -> 75 us in pairs of neighbours, 4.5 TB/s).
    const bool copy = at >= rot;
    const float2* cs = trig + tok * half;
    const int e = copy ? a.r + (at - rot) * wide : at * (HALF ? VEC : (VEC > 1 ? VEC : 2));
    if constexpr (VEC == 1) {
      const int e1 = HALF && !copy ? e + half : e + 1;
      const bool two = e1 < a.d;
      const float2 z = copy ? make_float2(1.f, 0.f) : cs[at];
      const float u = load_elem<S>(x, e), v = two ? load_elem<S>(x, e1) : 0.f;
      store_elem<S>(y, e, copy ? u : u * z.x - v * z.y);
      if (two) store_elem<S>(y, e1, copy ? v : u * z.y + v * z.x);
    } else if constexpr (HALF) {
      using P = Piece<S, VEC == Store<S>::VEC>;
      const int e1 = copy ? e + VEC : e + half;
      const bool two = e1 < a.d;
      const typename P::T wu = P::load(x + e), wv = P::load(x + (two ? e1 : e));
      float u[VEC], v[VEC], p[VEC], q[VEC];
      P::unpack(wu, u);
      P::unpack(wv, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float2 z = cs[copy ? 0 : e + j];
        p[j] = u[j] * z.x - v[j] * z.y;
        q[j] = u[j] * z.y + v[j] * z.x;
      }
      P::store(y + e, copy ? wu : P::pack(p));
      if (two) P::store(y + e1, copy ? wv : P::pack(q));
    } else {
      using P = Piece<S, VEC == Store<S>::VEC>;
      const typename P::T wu = P::load(x + e);
      float u[VEC], p[VEC];
      P::unpack(wu, u);
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        const float2 z = cs[copy ? 0 : (e + j) / 2];
        p[j] = u[j] * z.x - u[j + 1] * z.y;
        p[j + 1] = u[j] * z.y + u[j + 1] * z.x;
      }
      P::store(y + e, copy ? wu : P::pack(p));
    }
    at += step_at;
    const int more = at >= per;
    at -= more ? per : 0;
    th += step_h + more;
    const int wrap = th >= heads;
    th -= wrap ? heads : 0;
    tok += step_i + wrap;
  }
}

template <typename S, int VEC>
int rotary_launch(const RotArgs& a, bool half_layout, hipStream_t st) {
  const int half = a.r / 2;
  // four tokens a block (a wave a token's angles) where there are blocks enough
  int tokens = a.T >= (int64_t)device_cu_count() * 16 ? 4 : 1;
  while (tokens > 1 && tokens * half > kTrig) tokens /= 2;
  const int64_t blocks = (a.T + tokens - 1) / tokens;
  if (blocks > 0xffffffffll / kThreads)
    return set_error(MHC_ERR_UNSUPPORTED, "rotary: %lld rows exceed a dispatch", (long long)a.T);
  const dim3 g((unsigned)blocks), b(kThreads);
  if (half_layout) hipLaunchKernelGGL((rotary_kernel<S, VEC, true>), g, b, 0, st, a, tokens);
  else hipLaunchKernelGGL((rotary_kernel<S, VEC, false>), g, b, 0, st, a, tokens);
  return check_launch("rotary");
}

// 16 bytes an access where a head's parts are whole ones, else 8 (heads of 80
// with 40 turned in halves, 16384 x 64, bf16: 105 us, single elements 243 us),
// else single elements.  Addresses need no alignment (16384 x 64 heads of 128
// from an odd address: 119 us, 109 us from a whole 16 bytes, 4.9 TB/s).
template <typename S>
int rotary_run(const RotArgs& a, bool half_layout, hipStream_t st) {
  constexpr int VEC = Store<S>::VEC;
  const int part = half_layout ? a.r / 2 : a.r, rest = a.d - a.r;
  if (part % VEC == 0 && rest % VEC == 0) return rotary_launch<S, VEC>(a, half_layout, st);
  if (part % (VEC / 2) == 0 && rest % (VEC / 2) == 0) return rotary_launch<S, VEC / 2>(a, half_layout, st);
  return rotary_launch<S, 1>(a, half_layout, st);
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" int mhc_rotary(const mhc_rotary_args* c, void* stream) {
  clear_error();
  if (!c) return set_error(MHC_ERR_INVALID, "rotary: null arguments");
  if (c->rows < 0 || c->heads < 1 || c->heads_k < 0 || c->d < 1 || c->r < 0 || c->r > c->d || c->r % 2 ||
      (c->layout != MHC_ROTARY_HALF && c->layout != MHC_ROTARY_INTERLEAVED))
    return set_error(MHC_ERR_INVALID, "rotary: rows=%lld heads=%d heads_k=%d d=%d r=%d layout=%d", (long long)c->rows, c->heads,
                     c->heads_k, c->d, c->r, c->layout);
  if (c->flags & ~(MHC_ROTARY_WIDE_POSITIONS | MHC_ROTARY_INVERSE))
    return set_error(MHC_ERR_INVALID, "rotary: flags 0x%x", c->flags);
  if (c->dtype != MHC_DTYPE_F32 && c->dtype != MHC_DTYPE_BF16 && c->dtype != MHC_DTYPE_F16)
    return set_error(MHC_ERR_UNSUPPORTED, "rotary: dtype %d not supported", c->dtype);
  if (c->r > 2 * kTrig) return set_error(MHC_ERR_UNSUPPORTED, "rotary: r=%d above the supported %d", c->r, 2 * kTrig);
  // a block's items are counted in 32 bits
  if (((int64_t)c->heads + c->heads_k) * c->d > (1 << 28))
    return set_error(MHC_ERR_UNSUPPORTED, "rotary: heads=%d heads_k=%d d=%d above the supported sizes", c->heads, c->heads_k, c->d);
  if (c->q_row < 0 || c->q_head < 0 || c->k_row < 0 || c->k_head < 0)
    return set_error(MHC_ERR_INVALID, "rotary: negative stride");
  if (!c->positions && !c->cu_seqlens && c->length < 1)
    return set_error(MHC_ERR_INVALID, "rotary: length %lld", (long long)c->length);
  if (c->cu_seqlens && c->sequences < 0) return set_error(MHC_ERR_INVALID, "rotary: sequences %d", c->sequences);
  if (c->rows == 0) return MHC_OK;
  if (!c->q || !c->q_out || (c->heads_k && (!c->k || !c->k_out)) || (c->r && !c->freqs))
    return set_error(MHC_ERR_INVALID, "rotary: null pointer");
  const RotArgs a = {{c->q, c->k}, {c->q_out, c->k_out}, {c->q_row, c->k_row}, {c->q_head, c->k_head}, {c->heads, c->heads_k},
                     c->freqs, c->positions, c->cu_seqlens, c->rows, c->length, (c->flags & MHC_ROTARY_WIDE_POSITIONS) != 0,
                     c->sequences, c->d, c->r, c->amplitude, c->flags & MHC_ROTARY_INVERSE ? -1 : 1};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (c->dtype == MHC_DTYPE_F32) return rotary_run<float>(a, c->layout == MHC_ROTARY_HALF, st);
  if (c->dtype == MHC_DTYPE_BF16) return rotary_run<bf16_t>(a, c->layout == MHC_ROTARY_HALF, st);
  return rotary_run<f16_t>(a, c->layout == MHC_ROTARY_HALF, st);
}
