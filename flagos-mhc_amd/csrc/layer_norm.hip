// Layer norm of (T, D) rows, forward and backward.
//
//   y = (x - mean) rstd w + b,  mean = sum x / D,  rstd = (sum (x - mean)^2 / D + eps)^-1/2
//   with xhat = (x - mean) rstd and g = dy w:
//   dx = rstd (g - sum(g) / D - xhat sum(g xhat) / D),  dw = sum_t dy xhat,  db = sum_t dy
//
// Both passes are bound by HBM.  A row is read once into the registers of G
// lanes (a wave, or a block of 256 to 1024 threads, by the row's length), so
// the variance is the sum of squares about the mean that was just formed and
// never a difference of two sums.  Blocks walk rows with a fixed stride, the
// next row's loads started before a row is worked on; a thread has the same
// columns in every row and keeps their weight and bias.  The backward adds its
// columns' dw and db in fp32 registers, each block writes its sums once, and a
// second kernel adds the blocks' sums in a fixed order: no atomics, the same
// bits in every run.  T = 65536, D = 7168 bf16: forward 336 us (5.6 TB/s),
// backward 527 us (5.3 TB/s).  Rows longer than 4096 16-byte vectors (the
// backward: 2048) are read from memory again for each sum (they come from the
// L2), element by element, and the backward's dw and db are added in memory: T =
// 4096, D = 12288 fp32 467 us, a quarter of the rate (forward, in registers, 70).
#include "common.hpp"
#include "mhc_launch.hpp"

namespace mhc {
namespace {

// VEC elements from element `e` of a row of D >= VEC elements, as fp32; rows
// start at any element, so accesses are unaligned 16-byte ones.  W is the
// activations' type or fp32, so VEC is one or two of its vectors.
template <typename W, int VEC>
__device__ __forceinline__ void load_f32(const W* row, int64_t e, float* o) {
  constexpr int V = Store<W>::VEC;
  static_assert(VEC % V == 0, "whole vectors");
#pragma unroll
  for (int i = 0; i < VEC / V; ++i) {
    const u32x4 v = *reinterpret_cast<const u32x4_a2*>(row + e + i * V);
    Store<W>::unpack(v, o + i * V);
  }
}

// The v-th vector of a row of D elements: the last one of a row whose width
// is no multiple of VEC starts at D - VEC instead and repeats `skip` elements
// of the vector before it.
template <int VEC>
__device__ __forceinline__ int vec_start(int v, int D, int* skip) {
  const int e = v * VEC, s = e + VEC <= D ? e : D - VEC;
  *skip = e - s;
  return s;
}

// Sum over the G lanes of a row group.  red: G / 64 floats of LDS that no
// lane still reads from an earlier sum (callers alternate two).
template <int G>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = group_sum<63>(v);
  if constexpr (G == 64) return v;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) red[wave] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < G / 64; ++i) s += red[i];
  return s;
}

template <int G>
constexpr int kRowsPerBlock = G == 64 ? 4 : 1;
template <int G>
constexpr int kBlockThreads = G == 64 ? 256 : G;

struct NormFwdArgs {
  const void* x;
  const void* w;
  const void* b;
  void* y;
  float* mean;
  float* rstd;
  int64_t T;
  int D;
  float eps;
};

template <typename S, typename W, int G, int NV>
__global__ __launch_bounds__(kBlockThreads<G>) void norm_fwd_kernel(NormFwdArgs a) {
  constexpr int VEC = Store<S>::VEC;
  __shared__ float red[2][16];
  const int r = G == 64 ? threadIdx.x >> 6 : 0, t = G == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int D = a.D, nv = (D + VEC - 1) / VEC;
  const float inv_d = 1.f / (float)D;
  const S* x = static_cast<const S*>(a.x);
  S* y = static_cast<S*>(a.y);
  const int64_t step = (int64_t)gridDim.x * kRowsPerBlock<G>;
  int64_t row = (int64_t)blockIdx.x * kRowsPerBlock<G> + r;
  int e[NV], skip[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = t + i * G;
    e[i] = v < nv ? vec_start<VEC>(v, D, &skip[i]) : -1;
  }
  u32x4 raw[NV];
  const auto load = [&](int64_t rr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      raw[i] = {0u, 0u, 0u, 0u};
      if (e[i] >= 0) raw[i] = ld16nt_u(x + rr * D + e[i]);
    }
  };
  if (row < a.T) load(row);
  // weight and bias once a thread: read again for every row they are four times
  // the row's bytes (the longest rows leave no registers for them)
  constexpr bool kHold = NV * VEC * kBlockThreads<G> <= 16384;
  float w[kHold ? NV : 1][VEC], b[kHold ? NV : 1][VEC];
  const auto params = [&](int i, float* wv, float* bv) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) wv[j] = 1.f, bv[j] = 0.f;
    if (e[i] >= 0 && a.w) load_f32<W, VEC>(static_cast<const W*>(a.w), e[i], wv);
    if (e[i] >= 0 && a.b) load_f32<W, VEC>(static_cast<const W*>(a.b), e[i], bv);
  };
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < NV; ++i) params(i, w[i], b[i]);
  }
  // G > 64: every thread of the block has the same row, so barriers are met by all
  for (; row < a.T; row += step) {
    float f[NV][VEC];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) Store<S>::unpack(raw[i], f[i]);
    if (row + step < a.T) load(row + step);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (e[i] >= 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += j >= skip[i] ? f[i][j] : 0.f;
      }
    const float mean = row_sum<G>(s, red[0]) * inv_d;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (e[i] >= 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          f[i][j] -= mean;
          q += j >= skip[i] ? f[i][j] * f[i][j] : 0.f;
        }
      }
    const float var = row_sum<G>(q, red[1]) * inv_d;
    const float rstd = 1.f / sqrtf(var + a.eps);
    if (t == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (e[i] >= 0) {
        constexpr int H = kHold ? NV : 1;
        if constexpr (!kHold) params(i, w[0], b[0]);
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = f[i][j] * rstd * w[i % H][j] + b[i % H][j];
        st16nt_u(y + row * D + e[i], Store<S>::pack(o));
      }
  }
}

// Rows of any length, element by element: rows shorter than a vector, and
// rows too long for the registers.
template <typename S, typename W>
__global__ __launch_bounds__(1024) void norm_fwd_loop_kernel(NormFwdArgs a) {
  __shared__ float red[2][16];
  const int64_t row = blockIdx.x;
  const int D = a.D;
  const S* x = static_cast<const S*>(a.x) + row * D;
  S* y = static_cast<S*>(a.y) + row * D;
  float s = 0.f;
  for (int i = threadIdx.x; i < D; i += 1024) s += load_elem<S>(x, i);
  const float inv_d = 1.f / (float)D;
  const float mean = row_sum<1024>(s, red[0]) * inv_d;
  float q = 0.f;
  for (int i = threadIdx.x; i < D; i += 1024) {
    const float d = load_elem<S>(x, i) - mean;
    q += d * d;
  }
  const float var = row_sum<1024>(q, red[1]) * inv_d;
  const float rstd = 1.f / sqrtf(var + a.eps);
  if (threadIdx.x == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  for (int i = threadIdx.x; i < D; i += 1024) {
    const float w = a.w ? load_elem<W>(static_cast<const W*>(a.w), i) : 1.f;
    const float b = a.b ? load_elem<W>(static_cast<const W*>(a.b), i) : 0.f;
    store_elem<S>(y, i, (load_elem<S>(x, i) - mean) * rstd * w + b);
  }
}

struct NormBwdArgs {
  float* gw;  // where one launch does all: the weights' gradients (null: not wanted), its row blocks
  float* gb;
  int row_blocks;
  const void* gy;
  const void* x;
  const void* w;
  const float* mean;
  const float* rstd;
  void* gx;
  float* part;  // [blocks][2][D]: dw, then db of the block's rows (null: neither is wanted)
  int64_t T;
  int D;
};

template <typename S, typename W, int G, int NV>
__device__ __forceinline__ void norm_bwd_rows(const NormBwdArgs& a, int blocks) {
  constexpr int VEC = Store<S>::VEC, R = kRowsPerBlock<G>;
  __shared__ float red[2][2][16];
  const int r = G == 64 ? threadIdx.x >> 6 : 0, t = G == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int D = a.D, nv = (D + VEC - 1) / VEC;
  const float inv_d = 1.f / (float)D;
  const S* x = static_cast<const S*>(a.x);
  const S* gy = static_cast<const S*>(a.gy);
  S* gx = static_cast<S*>(a.gx);
  int e[NV], skip[NV];
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = t + i * G;
    e[i] = v < nv ? vec_start<VEC>(v, D, &skip[i]) : -1;
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[i][j] = 1.f, dw[i][j] = 0.f, db[i][j] = 0.f;
    if (e[i] >= 0 && a.w) load_f32<W, VEC>(static_cast<const W*>(a.w), e[i], w[i]);
  }
  const int64_t step = (int64_t)blocks * R;
  int64_t row = (int64_t)blockIdx.x * R + r;
  u32x4 xr[NV], gr[NV];
  float mean = 0.f, rstd = 0.f;
  const auto load = [&](int64_t rr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      xr[i] = gr[i] = {0u, 0u, 0u, 0u};
      if (e[i] >= 0) {
        xr[i] = ld16nt_u(x + rr * D + e[i]);
        gr[i] = ld16nt_u(gy + rr * D + e[i]);
      }
    }
    mean = a.mean[rr];
    rstd = a.rstd[rr];
  };
  if (row < a.T) load(row);
  int buf = 0;
  // G > 64: every thread of the block has the same row, so barriers are met by all
  for (; row < a.T; row += step) {
    float h[NV][VEC], g[NV][VEC];
    float s0 = 0.f, s1 = 0.f;
    const float mu = mean, rs = rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Store<S>::unpack(xr[i], h[i]);
      Store<S>::unpack(gr[i], g[i]);
    }
    if (row + step < a.T) load(row + step);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (e[i] >= 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          h[i][j] = (h[i][j] - mu) * rs;
          db[i][j] += g[i][j];
          dw[i][j] += g[i][j] * h[i][j];
          g[i][j] *= w[i][j];
          s0 += j >= skip[i] ? g[i][j] : 0.f;
          s1 += j >= skip[i] ? g[i][j] * h[i][j] : 0.f;
        }
      }
    float m0, m1;
    s0 = group_sum<63>(s0);
    s1 = group_sum<63>(s1);
    if constexpr (G == 64) {
      m0 = s0;
      m1 = s1;
    } else {
      if ((threadIdx.x & 63) == 0) {
        red[buf][0][threadIdx.x >> 6] = s0;
        red[buf][1][threadIdx.x >> 6] = s1;
      }
      __syncthreads();
      m0 = m1 = 0.f;
#pragma unroll
      for (int k = 0; k < G / 64; ++k) m0 += red[buf][0][k], m1 += red[buf][1][k];
      buf ^= 1;  // the other half: a slow wave may still read this one
    }
    m0 *= inv_d;
    m1 *= inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (e[i] >= 0) {
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = rs * (g[i][j] - m0 - h[i][j] * m1);
        st16nt_u(gx + row * D + e[i], Store<S>::pack(o));
      }
  }
  if (!a.part) return;
  if constexpr (G == 64) {
    // the block's four waves add theirs up in order: a quarter of the sums to write and read back
    __shared__ float sums[R - 1][2 * NV * VEC][64];
    if (r > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          sums[r - 1][i * VEC + j][t] = dw[i][j];
          sums[r - 1][(NV + i) * VEC + j][t] = db[i][j];
        }
    }
    __syncthreads();
    if (r > 0) return;
#pragma unroll
    for (int k = 0; k < R - 1; ++k)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          dw[i][j] += sums[k][i * VEC + j][t];
          db[i][j] += sums[k][(NV + i) * VEC + j][t];
        }
  }
  // a repeated element of the last vector is the owner's to write: both hold the same sum
  float* part = a.part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (e[i] >= 0) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        part[e[i] + j] = dw[i][j];
        part[D + e[i] + j] = db[i][j];
      }
    }
}

template <typename S, typename W, int G, int NV>
__global__ __launch_bounds__(kBlockThreads<G>) void norm_bwd_kernel(NormBwdArgs a) {
  norm_bwd_rows<S, W, G, NV>(a, gridDim.x);
}

// Few rows: one launch.  dw and db need nothing of the row sums that dx does
// (mean and rstd are there), so the blocks past the rows' add up a slab of
// four vectors' columns each: lane l of a wave has vector l % 4 of row l / 4 of
// its 16; x and grad_y come from the L2 the second time.  Saves the launch of
// the sums kernel, which is as long as the work here (T = 1024, D = 256 fp32,
// forward + backward of an eager program: 27 -> 20 us).
constexpr int kSlab = 4;
template <typename S, typename W, int G, int NV>
__global__ __launch_bounds__(kBlockThreads<G>) void norm_bwd_one_kernel(NormBwdArgs a) {
  if ((int)blockIdx.x < a.row_blocks) {
    norm_bwd_rows<S, W, G, NV>(a, a.row_blocks);
    return;
  }
  constexpr int VEC = Store<S>::VEC, kWaves = kBlockThreads<G> / 64, kRows = 64 / kSlab, kStep = kRows * kWaves, kUnroll = 8;
  __shared__ float sums[kWaves][2 * VEC][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int D = a.D, nv = (D + VEC - 1) / VEC, v = (blockIdx.x - a.row_blocks) * kSlab + lane % kSlab;
  int skip;
  const int e = v < nv ? vec_start<VEC>(v, D, &skip) : -1;
  const S* x = static_cast<const S*>(a.x);
  const S* gy = static_cast<const S*>(a.gy);
  float dw[VEC] = {}, db[VEC] = {};
  for (int64_t r0 = wave * kRows + lane / kSlab; r0 < a.T; r0 += kUnroll * kStep) {
    u32x4 xr[kUnroll], gr[kUnroll];
    float mean[kUnroll], rstd[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int64_t r = r0 + k * kStep;
      xr[k] = gr[k] = {0u, 0u, 0u, 0u};
      mean[k] = rstd[k] = 0.f;
      if (e >= 0 && r < a.T) {
        xr[k] = *reinterpret_cast<const u32x4_a2*>(x + r * D + e);
        gr[k] = *reinterpret_cast<const u32x4_a2*>(gy + r * D + e);
        mean[k] = a.mean[r];
        rstd[k] = a.rstd[r];
      }
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {  // rows past the last one add zeros
      float f[VEC], g[VEC];
      Store<S>::unpack(xr[k], f);
      Store<S>::unpack(gr[k], g);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        db[j] += g[j];
        dw[j] += g[j] * ((f[j] - mean[k]) * rstd[k]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    sums[wave][j][lane] = dw[j];
    sums[wave][VEC + j][lane] = db[j];
  }
  __syncthreads();
  // thread: one of the slab's 2 x VEC x kSlab sums, over waves and rows in order
  for (int t = threadIdx.x; t < 2 * VEC * kSlab; t += kBlockThreads<G>) {
    const int j = t / kSlab, q = t % kSlab;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
      for (int r = 0; r < kRows; ++r) s += sums[w][j][r * kSlab + q];
    const int vq = (blockIdx.x - a.row_blocks) * kSlab + q;
    if (vq >= nv) continue;
    int unused;
    float* o = j < VEC ? a.gw : a.gb;
    // a column that two vectors hold has the same sum in both
    if (o) o[vec_start<VEC>(vq, D, &unused) + j % VEC] = s;
  }
}

template <typename S, typename W>
__global__ __launch_bounds__(1024) void norm_bwd_loop_kernel(NormBwdArgs a) {
  __shared__ float red[2][2][16];
  const int D = a.D;
  const float inv_d = 1.f / (float)D;
  const S* x = static_cast<const S*>(a.x);
  const S* gy = static_cast<const S*>(a.gy);
  float* part = a.part ? a.part + (int64_t)blockIdx.x * 2 * D : nullptr;
  if (part)  // zeroed before the barrier; from then on column i of both sums is thread i % 1024's
    for (int i = threadIdx.x; i < 2 * D; i += 1024) part[i] = 0.f;
  __syncthreads();
  int buf = 0;
  for (int64_t row = blockIdx.x; row < a.T; row += gridDim.x) {
    const float mu = a.mean[row], rs = a.rstd[row];
    float s0 = 0.f, s1 = 0.f;
    for (int i = threadIdx.x; i < D; i += 1024) {
      const float gv = load_elem<S>(gy, row * D + i), h = (load_elem<S>(x, row * D + i) - mu) * rs;
      const float g = gv * (a.w ? load_elem<W>(static_cast<const W*>(a.w), i) : 1.f);
      s0 += g;
      s1 += g * h;
      if (part) {
        part[i] += gv * h;
        part[D + i] += gv;
      }
    }
    const float m0 = row_sum<1024>(s0, red[buf][0]) * inv_d;
    const float m1 = row_sum<1024>(s1, red[buf][1]) * inv_d;
    buf ^= 1;
    for (int i = threadIdx.x; i < D; i += 1024) {
      const float h = (load_elem<S>(x, row * D + i) - mu) * rs;
      const float g = load_elem<S>(gy, row * D + i) * (a.w ? load_elem<W>(static_cast<const W*>(a.w), i) : 1.f);
      store_elem<S>(static_cast<S*>(a.gx), row * D + i, rs * (g - m0 - h * m1));
    }
  }
}

// Adds n rows of [2][D] sums: block = 64 columns of dw (blockIdx.y = 0) or db
// (1), 16 waves that each add every 16th row, then the waves in order.
__global__ __launch_bounds__(1024) void norm_bwd_sums_kernel(const float* part, int n, int D, float* gw, float* gb) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < D) {
    const float* p = part + (int64_t)blockIdx.y * D + c;
#pragma unroll 8
    for (int i = wave; i < n; i += 16) s += p[(int64_t)i * 2 * D];
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < D) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += red[k][lane];
    float* o = blockIdx.y ? gb : gw;
    if (o) o[c] = s;
  }
}

// ---- host -------------------------------------------------------------------

// Lanes a row and vectors a lane for rows of nv 16-byte vectors (0: the loop).
struct NormPlan {
  int G, NV;
};
NormPlan norm_plan(int64_t D, int vec, bool backward) {
  const int64_t nv = (D + vec - 1) / vec;
  // the backward holds twice the row and its columns' sums: 2048 vectors fill 512 threads' registers
  if (D < vec || nv > (backward ? 2048 : 4096)) return {0, 0};
  if (nv <= 64) return {64, 1};
  if (nv <= 128) return {64, 2};
  if (nv <= 256) return {256, 1};
  if (nv <= 512) return {256, 2};
  if (nv <= 1024) return {256, 4};
  if (backward) return {512, 4};
  if (nv <= 2048) return {1024, 2};
  return {1024, 4};
}

int vec_of(int32_t dtype) { return dtype == MHC_DTYPE_F32 ? 4 : 8; }

// Blocks a CU: the fewest whose rows in flight fill the memory's latency, by
// the vectors a thread has of each (T = 65536 bf16, forward and backward in us
// with 1, 2, 4 and 8 blocks: D = 512 103, 73, 67, 74; D = 1536 407, 240, 203,
// 204; D = 4096 535, 450, 506, 520; D = 7168 backward 525, 564 with 1 and 2;
// more blocks also mean more of the backward's sums to write and read back,
// 8 D bytes each).
int blocks_per_cu(const NormPlan& p, bool backward) {
  if (p.NV == 1) return backward ? 4 : 8;
  if (p.NV == 2 && p.G < 1024) return 2;
  return backward || p.G == 1024 ? 1 : 2;
}

int norm_bwd_blocks(int64_t T, const NormPlan& p) {
  const int rows = p.G == 64 ? 4 : 1;
  const int64_t most = (int64_t)device_cu_count() * blocks_per_cu(p, true);
  const int64_t want = (T + rows - 1) / rows;
  return (int)(want < most ? want : most);
}

template <typename S, typename W>
int launch_norm_fwd(const NormFwdArgs& a, hipStream_t st) {
  const NormPlan p = norm_plan(a.D, Store<S>::VEC, false);
  const int rows = p.G == 64 ? 4 : 1, threads = p.G == 64 ? 256 : (p.G ? p.G : 1024);
  // blocks that walk the rows; the loop form has one a row
  const int64_t want = (a.T + rows - 1) / rows, most = (int64_t)device_cu_count() * blocks_per_cu(p, false);
  const dim3 g((unsigned)(p.G && want > most ? most : want)), b(threads);
  if (const int rc = check_grid(g, b, "layer_norm")) return rc;
#define MHC_NORM(GG, NN) \
  if (p.G == GG && p.NV == NN) hipLaunchKernelGGL((norm_fwd_kernel<S, W, GG, NN>), g, b, 0, st, a)
  MHC_NORM(64, 1);
  MHC_NORM(64, 2);
  MHC_NORM(256, 1);
  MHC_NORM(256, 2);
  MHC_NORM(256, 4);
  MHC_NORM(1024, 2);
  MHC_NORM(1024, 4);
#undef MHC_NORM
  if (p.G == 0) hipLaunchKernelGGL((norm_fwd_loop_kernel<S, W>), g, b, 0, st, a);
  return check_launch("layer_norm");
}

// The one-launch form: rows that the second reading finds in the L2, few
// enough that a slab's walk over them is no longer than a launch or two.  One
// launch and two, us in a replayed graph: fp32 D = 256 T = 1024 4.3, 5.6, T = 2048
// 6.5, 6.9, T = 4096 11.1, 10.3; bf16 D = 256 T = 1536 6.7, 6.7, T = 2048 8.5, 7.3;
// fp16 D = 1003 T = 1536 10.8, 11.0, T = 2048 16.5, 12.4.  By bytes of x and grad_y:
// bf16 D = 4096 8 MB 5.5, 24.8, 16 MB 14.6, 25.5; fp32 D = 2048 16 MB 13.8, 14.4, 24 MB
// 24.4, 16.4 (the limit leaves what one launch would gain up to 16 MB).
bool norm_bwd_in_one(int64_t T, int64_t D, size_t es, const NormPlan& p) {
  return p.G > 0 && T <= 1536 && 2 * T * D * (int64_t)es <= (8 << 20);
}

template <typename S, typename W>
int launch_norm_bwd(NormBwdArgs a, float* gw, float* gb, hipStream_t st) {
  const NormPlan p = norm_plan(a.D, Store<S>::VEC, true);
  if (a.part && norm_bwd_in_one(a.T, a.D, sizeof(S), p)) {
    a.part = nullptr;
    a.gw = gw, a.gb = gb;
    const int rows = p.G == 64 ? 4 : 1;
    const int64_t want = (a.T + rows - 1) / rows, most = (int64_t)device_cu_count() * 8;
    a.row_blocks = (int)(want < most ? want : most);
    const int slabs = (a.D + kSlab * Store<S>::VEC - 1) / (kSlab * Store<S>::VEC);
    const dim3 g(a.row_blocks + slabs), b(p.G == 64 ? 256 : p.G);
#define MHC_NORM(GG, NN) \
  if (p.G == GG && p.NV == NN) hipLaunchKernelGGL((norm_bwd_one_kernel<S, W, GG, NN>), g, b, 0, st, a)
    MHC_NORM(64, 1);
    MHC_NORM(64, 2);
    MHC_NORM(256, 1);
    MHC_NORM(256, 2);
    MHC_NORM(256, 4);
    MHC_NORM(512, 4);
#undef MHC_NORM
    return check_launch("layer_norm_backward");
  }
  const int blocks = norm_bwd_blocks(a.T, p), threads = p.G == 64 ? 256 : (p.G ? p.G : 1024);
  const dim3 g(blocks), b(threads);
#define MHC_NORM(GG, NN) \
  if (p.G == GG && p.NV == NN) hipLaunchKernelGGL((norm_bwd_kernel<S, W, GG, NN>), g, b, 0, st, a)
  MHC_NORM(64, 1);
  MHC_NORM(64, 2);
  MHC_NORM(256, 1);
  MHC_NORM(256, 2);
  MHC_NORM(256, 4);
  MHC_NORM(512, 4);
#undef MHC_NORM
  if (p.G == 0) hipLaunchKernelGGL((norm_bwd_loop_kernel<S, W>), g, b, 0, st, a);
  if (const int rc = check_launch("layer_norm_backward")) return rc;
  if (a.part) {
    const dim3 sg((unsigned)((a.D + 63) / 64), 2);
    hipLaunchKernelGGL(norm_bwd_sums_kernel, sg, dim3(1024), 0, st, a.part, blocks, a.D, gw, gb);
    return check_launch("layer_norm_backward sums");
  }
  return MHC_OK;
}

// The loop kernels count a row's elements, and the backward's two sums of
// each, in 32 bits and steps of 1024.
constexpr int32_t kMaxRow = (1 << 30) - 512;

bool known_dtype(int32_t d) { return d == MHC_DTYPE_F32 || d == MHC_DTYPE_BF16 || d == MHC_DTYPE_F16; }

int check_norm(const char* who, int64_t T, int64_t D, int32_t x_dtype, int32_t w_dtype) {
  if (T < 0 || D < 1) return set_error(MHC_ERR_INVALID, "%s: T=%lld D=%lld", who, (long long)T, (long long)D);
  if (D > kMaxRow)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: rows of %lld elements, above the supported %d", who, (long long)D, kMaxRow);
  if (const int rc = check_tokens(T, who)) return rc;
  if (!known_dtype(x_dtype)) return set_error(MHC_ERR_UNSUPPORTED, "%s: dtype %d not supported", who, x_dtype);
  if (w_dtype != x_dtype && w_dtype != MHC_DTYPE_F32)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: weight dtype %d is neither the rows' nor fp32", who, w_dtype);
  return MHC_OK;
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" int mhc_layer_norm_fwd(const void* x, int32_t x_dtype, const void* weight, const void* bias,
                                  int32_t w_dtype, float eps, void* y, float* mean, float* rstd, int64_t T,
                                  int32_t D, void* stream) {
  clear_error();
  if (const int rc = check_norm("layer_norm", T, D, x_dtype, w_dtype)) return rc;
  if (!mean != !rstd) return set_error(MHC_ERR_INVALID, "layer_norm: mean and rstd go together");
  if (T == 0) return MHC_OK;
  if (!x || !y) return set_error(MHC_ERR_INVALID, "layer_norm: null pointer");
  const NormFwdArgs a = {x, weight, bias, y, mean, rstd, T, D, eps};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (x_dtype == MHC_DTYPE_F32) return launch_norm_fwd<float, float>(a, st);
  if (x_dtype == MHC_DTYPE_BF16)
    return w_dtype == MHC_DTYPE_F32 ? launch_norm_fwd<bf16_t, float>(a, st) : launch_norm_fwd<bf16_t, bf16_t>(a, st);
  return w_dtype == MHC_DTYPE_F32 ? launch_norm_fwd<f16_t, float>(a, st) : launch_norm_fwd<f16_t, f16_t>(a, st);
}

extern "C" size_t mhc_layer_norm_bwd_workspace_size(int64_t T, int32_t D, int32_t x_dtype) {
  if (T <= 0 || D < 1 || D > kMaxRow || T > kMaxTokens || !known_dtype(x_dtype)) return 0;
  return (size_t)norm_bwd_blocks(T, norm_plan(D, vec_of(x_dtype), true)) * 2 * (size_t)D * sizeof(float);
}

extern "C" int mhc_layer_norm_bwd(const void* grad_y, const void* x, int32_t x_dtype, const void* weight,
                                  int32_t w_dtype, const float* mean, const float* rstd, void* grad_x,
                                  float* grad_weight, float* grad_bias, void* workspace, size_t workspace_bytes,
                                  int64_t T, int32_t D, void* stream) {
  clear_error();
  if (const int rc = check_norm("layer_norm_backward", T, D, x_dtype, w_dtype)) return rc;
  if (T == 0) return MHC_OK;
  if (!grad_y || !x || !mean || !rstd || !grad_x)
    return set_error(MHC_ERR_INVALID, "layer_norm_backward: null pointer");
  const bool sums = grad_weight || grad_bias;
  const size_t need = mhc_layer_norm_bwd_workspace_size(T, D, x_dtype);
  if (sums && (!workspace || workspace_bytes < need))
    return set_error(MHC_ERR_INVALID, "layer_norm_backward: workspace too small (%zu < %zu bytes)",
                     workspace ? workspace_bytes : (size_t)0, need);
  const NormBwdArgs a = {nullptr, nullptr, 0, grad_y, x, weight, mean, rstd, grad_x, sums ? static_cast<float*>(workspace) : nullptr, T, D};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (x_dtype == MHC_DTYPE_F32) return launch_norm_bwd<float, float>(a, grad_weight, grad_bias, st);
  if (x_dtype == MHC_DTYPE_BF16)
    return w_dtype == MHC_DTYPE_F32 ? launch_norm_bwd<bf16_t, float>(a, grad_weight, grad_bias, st)
                                    : launch_norm_bwd<bf16_t, bf16_t>(a, grad_weight, grad_bias, st);
  return w_dtype == MHC_DTYPE_F32 ? launch_norm_bwd<f16_t, float>(a, grad_weight, grad_bias, st)
                                  : launch_norm_bwd<f16_t, f16_t>(a, grad_weight, grad_bias, st);
}
