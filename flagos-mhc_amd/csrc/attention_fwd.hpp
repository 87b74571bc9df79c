// Attention forward: a block takes 32 NW / KS queries of one head, a wave 32 of
// them, and walks the keys they see in tiles of 32 NB, one pass with a running
// maximum and sum.
//
// Keys and values go through registers to LDS one tile ahead, in the rows they
// have in memory: k is read back as rows (first operand of K Q^T), v as columns
// (of V^T P^T) with the transposing read, so nothing is turned in memory.  What
// bounds it is the matrix instructions together with the exponentials between
// them (16 a product of 32 x 32, at a quarter of the others' rate): two waves a
// SIMD unit take turns.  32768 tokens, 32 heads of 128 over 8, causal, bf16:
// 8.2 and 8.5 ms (medians on two cards), 1.07 and 1.03 PFLOP/s (a large library
// product reaches 1.42); with the loads of keys and values left out it is 17 %
// faster.
//
// KS = 2: two waves share 32 queries, each takes every other
// tile, and their sums meet at the end: a long row is done in half the steps,
// which is what a call of few blocks waits for.
#pragma once

#include "attention.hpp"

namespace mhc {

// Items (tile of queries, head): an XCD walks a contiguous run of key heads, so
// that the blocks it runs at a time read the same keys and values from its L2;
// within a key head the tiles go from the last to the first, each for all heads
// of the group, since under a causal mask the last ones are the longest.
__device__ __forceinline__ void att_item(const AttDims& n, int64_t slots, int64_t& slot, int& h) {
  const int64_t item = xcd_contig(blockIdx.x, gridDim.x);
  const int G = n.H / n.Hk;
  const int64_t of = item / G;
  h = (int)(of / slots) * G + (int)(item % G);
  slot = slots - 1 - of % slots;
}

template <typename S, int DB>
__device__ __forceinline__ void store_none(S* row, bool live, int d, int lane) {
  floatx16 z[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) z[db][i] = 0.f;
  store_rows<S, DB>(z, 0.f, row, live, d, lane);
}

template <typename S, int DB, int NW, int KS, int NB, int WPE>
__global__ __launch_bounds__(64 * NW, WPE) void att_fwd_kernel(AttArgs a, int64_t slots) {
  using T = Tile<S, DB>;
  constexpr int RW = NW / KS, BN = 32 * NB, BS = BN * KS, BM = 32 * RW, NT = 64 * NW, ES = (int)sizeof(S);
  constexpr int kTileBytes = BS * T::kPitch;  // KS tiles
  extern __shared__ __attribute__((aligned(256))) char smem[];  // 2 x (K, V); at the end the sums of KS - 1 waves a row
  const int tid = threadIdx.x, lane = tid & 63, id = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave = id % RW, part = id / RW;
  int64_t slot;
  int h, first;
  att_item(a.n, slots, slot, h);
  const AttSeq s = q_tile(a.n, slot, BM, first);
  if (first >= s.lq) return;
  const int hk = h / (a.n.H / a.n.Hk), d = a.n.d, dc = d * ES / 16;
  const int row = first + 32 * wave + (lane & 31);  // the lane's query
  const bool live = row < s.lq;
  S* out = static_cast<S*>(a.out) + ((s.row0 + row) * a.n.H + h) * (int64_t)d;
  const int shift = s.lk - s.lq;
  // keys that the block's last query sees, and this lane's
  const int block_last = (first + BM < s.lq ? first + BM : s.lq) - 1;
  const int keys = s.none ? 0 : (a.n.causal ? min(s.lk, block_last + shift + 1) : s.lk);
  if (keys <= 0) {
    store_none<S, DB>(out, live, d, lane);
    if (a.lse && live && lane < 32) a.lse[(int64_t)h * a.n.Tq + s.row0 + row] = -__builtin_inff();
    return;
  }
  const int lim = a.n.causal ? min(s.lk - 1, row + shift) : s.lk - 1;  // last key the lane sees
  const int wave_first = first + 32 * wave;
  const int wave_lo = a.n.causal ? min(s.lk - 1, wave_first + shift) : s.lk - 1;       // seen by all of the wave
  const int wave_hi = a.n.causal ? min(s.lk - 1, wave_first + 31 + shift) : s.lk - 1;  // by any

  const int q_ts = (int)(a.q.ts * ES), k_ts = (int)(a.k.ts * ES), v_ts = (int)(a.v.ts * ES);
  u32x4 q[T::kSteps];
  load_rows<S, DB>(row_ptr(a.q, a.n.cu_q, s.row0, s.b, wave_first, h, ES), q_ts, s.lq - wave_first, dc, lane, q);
  const char* kp = uniform(row_ptr(a.k, a.n.cu_k, s.k0, s.b, 0, hk, ES));
  const char* vp = uniform(row_ptr(a.v, a.n.cu_k, s.k0, s.b, 0, hk, ES));
  const int lk = __builtin_amdgcn_readfirstlane(s.lk);
  const int64_t k_step = (int64_t)BS * k_ts, v_step = (int64_t)BS * v_ts;

  TileStage<S, DB, BS, NT> sk, sv;
  uint32_t k_off = sk.offset(k_ts, dc, tid), v_off = sv.offset(v_ts, dc, tid);
  const uint32_t lds = lds_addr(smem);
  sk.load(kp, k_ts, lk, k_off);
  sv.load(vp, v_ts, lk, v_off);
  // tiles with keys from here on are hidden from some of the block's queries
  const int zone = a.n.causal ? max(0, first + shift + 1) : 0x7fffffff;
  bool bad = false;
  auto stage = [&](int t) {
    if ((t + 1) * BS > zone) bad |= sv.clean();
    const uint32_t to = lds + (t & 1) * 2 * kTileBytes;
    sk.store(to, tid);
    sv.store(to + kTileBytes, tid);
  };
  stage(0);
  __syncthreads();
  T at(lane);

  floatx16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
  float m = -__builtin_inff(), l = 0.f;  // reference point (powers of two) and the lane's share of the sum
  const float c = a.scale2;
  const int tiles = (keys + BS - 1) / BS, half = lane >> 5;
  for (int t = 0; t < tiles; ++t) {
    const uint32_t tk = lds + (t & 1) * 2 * kTileBytes + part * BN * T::kPitch, tv = tk + kTileBytes;
    at.keep();
    const int k0 = t * BS + part * BN;
    if (t + 1 < tiles) {
      sk.load(kp + (t + 1) * k_step, k_ts, lk - (t + 1) * BS, k_off);
      sv.load(vp + (t + 1) * v_step, v_ts, lk - (t + 1) * BS, v_off);
    }
    if (k0 <= wave_hi) {
      floatx16 sc[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) sc[b] = row_products<S, DB>(at, tk, b, q);
      const bool masked = k0 + BN - 1 > wave_lo;
      if (masked) {
        stay();
        const int left = lim - k0 - 4 * half;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[b][i] = 32 * b + acc_row(i, 0) <= left ? sc[b][i] : -__builtin_inff();
      }
      float top = sc[0][0];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[b][i]);
      top = max_xor32(top) * c - kBelowMax<S>;
      if (__any(top > m + kLazyMax || m == -__builtin_inff())) {
        const float mn = fmaxf(m, top);
        const float f = mn == -__builtin_inff() ? 1.f : hw_exp2(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[db][i] *= f;
      }
      const float ref = m == -__builtin_inff() ? 0.f : m;
      u32x4 p[NB][T::kColSteps];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sc[b][i] = hw_exp2(__builtin_fmaf(sc[b][i], c, -ref));
          l += sc[b][i];
        }
        // p is rounded to the type of v, the sum is of the unrounded values
#pragma unroll
        for (int u = 0; u < T::kColSteps; ++u) p[b][u] = acc_frag<S>(sc[b], u);
      }
      add_columns<S, DB, NB>(acc, at, tv, p);
    }
    if (t + 1 < tiles) {
      stage(t + 1);
      __syncthreads();
    }
  }
  bad = __syncthreads_or(bad);
  if constexpr (KS == 2) {
    // the second wave's sums to the first, both from the larger reference point
    float* other = reinterpret_cast<float*>(smem) + wave * (DB * 16 + 2) * 64 + lane;
    if (part == 1) {
      other[0] = m;
      other[64] = l;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) other[(2 + db * 16 + i) * 64] = acc[db][i];
    }
    __syncthreads();
    if (part == 1) return;
    const float m1 = other[0], top = fmaxf(m, m1), ref = top == -__builtin_inff() ? 0.f : top;
    const float f0 = hw_exp2(m - ref), f1 = hw_exp2(m1 - ref);
    m = top;
    l = l * f0 + other[64] * f1;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] = acc[db][i] * f0 + other[(2 + db * 16 + i) * 64] * f1;
  }
  if (bad) {
    const int z = zone / BS * BS;
    add_nonfinite<S, DB, false>(acc, vp + (int64_t)z * v_ts, v_ts, keys - z, d, lane, [&](int r) { return z + r <= lim; });
  }
  l = add_xor32(l);
  // (a NaN among the scores leaves l NaN: not the empty row's zero)
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  store_rows<S, DB>(acc, inv, out, live, d, lane);
  if (a.lse && live && lane < 32)
    a.lse[(int64_t)h * a.n.Tq + s.row0 + row] = l == 0.f ? -__builtin_inff() : m * kLn2 + __logf(l);
}

}  // namespace mhc
