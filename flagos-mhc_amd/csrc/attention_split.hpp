// Attention forward for few queries: single tokens over a cache, short chunks
// over long contexts.
//
// Rows are (query, head of the group) pairs, so that a key head's keys and
// values are read once for every head that shares them.  A block takes 32
// rows and one part of their keys, its four waves every fourth tile of 32
// keys of that part; their sums meet in LDS at the end.  Where there are too
// few rows for the GPU the keys are split further over blocks, and a second
// kernel joins the parts, in their order.  A wave keeps its tile of keys in
// registers, loaded as the operand it is, and turns the values through 8 KB
// of LDS of its own: no wave waits for another, and 16 KB a wave are in
// flight while it computes.
//
// Reading the cache bounds it: 64 sequences of up to 8192 keys, 32 heads of 128
// over 8, bf16: 286 us, 5.6 TB/s; one of 32768: 26 us, 5.2 TB/s, and 4 us for
// the join (medians; a copy of large tensors moves 4.96 TB/s, read and written).
#pragma once

#include "attention.hpp"
#include "attention_bwd.hpp"
#include "attention_fwd.hpp"

namespace mhc {

constexpr int kSplitWaves = 4;

// Bytes of LDS: a wave's tile of values, later its sums.
template <typename S, int DB>
constexpr size_t split_lds() {
  constexpr size_t tile = 32 * Tile<S, DB>::kPitch, sums = DB * 4096;
  return kSplitWaves * ((tile > sums ? tile : sums) + 32 * 2 * 4);
}

// Tile of 32 rows (query * G + head of the group) that slot `slot` stands for:
// its sequence and first row (lq * G or more: nothing to do).
__device__ __forceinline__ AttSeq group_tile(const AttDims& n, int64_t slot, int64_t& first) {
  const int G = n.H / n.Hk;
  if (!n.cu_q) {
    const int64_t per = ((int64_t)n.Sq * G + 31) / 32;
    first = slot % per * 32;
    return att_seq(n, (int)(slot / per));
  }
  // the slots of tiles of 32 of G rows a query, as slot_sequence's
  const int lane = threadIdx.x & 63;
  int lo = 0, m = n.B + 1;
  while (m > 1) {
    const int step = (m + 63) / 64, c = lane * step;
    int hit = __popcll(__ballot(c < m && cu_at(n.cu_q, lo + c, n.Tq) * G / 32 + lo + c <= slot));
    hit = hit < 1 ? 1 : hit;
    const int skip = (hit - 1) * step;
    lo += skip;
    m = m - skip < step ? m - skip : step;
  }
  const int b = __builtin_amdgcn_readfirstlane(lo);
  const AttSeq s = att_seq(n, b);
  first = (slot - (s.row0 * G / 32 + b)) * 32;
  if (first < 0) first = (int64_t)s.lq * G;  // (decreasing starts)
  return s;
}

// A lane's own row as fragments; zero if there is none.
template <typename S, int DB>
__device__ __forceinline__ void lane_row(const char* p, bool live, int d_chunks, int lane, u32x4 (&f)[Tile<S, DB>::kSteps]) {
#pragma unroll
  for (int t = 0; t < Tile<S, DB>::kSteps; ++t) {
    const int c = 2 * t + (lane >> 5);
    f[t] = u32x4{0u, 0u, 0u, 0u};
    if (live && c < d_chunks) f[t] = ld16(p + c * 16);
  }
}

template <typename S, int DB, int WPE>
__global__ __launch_bounds__(64 * kSplitWaves, WPE) void att_split_kernel(AttArgs a, int64_t slots, int splits) {
  using T = Tile<S, DB>;
  constexpr int ES = (int)sizeof(S);
  constexpr size_t kRegion = split_lds<S, DB>() / kSplitWaves - 256;
  extern __shared__ __attribute__((aligned(256))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  // the parts of one tile of rows lie side by side: they read neighbouring keys
  const int64_t item = blockIdx.x;
  const int part = (int)(item % splits);
  const int hk = (int)(item / splits % a.n.Hk);
  const int64_t slot = item / splits / a.n.Hk;
  const int G = a.n.H / a.n.Hk, d = a.n.d, dc = d * ES / 16;
  int64_t first;  // first row (query * G + head)
  const AttSeq s = group_tile(a.n, slot, first);
  if (first >= (int64_t)s.lq * G) return;
  const int64_t r = first + (lane & 31);
  const int i = (int)(r / G), g = (int)(r % G), h = hk * G + g;
  const bool live = i < s.lq;
  const int64_t orow = (s.row0 + i) * a.n.H + h;
  const int shift = s.lk - s.lq;
  const int lim = s.none || !live ? -1 : (a.n.causal ? min(s.lk - 1, i + shift) : s.lk - 1);
  // the block's part of the keys that its last row sees
  const int last = (int)min((int64_t)s.lq - 1, (first + 31) / G);
  const int keys = s.none ? 0 : max(0, a.n.causal ? min(s.lk, last + shift + 1) : s.lk);
  const int chunk = ((keys + splits - 1) / splits + 31) / 32 * 32;
  const int from = (int)min((int64_t)keys, (int64_t)part * chunk), to = min(keys, from + chunk);
  const int tiles = (to - from + 31) / 32;

  u32x4 q[T::kSteps];
  lane_row<S, DB>(row_ptr(a.q, a.n.cu_q, s.row0, s.b, live ? i : 0, h, ES), live && !s.none, dc, lane, q);
  const int k_ts = (int)(a.k.ts * ES), v_ts = (int)(a.v.ts * ES);
  const char* kp = row_ptr(a.k, a.n.cu_k, s.k0, s.b, from, hk, ES);
  const char* vp = row_ptr(a.v, a.n.cu_k, s.k0, s.b, from, hk, ES);
  char* mine = smem + wave * kRegion;
  const uint32_t tile = lds_addr(mine);

  floatx16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[db][j] = 0.f;
  float m = -__builtin_inff(), l = 0.f;
  const float c = a.scale2;
  u32x4 k[T::kSteps];
  TileStage<S, DB, 32, 64> sv;
  const uint32_t v_off = sv.offset(v_ts, dc, lane);
  T at(lane);
  const int have = to - from;
  // tiles from here on are hidden from some of the rows
  const int zone = a.n.causal ? max(0, (int)(first / G) + shift + 1) : 0x7fffffff;
  bool bad = false;
  if (wave < tiles) {
    load_rows<S, DB>(kp + (int64_t)wave * 32 * k_ts, k_ts, have - wave * 32, dc, lane, k);
    sv.load(vp + (int64_t)wave * 32 * v_ts, v_ts, have - wave * 32, v_off);
  }
  for (int t = wave; t < tiles; t += kSplitWaves) {
    const int next = t + kSplitWaves, k0 = from + t * 32;
    at.keep();
    int ln = lane;
    asm volatile("" : "+v"(ln));
    floatx16 sc;
#pragma unroll
    for (int j = 0; j < 16; ++j) sc[j] = 0.f;
#pragma unroll
    for (int u = 0; u < T::kSteps; ++u) sc = Mma32<S>::fma(k[u], q[u], sc);
    if (next < tiles) load_rows<S, DB>(kp + (int64_t)next * 32 * k_ts, k_ts, have - next * 32, dc, lane, k);
    const int left = min(lim, to - 1) - k0 - 4 * half;
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      sc[j] = acc_row(j, 0) <= left ? sc[j] : -__builtin_inff();
      top = fmaxf(top, sc[j]);
    }
    top = max_xor32(top) * c - kBelowMax<S>;
    if (__any(top > m + kLazyMax || m == -__builtin_inff())) {
      const float mn = fmaxf(m, top);
      const float f = mn == -__builtin_inff() ? 1.f : hw_exp2(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[db][j] *= f;
    }
    const float ref = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      sc[j] = hw_exp2(__builtin_fmaf(sc[j], c, -ref));
      l += sc[j];
    }
    u32x4 p[1][T::kColSteps];
#pragma unroll
    for (int u = 0; u < T::kColSteps; ++u) p[0][u] = acc_frag<S>(sc, u);
    if (k0 + 32 > zone) bad |= sv.clean();
    sv.store(tile, ln & 63);
    if (next < tiles) sv.load(vp + (int64_t)next * 32 * v_ts, v_ts, have - next * 32, v_off);
    add_columns<S, DB, 1>(acc, at, tile, p);
  }

  // the four waves' sums, each from its own reference point to the largest
  float* stats = reinterpret_cast<float*>(smem + kSplitWaves * kRegion);
  l = add_xor32(l);
  if (lane < 32) {
    stats[wave * 64 + lane] = m;
    stats[wave * 64 + 32 + lane] = l;
  }
  bad = __syncthreads_or(bad);
  float top = m, sum = 0.f;
#pragma unroll
  for (int w = 0; w < kSplitWaves; ++w) top = fmaxf(top, stats[w * 64 + (lane & 31)]);
  const float ref = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
  for (int w = 0; w < kSplitWaves; ++w) sum += stats[w * 64 + 32 + (lane & 31)] * hw_exp2(stats[w * 64 + (lane & 31)] - ref);
  const float f = hw_exp2(m - ref);
  float* region = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int j = 0; j < 16; ++j) region[(db * 16 + j) * 64 + lane] = acc[db][j] * f;
  __syncthreads();
  const float inv = splits > 1 ? 1.f : (sum == 0.f ? 0.f : 1.f / sum);
  if (splits > 1) {
    float* ml = a.part + (int64_t)splits * a.n.Tq * a.n.H * d;
    const int64_t to_ml = (int64_t)part * a.n.Tq * a.n.H + orow;
    if (wave == 0 && live && lane < 32) {
      ml[2 * to_ml] = top;
      ml[2 * to_ml + 1] = sum;
    }
  } else if (a.lse && wave == 0 && live && lane < 32) {
    a.lse[(int64_t)h * a.n.Tq + s.row0 + i] = sum == 0.f ? -__builtin_inff() : top * kLn2 + logf(sum);
  }
  for (int db = wave; db < DB; db += kSplitWaves) {
    floatx16 z[1];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kSplitWaves; ++w) v += reinterpret_cast<const float*>(smem + w * kRegion)[(db * 16 + j) * 64 + lane];
      z[0][j] = v;
    }
    if (bad) {
      // the parts' tiles of 32 begin at `from`
      const int z0 = from + max(0, zone - from) / 32 * 32;
      add_nonfinite<S, 1, false>(z, vp + (int64_t)(z0 - from) * v_ts + 32 * db * ES, v_ts, to - z0, d - 32 * db, lane,
                                 [&](int row) { return z0 + row <= lim; });
    }
    if (splits > 1)
      store_rows<float, 1>(z, 1.f, a.part + ((int64_t)part * a.n.Tq * a.n.H + orow) * d + 32 * db, live, d - 32 * db, lane);
    else
      store_rows<S, 1>(z, inv, static_cast<S*>(a.out) + orow * d + 32 * db, live, d - 32 * db, lane);
  }
}

// dq, and D, for the same rows: a backward of few queries, or of too few blocks
// of 128.  Each of the four waves adds what its tiles of keys give; the four
// sums meet in LDS.  k is turned through LDS, v comes as the operand it is.
template <typename S, int DB, int WPE>
__global__ __launch_bounds__(64 * kSplitWaves, WPE) void att_dq_split_kernel(AttArgs a, int64_t slots) {
  using T = Tile<S, DB>;
  constexpr int ES = (int)sizeof(S);
  constexpr size_t kRegion = split_lds<S, DB>() / kSplitWaves - 256;
  extern __shared__ __attribute__((aligned(256))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int hk = (int)(blockIdx.x % a.n.Hk);
  const int64_t slot = slots - 1 - blockIdx.x / a.n.Hk;
  const int G = a.n.H / a.n.Hk, d = a.n.d, dc = d * ES / 16;
  int64_t first;
  const AttSeq s = group_tile(a.n, slot, first);
  if (first >= (int64_t)s.lq * G) return;
  const int64_t r = first + (lane & 31);
  const int i = (int)(r / G), h = hk * G + (int)(r % G);
  const bool live = i < s.lq;
  const int64_t orow = (s.row0 + i) * a.n.H + h, stat = (int64_t)h * a.n.Tq + s.row0 + i;
  const int shift = s.lk - s.lq;
  const int lim = s.none || !live ? -1 : (a.n.causal ? min(s.lk - 1, i + shift) : s.lk - 1);
  const int last = (int)min((int64_t)s.lq - 1, (first + 31) / G);
  const int keys = s.none ? 0 : max(0, a.n.causal ? min(s.lk, last + shift + 1) : s.lk);
  const int tiles = (keys + 31) / 32;

  u32x4 q[T::kSteps], go[T::kSteps];
  const bool load = live && !s.none;
  const int at_row = live ? i : 0;
  lane_row<S, DB>(row_ptr(a.q, a.n.cu_q, s.row0, s.b, at_row, h, ES), load, dc, lane, q);
  lane_row<S, DB>(row_ptr(a.go, a.n.cu_q, s.row0, s.b, at_row, h, ES), load, dc, lane, go);
  const int sum = keys <= kSumKeys ? tiles : 0;  // as in att_dq_kernel
  float delta = 0.f;
  if (sum == 0) {
    u32x4 o[T::kSteps];
    lane_row<S, DB>(row_ptr(a.o, a.n.cu_q, s.row0, s.b, at_row, h, ES), load, dc, lane, o);
#pragma unroll
    for (int t = 0; t < T::kSteps; ++t) {
      float x[Store<S>::VEC], y[Store<S>::VEC];
      Store<S>::unpack(o[t], x);
      Store<S>::unpack(go[t], y);
#pragma unroll
      for (int j = 0; j < Store<S>::VEC; ++j) delta = __builtin_fmaf(x[j], y[j], delta);
    }
    delta = add_xor32(delta);
    if (live && wave == 0 && lane < 32) a.delta[stat] = delta;
  }
  const float lse = load ? a.lse[stat] : -__builtin_inff();
  const float lse2 = lse == -__builtin_inff() ? __builtin_inff() : lse * kLog2e;

  const int k_ts = (int)(a.k.ts * ES), v_ts = (int)(a.v.ts * ES);
  const char* kp = row_ptr(a.k, a.n.cu_k, s.k0, s.b, 0, hk, ES);
  const char* vp = row_ptr(a.v, a.n.cu_k, s.k0, s.b, 0, hk, ES);
  const uint32_t tile = lds_addr(smem) + wave * kRegion;
  const int zone = a.n.causal ? max(0, (int)(first / G) + shift + 1) : 0x7fffffff;
  bool bad = false;
  floatx16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[db][j] = 0.f;
  const float c = a.scale2;
  u32x4 v[T::kSteps];
  TileStage<S, DB, 32, 64> sk;
  const uint32_t k_off = sk.offset(k_ts, dc, lane);
  T at(lane);
  // tile t's dS (P (go v^T) while delta is 0); the next tile's loads are begun on the way
  const auto first_loads = [&]() {
    if (wave >= tiles) return;
    sk.load(kp + (int64_t)wave * 32 * k_ts, k_ts, s.lk - wave * 32, k_off);
    load_rows<S, DB>(vp + (int64_t)wave * 32 * v_ts, v_ts, s.lk - wave * 32, dc, lane, v);
  };
  const auto scores = [&](int t) __attribute__((always_inline)) {
    const int next = t + kSplitWaves, k0 = t * 32;
    at.keep();
    int ln = lane;
    asm volatile("" : "+v"(ln));
    if (k0 + 32 > zone) bad |= sk.clean();
    sk.store(tile, ln & 63);
    if (next < tiles) sk.load(kp + (int64_t)next * 32 * k_ts, k_ts, s.lk - next * 32, k_off);
    floatx16 dp;
#pragma unroll
    for (int j = 0; j < 16; ++j) dp[j] = 0.f;
#pragma unroll
    for (int u = 0; u < T::kSteps; ++u) dp = Mma32<S>::fma(v[u], go[u], dp);
    if (next < tiles) load_rows<S, DB>(vp + (int64_t)next * 32 * v_ts, v_ts, s.lk - next * 32, dc, lane, v);
    const floatx16 sc = row_products<S, DB>(at, tile, 0, q);
    const int left = lim - k0 - 4 * half;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float x = hw_exp2(__builtin_fmaf(sc[j], c, -lse2)) * (dp[j] - delta);
      dp[j] = acc_row(j, 0) <= left ? x : 0.f;
    }
    return dp;
  };
  first_loads();
  if (sum) {
    float total = 0.f;
    for (int t = wave; t < tiles; t += kSplitWaves) {
      const floatx16 x = scores(t);
#pragma unroll
      for (int j = 0; j < 16; ++j) total += x[j];
    }
    first_loads();
    float* sums = reinterpret_cast<float*>(smem + kSplitWaves * kRegion);
    total = add_xor32(total);
    if (lane < 32) sums[wave * 32 + lane] = total;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSplitWaves; ++w) delta += sums[w * 32 + (lane & 31)];
    if (live && wave == 0 && lane < 32) a.delta[stat] = delta;
  }
  Lift<S> lift;
  for (int t = wave; t < tiles; t += kSplitWaves) {
    floatx16 dp = scores(t);
    lift.template fit<WPE == 1>(dp, acc);
    u32x4 p[1][T::kColSteps];
#pragma unroll
    for (int u = 0; u < T::kColSteps; ++u) p[0][u] = acc_frag<S>(dp, u);
    add_columns<S, DB, 1>(acc, at, tile, p);
  }

  bad = __syncthreads_or(bad);
  float* region = reinterpret_cast<float*>(smem + wave * kRegion);
  const float back = lift.back();
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int j = 0; j < 16; ++j) region[(db * 16 + j) * 64 + lane] = acc[db][j] * back;
  __syncthreads();
  for (int db = wave; db < DB; db += kSplitWaves) {
    floatx16 z[1];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kSplitWaves; ++w) x += reinterpret_cast<const float*>(smem + w * kRegion)[(db * 16 + j) * 64 + lane];
      z[0][j] = x;
    }
    if (bad) {
      // whole rows become NaN: every column of the row is looked at, this block of 32 written
      const int z0 = zone / 32 * 32;
      for (int row = 0; row < keys - z0; ++row) {
        float any = 0.f;
        for (int e = 0; e < d; ++e) {
          const float x = load_elem<S>(reinterpret_cast<const S*>(kp + (int64_t)(z0 + row) * k_ts), e);
          any = (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? 1.f : any;
        }
        if (any != 0.f && z0 + row <= lim) {
#pragma unroll
          for (int j = 0; j < 16; ++j) z[0][j] = __builtin_nanf("");
        }
      }
    }
    store_rows<S, 1>(z, a.scale, static_cast<S*>(a.out) + orow * d + 32 * db, live, d - 32 * db, lane);
  }
}

// out = sum over parts of 2^(m - M) O / sum of 2^(m - M) l: a block a row and
// head (or every so many of them, where a dispatch holds fewer blocks), 16, 32
// or 64 lanes a part (four elements each), so that 4 to 16 parts are read at a
// time; their sums meet in LDS, always in the same order.
template <typename S>
__global__ __launch_bounds__(256) void att_join_kernel(AttArgs a, int64_t rows, int splits) {
  __shared__ float sums[256 * 5];
  const int tid = threadIdx.x, lane = tid & 63;
  const int d = a.n.d, per = d <= 64 ? 16 : (d <= 128 ? 32 : 64), groups = 256 / per;
  const int mine = tid / per, e = tid % per * 4;
  const float* ml = a.part + (int64_t)splits * rows * d;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {  // (row of q, head)
    float top = -__builtin_inff();
    for (int p = lane; p < splits; p += 64) top = fmaxf(top, ml[2 * ((int64_t)p * rows + row)]);
    top = group_max<63>(top);
    const float ref = top == -__builtin_inff() ? 0.f : top;
    float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int kAhead = 4;
    for (int p0 = mine; p0 < splits; p0 += groups * kAhead) {
      float m[kAhead], l[kAhead];
      floatx4 o[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int p = p0 + u * groups;
        const int64_t at = (int64_t)(p < splits ? p : p0) * rows + row;
        m[u] = ml[2 * at];
        l[u] = p < splits ? ml[2 * at + 1] : 0.f;
        o[u] = e < d ? *reinterpret_cast<const floatx4*>(a.part + at * d + e) : floatx4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (l[u] == 0.f) continue;  // no keys in this part: it left its sums as they were
        const float f = hw_exp2(m[u] - ref);
        sum += l[u] * f;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += o[u][j] * f;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[j * 256 + tid] = v[j];
    sums[1024 + tid] = sum;
    __syncthreads();
    if (tid < per) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = 0.f;
      sum = 0.f;
      for (int g = 0; g < groups; ++g) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += sums[j * 256 + g * per + tid];
        sum += sums[1024 + g * per + tid];
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      S* out = static_cast<S*>(a.out) + row * d + e;
      if (e < d) {
#pragma unroll
        for (int j = 0; j < 4; ++j) store_elem<S>(out, j, v[j] * inv);
      }
      if (a.lse && tid == 0)
        a.lse[row % a.n.H * a.n.Tq + row / a.n.H] = sum == 0.f ? -__builtin_inff() : top * kLn2 + logf(sum);
    }
    __syncthreads();  // the sums are read before the next row's are written
  }
}

}  // namespace mhc
