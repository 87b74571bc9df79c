// Attention backward, from the forward's lse.
//
//   D_i = go_i . o_i,  P = exp(scale q k - lse),  dS = P (go v^T - D)
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T go
//
// Two kernels, each of which recomputes P: one whose waves own 32 queries and
// walk the keys (dq; it computes D first, for itself and the other), one
// whose waves own 32 keys and walk the queries of every head that shares them
// (dk, dv).  That is seven products instead of the five of one kernel, but no
// sum is taken by atomics or in memory: results do not depend on an order,
// and nothing but the gradients is written.
//
// D from o, which is rounded, is off by half a step of |go| |o|, the same for
// all of a query's keys: of n keys that is about 1 / sqrt(n) of what rounding dS
// does to dq, so it is taken where a block's queries see more than 256 keys.
// Those that see fewer take sum_j P (go v^T) in a first round over them (dq and
// dk of short sequences: errors of 0.0036 -> 0.0024 relative in bf16, where
// rounding the exact result gives 0.0017).
//
// P and dS are rounded to the operands' type for the products that sum them, in
// fp16 times powers of two that keep them within its range (Lift).
//
// Both are bound as the forward is.  16384 tokens, 56 heads of 128 over 8,
// causal, bf16: dq 5.4 and 5.6 ms, dk and dv 7.2 and 7.4 ms (medians on two
// cards), 1.02 to 1.07 PFLOP/s each.
#pragma once

#include "attention.hpp"
#include "attention_fwd.hpp"

namespace mhc {

constexpr int kSumKeys = 256;

// dq, and D.  KS as in the forward.
template <typename S, int DB, int NW, int KS, int NB, int WPE>
__global__ __launch_bounds__(64 * NW, WPE) void att_dq_kernel(AttArgs a, int64_t slots) {
  using T = Tile<S, DB>;
  constexpr int RW = NW / KS, BN = 32 * NB, BS = BN * KS, BM = 32 * RW, NT = 64 * NW, ES = (int)sizeof(S);
  constexpr int kTileBytes = BS * T::kPitch;
  extern __shared__ __attribute__((aligned(256))) char smem[];  // 2 x (K, V); at the end the sums of KS - 1 waves a row
  const int tid = threadIdx.x, lane = tid & 63, id = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave = id % RW, part = id / RW;
  int64_t slot;
  int h, first;
  att_item(a.n, slots, slot, h);
  const AttSeq s = q_tile(a.n, slot, BM, first);
  if (first >= s.lq) return;
  const int hk = h / (a.n.H / a.n.Hk), d = a.n.d, dc = d * ES / 16;
  const int row = first + 32 * wave + (lane & 31);
  const bool live = row < s.lq;
  S* out = static_cast<S*>(a.out) + ((s.row0 + row) * a.n.H + h) * (int64_t)d;
  const int64_t stat = (int64_t)h * a.n.Tq + s.row0 + row;
  const int shift = s.lk - s.lq;
  const int block_last = (first + BM < s.lq ? first + BM : s.lq) - 1;
  const int keys = s.none ? 0 : (a.n.causal ? min(s.lk, block_last + shift + 1) : s.lk);
  if (keys <= 0) {
    store_none<S, DB>(out, live, d, lane);
    if (live && lane < 32) a.delta[stat] = 0.f;
    return;
  }
  const int lim = a.n.causal ? min(s.lk - 1, row + shift) : s.lk - 1;
  const int wave_first = first + 32 * wave;
  const int wave_lo = a.n.causal ? min(s.lk - 1, wave_first + shift) : s.lk - 1;
  const int wave_hi = a.n.causal ? min(s.lk - 1, wave_first + 31 + shift) : s.lk - 1;

  const int q_ts = (int)(a.q.ts * ES), k_ts = (int)(a.k.ts * ES), v_ts = (int)(a.v.ts * ES), go_ts = (int)(a.go.ts * ES);
  const char* kp = row_ptr(a.k, a.n.cu_k, s.k0, s.b, 0, hk, ES);
  const char* vp = row_ptr(a.v, a.n.cu_k, s.k0, s.b, 0, hk, ES);
  const int64_t k_step = (int64_t)BS * k_ts, v_step = (int64_t)BS * v_ts;
  TileStage<S, DB, BS, NT> sk, sv;
  const uint32_t k_off = sk.offset(k_ts, dc, tid), v_off = sv.offset(v_ts, dc, tid), lds = lds_addr(smem);
  sk.load(kp, k_ts, s.lk, k_off);
  sv.load(vp, v_ts, s.lk, v_off);

  u32x4 q[T::kSteps], go[T::kSteps];
  const int left = s.lq - wave_first;
  load_rows<S, DB>(row_ptr(a.q, a.n.cu_q, s.row0, s.b, wave_first, h, ES), q_ts, left, dc, lane, q);
  load_rows<S, DB>(row_ptr(a.go, a.n.cu_q, s.row0, s.b, wave_first, h, ES), go_ts, left, dc, lane, go);
  const int tiles = (keys + BS - 1) / BS, half = lane >> 5;
  const int sum = keys <= kSumKeys ? tiles : 0;  // a round over the tiles for D
  float delta = 0.f;
  if (sum == 0) {
    u32x4 o[T::kSteps];
    load_rows<S, DB>(row_ptr(a.o, a.n.cu_q, s.row0, s.b, wave_first, h, ES), (int)(a.o.ts * ES), left, dc, lane, o);
#pragma unroll
    for (int t = 0; t < T::kSteps; ++t) {
      float x[Store<S>::VEC], y[Store<S>::VEC];
      Store<S>::unpack(o[t], x);
      Store<S>::unpack(go[t], y);
#pragma unroll
      for (int j = 0; j < Store<S>::VEC; ++j) delta = __builtin_fmaf(x[j], y[j], delta);
    }
    delta = add_xor32(delta);
    if (live && lane < 32) a.delta[stat] = delta;
  }
  const float lse = live ? a.lse[stat] : -__builtin_inff();
  const float lse2 = lse == -__builtin_inff() ? __builtin_inff() : lse * kLog2e;  // an empty row: P = 0

  const int zone = a.n.causal ? max(0, first + shift + 1) : 0x7fffffff;  // as in the forward, for the keys
  bool bad = false;
  auto stage = [&](int it, int t) {
    if ((t + 1) * BS > zone) bad |= sk.clean();
    const uint32_t to = lds + (it & 1) * 2 * kTileBytes;
    sk.store(to, tid);
    sv.store(to + kTileBytes, tid);
  };
  stage(0, 0);
  __syncthreads();
  T at(lane);

  floatx16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
  const float c = a.scale2;
  float total = 0.f;
  Lift<S> lift;
  for (int it = 0; it < sum + tiles; ++it) {
    const uint32_t tk = lds + (it & 1) * 2 * kTileBytes + part * BN * T::kPitch, tv = tk + kTileBytes;
    at.keep();
    const int k0 = (it < sum ? it : it - sum) * BS + part * BN;
    const int next = it + 1 < sum ? it + 1 : it + 1 - sum;
    if (it + 1 < sum + tiles) {
      sk.load(kp + next * k_step, k_ts, s.lk - next * BS, k_off);
      sv.load(vp + next * v_step, v_ts, s.lk - next * BS, v_off);
    }
    if (k0 <= wave_hi) {
      const bool masked = k0 + BN - 1 > wave_lo;
      u32x4 p[NB][T::kColSteps];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        floatx16 sc = row_products<S, DB>(at, tk, b, q);
        floatx16 dp = row_products<S, DB>(at, tv, b, go);
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] = hw_exp2(__builtin_fmaf(sc[i], c, -lse2)) * (dp[i] - delta);
        if (masked) {
          stay();
          const int left = lim - k0 - 4 * half;
#pragma unroll
          for (int i = 0; i < 16; ++i) dp[i] = 32 * b + acc_row(i, 0) <= left ? dp[i] : 0.f;
        }
        if (it < sum) {
          stay();
#pragma unroll
          for (int i = 0; i < 16; ++i) total += dp[i];
        }
        if constexpr (Lift<S>::kOn) {
          // (a block of 32 keys at a time: the next one may move the sums)
          if (it < sum) continue;
          lift.template fit<WPE == 1>(dp, acc);
          u32x4 one[1][T::kColSteps];
#pragma unroll
          for (int u = 0; u < T::kColSteps; ++u) one[0][u] = acc_frag<S>(dp, u);
          add_columns<S, DB, 1>(acc, at, tk + b * 32 * T::kPitch, one);
        } else {
#pragma unroll
          for (int u = 0; u < T::kColSteps; ++u) p[b][u] = acc_frag<S>(dp, u);
        }
      }
      if constexpr (!Lift<S>::kOn)
        if (it >= sum) add_columns<S, DB, NB>(acc, at, tk, p);
    }
    if (it + 1 == sum) {
      delta = add_xor32(total);
      if constexpr (KS == 2) {
        __shared__ float sums[KS][BM];
        sums[part][32 * wave + (lane & 31)] = delta;
        __syncthreads();
        delta = sums[0][32 * wave + (lane & 31)] + sums[1][32 * wave + (lane & 31)];
      }
      if (live && lane < 32) a.delta[stat] = delta;
    }
    if (it + 1 < sum + tiles) {
      stage(it + 1, next);
      __syncthreads();
    }
  }
  if constexpr (Lift<S>::kOn) {
    const float back = lift.back();
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] *= back;
  }
  bad = __syncthreads_or(bad);
  if constexpr (KS == 2) {
    float* other = reinterpret_cast<float*>(smem) + wave * DB * 16 * 64 + lane;
    if (part == 1) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) other[(db * 16 + i) * 64] = acc[db][i];
    }
    __syncthreads();
    if (part == 1) return;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] += other[(db * 16 + i) * 64];
  }
  if (bad) {
    const int z = zone / BS * BS;
    add_nonfinite<S, DB, true>(acc, kp + (int64_t)z * k_ts, k_ts, keys - z, d, lane, [&](int r) { return z + r <= lim; });
  }
  store_rows<S, DB>(acc, a.scale, out, live, d, lane);
}

// A float of the `bytes` at p; zero past them.
__device__ __forceinline__ float buffer_f32(const float* p, int bytes, uint32_t off) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p), 0, uniform(max(bytes, 0)), 0x00020000);
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0));
}

// dk and dv, or, of `splits` parts of the queries, a part's share of them in
// fp32, for att_dkv_join_kernel.  VLDS: the block's own rows of v are in LDS,
// and read as they are needed, instead of in registers: with those two waves
// fit a SIMD unit (16384 x 56 heads, forward and backward: 24.6 -> 18.6 ms).
// Heads of 64 keep them in registers: 64 queries a step fit as well (three waves
// a SIMD unit, 32 queries a step: 2.53 -> 2.98 ms the whole backward of 16384 in two, 32 heads).
template <typename S, int DB, int NW, int NB, int WPE, bool VLDS>
__global__ __launch_bounds__(64 * NW, WPE) void att_dkv_kernel(AttArgs a, int64_t slots, int splits) {
  using T = Tile<S, DB>;
  constexpr int BQ = 32 * NB, BK = 32 * NW, NT = 64 * NW, ES = (int)sizeof(S);
  constexpr int kTileBytes = BQ * T::kPitch, kStage = 2 * kTileBytes + (2 * BQ * 4 + 255) / 256 * 256;
  static_assert(BQ <= NT, "a thread a row's lse and D");
  constexpr int kOwn = VLDS ? BK * T::kPitch : 0;
  extern __shared__ __attribute__((aligned(256))) char smem[];  // own V, 2 x (Q, dO, lse, D)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t slot, row0;
  int hk, first, rows;
  const int64_t item = xcd_contig(blockIdx.x, gridDim.x) / splits;
  const int part = (int)(xcd_contig(blockIdx.x, gridDim.x) % splits);
  hk = (int)(item / slots);
  slot = item % slots;  // a head's first keys are seen by the most queries
  const AttSeq s = k_tile(a.n, slot, BK, first, rows, row0);
  if (first >= rows) return;
  const int G = a.n.H / a.n.Hk, d = a.n.d, dc = d * ES / 16;
  const int key = first + 32 * wave + (lane & 31);
  const bool live = key < rows;
  const int shift = s.lk - s.lq;
  // the first query that sees the block's first key
  const int q_first = a.n.causal ? max(0, first - shift) : 0;
  const int t0 = q_first / BQ, tiles = s.none || first >= s.lk || q_first >= s.lq ? 0 : (s.lq + BQ - 1) / BQ - t0;
  if (tiles <= 0) {
    const int64_t place = ((row0 + key) * a.n.Hk + hk) * (int64_t)d, all = a.n.Tk * a.n.Hk * d;
    if (splits > 1) {
      store_none<float, DB>(a.part + 2 * part * all + place, live, d, lane);
      store_none<float, DB>(a.part + (2 * part + 1) * all + place, live, d, lane);
    } else {
      store_none<S, DB>(static_cast<S*>(a.dk) + place, live, d, lane);
      store_none<S, DB>(static_cast<S*>(a.dv) + place, live, d, lane);
    }
    return;
  }
  int wave_first = first + 32 * wave;
  const int q_ts = (int)(a.q.ts * ES), go_ts = (int)(a.go.ts * ES);
  u32x4 k[T::kSteps], v[VLDS ? 1 : T::kSteps];
  load_rows<S, DB>(row_ptr(a.k, a.n.cu_k, s.k0, s.b, wave_first, hk, ES), (int)(a.k.ts * ES), s.lk - wave_first, dc, lane, k);
  if constexpr (VLDS) {
    // (a wave reads back its own rows alone)
    TileStage<S, DB, 32, 64> own;
    own.load(row_ptr(a.v, a.n.cu_k, s.k0, s.b, wave_first, hk, ES), (int)(a.v.ts * ES), s.lk - wave_first,
             own.offset((int)(a.v.ts * ES), dc, lane));
    own.store(lds_addr(smem) + wave * 32 * T::kPitch, lane);
  } else {
    load_rows<S, DB>(row_ptr(a.v, a.n.cu_k, s.k0, s.b, wave_first, hk, ES), (int)(a.v.ts * ES), s.lk - wave_first, dc, lane, v);
  }

  // Items: the tiles of queries of every head that shares the keys.  What is
  // loaded next is kept as pointers: divisions and 64-bit products an item cost
  // as many instructions as a tile of 64-wide heads.
  const int items = tiles * G, it0 = (int)((int64_t)items * part / splits), it1 = (int)((int64_t)items * (part + 1) / splits);
  const int h0 = hk * G + it0 / tiles, end = t0 + tiles;
  int t = t0 + it0 % tiles;
  const char* qp = uniform(row_ptr(a.q, a.n.cu_q, s.row0, s.b, (int64_t)t * BQ, h0, ES));
  const char* gp = uniform(row_ptr(a.go, a.n.cu_q, s.row0, s.b, (int64_t)t * BQ, h0, ES));
  int64_t sp = (int64_t)uniform(reinterpret_cast<const char*>((int64_t)h0 * a.n.Tq + s.row0 + (int64_t)t * BQ));
  const int lq = __builtin_amdgcn_readfirstlane(s.lq);
  TileStage<S, DB, BQ, NT> sq, sg;
  const uint32_t q_off = sq.offset(q_ts, dc, tid), go_off = sg.offset(go_ts, dc, tid), lds = lds_addr(smem) + kOwn;
  float st_lse = 0.f, st_delta = 0.f;  // of query `lane` of the tile, in wave 0
  auto load = [&]() {
    const int left = lq - t * BQ;
    sq.load(qp, q_ts, left, q_off);
    sg.load(gp, go_ts, left, go_off);
    if (wave == 0) {
      const int bytes = min(left, BQ) * 4;
      st_lse = buffer_f32(a.lse + sp, bytes, lane * 4);
      st_delta = buffer_f32(a.delta + sp, bytes, lane * 4);
    }
  };
  // queries before `zone` see not all of the block's keys: as in the forward,
  // for q and the output's gradient
  const int zone = a.n.causal ? first + BK - 1 - shift : 0;
  bool bad = false;
  auto store = [&](int it) {
    const int buf = it & 1;
    if (t * BQ < zone) {
      bad |= sq.clean();
      bad |= sg.clean();
    }
    sq.store(lds + buf * kStage, tid);
    sg.store(lds + buf * kStage + kTileBytes, tid);
    if (tid < BQ) {
      float* to = reinterpret_cast<float*>(smem + kOwn + buf * kStage + 2 * kTileBytes);
      // no such row, or an empty one: P = 0
      to[tid] = t * BQ + tid >= lq || st_lse == -__builtin_inff() ? __builtin_inff()
                                                                  : __builtin_fmaf(st_lse, kLog2e, -Lift<S>::kWeights);
      to[BQ + tid] = st_delta;
    }
  };
  auto advance = [&]() {
    ++t;
    qp += (int64_t)BQ * q_ts;
    gp += (int64_t)BQ * go_ts;
    sp += BQ;
    if (t == end) {
      t = t0;
      qp += a.q.hs * ES - (int64_t)tiles * BQ * q_ts;
      gp += a.go.hs * ES - (int64_t)tiles * BQ * go_ts;
      sp += a.n.Tq - (int64_t)tiles * BQ;
    }
  };
  load();
  store(it0);
  __syncthreads();
  T at(lane);

  floatx16 ak[DB], av[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) ak[db][i] = av[db][i] = 0.f;
  const float c = a.scale2;
  Lift<S> lift;
  const int half = lane >> 5;
  const uint32_t own_v = lds_addr(smem) + wave * 32 * T::kPitch;
  for (int it = it0; it < it1; ++it) {
    const uint32_t tq = lds + (it & 1) * kStage, tg = tq + kTileBytes;
    const float* stats = reinterpret_cast<const float*>(smem + kOwn + (it & 1) * kStage + 2 * kTileBytes);
    at.keep();
    const int q0 = t * BQ;
    if (it + 1 < it1) {
      advance();
      load();
    }
    // queries from here on see the lane's key; all of the wave's keys are seen by the tile or none
    const int lim = a.n.causal ? key - shift : 0;
    const bool any = wave_first < s.lk && (!a.n.causal || q0 + BQ - 1 >= wave_first - shift);
    if (any) {
      const bool masked = a.n.causal && q0 < wave_first + 31 - shift;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        floatx16 sc = row_products<S, DB>(at, tq, b, k);
        floatx16 dp;
        if constexpr (VLDS) {
#pragma unroll
          for (int i = 0; i < 16; ++i) dp[i] = 0.f;
#pragma unroll
          for (int u = 0; u < T::kSteps; ++u) dp = Mma32<S>::fma(at.row_frag(tg, b, u), at.row_frag(own_v, 0, u), dp);
        } else {
          dp = row_products<S, DB>(at, tg, b, v);
        }
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const floatx4 lse = *reinterpret_cast<const floatx4*>(stats + 32 * b + acc_row(i, half));
          const floatx4 del = *reinterpret_cast<const floatx4*>(stats + BQ + 32 * b + acc_row(i, half));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sc[i + j] = hw_exp2(__builtin_fmaf(sc[i + j], c, -lse[j]));
            dp[i + j] = sc[i + j] * (dp[i + j] - del[j]);
          }
        }
        if (masked) {
          stay();
          const int from = lim - q0 - 4 * half;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const bool in = 32 * b + acc_row(i, 0) >= from;
            sc[i] = in ? sc[i] : 0.f;
            dp[i] = in ? dp[i] : 0.f;
          }
        }
        lift.template fit<WPE == 1>(dp, ak);
        u32x4 p[1][T::kColSteps], ds[1][T::kColSteps];
#pragma unroll
        for (int u = 0; u < T::kColSteps; ++u) {
          p[0][u] = acc_frag<S>(sc, u);
          ds[0][u] = acc_frag<S>(dp, u);
        }
        add_columns<S, DB, 1>(av, at, tg + b * 32 * T::kPitch, p);
        add_columns<S, DB, 1>(ak, at, tq + b * 32 * T::kPitch, ds);
      }
    }
    if (it + 1 < it1) {
      store(it + 1);
      __syncthreads();
    }
  }
  // (heads of 64, 8192 in nine: the whole backward 148 -> 139 us; of 192, 4096 in two: 525 -> 495 us)
  const AttArgs e = args_again();
  if (__syncthreads_or(bad)) {
    for (int it = it0; it < it1; ++it) {
      const int h = hk * (e.n.H / e.n.Hk) + it / tiles, q0 = (t0 + it % tiles) * BQ, n = min(BQ, lq - q0);
      if (q0 >= zone) continue;
      const auto seen = [&](int r) { return q0 + r >= key - shift; };
      add_nonfinite<S, DB, false>(av, row_ptr(e.go, e.n.cu_q, s.row0, s.b, q0, h, ES), (int)(e.go.ts * ES), n, e.n.d, lane, seen);
      add_nonfinite<S, DB, true>(ak, row_ptr(e.q, e.n.cu_q, s.row0, s.b, q0, h, ES), (int)(e.q.ts * ES), n, e.n.d, lane, seen);
    }
  }
  // keys past the sequence's are zero rows of k, but no zero rows of dk
  const bool has = key < s.lk;
  if (!has) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) ak[db][i] = av[db][i] = 0.f;
  }
  // (P's factor is in dS too)
  constexpr float kBack = Lift<S>::kOn ? 0x1p-14f : 1.0f;
  static_assert(!Lift<S>::kOn || Lift<S>::kWeights == 14.0f, "P's factor");
  const float ak_f = e.scale * (lift.back() * kBack);
  const int d_end = e.n.d;
  const int64_t place = ((row0 + key) * e.n.Hk + hk) * (int64_t)d_end, all = e.n.Tk * e.n.Hk * d_end;
  if (splits > 1) {
    store_rows<float, DB>(ak, ak_f, e.part + 2 * part * all + place, live, d_end, lane);
    store_rows<float, DB>(av, kBack, e.part + (2 * part + 1) * all + place, live, d_end, lane);
  } else {
    store_rows<S, DB>(ak, ak_f, static_cast<S*>(e.dk) + place, live, d_end, lane);
    store_rows<S, DB>(av, kBack, static_cast<S*>(e.dv) + place, live, d_end, lane);
  }
}

// dk, dv: the parts' shares added in their order, four elements a thread: 3
// parts of 4099 keys, 8 heads of 128: 118 MB in 18 us (some from the caches).
template <typename S>
__global__ __launch_bounds__(256) void att_dkv_join_kernel(AttArgs a, int64_t all, int splits) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;  // of 2 `all`: dk, then dv
  if (e >= 2 * all) return;
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < splits; ++p) sum += *reinterpret_cast<const floatx4*>(a.part + 2 * p * all + e);
  S* out = e < all ? static_cast<S*>(a.dk) + e : static_cast<S*>(a.dv) + (e - all);
  if constexpr (sizeof(S) == 2)
    *reinterpret_cast<u32x2*>(out) = u32x2{Mma32<S>::pack2(sum[0], sum[1]), Mma32<S>::pack2(sum[2], sum[3])};
  else
    *reinterpret_cast<floatx4*>(out) = sum;
}

}  // namespace mhc
