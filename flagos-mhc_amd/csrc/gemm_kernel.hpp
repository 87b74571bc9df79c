// The matrix products' kernels: what they compute, their epilogues, and the
// tile kernel that runs every shape, type and layout.
#pragma once

#include "gemm_plan.hpp"
#include "gemm_tile.hpp"

namespace mhc {

// ---- what a product is ----------------------------------------------------------

// kEpiStore: out0 = C.  kEpiGated (two B operands, g = A B0^T, u = A B1^T):
// out0 = act(g) u, and g and u where gate and up are given.  kEpiGatedGrad
// (C is the gradient of act(g) u): out0 = C u act'(g), out1 = C act(g).
enum { kActSilu = 0, kActGelu = 1, kActGeluTanh = 2, kActRelu = 3 };

struct GemmArgs {
  const void* A[2];  // second: the next segment of k, or of the next product of the batch
  const void* B[2];  // second: the next segment of k, or the gated form's other operand
  int64_t lda, ldb;  // elements between lines
  int M, N, K;       // K of one segment
  int segments;      // of k: C = A0 B0^T (+ A1 B1^T)
  int batch;         // 2: also out1 = A1 B0^T
  void* out0;
  void* out1;
  int64_t ldo;       // of out0 and out1; columns N .. ldo - 1 are written as zero
  float* gate;       // (M, N)
  float* up;
  int act;
  // How the tiles are dealt out: whole ones to the first blocks, one each; the
  // steps of the others in equal runs to `run_blocks` more, whose parts of
  // tiles go to `part` ([2 a block][tile]) and are added by the join kernel.
  int whole_tiles, run_tiles, run_blocks;
  float* part;
};

// 1 / (1 + exp(-z)).  16-bit results: by the hardware's exp2 and reciprocal,
// whose errors (1 ulp each, and |z| half ulps of the exponent's rounding, where
// the result is not yet 1) stay below 2^-17 for z >= -87.3.  Below, 1 + exp(-z)
// is above 2^126, whose reciprocal is subnormal and comes out as 0: off by less
// than 2^-126, z times it by 1.1e-36.  The accurate functions cost four times
// the instructions, a tenth of a large product with this epilogue.
template <bool FAST>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (FAST) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z));
  return 1.f / (1.f + expf(-z));
}

// act(g) and act'(g) in fp32.
template <int KIND, bool FAST>
__device__ __forceinline__ void act_both(float g, float* a, float* d) {
  if constexpr (KIND == kActSilu) {
    const float s = sigmoid<FAST>(g);
    *a = g * s;
    *d = s * (1.f + g * (1.f - s));
  } else if constexpr (KIND == kActGelu) {
    const float p = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    *a = g * p;
    *d = p + g * 0.39894228040143268f * expf(-0.5f * g * g);
  } else if constexpr (KIND == kActGeluTanh) {
    // 0.5 (1 + tanh v) = 1 / (1 + exp(-2 v))
    const float v = 0.79788456080286536f * (g + 0.044715f * g * g * g);
    const float s = sigmoid<FAST>(2.f * v);
    *a = g * s;
    *d = s + g * 2.f * s * (1.f - s) * 0.79788456080286536f * (1.f + 0.134145f * fminf(g * g, 1e30f));
  } else {
    *a = g > 0.f ? g : (g != g ? g : 0.f);
    *d = g > 0.f ? 1.f : 0.f;
  }
}
// The same for N gates and a kind known at run time; S: the results' type.
template <typename S, int N>
__device__ __forceinline__ void act_all(int kind, const float* g, float* a, float* d) {
  constexpr bool kFast = sizeof(S) == 2;
  if (kind == kActSilu) {
#pragma unroll
    for (int i = 0; i < N; ++i) act_both<kActSilu, kFast>(g[i], a + i, d + i);
  } else if (kind == kActGelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) act_both<kActGelu, kFast>(g[i], a + i, d + i);
  } else if (kind == kActGeluTanh) {
#pragma unroll
    for (int i = 0; i < N; ++i) act_both<kActGeluTanh, kFast>(g[i], a + i, d + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) act_both<kActRelu, kFast>(g[i], a + i, d + i);
  }
}

// ---- epilogues -------------------------------------------------------------------

typedef floatx4 floatx4_a4 __attribute__((aligned(4)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));

// Four consecutive elements of a row of `len`, the first at n.  STREAM: not
// kept in the caches (gate and up are larger than they are and next read by
// the backward: 1 to 3% of a forward and backward pass).
template <typename S, bool STREAM = false>
__device__ __forceinline__ void store4(S* row, int64_t n, int64_t len, const floatx4& c) {
  if (n + 4 <= len) {
    if constexpr (STREAM) {
      static_assert(sizeof(S) == 4, "gate and up");
      __builtin_nontemporal_store(c, reinterpret_cast<floatx4_a4*>(row + n));
    } else if constexpr (sizeof(S) == 4) {
      *reinterpret_cast<floatx4_a4*>(row + n) = c;
    } else {
      const u32x2 v = {(uint32_t)Store<S>::from_f32(c[0]) | (uint32_t)Store<S>::from_f32(c[1]) << 16,
                       (uint32_t)Store<S>::from_f32(c[2]) | (uint32_t)Store<S>::from_f32(c[3]) << 16};
      *reinterpret_cast<u32x2_a2*>(row + n) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < len) store_elem<S>(row, n + i, c[i]);
  }
}
__device__ __forceinline__ floatx4 load4(const float* row, int64_t n, int64_t len) {
  if (n + 4 <= len) return __builtin_nontemporal_load(reinterpret_cast<const floatx4_a4*>(row + n));
  floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < len) v[i] = row[n + i];
  return v;
}

// c with zeros from column `len` on; c[0] is column n.
__device__ __forceinline__ floatx4 zero_past(floatx4 c, int64_t n, int64_t len) {
  if (n + 4 > len) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i >= len) c[i] = 0.f;
  }
  return c;
}

// Row m, columns n .. n + 3 of the product (c; gated: c0 = g, c1 = u); z is
// the product of the batch.  The gated forms' results are operands of the next
// product, which reads whole chunks of k: their columns from N on are set to
// zero, as the sums there are NaN in rows with a NaN or an infinity (times the
// zeros that stand for operands out of range).
template <typename S, int EPI>
__device__ __forceinline__ void epilogue(const GemmArgs& a, int z, int64_t m, int n, const floatx4& c0, const floatx4& c1) {
  if (m >= a.M || n >= a.ldo) return;
  S* o0 = static_cast<S*>(z ? a.out1 : a.out0) + m * a.ldo;
  if constexpr (EPI == kEpiStore) {
    store4<S>(o0, n, a.ldo, c0);
  } else if constexpr (EPI == kEpiGated) {
    const float g[4] = {c0[0], c0[1], c0[2], c0[3]};
    float v[4], d[4];
    act_all<S, 4>(a.act, g, v, d);
    store4<S>(o0, n, a.ldo, zero_past(floatx4{v[0] * c1[0], v[1] * c1[1], v[2] * c1[2], v[3] * c1[3]}, n, a.N));
    if (a.gate) {
      store4<float, true>(a.gate + m * a.N, n, a.N, c0);
      store4<float, true>(a.up + m * a.N, n, a.N, c1);
    }
  } else {
    const floatx4 g = load4(a.gate + m * a.N, n, a.N), u = load4(a.up + m * a.N, n, a.N);
    const float ga[4] = {g[0], g[1], g[2], g[3]};
    float v[4], d[4];
    act_all<S, 4>(a.act, ga, v, d);
    floatx4 dg, du;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      dg[i] = c0[i] * u[i] * d[i];
      du[i] = c0[i] * v[i];
    }
    store4<S>(o0, n, a.ldo, zero_past(dg, n, a.N));
    store4<S>(static_cast<S*>(a.out1) + m * a.ldo, n, a.ldo, zero_past(du, n, a.N));
  }
}

// ---- order of the tiles ------------------------------------------------------------

// Tile (mt, nt) of product z for the t-th of batch x tm x tn: down groups of 8
// tile rows, so that the tiles an XCD works on at one time (contiguous runs of
// the order) share their operands in its L2.
__device__ __forceinline__ void tile_of(int t, int tm, int tn, int* mt, int* nt, int* z) {
  constexpr int kGroup = 8;
  const int q = t / (tm * tn);
  t -= q * tm * tn;
  const int per = kGroup * tn, g = t / per, r = t % per;
  const int rows = tm - g * kGroup < kGroup ? tm - g * kGroup : kGroup;
  // (the compiler divides in vector registers)
  *z = __builtin_amdgcn_readfirstlane(q);
  *mt = __builtin_amdgcn_readfirstlane(g * kGroup + r % rows);
  *nt = __builtin_amdgcn_readfirstlane(r / rows);
}

// A block's i-th piece of work: steps s0 .. s1 - 1 of a tile, or none.
struct Piece {
  int tile, s0, s1;
  int slot;  // of the partial sums; -1: the whole tile
};
__device__ __forceinline__ bool piece_of(const GemmArgs& a, int steps, int i, Piece* p) {
  const int bid = blockIdx.x;
  const auto uniform = [](int64_t v) { return __builtin_amdgcn_readfirstlane((int)v); };
  if (bid < a.whole_tiles) {
    *p = {uniform(xcd_contig(bid, a.whole_tiles)), 0, steps, -1};
    return i == 0;
  }
  RunPiece r;
  if (!run_piece(xcd_contig(bid - a.whole_tiles, a.run_blocks), i, a.run_tiles, steps, a.run_blocks, &r)) return false;
  *p = {uniform(a.whole_tiles + r.tile), uniform(r.s0), uniform(r.s1), uniform(r.slot)};
  return true;
}

// Row r, columns c .. c + 3 of the tile at (m0, n0): through the epilogue, or
// to the piece's partial sums ([BM][columns, then those of the gated form's
// second operand]).
template <typename C>
__device__ __forceinline__ void finish(const GemmArgs& a, const Piece& p, int z, int m0, int n0, int r, int c,
                                       const floatx4& c0, const floatx4& c1) {
  if (p.slot < 0) {
    epilogue<typename C::S, C::EPI>(a, z, (int64_t)m0 + r, n0 + c, c0, c1);
  } else if (m0 + r < a.M) {
    float* q = a.part + ((int64_t)p.slot * C::BM + r) * C::BN + c;
    *reinterpret_cast<floatx4*>(q) = c0;
    if constexpr (C::EPI == kEpiGated) *reinterpret_cast<floatx4*>(q + C::kCols) = c1;
  }
}

// ROWS rows of a tile's sums, from its row `first` on, out of LDS: a wave has
// whole rows, so that what it writes (and the gated gradient reads) are long
// runs.  16-byte chunks are exclusive-ored with the row for the banks.
template <typename C, int ROWS, int THREADS>
__device__ __forceinline__ void stream_rows(const GemmArgs& a, const Piece& p, int z, int m0, int n0, int first,
                                            const floatx4* cs) {
  constexpr int kRow4 = C::BN / 4, kCols4 = C::kCols / 4, kTurn = THREADS / kCols4;  // rows a turn
  static_assert(ROWS % kTurn == 0, "whole turns");
  constexpr int kTurns = ROWS / kTurn, kUnroll = kTurns < 4 ? kTurns : 4;
  const int r0 = threadIdx.x / kCols4, c = threadIdx.x % kCols4;
#pragma unroll kUnroll
  for (int i = 0; i < kTurns; ++i) {
    const int r = i * kTurn + r0;
    const floatx4 c0 = cs[r * kRow4 + (c ^ (r & 15))];
    const floatx4 c1 = C::EPI == kEpiGated ? cs[r * kRow4 + ((kCols4 + c) ^ (r & 15))] : c0;
    finish<C>(a, p, z, m0, n0, first + r, c * 4, c0, c1);
  }
}

// Where a block's next tiles of A and B start, and how many k are left there
// (0 past the block's steps).
template <typename C>
struct KCursor {
  using S = typename C::S;
  const S *pa, *pb, *pb2;  // pb2: the gated form's second operand
  int s, left;

  static __device__ __forceinline__ int64_t at(int layout, int64_t ld, int first, int kt) {
    const int64_t k = (int64_t)kt * kStep<S>;
    return layout == kRow ? first * ld + k : k * ld + first;
  }
  __device__ __forceinline__ void segment(const GemmArgs& a, int z, int m0, int n0, int seg, int kt) {
    pa = static_cast<const S*>(seg | z ? a.A[1] : a.A[0]) + at(C::LA, a.lda, m0, kt);
    pb = static_cast<const S*>(seg ? a.B[1] : a.B[0]) + at(C::LB, a.ldb, n0, kt);
    if constexpr (C::EPI == kEpiGated) pb2 = static_cast<const S*>(a.B[1]) + at(C::LB, a.ldb, n0, kt);
    left = a.K - kt * kStep<S>;
  }
  __device__ __forceinline__ KCursor(const GemmArgs& a, int z, int m0, int n0, int nk, int s0, int s1) : pb2(nullptr), s(s0) {
    segment(a, z, m0, n0, s0 >= nk, s0 >= nk ? s0 - nk : s0);
    if (s0 >= s1) left = 0;
  }
  __device__ __forceinline__ void advance(const GemmArgs& a, int z, int m0, int n0, int nk, int s1) {
    ++s;
    pa += C::LA == kRow ? (int64_t)kStep<S> : kStep<S> * a.lda;
    pb += C::LB == kRow ? (int64_t)kStep<S> : kStep<S> * a.ldb;
    if constexpr (C::EPI == kEpiGated) pb2 += C::LB == kRow ? (int64_t)kStep<S> : kStep<S> * a.ldb;
    left -= kStep<S>;
    if (a.segments == 2 && s == nk) segment(a, z, m0, n0, 1, 0);
    if (s >= s1) left = 0;
  }
};

// ---- the tile kernel -----------------------------------------------------------------
// Four waves hold a BM x BN tile of C in registers (WM x WN waves); tiles of A
// and B go through LDS in STAGES slots.  DMA: loads go straight to LDS,
// STAGES - 1 tiles ahead; otherwise through registers, for operands whose rows
// are not multiples of 16 bytes.  128 x 128 (the waves 2 x 2) and 64 x 64 run
// two and four blocks a CU, so that one's products cover another's waits and
// its results' way to memory: two 5632 x 2048 x 4099 bf16 products 193 us (0.98
// PFLOP/s; 179 at best); fp32, bound by its matrix instructions, 126 and 135
// TFLOP/s at 2048 and 4096 tokens.  16 and 64 rows x 128 are bound by B's bytes:
// one block a CU with 80 KB or more on their way (T = 64, 180 MB of weights in 41
// us, 4.4 TB/s).

template <typename S_, int LA_, int LB_, int BM_, int BN_, int WAVES_M_, int STAGES_, int PER_CU_, int EPI_, bool DMA_>
struct TileCfg {
  using S = S_;
  static constexpr int LA = LA_, LB = LB_, BM = BM_, BN = BN_, STAGES = STAGES_, EPI = EPI_;
  static constexpr bool DMA = DMA_;
  static constexpr int NW = 4, WAVES_M = WAVES_M_, WAVES_N = NW / WAVES_M_;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;  // a wave's tile
  static constexpr int NFA = WM / 16, NFB = WN / 16;
  static constexpr int kNB = EPI == kEpiGated ? 2 : 1;         // B operands
  static constexpr int kCols = BN / kNB;                       // columns of C
  static constexpr int kSlot = (BM + BN) * 128;
  static constexpr int kPerCu = PER_CU_;  // blocks
  static_assert(STAGES >= 2 && kPerCu * STAGES * kSlot <= 160 * 1024, "LDS");
  static_assert(DMA || STAGES == 2, "register staging has two slots");
  static_assert(EPI != kEpiGated || LB == kRow, "the gated form's weights are rows of k");
};

template <typename C>
__device__ __forceinline__ void gemm_tile_piece(const GemmArgs& a, const Piece& piece, int nk, char* smem) {
  using S = typename C::S;
  const uint32_t lds = lds_addr(smem);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WAVES_M, wn = wave / C::WAVES_M;
  int mt, nt, z;
  tile_of(piece.tile, (a.M + C::BM - 1) / C::BM, (int)((a.ldo + C::kCols - 1) / C::kCols), &mt, &nt, &z);
  const int m0 = mt * C::BM, n0 = nt * C::kCols, s0 = piece.s0, s1 = piece.s1;
  using LdA = TileLoader<S, C::LA, C::BM, C::NW>;
  using LdB = TileLoader<S, C::LB, C::BN, C::NW>;
  const auto row_a = [](int l) { return l; };
  // gated: each wave's columns are WN / 2 of the gate's, then the same of the other operand's
  const auto row_b = [](int l) {
    if constexpr (C::kNB == 2) return l / C::WN * (C::WN / 2) + l % (C::WN / 2);
    return l;
  };
  const auto second_b = [](int l) { return C::kNB == 2 && l % C::WN >= C::WN / 2; };
  // kCol operands: columns up to the line's end may be read (whole chunks)
  const int rows_a = C::LA == kRow || !C::DMA ? a.M - m0 : (int)(a.lda - m0);
  const int rows_b = C::LB == kRow || !C::DMA ? a.N - n0 : (int)(a.ldb - n0);
  const auto corner = [&](const void* p, int layout, int64_t ld, int first, int kt) {
    const int64_t k = (int64_t)kt * kStep<S>;
    return static_cast<const S*>(p) + (layout == kRow ? first * ld + k : k * ld + first);
  };

  FragReader<S, C::LA, C::BM, C::NFA> ra;
  FragReader<S, C::LB, C::BN, C::NFB> rb;
  ra.init(wm * C::WM, lane);
  rb.init(wn * C::WN, lane);
  floatx4 acc[C::NFA][C::NFB];
#pragma unroll
  for (int i = 0; i < C::NFA; ++i)
#pragma unroll
    for (int j = 0; j < C::NFB; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  const auto multiply = [&](int slot) {
    u32x4 fa[2][C::NFA], fb[2][C::NFB];
    const uint32_t t = lds + slot * C::kSlot;
    ra.read(fa, t);
    rb.read(fb, t + C::BM * 128);
    mma_frags<S>(acc, fa, fb);
  };

  if constexpr (C::DMA) {
    LdA la;
    LdB lb;
    la.init(a.lda, 0, rows_a, wave, lane, row_a);
    lb.init(a.ldb, 0, rows_b, wave, lane, row_b);
    KCursor<C> cur(a, z, m0, n0, nk, s0, s1);
    const auto issue = [&](int slot) {
      const uint32_t t = lds + slot * C::kSlot;
      la.issue(cur.pa, a.lda, cur.left, t, wave);
      if constexpr (C::kNB == 2)
        lb.issue_two(cur.pb, cur.pb2, a.ldb, cur.left, t + C::BM * 128, wave, second_b);
      else
        lb.issue(cur.pb, a.ldb, cur.left, t + C::BM * 128, wave);
      cur.advance(a, z, m0, n0, nk, s1);
    };
#pragma unroll
    for (int i = 0; i < C::STAGES - 1; ++i) issue(i);
    int slot = 0;
    for (int s = s0; s < s1; ++s) {
      wait_vmcnt<(C::STAGES - 2) * (LdA::kLoads + LdB::kLoads)>();
      // every wave's part of slot s is there, and every wave has read slot s - 1
      __builtin_amdgcn_s_barrier();
      issue(slot == 0 ? C::STAGES - 1 : slot - 1);
      multiply(slot);
      slot = slot == C::STAGES - 1 ? 0 : slot + 1;
    }
    wait_vmcnt<0>();  // no load may still be on its way to LDS when the block ends
  } else {
    TileRegs<S, C::LA, C::BM, C::NW> va;
    TileRegs<S, C::LB, C::BN, C::NW> vb;
    const auto load = [&](int s) {
      const int seg = s >= nk, kt = s - seg * nk;
      const int left = s < s1 ? a.K - kt * kStep<S> : 0;
      va.load(corner(a.A[seg | z], C::LA, a.lda, m0, kt), a.lda, rows_a, left, wave, lane, row_a);
      if constexpr (C::kNB == 2)
        vb.load_two(corner(a.B[0], C::LB, a.ldb, n0, kt), corner(a.B[1], C::LB, a.ldb, n0, kt), a.ldb, rows_b, left,
                    wave, lane, row_b, second_b);
      else
        vb.load(corner(a.B[seg], C::LB, a.ldb, n0, kt), a.ldb, rows_b, left, wave, lane, row_b);
    };
    const auto store = [&](int slot) {
      va.store(lds + slot * C::kSlot, wave, lane);
      vb.store(lds + slot * C::kSlot + C::BM * 128, wave, lane);
    };
    load(s0);
    store(0);
    load(s0 + 1);
    int slot = 0;
    for (int s = s0; s < s1; ++s) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      if (s + 1 < s1) store(slot ^ 1);
      if (s + 2 < s1) load(s + 2);
      multiply(slot);
      slot ^= 1;
    }
  }

  // lane: row l % 16 of a fragment of A, columns 4 (l / 16) .. + 3 of one of B.
  // Through LDS, as rows of [columns, those of the gated form's second operand].
  constexpr int NC = C::NFB / C::kNB, kRow4 = C::BN / 4;
  static_assert(C::BM * C::BN * 4 <= C::STAGES * C::kSlot, "the tile's sums fit the slots");
  floatx4* const cs = reinterpret_cast<floatx4*>(smem);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < C::NFA; ++i)
#pragma unroll
    for (int j = 0; j < C::NFB; ++j) {
      const int r = wm * C::WM + 16 * i + (lane & 15);
      const int c = j / NC * (C::kCols / 4) + wn * (C::WN / C::kNB / 4) + j % NC * 4 + (lane >> 4);
      cs[r * kRow4 + (c ^ (r & 15))] = acc[i][j];
    }
  __syncthreads();
  stream_rows<C, C::BM, 256>(a, piece, z, m0, n0, 0, cs);
}

template <typename C>
__global__ __launch_bounds__(256, C::kPerCu) void gemm_tile_kernel(GemmArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[C::STAGES * C::kSlot];
  const int nk = (a.K + kStep<typename C::S> - 1) / kStep<typename C::S>;
  Piece piece;
  for (int i = 0; piece_of(a, nk * a.segments, i, &piece); ++i) {
    if (i) __syncthreads();  // every wave is through with the last piece's LDS
    gemm_tile_piece<C>(a, piece, nk, smem);
  }
}

// ---- the large tiles' kernel ----------------------------------------------------------
// BM x 256 of C in the registers of eight waves (2 x 4), one block per CU, BM
// = 256 or 128.  The tile's rows are halves of 128 (one or two), its columns
// two (the gated form: B's halves are its two operands); a wave has 64 rows
// and 32 columns of every half.  A step of k is a phase for each half of A:
//
//   phase  LDS reads     products       loads started (BM = 256)
//     1    A0, B0, B1    A0 x B0, B1    A1 of step k + 1
//     2    A1            A1 x B0, B1    A0, B0, B1 of step k + 2
//
// With two slots a half's is free as soon as the phase that reads it is over,
// so loads run a whole step ahead (64 KB a CU on their way).  BM = 128 has
// three slots and starts the loads of step k + 2 in its only phase.  Every
// phase is reads, barrier, products, barrier, and waves 4 .. 7 run one barrier
// behind waves 0 .. 3: of the two waves on a SIMD one reads while the other
// multiplies.  16384 x 7168 x 18432 bf16: 2.94 ms, 1.47 PFLOP/s, the matrix
// instructions busy 82% of the cycles at the 1.57 GHz that the card's power
// leaves them; with a phase for each quadrant, and twice the barriers, a forward
// and backward at this size took 36.3 ms instead of 29.3.  BM = 128 is a seventh
// slower for its products and leaves fewer CUs without a tile.

template <typename S_, int LA_, int LB_, int BM_, int EPI_>
struct WideCfg {
  using S = S_;
  static constexpr int LA = LA_, LB = LB_, EPI = EPI_, BM = BM_, BN = 256;
  static constexpr int kCols = EPI == kEpiGated ? 128 : 256;  // columns of C
  static constexpr int kHalf = 128 * 128;                     // bytes of a half in LDS
  static constexpr int kHalves = BM / 128;                    // of A
  static constexpr int kA0 = 0, kA1 = kHalf, kB0 = kHalves * kHalf, kB1 = kB0 + kHalf, kSlot = kB1 + kHalf;
  static constexpr int kSlots = kHalves == 2 ? 2 : 3;
  static constexpr int kPerCu = 1;
};

template <typename C>
__device__ __forceinline__ void gemm_wide_piece(const GemmArgs& a, const Piece& piece, int nk, char* smem) {
  using S = typename C::S;
  const uint32_t lds = lds_addr(smem);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = (wave >> 1) & 1, wn = (wave & 1) | ((wave >> 2) << 1);
  int mt, nt, z;
  tile_of(piece.tile, (a.M + C::BM - 1) / C::BM, (int)((a.ldo + C::kCols - 1) / C::kCols), &mt, &nt, &z);
  const int m0 = mt * C::BM, n0 = nt * C::kCols, s0 = piece.s0, s1 = piece.s1;
  using LdA = TileLoader<S, C::LA, 128, 8>;
  using LdB = TileLoader<S, C::LB, 128, 8>;
  constexpr bool kPair = C::EPI == kEpiGated;
  const int rows_a = C::LA == kRow ? a.M - m0 : (int)(a.lda - m0);
  const int rows_b = C::LB == kRow ? a.N - n0 : (int)(a.ldb - n0);
  const auto same = [](int l) { return l; };
  LdA la0, la1;
  LdB lb0, lb1;
  la0.init(a.lda, 0, rows_a, wave, lane, same);
  if constexpr (C::kHalves == 2) la1.init(a.lda, 128, rows_a - 128, wave, lane, same);
  lb0.init(a.ldb, 0, rows_b, wave, lane, same);
  if constexpr (!kPair) lb1.init(a.ldb, 128, rows_b - 128, wave, lane, same);
  KCursor<C> cur(a, z, m0, n0, nk, s0, s1);
  const auto issue_first = [&](uint32_t slot) {
    la0.issue(cur.pa, a.lda, cur.left, slot + C::kA0, wave);
    lb0.issue(cur.pb, a.ldb, cur.left, slot + C::kB0, wave);
    (kPair ? lb0 : lb1).issue(kPair ? cur.pb2 : cur.pb, a.ldb, cur.left, slot + C::kB1, wave);
  };
  const auto issue_second = [&](uint32_t slot) {
    if constexpr (C::kHalves == 2) la1.issue(cur.pa, a.lda, cur.left, slot + C::kA1, wave);
    cur.advance(a, z, m0, n0, nk, s1);
  };

  FragReader<S, C::LA, 128, 4> ra;
  FragReader<S, C::LB, 128, 2> rb;
  ra.init(wm * 64, lane);
  rb.init(wn * 32, lane);
  floatx4 acc[C::kHalves][4][4];  // [half of A][fragment][two of B0, two of B1]
#pragma unroll
  for (int i = 0; i < C::kHalves; ++i)
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[i][p][q] = {0.f, 0.f, 0.f, 0.f};

  const auto barrier = [] {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  u32x4 fa[2][4], fb[2][4];
  const auto products = [&](floatx4 (&c)[4][4]) {
    barrier();
    __builtin_amdgcn_s_setprio(1);
    mma_frags<S>(c, fa, fb);
    __builtin_amdgcn_s_setprio(0);
    barrier();
  };
  if constexpr (C::kHalves == 2) {
    // the loads younger than those a phase waits for: four halves
    constexpr int kYounger = 2 * LdA::kLoads + 2 * LdB::kLoads;
    issue_first(lds);
    issue_second(lds);
    issue_first(lds + C::kSlot);
    wait_vmcnt<kYounger>();
    barrier();
    if (wave >= 4) barrier();
    uint32_t t = lds, o = lds + C::kSlot;
    for (int s = s0; s < s1; ++s) {
      issue_second(o);
      read_all<S, C::LA, C::LB>(fa, fb, ra, rb, t + C::kA0, t + C::kB0);
      wait_vmcnt<kYounger>();  // A1 of this step, for the next phase
      products(acc[0]);

      issue_first(t);
      ra.read(fa, t + C::kA1);
      wait_vmcnt<kYounger>();  // A0, B0 and B1 of the next step
      products(acc[1]);
      const uint32_t n = t;
      t = o;
      o = n;
    }
  } else {
    constexpr int kYounger = LdA::kLoads + 2 * LdB::kLoads;  // a step's
    const auto issue = [&](uint32_t slot) {
      issue_first(slot);
      issue_second(slot);
    };
    issue(lds);
    issue(lds + C::kSlot);
    wait_vmcnt<kYounger>();
    barrier();
    if (wave >= 4) barrier();
    // a step's slot, and that of the step before it, which nobody reads any more
    uint32_t t = lds, free = lds + 2 * C::kSlot;
    for (int s = s0; s < s1; ++s) {
      issue(free);
      read_all<S, C::LA, C::LB>(fa, fb, ra, rb, t + C::kA0, t + C::kB0);
      wait_vmcnt<kYounger>();  // the next step
      products(acc[0]);
      free = t;
      t = t == lds + 2 * C::kSlot ? lds : t + C::kSlot;
    }
  }
  if (wave < 4) barrier();
  wait_vmcnt<0>();  // no load may still be on its way to LDS when the block ends

  // 128 rows of C at a time through LDS
  floatx4* const cs = reinterpret_cast<floatx4*>(smem);
#pragma unroll
  for (int i = 0; i < C::kHalves; ++i) {
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = wm * 64 + p * 16 + (lane & 15), c = (q >> 1) * 32 + wn * 8 + (q & 1) * 4 + (lane >> 4);
        cs[r * 64 + (c ^ (r & 15))] = acc[i][p][q];
      }
    __syncthreads();
    stream_rows<C, 128, 512>(a, piece, z, m0, n0, i * 128, cs);
  }
}

template <typename C>
__global__ __launch_bounds__(512, 2) void gemm_wide_kernel(GemmArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[C::kSlots * C::kSlot];
  const int nk = (a.K + kStep<typename C::S> - 1) / kStep<typename C::S>;
  Piece piece;
  for (int i = 0; piece_of(a, nk * a.segments, i, &piece); ++i) {
    if (i) __syncthreads();  // every wave is through with the last piece's LDS
    gemm_wide_piece<C>(a, piece, nk, smem);
  }
}

// Adds the pieces of the tiles that several blocks have parts of, in order of
// k, and runs the epilogue; a thread has four columns of a row.
template <typename C>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmArgs a) {
  const int steps = (a.K + kStep<typename C::S> - 1) / kStep<typename C::S> * a.segments;
  constexpr int kRowThreads = C::kCols / 4, kBlocks = C::BM * kRowThreads / 256;  // a tile's
  static_assert(C::BM * kRowThreads % 256 == 0, "whole blocks");
  const int t = blockIdx.x / kBlocks, i = blockIdx.x % kBlocks * 256 + threadIdx.x;
  const int r = i / kRowThreads, c = i % kRowThreads * 4;
  int mt, nt, z;
  tile_of(a.whole_tiles + t, (a.M + C::BM - 1) / C::BM, (int)((a.ldo + C::kCols - 1) / C::kCols), &mt, &nt, &z);
  const int64_t m = (int64_t)mt * C::BM + r;
  if (m >= a.M) return;
  const RunBlocks rb = run_blocks_of(t, a.run_tiles, steps, a.run_blocks);
  if (rb.first == rb.last) return;  // one block has the whole tile, and has finished it
  const int64_t stride = 2 * (int64_t)C::BM * C::BN;
  const float* q = a.part + rb.first * stride + (int64_t)r * C::BN + c;
  if (rb.begun_before) q += stride / 2;
  floatx4 c0 = *reinterpret_cast<const floatx4*>(q), c1 = c0;
  if constexpr (C::EPI == kEpiGated) c1 = *reinterpret_cast<const floatx4*>(q + C::kCols);
  q = a.part + (rb.first + 1) * stride + (int64_t)r * C::BN + c;
  const auto add = [&](int n) {  // n runs, their loads first
    floatx4 u[8], v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) {
        u[k] = *reinterpret_cast<const floatx4*>(q + k * stride);
        if constexpr (C::EPI == kEpiGated) v[k] = *reinterpret_cast<const floatx4*>(q + k * stride + C::kCols);
      }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) {
        c0 += u[k];
        if constexpr (C::EPI == kEpiGated) c1 += v[k];
      }
    q += n * stride;
  };
  int64_t left = rb.last - rb.first - 1;
  for (; left >= 8; left -= 8) add(8);
  if (left > 0) add((int)left);
  epilogue<typename C::S, C::EPI>(a, z, m, nt * C::kCols + c, c0, c1);
}

// ---- few rows -------------------------------------------------------------------------
// The forward's products for up to four rows of A (kRow operands): bound by
// the reading of B's rows, once.  A block has the four rows B(n) .. B(n + 3)
// (the gated form: two of each operand) and its four waves every fourth KB of
// them, 1 KB a load; fp32 products and sums, the lanes' sums are added at the
// end.  No LDS on the way, so that a CU holds up to 32 waves, each with eight
// loads under way: 528 MB of gate and up weights in 73 us (7.2 TB/s), where
// tiles of 16 rows take 92 and a join.
template <typename S, int ROWS, int EPI>
__global__ __launch_bounds__(256) void few_rows_kernel(GemmArgs a) {
  constexpr int V = kVec<S>, kB = 4, kChunk = kWave * V;
  constexpr int kCols = EPI == kEpiGated ? 2 : 4;  // columns of C
  __shared__ float red[4][kB * ROWS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * kCols;
  const S* A = static_cast<const S*>(a.A[0]);
  const S* row[kB];  // rows past the last one repeat it
#pragma unroll
  for (int j = 0; j < kB; ++j) {
    const int64_t n = n0 + (EPI == kEpiGated ? j & 1 : j);
    row[j] = static_cast<const S*>(EPI == kEpiGated && j >= 2 ? a.B[1] : a.B[0]) + (n < a.N ? n : a.N - 1) * a.ldb;
  }
  float acc[kB][ROWS] = {};
  const auto dot = [&](const u32x4 (&w)[kB], const u32x4 (&x)[ROWS]) {
    float fx[ROWS][V];
#pragma unroll
    for (int t = 0; t < ROWS; ++t) Store<S>::unpack(x[t], fx[t]);
#pragma unroll
    for (int j = 0; j < kB; ++j) {
      float fw[V];
      Store<S>::unpack(w[j], fw);
#pragma unroll
      for (int t = 0; t < ROWS; ++t)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[j][t] = fmaf(fw[i], fx[t][i], acc[j][t]);
    }
  };
  const auto fetch = [&](int64_t k, u32x4 (&w)[kB], u32x4 (&x)[ROWS]) {
#pragma unroll
    for (int j = 0; j < kB; ++j) w[j] = ld16nt_u(row[j] + k);
#pragma unroll
    for (int t = 0; t < ROWS; ++t) x[t] = *reinterpret_cast<const u32x4_a2*>(A + (t < a.M ? t : 0) * a.lda + k);
  };
  const int64_t whole = a.K / kChunk;
  int64_t c = wave;
  for (; c + 4 < whole; c += 8) {
    u32x4 w0[kB], w1[kB], x0[ROWS], x1[ROWS];
    fetch(c * kChunk + lane * V, w0, x0);
    fetch((c + 4) * kChunk + lane * V, w1, x1);
    dot(w0, x0);
    dot(w1, x1);
  }
  for (; c < whole; c += 4) {
    u32x4 w0[kB], x0[ROWS];
    fetch(c * kChunk + lane * V, w0, x0);
    dot(w0, x0);
  }
  if (c == whole && whole * kChunk < a.K) {  // the last, shorter KB: one wave's, its lanes' chunks whole, cut or empty
    const int64_t k = whole * kChunk + lane * V, have = a.K - k;
    u32x4 w0[kB] = {}, x0[ROWS] = {};
    if (have >= V) {
      fetch(k, w0, x0);
    } else if (have > 0) {
#pragma unroll
      for (int j = 0; j < kB; ++j) w0[j] = ld16_elems<S>(row[j] + k, (int)have);
#pragma unroll
      for (int t = 0; t < ROWS; ++t) x0[t] = ld16_elems<S>(A + (t < a.M ? t : 0) * a.lda + k, (int)have);
    }
    dot(w0, x0);
  }
#pragma unroll
  for (int j = 0; j < kB; ++j)
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
      const float s = group_sum<63>(acc[j][t]);
      if (lane == 0) red[wave][j * ROWS + t] = s;
    }
  __syncthreads();
  // thread t: row t
  const int t = threadIdx.x;
  if (t >= ROWS || t >= a.M) return;
  float s[kB];
#pragma unroll
  for (int j = 0; j < kB; ++j) s[j] = red[0][j * ROWS + t] + red[1][j * ROWS + t] + red[2][j * ROWS + t] + red[3][j * ROWS + t];
  S* out = static_cast<S*>(a.out0) + t * a.ldo;
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    const int64_t n = n0 + j;
    if (n >= a.ldo) continue;
    if constexpr (EPI == kEpiGated) {
      float v = 0.f, d;
      if (n < a.N) {
        act_all<S, 1>(a.act, &s[j], &v, &d);
        v *= s[j + 2];
        if (a.gate) a.gate[t * (int64_t)a.N + n] = s[j], a.up[t * (int64_t)a.N + n] = s[j + 2];
      }
      store_elem<S>(out, n, v);
    } else {
      store_elem<S>(out, n, s[j]);
    }
  }
}

}  // namespace mhc
