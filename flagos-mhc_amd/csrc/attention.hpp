// Attention over sequences of different lengths: arguments, the map from
// blocks to sequences, tiles in LDS and the matrix operands read from them.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j - lse_i),  lse_i = ln sum_j exp(scale q_i . k_j)
//
// over the keys j that query i sees: j < Lk and, if causal, j <= i + Lk - Lq
// (the queries are the last Lq of the Lk positions).
//
// Every product keeps the index that is summed last in a lane's own
// registers: with 32x32 products, S^T = K Q^T leaves lane l with query l % 32
// and keys 8 (i / 4) + 4 (l / 32) + i % 4, i = 0..15, which is, packed, the
// second operand of O^T = V^T P^T with its k order permuted; the first operand
// is read in that order.  Maxima and sums over keys are then a lane's own but
// for one exchange with lane l ^ 32, factors of a query are one register, and
// P never goes through LDS.
#pragma once

#include "attention_plan.hpp"
#include "common.hpp"
#include "lds_dma.hpp"

namespace mhc {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8_att __attribute__((ext_vector_type(8)));
typedef short s16x4_att __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// A new row maximum moves the reference point only where it exceeds the old one
// by more than this (in powers of two), so that sums are rescaled a few times a
// row and not once a tile.  Weights are then at most 2^8 instead of 1: within
// every type's range, and as many bits are left to them.
constexpr float kLazyMax = 8.0f;
// fp16 weights lose bits below 2^-14 and are 0 below 2^-25, though many of them
// may make a result.  Its numbers reach 65504, so its reference point lies this
// far below the row's maximum: weights are at most 2^15, and keep all bits down
// to 2^-21 of the row's largest (1024 keys of 2^-18.4, the largest's value 0:
// off by 1.1 % before).  bf16 and fp32 have fp32's range.
template <typename S> inline constexpr float kBelowMax = 0.0f;
template <> inline constexpr float kBelowMax<f16_t> = 7.0f;

// One of q, k, v or a gradient: element (sequence's row t, head h, i) at
// p[b * bs + t * ts + h * hs + i]; packed sequences have bs = 0 and rows
// counted from the first sequence's start.
struct AttRows {
  const void* p;
  int64_t bs, ts, hs;  // elements
};

struct AttArgs {
  AttRows q, k, v, go, o;  // go, o: backward; o contiguous
  void* out;               // (rows of q, H, d), forward: o, backward: dq
  void *dk, *dv;           // (rows of k, Hk, d)
  float* lse;              // (H, rows of q)
  float* delta;            // (H, rows of q): sum_d go o, backward
  float* part;             // partial results of splits
  AttDims n;
  float scale, scale2;     // scale, scale * log2(e)
};

// The kernel's arguments (its first parameter) read once more: what only the
// end of a kernel uses is not to hold scalar registers over its loop, which are
// otherwise kept in lanes of vector registers and read back in every step.
__device__ __forceinline__ AttArgs args_again() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const AttArgs*)p;
}

// ---- sequences ---------------------------------------------------------------

struct AttSeq {
  int64_t row0;  // first row in the outputs' and lse's order
  int64_t k0;    // first row of packed keys
  int lq, lk;    // rows; lq counts output rows of the sequence behind the last one too
  int b;
  bool none;     // rows behind the last sequence: zeros are written
};

// A value that is the same for the wave, known to be so: what a scalar register
// holds costs no vector instruction, and a branch on it no mask.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ int64_t cu_at(const int32_t* cu, int b, int64_t T) {
  const int64_t c = b == 0 ? 0 : (int64_t)cu[b];
  return c < 0 ? 0 : (c > T ? T : c);
}

// First slot of sequence b, where tiles of R rows are dealt to slots: sequence
// b's tiles begin at slot cu[b] / R + b, which leaves each the ceil(L / R) it
// needs without a sum over the sequences before it.
__device__ __forceinline__ int64_t slot_start(const int32_t* cu, int b, int64_t T, int R) { return cu_at(cu, b, T) / R + b; }

// The sequence whose slots hold `slot`, of B + 1 (the last: rows behind the
// sequences): 64 candidates a step, one a lane.
__device__ __forceinline__ int slot_sequence(const int32_t* cu, int B, int64_t T, int R, int64_t slot) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = B + 1;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int c = lane * step;
    const bool in = c < n && slot_start(cu, lo + c, T, R) <= slot;
    int hit = __popcll(__ballot(in));
    hit = hit < 1 ? 1 : hit;
    const int skip = (hit - 1) * step;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The rows of sequence b, and where its keys are.
__device__ __forceinline__ AttSeq att_seq(const AttDims& n, int b) {
  AttSeq s;
  s.b = b;
  s.none = b >= n.B;
  if (n.cu_q) {
    s.row0 = cu_at(n.cu_q, b, n.Tq);
    const int64_t e = s.none ? n.Tq : cu_at(n.cu_q, b + 1, n.Tq);
    s.lq = e > s.row0 ? (int)(e - s.row0) : 0;
  } else {
    s.row0 = (int64_t)b * n.Sq;
    s.lq = n.Sq;
  }
  s.lk = 0;
  s.k0 = 0;
  if (!s.none) {
    if (n.cu_k) {
      s.k0 = cu_at(n.cu_k, b, n.Tk);
      const int64_t e = cu_at(n.cu_k, b + 1, n.Tk);
      s.lk = e > s.k0 ? (int)(e - s.k0) : 0;
    } else {
      s.lk = n.Sk;
      if (n.len_k) {
        const int l = n.len_k[b];
        s.lk = l < 0 ? 0 : (l < n.Sk ? l : n.Sk);
      }
    }
  }
  s.row0 = uniform(s.row0);
  s.k0 = uniform(s.k0);
  s.lq = uniform(s.lq);
  s.lk = uniform(s.lk);
  return s;
}

// Tile of `R` query rows that slot `slot` stands for: its sequence and first
// row (lq or more: nothing to do).  Starts that decrease can lead to a sequence
// whose slots begin later: no tile of it.
__device__ __forceinline__ AttSeq q_tile(const AttDims& n, int64_t slot, int R, int& first) {
  if (!n.cu_q) {
    const int per = (n.Sq + R - 1) / R;
    const int b = (int)(slot / per);
    first = (int)(slot % per) * R;
    return att_seq(n, b);
  }
  const int b = slot_sequence(n.cu_q, n.B, n.Tq, R, slot);
  const int64_t t = slot - slot_start(n.cu_q, b, n.Tq, R);
  AttSeq s = att_seq(n, b);
  first = uniform(t >= 0 && t * R < s.lq ? (int)(t * R) : s.lq);
  return s;
}

// The same for key rows; rows is how many of dk and dv the sequence has
// (those past lk are zero).
__device__ __forceinline__ AttSeq k_tile(const AttDims& n, int64_t slot, int R, int& first, int& rows, int64_t& row0) {
  if (!n.cu_k) {
    const int per = (n.Sk + R - 1) / R;
    const int b = (int)(slot / per);
    first = (int)(slot % per) * R;
    rows = n.Sk;
    row0 = (int64_t)b * n.Sk;
    return att_seq(n, b);
  }
  const int b = slot_sequence(n.cu_k, n.B, n.Tk, R, slot);
  const int64_t t = slot - slot_start(n.cu_k, b, n.Tk, R);
  AttSeq s = att_seq(n, b);
  row0 = cu_at(n.cu_k, b, n.Tk);
  const int64_t e = s.none ? n.Tk : cu_at(n.cu_k, b + 1, n.Tk);
  rows = e > row0 ? (int)(e - row0) : 0;
  rows = uniform(rows);
  row0 = uniform(row0);
  first = uniform(t >= 0 && t * R < rows ? (int)(t * R) : rows);
  return s;
}

// Address of row `t` of sequence s for head h.  (Packed rows are counted from
// the buffer's first.)
__device__ __forceinline__ const char* row_ptr(const AttRows& r, const int32_t* cu, int64_t start, int b, int64_t t, int h, int es) {
  const int64_t at = (cu ? start + t : t) * r.ts + (cu ? 0 : (int64_t)b * r.bs) + (int64_t)h * r.hs;
  return static_cast<const char*>(r.p) + at * es;
}

// ---- operands -----------------------------------------------------------------
// A fragment is 16 bytes a lane: E elements of the summed index for one of 32
// rows.  Two lane halves make a step of 2 E: 16 (16-bit types, one 32x32x16
// product) or 8 (fp32, four 32x32x2 products, element j of both halves each).

template <typename S> struct Mma32;
template <> struct Mma32<bf16_t> {
  static constexpr int E = 8;
  __device__ static floatx16 fma(const u32x4& a, const u32x4& b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  __device__ static uint32_t pack2(float lo, float hi) { return pack_bf16x2(lo, hi); }
  // w with infinities and NaNs as zero
  __device__ static uint32_t finite(uint32_t w) {
    w = (w & 0x7f800000u) == 0x7f800000u ? w & 0xffffu : w;
    return (w & 0x7f80u) == 0x7f80u ? w & 0xffff0000u : w;
  }
};
template <> struct Mma32<f16_t> {
  static constexpr int E = 8;
  __device__ static floatx16 fma(const u32x4& a, const u32x4& b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_att, a), __builtin_bit_cast(f16x8_att, b), c, 0, 0, 0);
  }
  __device__ static uint32_t pack2(float lo, float hi) { return f32_to_f16_bits(lo) | (f32_to_f16_bits(hi) << 16); }
  __device__ static uint32_t finite(uint32_t w) {
    w = (w & 0x7c000000u) == 0x7c000000u ? w & 0xffffu : w;
    return (w & 0x7c00u) == 0x7c00u ? w & 0xffff0000u : w;
  }
};
template <> struct Mma32<float> {
  static constexpr int E = 4;
  __device__ static floatx16 fma(const u32x4& a, const u32x4& b, floatx16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
  __device__ static uint32_t finite(uint32_t w) { return (w & 0x7f800000u) == 0x7f800000u ? 0u : w; }
};

// The fragment of elements E t .. E t + E - 1 of the 16 that a product left a
// lane: step t of that block of 32.
template <typename S>
__device__ __forceinline__ u32x4 acc_frag(const floatx16& s, int t) {
  u32x4 f;
  if constexpr (sizeof(S) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = Mma32<S>::pack2(s[8 * t + 2 * i], s[8 * t + 2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __float_as_uint(s[4 * t + i]);
  }
  return f;
}

// Row of a block of 32 that element i of a product is, for the lane's half.
__device__ __forceinline__ int acc_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// ---- tiles ----------------------------------------------------------------------
// R rows of a head as they lie in memory, in chunks of 16 bytes whose position
// within the row is exclusive-ored with a function of the row.  Two kinds of
// reads have to meet all 64 banks: 16 rows of one chunk (row fragments), and
// 4 rows of 4 chunks (16-bit columns, one transposing read of 32 lanes) or
// rows j and j + 4 of 8 chunks (fp32 columns).  Rows of 256 bytes start at
// the same bank, those of 128 at alternating halves.
//
// Addresses are a lane's two base registers and the tile's place (whole 256
// bytes), exclusive-ored with constants, plus constants that the instructions
// hold: one instruction for every few reads, computed where they are read (all
// of them hoisted out of a loop would cost a register each).

typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) const uint32_t lds_u32;
typedef __attribute__((address_space(3))) s16x4_att lds_s16x4;

template <typename S, int DB>
struct Tile {
  static constexpr int kEs = (int)sizeof(S);
  static constexpr int kE = Mma32<S>::E;
  static constexpr int kD = 32 * DB;                 // columns held
  static constexpr int kPitch = att_pitch(kEs, DB);  // bytes from row to row
  static constexpr int kChunks = kPitch / 16;
  static constexpr int kUsed = kD * kEs / 16;    // chunks that are read
  static constexpr int kSteps = kUsed / 2;       // row fragments
  static constexpr int kColSteps = 16 / kE;      // column fragments of 32 rows
  static constexpr int kLow = kChunks >= 16 ? 16 : 8;  // chunks whose position is exclusive-ored

  static __device__ __forceinline__ int swizzle(int r) {
    if constexpr (kEs == 4) return ((r & 4) << 1) | ((r & 8) >> 1) | (r & 3);
    if constexpr (kChunks == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
    return ((r & 3) << 2) | ((r >> 2) & 3);
  }
  static __device__ __forceinline__ uint32_t at(int r, int c) { return (uint32_t)(r * kPitch + ((c ^ swizzle(r)) * 16)); }

  uint32_t row, col;  // a lane's base addresses

  __device__ __forceinline__ explicit Tile(int lane) {
    const int h = lane >> 5, i = lane & 15, g = (lane >> 4) & 1;
    row = at(lane & 31, h);
    if constexpr (kEs == 2) col = at(4 * h + (i >> 2), 2 * g + ((i & 3) >> 1)) + (i & 1) * 8;
    else col = at(4 * h, (lane & 31) >> 2) + (lane & 3) * 4;
  }
  // What follows is not to be computed before a loop that this stands in.
  __device__ __forceinline__ void keep() { asm volatile("" : "+v"(row), "+v"(col)); }

  // Row fragment: row 32 blk + l % 32, chunk 2 step + l / 32.
  __device__ __forceinline__ u32x4 row_frag(uint32_t tile, int blk, int step) const {
    const int c = 2 * step;
    return *(lds_u32x4*)(uintptr_t)(((row + tile) ^ (uint32_t)((c % kLow) * 16)) + blk * 32 * kPitch + (c / kLow) * kLow * 16);
  }

  // Column fragment: column 32 db + l % 32; rows of step t of block blk in the
  // order of acc_frag.
  __device__ __forceinline__ u32x4 col_frag(uint32_t tile, int blk, int t, int db) const {
    u32x4 f;
    if constexpr (kEs == 2) {
      constexpr int kDbs = kLow / 4;  // blocks of 32 columns within the exclusive-ored bits
      const uint32_t at = (blk * 32 + t * 16) * kPitch + (db / kDbs) * kLow * 16;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const s16x4_att v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4*)(uintptr_t)(((col + tile) ^ (uint32_t)((db % kDbs) * 64 + 32 * u)) + at + 8 * u * kPitch));
        const u32x2 w = __builtin_bit_cast(u32x2, v);
        f[2 * u] = w[0];
        f[2 * u + 1] = w[1];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = *(lds_u32*)(uintptr_t)(((col + tile) ^ (uint32_t)(((db & 1) * 8 + (t & 1) * 4 + j) * 16)) +
                                      (blk * 32 + 8 * t + j) * kPitch + (db >> 1) * 256);
    }
    return f;
  }
};

// A pointer that is the same for the wave, known to be so: resources made of
// one that the compiler cannot prove uniform are loaded with in a loop over
// their values.
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t a = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return reinterpret_cast<const char*>((uintptr_t)((uint64_t)hi << 32 | lo));
}

// Rows of a head on their way from memory to a tile, through registers: NT
// threads hold the next tile while this one is computed with.  `left` rows
// exist (others read zero without touching memory), chunks past `d` too.  A
// thread's loads differ in the resource's base alone.
template <typename S, int DB, int R, int NT>
struct TileStage {
  using T = Tile<S, DB>;
  static_assert(NT % T::kChunks == 0 && R * T::kChunks % NT == 0, "a thread keeps its chunk");
  static constexpr int kRows = NT / T::kChunks;  // of a load
  static constexpr int kLoads = R / kRows;
  u32x4 v[kLoads];

  static __device__ __forceinline__ uint32_t offset(int ts_bytes, int d_chunks, int tid) {
    const int c = tid % T::kChunks;
    return c < d_chunks ? (uint32_t)(tid / T::kChunks * ts_bytes + c * 16) : kBufferOob;
  }
  __device__ __forceinline__ void load(const char* base, int ts_bytes, int left, uint32_t off) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      // (uniform: the minimum of a maximum is a vector instruction)
      const int rows = uniform(min(max(left - i * kRows, 0), kRows));
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(base + (int64_t)(i * kRows) * ts_bytes), 0, rows * ts_bytes, 0x00020000);
      v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
    }
  }
  // Infinities and NaNs become zero; whether the thread had any.
  __device__ __forceinline__ bool clean() {
    bool any = false;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = Mma32<S>::finite(v[i][j]);
        any |= w != v[i][j];
        v[i][j] = w;
      }
    return any;
  }
  __device__ __forceinline__ void store(uint32_t tile, int tid) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(tile + T::at(tid / T::kChunks + i * kRows, tid % T::kChunks)) = v[i];
  }
};

// A wave's own 32 rows as fragments (row l % 32), from memory; rows from `left`
// on and chunks from d_chunks on are zero.
template <typename S, int DB>
__device__ __forceinline__ void load_rows(const char* base, int ts_bytes, int left, int d_chunks, int lane,
                                          u32x4 (&f)[Tile<S, DB>::kSteps]) {
  const int rows = uniform(min(max(left, 0), 32));
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, rows * ts_bytes, 0x00020000);
  const uint32_t off = (uint32_t)((lane & 31) * ts_bytes + (lane >> 5) * 16);
  if (d_chunks == Tile<S, DB>::kUsed) {
#pragma unroll
    for (int s = 0; s < Tile<S, DB>::kSteps; ++s)
      f[s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off + s * 32, 0, 0));
  } else {
    asm volatile("" : "+s"(d_chunks));  // the offsets are not to be kept over a loop
#pragma unroll
    for (int s = 0; s < Tile<S, DB>::kSteps; ++s)
      f[s] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, 2 * s + (lane >> 5) < d_chunks ? off + s * 32 : kBufferOob, 0, 0));
  }
}

// The backward's P and dS = P (dP - D) in fp16, whose full precision is that of
// 2^-14 .. 65504: a row's weights are 2^-14 at 16384 keys, and dS is as small,
// or large, as these times the output's gradient, whatever dq and dk come to
// (8192 keys, gradients of 1e-4: dq was off by 10 %; two keys, gradients of
// 1.2e4: infinite).  So P is taken 2^14 times as large (at most 2^14, for the sum
// over queries that is dv), and dS times a power of two of the lane's own, 2^e:
// the lane's query in dq, its key in dk, for which its products add up.  e is
// found as the forward's reference point is: where the largest of a tile's dS
// comes past 2^15, it moves to put that at 2^8, and the lane's sums with it.  Both
// are taken back from the fp32 sums at the end.  It costs a maximum and a product
// an element (backward of 4096 in two, 16 heads over 4, fp16: of 64 158 -> 174 us,
// of 128 262 -> 276, of 256 608 -> 681).  bf16 and fp32 have fp32's range.
template <typename S> struct Lift {
  static constexpr bool kOn = false;
  static constexpr float kWeights = 0.0f;  // log2 of P's factor
  template <bool ACC, int DB> __device__ __forceinline__ void fit(floatx16&, floatx16 (&)[DB]) {}
  __device__ __forceinline__ float back() const { return 1.0f; }
};
template <> struct Lift<f16_t> {
  static constexpr bool kOn = true;
  static constexpr float kWeights = 14.0f;
  float f = 0x1p126f;  // 2^e

  // x: a tile's dS of the lane, in place; acc: the lane's sums of the tiles before.
  // ACC: they fill accumulation registers (kernels of one wave a SIMD unit) and
  // are to stay there but for the factor.
  template <bool ACC, int DB>
  __device__ __forceinline__ void fit(floatx16& x, floatx16 (&acc)[DB]) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));  // (passes over NaN)
    top = max_xor32(top);
    const bool over = top * f > 0x1p15f;
    if (__any(over)) {
      // (an infinite dS has exponent 0 here, and stays infinite)
      const int e = __builtin_amdgcn_frexp_expf(f) - 1, to = over ? min(e, 9 - __builtin_amdgcn_frexp_expf(top)) : e;
      const float r = ldexpf(1.0f, to - e);
      f = ldexpf(1.0f, to);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        if constexpr (ACC) asm volatile("" : "+a"(acc[db]));
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] *= r;
        if constexpr (ACC) asm volatile("" : "+a"(acc[db]));
        __builtin_amdgcn_sched_barrier(0);  // rare: not to cost the kernel registers
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] *= f;
  }
  __device__ __forceinline__ float back() const { return ldexpf(1.0f, 1 - __builtin_amdgcn_frexp_expf(f)); }
};

// The transposed 32 x 32 DB result of a wave (lane: row l % 32 of the output,
// its columns 32 db + 8 (i / 4) + 4 (l / 32) + i % 4) to rows of `ts` elements.
template <typename S, int DB>
__device__ __forceinline__ void store_rows(const floatx16 (&acc)[DB], float f, S* row, bool live, int d, int lane) {
  const int h = lane >> 5;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    if constexpr (sizeof(S) == 2) {
#pragma unroll
      for (int i = 0; i < 16; i += 8) {
        // lanes l and l + 32 hold columns 0..3 | 4..7 and 8..11 | 12..15: exchanged, 0..7 and 8..15
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = Mma32<S>::pack2(acc[db][i + 2 * j] * f, acc[db][i + 2 * j + 1] * f);
        const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        const auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        const int col = 32 * db + 2 * i + 8 * h;
        if (live && col < d) *reinterpret_cast<u32x4*>(row + col) = u32x4{a[0], b[0], a[1], b[1]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int col = 32 * db + 2 * i + 4 * h;
        if (live && col < d)
          *reinterpret_cast<u32x4*>(row + col) = u32x4{__float_as_uint(acc[db][i] * f), __float_as_uint(acc[db][i + 1] * f),
                                                       __float_as_uint(acc[db][i + 2] * f), __float_as_uint(acc[db][i + 3] * f)};
      }
    }
  }
}

// acc[db] += (columns of the tile's rows)^T p over NB blocks of 32 rows; p: what
// the lane's own row weighs the tile's rows with.
template <typename S, int DB, int NB>
__device__ __forceinline__ void add_columns(floatx16 (&acc)[DB], const Tile<S, DB>& at, uint32_t tile,
                                            const u32x4 (&p)[NB][Tile<S, DB>::kColSteps]) {
#pragma unroll
  for (int blk = 0; blk < NB; ++blk)
#pragma unroll
    for (int t = 0; t < Tile<S, DB>::kColSteps; ++t)
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db] = Mma32<S>::fma(at.col_frag(tile, blk, t, db), p[blk][t], acc[db]);
}

// A row that a causal mask hides from some of the tile's queries, but that
// holds an infinity or NaN, must not reach them through 0 * inf.  Where a tile
// has hidden rows its infinities and NaNs are zero in LDS (TileStage::clean);
// if there were any, this adds them after the last tile, from memory, with
// weight 1 where they are seen (an infinity's weight is positive, and a NaN's
// does not matter).
// base: row 0 of the tile; seen(r): the lane sees row r.  WHOLE: rows that were
// operands of the scores too (k, q): all of the result becomes NaN, as the
// scores' weights are not those of the zeroed row.
template <typename S, int DB, bool WHOLE, typename F>
__device__ __forceinline__ void add_nonfinite(floatx16 (&acc)[DB], const char* base, int64_t ts_bytes, int rows, int d,
                                              int lane, F seen) {
  const int half = lane >> 5;
  const auto value = [&](int r, int col) {
    const float v = col + 4 * half < d ? load_elem<S>(reinterpret_cast<const S*>(base + r * ts_bytes) + 4 * half, col) : 0.f;
    return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? v : 0.f;
  };
#pragma unroll 1
  for (int r = 0; r < rows; ++r) {
    if constexpr (WHOLE) {
      float any = 0.f;
#pragma unroll 1
      for (int i = 0; i < 16 * DB; ++i) any = value(r, 8 * (i >> 2) + (i & 3)) != 0.f ? 1.f : any;
      if (max_xor32(any) != 0.f && seen(r)) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[db][i] = __builtin_nanf("");
      }
    } else if (seen(r)) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          acc[db][i] += value(r, 32 * db + acc_row(i, 0));
          if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // rare: not to cost the kernel registers
        }
    }
  }
}

// s = rows of block blk of the tile times the wave's own rows.
template <typename S, int DB>
__device__ __forceinline__ floatx16 row_products(const Tile<S, DB>& at, uint32_t tile, int blk,
                                                 const u32x4 (&own)[Tile<S, DB>::kSteps]) {
  floatx16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
  for (int t = 0; t < Tile<S, DB>::kSteps; ++t) s = Mma32<S>::fma(at.row_frag(tile, blk, t), own[t], s);
  return s;
}

// What follows stays behind the branch it stands in (selects over a whole tile
// are otherwise taken for every tile).
__device__ __forceinline__ void stay() { asm volatile(""); }

__device__ __forceinline__ float hw_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace mhc
