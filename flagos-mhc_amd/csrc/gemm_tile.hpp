// Building blocks of the matrix products: operand tiles in LDS, their loads
// and the fragments read from them.
//
// C[m][n] = sum_k A(m, k) B(n, k).  An operand is kRow (k is its contiguous
// index) or kCol (m or n is).  A tile holds R rows of 128 bytes of k (64
// 16-bit or 32 fp32 elements) as it lies in memory: R lines of 128 bytes
// (kRow) or one line of R elements per k (kCol), in 16-byte chunks whose
// position within the line is exclusive-ored with a function of the line, so
// that the lanes of one LDS read meet all banks.
//
// A fragment is 16 rows by 64 bytes of k, 16 bytes a lane: row lane % 16, the
// k of chunk lane / 16.  kRow tiles give it with one ds_read_b128, 16-bit kCol
// tiles with two transposing reads (ds_read_b64_tr_b16: lane i of 16 gets
// column i of four 16-element lines), fp32 kCol tiles with four ds_read_b32.
#pragma once

#include "common.hpp"
#include "gemm_plan.hpp"
#include "lds_dma.hpp"

namespace mhc {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// acc + the product of two fragments, accumulated in fp32: lane l's four
// values are rows 4 (l / 16) .. + 3 of `a` and row l % 16 of `b`.
template <typename S> struct Mma;
template <> struct Mma<bf16_t> {
  __device__ static floatx4 fma(int, const u32x4& a, const u32x4& b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mma<f16_t> {
  __device__ static floatx4 fma(int, const u32x4& a, const u32x4& b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
};
template <> struct Mma<float> {
  // chunk g of a fragment holds k = 4 g .. 4 g + 3: part j takes the j-th of each
  __device__ static floatx4 fma(int j, const u32x4& a, const u32x4& b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
  }
};

// acc[i][j] += a[.][i] b[.][j]^T over both halves of a tile's k.  fp32: the
// tile's 32 products are added by themselves first, so that the running sum
// is rounded once a tile (an error that grows with K / 32 additions, not
// K / 4; the additions are 1 / 64 of the matrix instructions' time).
template <typename S, int NA, int NB>
__device__ __forceinline__ void mma_frags(floatx4 (&acc)[NA][NB], const u32x4 (&a)[2][NA], const u32x4 (&b)[2][NB]) {
  if constexpr (sizeof(S) == 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = Mma<S>::fma(0, b[h][j], a[h][i], acc[i][j]);
  } else {
    constexpr int RI = NA > 1 && NB < 4 ? 2 : 1;  // rows at a time: four chains
#pragma unroll
    for (int i = 0; i < NA; i += RI) {
      floatx4 t[RI][NB];
#pragma unroll
      for (int r = 0; r < RI; ++r)
#pragma unroll
        for (int j = 0; j < NB; ++j) t[r][j] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int r = 0; r < RI; ++r)
#pragma unroll
            for (int j = 0; j < NB; ++j) t[r][j] = Mma<S>::fma(p, b[h][j], a[h][i + r], t[r][j]);
#pragma unroll
      for (int r = 0; r < RI; ++r)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i + r][j] += t[r][j];
    }
  }
}

template <typename S> constexpr int kVec = 16 / (int)sizeof(S);   // elements of a chunk
template <typename S> constexpr int kStep = 128 / (int)sizeof(S);  // k of a tile

// The exclusive-or of a line's chunk positions.  kRow: a read's 16 lanes are
// 16 lines of 128 bytes (two lines fill the 64 banks).  kCol: a read of 32
// lanes covers lines {0..3, 8..11} of 32 bytes each (16-bit), one of 64 lanes
// lines j, 4 + j, 8 + j, 12 + j of 64 bytes each (fp32).
__device__ __forceinline__ int row_swizzle(int r) { return (r >> 1) & 7; }
template <typename S, int R>
__device__ __forceinline__ int col_swizzle(int k) {
  static_assert(R >= 64, "kCol tiles hold 64 rows or more");
  if constexpr (sizeof(S) == 4) return 4 * ((k >> 2) & 3);
  if constexpr (R == 64) return 2 * (((k >> 1) & 1) | ((k >> 2) & 2));
  return 2 * ((k & 3) | ((k >> 1) & 4));
}

// One operand of a block: where a thread's chunks of a tile come from.  NW
// waves fetch the tile in units of 64 chunks (1 KB of LDS), wave w units w,
// w + NW, ... (counted modulo the tile's units, so that every wave issues the
// same number and small tiles are fetched twice).
template <typename S, int L, int R, int NW>
struct TileLoader {
  static constexpr int kUnits = R / 8;
  static constexpr int kLoads = (kUnits + NW - 1) / NW;
  static constexpr int kBytes = R * 128;
  static constexpr int kLineChunks = L == kRow ? 8 : R / kVec<S>;
  static_assert(kLineChunks <= 64, "a unit holds whole lines");

  uint32_t off[kLoads];  // byte offset of a thread's chunk from the tile's corner, or out of range
  int pos;               // kRow: the chunk's byte within the line

  static __device__ __forceinline__ int unit(int i, int wave) { return (wave + i * NW) % kUnits; }
  static __device__ __forceinline__ int line(int u, int lane) { return u * (64 / kLineChunks) + lane / kLineChunks; }
  static __device__ __forceinline__ int chunk(int u, int lane) {
    const int l = line(u, lane), p = lane % kLineChunks;
    if constexpr (L == kRow) return p ^ row_swizzle(l);
    else return p ^ col_swizzle<S, R>(l);
  }

  // first: the tile's first row from the corner; rows: how many of its rows
  // exist; row_of(line) maps a kRow tile's
  // line to its row from the corner (identity but for interleaved operands).
  template <typename F>
  __device__ __forceinline__ void init(int64_t ld, int first, int rows, int wave, int lane, F row_of) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int u = unit(i, wave), l = line(u, lane), c = chunk(u, lane);
      const bool ok = L == kRow ? row_of(l) < rows : c * kVec<S> < rows;
      const int line_bytes = (int)ld * (int)sizeof(S);
      const int at = L == kRow ? (first + row_of(l)) * line_bytes + c * 16 : l * line_bytes + first * (int)sizeof(S) + c * 16;
      off[i] = ok ? (uint32_t)at : kBufferOob;
    }
    // every unit of a wave has the same parity of 8 lines, so the same chunk
    static_assert(NW % 2 == 0, "units of a wave keep their parity");
    pos = L == kRow ? chunk(unit(0, wave), lane) * 16 : 0;
  }

  // Starts the loads of the tile at `base` (its corner) into LDS at `dst`;
  // `left` k exist from there on (0 or less: zeros, no memory is read).
  __device__ __forceinline__ void issue(const void* base, int64_t ld, int left, uint32_t dst, int wave) const {
    issue_two(base, base, ld, left, dst, wave, [](int) { return false; });
  }
  // Lines with second(line) come from the other corner (the same for a unit's lines).
  template <typename F>
  __device__ __forceinline__ void issue_two(const void* base, const void* other, int64_t ld, int left, uint32_t dst,
                                            int wave, F second) const {
    // kCol: lines from `left` on are beyond the range
    const int k = left < 0 ? 0 : (left < kStep<S> ? left : kStep<S>);
    const int bytes = __builtin_amdgcn_readfirstlane(L == kCol ? k * (int)(ld * (int)sizeof(S)) : (k > 0 ? 0x7fffffff : 0));
    const bool in = L == kCol || pos < left * (int)sizeof(S);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int u = unit(i, wave);
      const __amdgpu_buffer_rsrc_t rs =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(second(line(u, 0)) ? other : base), 0, bytes, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(uintptr_t)(dst + u * 1024), 16, in ? off[i] : kBufferOob, 0, 0, 0);
    }
  }
};

// The same through registers, for operands at any element alignment and
// width: whole chunks are unaligned 16-byte loads, those that end outside the
// operand are read element by element, the rest as zero.
template <typename S, int L, int R, int NW>
struct TileRegs {
  using T = TileLoader<S, L, R, NW>;
  u32x4 v[T::kLoads];

  template <typename F>
  __device__ __forceinline__ void load(const S* corner, int64_t ld, int rows, int left, int wave, int lane, F row_of) {
    load_two(corner, corner, ld, rows, left, wave, lane, row_of, [](int) { return false; });
  }
  template <typename F, typename G>
  __device__ __forceinline__ void load_two(const S* corner, const S* other, int64_t ld, int rows, int left, int wave,
                                           int lane, F row_of, G second) {
    if (rows >= R && left >= kStep<S>) {  // a whole tile: nothing to check
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) {
        const int u = T::unit(i, wave), l = T::line(u, lane);
        const S* p = (second(l) ? other : corner) + (int64_t)(L == kRow ? row_of(l) : l) * ld + T::chunk(u, lane) * kVec<S>;
        v[i] = *reinterpret_cast<const u32x4_a2*>(p);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      const int u = T::unit(i, wave), l = T::line(u, lane), c = T::chunk(u, lane);
      const int e = c * kVec<S>;
      // elements of the chunk that exist
      const int line_no = L == kRow ? row_of(l) : l;
      const int lines = L == kRow ? rows : left, len = L == kRow ? left : rows;
      const int have = line_no < lines ? len - e : 0;
      const S* p = (second(l) ? other : corner) + (int64_t)line_no * ld + e;
      v[i] = {0u, 0u, 0u, 0u};
      if (have >= kVec<S>)
        v[i] = *reinterpret_cast<const u32x4_a2*>(p);
      else if (have > 0)
        v[i] = ld16_elems<S>(p, have);
    }
  }
  __device__ __forceinline__ void store(uint32_t dst, int wave, int lane) const {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      const uint32_t a = dst + T::unit(i, wave) * 1024 + lane * 16;
      asm volatile("ds_write_b128 %0, %1" ::"v"(a), "v"(v[i]) : "memory");
    }
  }
};

// ---- fragments ---------------------------------------------------------------
// Each asm statement waits for its own reads before it ends.

__device__ __forceinline__ u32x4 join(const u32x2& a, const u32x2& b) { return {a[0], a[1], b[0], b[1]}; }

// kRow: NF fragments 2048 bytes apart, both halves of k (a0, a1).
template <int NF>
__device__ __forceinline__ void read_row_frags(u32x4 (&f)[2][NF], uint32_t a0, uint32_t a1) {
  if constexpr (NF == 1) {
    asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0][0]), "=&v"(f[1][0]) : "v"(a0), "v"(a1) : "memory");
  } else if constexpr (NF == 2) {
    asm volatile(
        "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:2048\n\t"
        "ds_read_b128 %2, %5\n\tds_read_b128 %3, %5 offset:2048\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(f[0][0]), "=&v"(f[0][1]), "=&v"(f[1][0]), "=&v"(f[1][1]) : "v"(a0), "v"(a1) : "memory");
  } else {
    static_assert(NF == 4, "1, 2 or 4 fragments");
    asm volatile(
        "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:2048\n\t"
        "ds_read_b128 %2, %8 offset:4096\n\tds_read_b128 %3, %8 offset:6144\n\t"
        "ds_read_b128 %4, %9\n\tds_read_b128 %5, %9 offset:2048\n\t"
        "ds_read_b128 %6, %9 offset:4096\n\tds_read_b128 %7, %9 offset:6144\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(f[0][0]), "=&v"(f[0][1]), "=&v"(f[0][2]), "=&v"(f[0][3]), "=&v"(f[1][0]), "=&v"(f[1][1]),
          "=&v"(f[1][2]), "=&v"(f[1][3])
        : "v"(a0), "v"(a1) : "memory");
  }
}

// kCol, 16 bits: two fragments, their addresses a and b; LINE bytes a line.
// Lines 0 and 4 (the lane's eight k in two reads) of both halves of k.
template <int LINE, int NF>
__device__ __forceinline__ void read_col16_frags(u32x4 (&f)[2][NF], int i, uint32_t a, uint32_t b) {
  u32x2 r[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%10\n\t"
      "ds_read_b64_tr_b16 %4, %8 offset:%11\n\tds_read_b64_tr_b16 %5, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:%11\n\tds_read_b64_tr_b16 %7, %9 offset:%12\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
      : "v"(a), "v"(b), "i"(4 * LINE), "i"(32 * LINE), "i"(36 * LINE) : "memory");
  f[0][i] = join(r[0], r[1]);
  f[0][i + 1] = join(r[2], r[3]);
  f[1][i] = join(r[4], r[5]);
  f[1][i + 1] = join(r[6], r[7]);
}
template <int LINE>
__device__ __forceinline__ void read_col16_frags4(u32x4 (&f)[2][4], const uint32_t (&a)[4]) {
  u32x2 r[16];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:%20\n\t"
      "ds_read_b64_tr_b16 %2, %17\n\tds_read_b64_tr_b16 %3, %17 offset:%20\n\t"
      "ds_read_b64_tr_b16 %4, %18\n\tds_read_b64_tr_b16 %5, %18 offset:%20\n\t"
      "ds_read_b64_tr_b16 %6, %19\n\tds_read_b64_tr_b16 %7, %19 offset:%20\n\t"
      "ds_read_b64_tr_b16 %8, %16 offset:%21\n\tds_read_b64_tr_b16 %9, %16 offset:%22\n\t"
      "ds_read_b64_tr_b16 %10, %17 offset:%21\n\tds_read_b64_tr_b16 %11, %17 offset:%22\n\t"
      "ds_read_b64_tr_b16 %12, %18 offset:%21\n\tds_read_b64_tr_b16 %13, %18 offset:%22\n\t"
      "ds_read_b64_tr_b16 %14, %19 offset:%21\n\tds_read_b64_tr_b16 %15, %19 offset:%22\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]),
        "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]), "=&v"(r[15])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(4 * LINE), "i"(32 * LINE), "i"(36 * LINE) : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[0][i] = join(r[2 * i], r[2 * i + 1]);
    f[1][i] = join(r[8 + 2 * i], r[9 + 2 * i]);
  }
}

// kCol, fp32: two fragments, at a and b, both halves of k.
template <int LINE, int NF>
__device__ __forceinline__ void read_col32_frags(u32x4 (&f)[2][NF], int i, uint32_t a, uint32_t b) {
  uint32_t r[16];
  asm volatile(
      "ds_read_b32 %0, %16\n\tds_read_b32 %1, %16 offset:%18\n\tds_read_b32 %2, %16 offset:%19\n\t"
      "ds_read_b32 %3, %16 offset:%20\n\tds_read_b32 %4, %16 offset:%21\n\tds_read_b32 %5, %16 offset:%22\n\t"
      "ds_read_b32 %6, %16 offset:%23\n\tds_read_b32 %7, %16 offset:%24\n\t"
      "ds_read_b32 %8, %17\n\tds_read_b32 %9, %17 offset:%18\n\tds_read_b32 %10, %17 offset:%19\n\t"
      "ds_read_b32 %11, %17 offset:%20\n\tds_read_b32 %12, %17 offset:%21\n\tds_read_b32 %13, %17 offset:%22\n\t"
      "ds_read_b32 %14, %17 offset:%23\n\tds_read_b32 %15, %17 offset:%24\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]),
        "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]), "=&v"(r[15])
      : "v"(a), "v"(b), "i"(LINE), "i"(2 * LINE), "i"(3 * LINE), "i"(16 * LINE), "i"(17 * LINE), "i"(18 * LINE),
        "i"(19 * LINE)
      : "memory");
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    f[0][i + k] = {r[8 * k], r[8 * k + 1], r[8 * k + 2], r[8 * k + 3]};
    f[1][i + k] = {r[8 * k + 4], r[8 * k + 5], r[8 * k + 6], r[8 * k + 7]};
  }
}

// The NF fragments of a wave, from row `first` (a multiple of 16 NF) of a tile of R rows.
template <typename S, int L, int R, int NF>
struct FragReader {
  static constexpr int kLine = R * (int)sizeof(S);  // kCol
  uint32_t a[L == kRow ? 2 : NF];

  __device__ __forceinline__ void init(int first, int lane) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (L == kRow) {
      a[0] = (uint32_t)((first + i) * 128 + ((g ^ row_swizzle(i)) * 16));
      a[1] = a[0] ^ 64u;
    } else {
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const int e = first + 16 * j;  // the fragment's first element of a line
        if constexpr (sizeof(S) == 2) {
          const int k = 8 * g + i / 4, c = (e >> 3) + (i & 3) / 2;
          a[j] = (uint32_t)(k * kLine + ((c ^ col_swizzle<S, R>(k)) * 16) + (i & 1) * 8);
        } else {
          const int k = 4 * g, c = (e >> 2) + i / 4;
          a[j] = (uint32_t)(k * kLine + ((c ^ col_swizzle<S, R>(k)) * 16) + (i & 3) * 4);
        }
      }
    }
  }
  __device__ __forceinline__ void read(u32x4 (&f)[2][NF], uint32_t tile) const {
    if constexpr (L == kRow) {
      read_row_frags<NF>(f, tile + a[0], tile + a[1]);
    } else if constexpr (sizeof(S) == 4) {
      static_assert(NF % 2 == 0, "pairs of fragments");
#pragma unroll
      for (int j = 0; j < NF; j += 2) read_col32_frags<kLine, NF>(f, j, tile + a[j], tile + a[j + 1]);
    } else if constexpr (NF == 4) {
      const uint32_t t[4] = {tile + a[0], tile + a[1], tile + a[2], tile + a[3]};
      read_col16_frags4<kLine>(f, t);
    } else {
      static_assert(NF % 2 == 0, "pairs of fragments");
#pragma unroll
      for (int j = 0; j < NF; j += 2) read_col16_frags<kLine, NF>(f, j, tile + a[j], tile + a[j + 1]);
    }
  }
};

// Four fragments of A and two of each half of B (16 KB apart) in one go, 16 bits.
#define MHC_ROW4(v, a, o1, o2, o3)                                                                     \
  "ds_read_b128 %[" v "0], %[" a "0]\n\tds_read_b128 %[" v "1], %[" a "0] offset:" o1 "\n\t"         \
  "ds_read_b128 %[" v "2], %[" a "0] offset:" o2 "\n\tds_read_b128 %[" v "3], %[" a "0] offset:" o3 "\n\t" \
  "ds_read_b128 %[" v "4], %[" a "1]\n\tds_read_b128 %[" v "5], %[" a "1] offset:" o1 "\n\t"         \
  "ds_read_b128 %[" v "6], %[" a "1] offset:" o2 "\n\tds_read_b128 %[" v "7], %[" a "1] offset:" o3 "\n\t"
#define MHC_COL2(v, w, a, o)                                                                          \
  "ds_read_b64_tr_b16 %[" v "0" w "], %[" a "] offset:" o "\n\t"                                       \
  "ds_read_b64_tr_b16 %[" v "1" w "], %[" a "] offset:" o "+1024\n\t"                                  \
  "ds_read_b64_tr_b16 %[" v "2" w "], %[" a "] offset:" o "+8192\n\t"                                  \
  "ds_read_b64_tr_b16 %[" v "3" w "], %[" a "] offset:" o "+9216\n\t"
#define MHC_OUT8(v, r) \
  [v##0] "=&v"(r[0]), [v##1] "=&v"(r[1]), [v##2] "=&v"(r[2]), [v##3] "=&v"(r[3]), [v##4] "=&v"(r[4]), \
  [v##5] "=&v"(r[5]), [v##6] "=&v"(r[6]), [v##7] "=&v"(r[7])
#define MHC_OUT4(v, w, r, i) \
  [v##0##w] "=&v"(r[4 * i]), [v##1##w] "=&v"(r[4 * i + 1]), [v##2##w] "=&v"(r[4 * i + 2]), [v##3##w] "=&v"(r[4 * i + 3])

// A: fragments of 128 lines at `ta`; B: those of the halves at `tb` and `tb` + 16 KB.
template <typename S, int LA, int LB>
__device__ __forceinline__ void read_all(u32x4 (&fa)[2][4], u32x4 (&fb)[2][4], const FragReader<S, LA, 128, 4>& ra,
                                         const FragReader<S, LB, 128, 2>& rb, uint32_t ta, uint32_t tb) {
  if constexpr (sizeof(S) == 4 && !(LA == kRow && LB == kRow)) {
    u32x4 b0[2][2], b1[2][2];
    ra.read(fa, ta);
    rb.read(b0, tb);
    rb.read(b1, tb + 16384);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) fb[h][j] = b0[h][j], fb[h][2 + j] = b1[h][j];
  } else if constexpr (LA == kRow && LB == kRow) {
    u32x4 x[8], y[8];
    asm volatile(MHC_ROW4("x", "a", "2048", "4096", "6144") MHC_ROW4("y", "b", "2048", "16384", "18432") "s_waitcnt lgkmcnt(0)"
                 : MHC_OUT8(x, x), MHC_OUT8(y, y)
                 : [a0] "v"(ta + ra.a[0]), [a1] "v"(ta + ra.a[1]), [b0] "v"(tb + rb.a[0]), [b1] "v"(tb + rb.a[1])
                 : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) fa[i / 4][i % 4] = x[i], fb[i / 4][i % 4] = y[i];
  } else if constexpr (LA == kRow) {
    u32x4 x[8];
    u32x2 y[16];
    asm volatile(MHC_ROW4("x", "a", "2048", "4096", "6144") MHC_COL2("y", "p", "b0", "0") MHC_COL2("y", "q", "b1", "0")
                     MHC_COL2("y", "r", "b0", "16384") MHC_COL2("y", "s", "b1", "16384") "s_waitcnt lgkmcnt(0)"
                 : MHC_OUT8(x, x), MHC_OUT4(y, p, y, 0), MHC_OUT4(y, q, y, 1), MHC_OUT4(y, r, y, 2), MHC_OUT4(y, s, y, 3)
                 : [a0] "v"(ta + ra.a[0]), [a1] "v"(ta + ra.a[1]), [b0] "v"(tb + rb.a[0]), [b1] "v"(tb + rb.a[1])
                 : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) fa[i / 4][i % 4] = x[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) fb[0][j] = join(y[4 * j], y[4 * j + 1]), fb[1][j] = join(y[4 * j + 2], y[4 * j + 3]);
  } else {
    static_assert(LB == kCol, "kCol A goes with kCol B");
    u32x2 x[16], y[16];
    asm volatile(MHC_COL2("x", "p", "a0", "0") MHC_COL2("x", "q", "a1", "0") MHC_COL2("x", "r", "a2", "0")
                     MHC_COL2("x", "s", "a3", "0") MHC_COL2("y", "p", "b0", "0") MHC_COL2("y", "q", "b1", "0")
                         MHC_COL2("y", "r", "b0", "16384") MHC_COL2("y", "s", "b1", "16384") "s_waitcnt lgkmcnt(0)"
                 : MHC_OUT4(x, p, x, 0), MHC_OUT4(x, q, x, 1), MHC_OUT4(x, r, x, 2), MHC_OUT4(x, s, x, 3),
                   MHC_OUT4(y, p, y, 0), MHC_OUT4(y, q, y, 1), MHC_OUT4(y, r, y, 2), MHC_OUT4(y, s, y, 3)
                 : [a0] "v"(ta + ra.a[0]), [a1] "v"(ta + ra.a[1]), [a2] "v"(ta + ra.a[2]), [a3] "v"(ta + ra.a[3]),
                   [b0] "v"(tb + rb.a[0]), [b1] "v"(tb + rb.a[1])
                 : "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      fa[0][j] = join(x[4 * j], x[4 * j + 1]), fa[1][j] = join(x[4 * j + 2], x[4 * j + 3]);
      fb[0][j] = join(y[4 * j], y[4 * j + 1]), fb[1][j] = join(y[4 * j + 2], y[4 * j + 3]);
    }
  }
}
#undef MHC_ROW4
#undef MHC_COL2
#undef MHC_OUT8
#undef MHC_OUT4

}  // namespace mhc
