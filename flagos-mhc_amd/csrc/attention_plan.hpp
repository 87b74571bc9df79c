// Sizes of an attention call and the plans of its launches: plain C++, so that
// they are tested without a GPU.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace mhc {

struct AttDims {
  const int32_t* cu_q;   // (B + 1,) first rows of packed queries, or null: B sequences of Sq rows
  const int32_t* cu_k;   // the same for keys
  const int32_t* len_k;  // (B,) keys in use of the Sk rows, or null: all
  int64_t Tq, Tk;        // rows of the buffers
  int B, Sq, Sk, H, Hk, d;
  int causal;
};

// Tiles of R rows a sequence list can have at most: packed sequences take
// their share of T / R and one more each, rows behind the last one too.
inline int64_t att_slots(bool packed, int64_t T, int B, int S, int R) {
  return packed ? T / R + B + 1 : (int64_t)B * ((S + R - 1) / R);
}

// Blocks of 128 queries; or of 256, where there are many: half the reads of k
// and v, but more queries past the sequences' ends, and less to choose from when
// blocks end (32768 x 32 heads of 128 bf16: 3 to 5 % faster; documents of 400 to
// 1300 tokens, 700 blocks: 10 % slower); or of 128 with two waves for every 32
// of them, where there are few (4096 x 16 heads over 8, 544 blocks: 110 -> 92 us
// forward, 368 -> 333 us backward; 4096 x 32, 1088 blocks: 172 -> 179 us).
enum AttBlocks { kBlocks128, kBlocks256, kBlocksPairs };
inline AttBlocks att_blocks(const AttDims& n, bool big, int cus) {
  if (big && att_slots(n.cu_q != nullptr, n.Tq, n.B, n.Sq, 256) * n.H >= 8 * (int64_t)cus) return kBlocks256;
  if (att_slots(n.cu_q != nullptr, n.Tq, n.B, n.Sq, 128) * n.H <= 3 * (int64_t)cus) return kBlocksPairs;
  return kBlocks128;
}

// Few queries, or few blocks of 128 (less than one a compute unit): the rows of
// a group's heads share tiles of 32, whose keys a block's waves split, and,
// where even those are few, `splits` blocks.
//   1024 tokens, 4 heads of 128 bf16 (36 blocks of 128): 30 -> 17 us; 777 in
//   three, 16 heads of 80 (160): 16.1 -> 13.7 us; 2048 in four, 16 heads of 128
//   (288): 27 us, split 32 us.
struct AttSplit {
  bool use;
  int splits;
  int64_t slots;
  size_t bytes(const AttDims& n) const {  // partial sums, maxima and sums of weights
    return use && splits > 1 ? (size_t)splits * n.Tq * n.H * (n.d + 2) * 4 : 0;
  }
};

inline AttSplit att_split(const AttDims& n, int cus) {
  const int G = n.H / n.Hk;
  AttSplit s = {false, 1, 0};
  if (n.B == 0 || n.Tq == 0 || n.Tk == 0) return s;
  const int64_t rows = (n.Tq + n.B - 1) / n.B * G;  // of a sequence, on average
  s.use = rows <= 64 || att_slots(n.cu_q != nullptr, n.Tq, n.B, n.Sq, 128) * n.H < cus;
  s.slots = n.cu_q ? n.Tq * G / 32 + n.B + 1 : (int64_t)n.B * (((int64_t)n.Sq * G + 31) / 32);
  const int64_t blocks = s.slots * n.Hk;
  const int64_t longest = n.cu_k ? (n.Tk + n.B - 1) / n.B : n.Sk;  // keys of a sequence, on average
  // As many parts as there are compute units for, of a tile a wave at least
  // (one token, 8 key heads, 32768 keys: 64 parts 30.2 us, 32 28.9 us, 8 54 us) ..
  int64_t parts = cus / blocks;
  if (parts > longest / 128) parts = longest / 128;
  // .. or, for few queries of many sequences, about 1024 keys each, so that
  // blocks end when others do (64 x 8192, one token, 8 key heads: 371 us whole,
  // 320 us in 8 parts).  An odd number: the parts of a head then fall to
  // different XCDs from head to head (7 parts 296 us, 9 parts 296 us).
  if (parts < 4 && rows <= 64 && longest >= 2048 && parts < (longest / 1024 | 1)) parts = longest / 1024 | 1;
  s.splits = parts < 1 ? 1 : (int)parts;
  return s;
}

// Backward, dk and dv: keys of a block, and parts of the queries that a block's
// keys are shared over.
struct AttBwdPlan {
  int keys, splits;
  int64_t slots;
  size_t delta_bytes, part_bytes;
};

// big: heads of 128 16-bit elements, whose kernel has a form of 256 keys a
// block (half the reads of q and the output's gradient; 16384 x 56 heads over 8:
// 14.1 -> 13.5 ms for the whole backward in two parts).
inline AttBwdPlan att_bwd_plan(const AttDims& n, bool fp32, bool big, int cus) {
  AttBwdPlan p = {128, 1, att_slots(n.cu_k != nullptr, n.Tk, n.B, n.Sk, 128), ((size_t)n.H * n.Tq * 4 + 255) / 256 * 256, 0};
  if (n.B == 0 || n.Tq == 0 || n.Tk == 0) return p;
  const int64_t tall = att_slots(n.cu_k != nullptr, n.Tk, n.B, n.Sk, 256);
  if (big && tall * n.Hk >= 2 * (int64_t)cus) {
    p.keys = 256;
    p.slots = tall;
  }
  const int64_t blocks = p.slots * n.Hk;
  const int64_t rows = (n.Tq + n.B - 1) / n.B * (n.H / n.Hk);  // queries of a key head and sequence, on average
  // three blocks a compute unit, and enough queries to be worth the sums' way through memory
  //   777 tokens in three, 16 heads over 4 of 80 (40 blocks): whole 110 us, 8 parts 46 us;
  //   4099 in five, 32 over 8 of 128 (304 blocks): whole 417 us, 3 parts 249 us, 8 parts 299 us
  int64_t want = (3 * (int64_t)cus + blocks - 1) / blocks;
  const int64_t most = rows / (fp32 ? 64 : 128);
  want = want < most ? want : most;
  p.splits = want < 1 ? 1 : (want > 16 ? 16 : (int)want);
  if (p.splits > 1) p.part_bytes = (size_t)p.splits * 2 * n.Tk * n.Hk * n.d * 4;
  return p;
}

// ---- LDS --------------------------------------------------------------------

// Bytes of a tile's row: DB blocks of 32 columns of `es` bytes, at a power of two.
constexpr int att_pitch(int es, int db) { return (db <= 2 ? 64 : (db <= 4 ? 128 : 256)) * es; }

// A block that asks for more than a compute unit has does not run, and nothing
// but the launch's error says so: every launch's bytes go through here, with
// room for what a kernel declares itself.
constexpr size_t kCuLds = 160 * 1024, kOwnLds = 2048;
template <size_t BYTES>
constexpr size_t att_fits() {
  static_assert(BYTES + kOwnLds <= kCuLds, "a block's LDS exceeds a compute unit's");
  return BYTES;
}

// dk and dv: two stages of `rows` rows of q and of the output's gradient, with
// lse and D, and the block's own rows of v if they are held there.
constexpr size_t att_dkv_lds(int es, int db, int waves, int rows, bool own) {
  return (size_t)2 * (2 * rows * att_pitch(es, db) + (2 * rows * 4 + 255) / 256 * 256) + (own ? 32 * waves * att_pitch(es, db) : 0);
}

inline bool att_big_head(const AttDims& n, bool fp32) { return !fp32 && n.d > 96 && n.d <= 128; }

}  // namespace mhc
