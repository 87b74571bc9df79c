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

// Few queries: the rows of a group's heads share tiles, and the keys of a tile
// are split into `splits` parts.
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
  s.use = rows <= 64;
  s.slots = n.cu_q ? n.Tq * G / 32 + n.B + 1 : (int64_t)n.B * (((int64_t)n.Sq * G + 31) / 32);
  const int64_t blocks = s.slots * n.Hk;
  const int64_t longest = n.cu_k ? n.Tk : n.Sk;
  int64_t want = (2 * (int64_t)cus + blocks - 1) / blocks;
  const int64_t most = (longest + 127) / 128;  // a tile for each wave
  if (want > most) want = most;
  s.splits = want < 1 ? 1 : (int)want;
  return s;
}

}  // namespace mhc
