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

}  // namespace mhc
