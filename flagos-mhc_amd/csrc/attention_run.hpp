// Launches of the attention kernels for one element type.
#pragma once

#include "attention_bwd.hpp"
#include "attention_fwd.hpp"
#include "attention_split.hpp"
#include "mhc_launch.hpp"

namespace mhc {

// A launch of `blocks` blocks; a size that the grid does not hold is refused.
template <typename K>
int att_launch(K kernel, const AttArgs& a, int64_t slots, int64_t heads, int threads, size_t lds, hipStream_t st, const char* what) {
  const int64_t blocks = slots * heads;
  if (blocks > 0xffffffffll / threads)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: %lld blocks exceed the 2^32 work-items of a dispatch", what, (long long)blocks);
  if (blocks == 0) return MHC_OK;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, st, a, slots);
  return check_launch(what);
}

// Waves of a block, tile height / 32 and waves a SIMD unit holds of each
// kernel, by the bytes of a head: registers hold a wave's own rows and its sums.
template <typename S, int DB> struct AttShape {
  static constexpr int kBytes = 32 * DB * (int)sizeof(S);
  static constexpr int kFwdNW = kBytes == 256 && sizeof(S) == 2 ? 8 : 4, kFwdNB = sizeof(S) == 2 && DB <= 4 ? 2 : 1, kFwdWPE = kBytes <= 256 ? 2 : 1;
  static constexpr int kDqNW = kBytes == 256 && sizeof(S) == 2 ? 8 : 4, kDqNB = 1, kDqWPE = kBytes <= 256 ? 2 : 1;
  static constexpr int kDkvNW = 4, kDkvNB = 1, kDkvWPE = kBytes <= 256 ? 2 : 1;
  static constexpr bool kDkvLds = kBytes >= 256;
};

template <typename S, int DB>
int att_split_width(const AttArgs& a, const AttSplit& p, hipStream_t st) {
  const int64_t blocks = p.slots * a.n.Hk * p.splits, rows = a.n.Tq * a.n.H;
  if (blocks > 0xffffffffll / 256 || rows > 0xffffffffll / 256)
    return set_error(MHC_ERR_UNSUPPORTED, "attention: %lld blocks exceed the 2^32 work-items of a dispatch", (long long)blocks);
  constexpr int WPE = AttShape<S, DB>::kBytes <= 256 ? 2 : 1;
  hipLaunchKernelGGL((att_split_kernel<S, DB, WPE>), dim3((unsigned)blocks), dim3(64 * kSplitWaves), (split_lds<S, DB>()), st, a,
                     p.slots, p.splits);
  if (const int rc = check_launch("attention")) return rc;
  if (p.splits == 1) return MHC_OK;
  hipLaunchKernelGGL(att_join_kernel<S>, dim3((unsigned)rows), dim3(256), 0, st, a, rows, p.splits);
  return check_launch("attention");
}

template <typename S, int DB>
int att_fwd_width(const AttArgs& a, hipStream_t st) {
  using A = AttShape<S, DB>;
  const AttSplit p = att_split(a.n, device_cu_count());
  if (p.use) return att_split_width<S, DB>(a, p, st);
  constexpr size_t lds = 4 * 32 * A::kFwdNB * Tile<S, DB>::kPitch;
  const int64_t slots = att_slots(a.n.cu_q != nullptr, a.n.Tq, a.n.B, a.n.Sq, 32 * A::kFwdNW);
  return att_launch(att_fwd_kernel<S, DB, A::kFwdNW, A::kFwdNB, A::kFwdWPE>, a, slots, a.n.H, 64 * A::kFwdNW, lds, st,
                    "attention");
}
template <typename S, int DB>
int att_bwd_width(const AttArgs& a, hipStream_t st) {
  using A = AttShape<S, DB>;
  constexpr size_t lds = 4 * 32 * A::kDqNB * Tile<S, DB>::kPitch;
  constexpr size_t lds2 = 2 * (2 * 32 * A::kDkvNB * Tile<S, DB>::kPitch + (2 * 32 * A::kDkvNB * 4 + 255) / 256 * 256) +
                          (A::kDkvLds ? 32 * A::kDkvNW * Tile<S, DB>::kPitch : 0);
  const int64_t slots = att_slots(a.n.cu_q != nullptr, a.n.Tq, a.n.B, a.n.Sq, 32 * A::kDqNW);
  if (const int rc = att_launch(att_dq_kernel<S, DB, A::kDqNW, A::kDqNB, A::kDqWPE>, a, slots, a.n.H, 64 * A::kDqNW, lds, st,
                                "attention_backward"))
    return rc;
  const int64_t slots_k = att_slots(a.n.cu_k != nullptr, a.n.Tk, a.n.B, a.n.Sk, 32 * A::kDkvNW);
  return att_launch(att_dkv_kernel<S, DB, A::kDkvNW, A::kDkvNB, A::kDkvWPE, A::kDkvLds>, a, slots_k, a.n.Hk, 64 * A::kDkvNW, lds2, st,
                    "attention_backward");
}

template <typename S>
int att_fwd(const AttArgs& a, hipStream_t st) {
  if (a.n.d <= 64) return att_fwd_width<S, 2>(a, st);
  if (a.n.d <= 128) return att_fwd_width<S, 4>(a, st);
  if constexpr (sizeof(S) == 2) return att_fwd_width<S, 8>(a, st);
  return MHC_ERR_UNSUPPORTED;  // (refused before)
}
template <typename S>
int att_bwd(const AttArgs& a, hipStream_t st) {
  if (a.n.d <= 64) return att_bwd_width<S, 2>(a, st);
  if (a.n.d <= 128) return att_bwd_width<S, 4>(a, st);
  if constexpr (sizeof(S) == 2) return att_bwd_width<S, 8>(a, st);
  return MHC_ERR_UNSUPPORTED;
}

}  // namespace mhc
