// Launches of the attention kernels for one element type.
#pragma once

#include "attention_bwd.hpp"
#include "attention_fwd.hpp"
#include "attention_split.hpp"
#include "mhc_launch.hpp"

namespace mhc {

// A launch of `blocks` blocks; a size that the grid does not hold is refused.
template <typename K, typename... X>
int att_launch(K kernel, const AttArgs& a, int64_t slots, int64_t per_slot, int threads, size_t lds, hipStream_t st,
               const char* what, X... x) {
  const int64_t blocks = slots * per_slot;
  if (blocks > 0xffffffffll / threads)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: %lld blocks exceed the 2^32 work-items of a dispatch", what, (long long)blocks);
  if (blocks == 0) return MHC_OK;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, st, a, slots, x...);
  return check_launch(what);
}

// What a head's bytes leave of the registers: two waves a SIMD unit, or one;
// tiles of 64 keys, or 32; the block's own values in LDS in the dk, dv kernel.
template <typename S, int DB> struct AttShape {
  static constexpr int kBytes = 32 * DB * (int)sizeof(S);
  static constexpr int kWPE = kBytes <= 256 ? 2 : 1;
  static constexpr int kFwdWPE = sizeof(S) == 2 || kBytes <= 256 ? 2 : 1;  // (fewer sums than the backward)
  static constexpr int kFwdNW = DB == 8 ? 8 : 4;  // heads of 256: 8 waves 489 us, 4 waves 627 us, one a SIMD unit 882 us (8192 in 2, 20 heads)
  static constexpr int kFwdNB = sizeof(S) == 2 && DB <= 4 ? 2 : 1;
  static constexpr int kBwdNB = sizeof(S) == 2 && DB <= 2 ? 2 : 1;
  static constexpr bool kDkvLds = kBytes > 128;
  static constexpr bool kBig = DB == 4 && sizeof(S) == 2;  // 256 rows a block are a choice (att_big_head)
};

// Blocks of 256 threads that a dispatch holds.
constexpr int64_t kMaxBlocks256 = 0xffffffffll / 256;

template <typename S, int DB>
int att_split_run(const AttArgs& a, const AttSplit& p, hipStream_t st) {
  const int64_t blocks = p.slots * a.n.Hk * p.splits, rows = a.n.Tq * a.n.H;
  if (blocks > kMaxBlocks256)
    return set_error(MHC_ERR_UNSUPPORTED, "attention: %lld blocks exceed the 2^32 work-items of a dispatch", (long long)blocks);
  constexpr int WPE = AttShape<S, DB>::kWPE;
  hipLaunchKernelGGL((att_split_kernel<S, DB, WPE>), dim3((unsigned)blocks), dim3(64 * kSplitWaves), (att_fits<split_lds<S, DB>()>()), st, a,
                     p.slots, p.splits);
  if (const int rc = check_launch("attention")) return rc;
  if (p.splits == 1) return MHC_OK;
  const int64_t joins = rows < kMaxBlocks256 ? rows : kMaxBlocks256;
  hipLaunchKernelGGL(att_join_kernel<S>, dim3((unsigned)joins), dim3(256), 0, st, a, rows, p.splits);
  return check_launch("attention");
}

// LDS of a kernel that holds two times `rows` rows of k and of v, and in the
// end the sums of half of its waves.
template <typename S, int DB, int NW, int KS>
constexpr size_t att_lds(int rows) {
  const size_t tiles = (size_t)4 * rows * Tile<S, DB>::kPitch, sums = KS == 2 ? (size_t)NW / 2 * (DB * 16 + 2) * 256 : 0;
  return tiles > sums ? tiles : sums;
}

template <typename S, int DB, int NW, int KS>
int att_fwd_run(const AttArgs& a, hipStream_t st) {
  using A = AttShape<S, DB>;
  constexpr int BM = 32 * NW / KS;
  return att_launch(att_fwd_kernel<S, DB, NW, KS, A::kFwdNB, A::kFwdWPE>, a, att_slots(a.n.cu_q != nullptr, a.n.Tq, a.n.B, a.n.Sq, BM),
                    a.n.H, 64 * NW, att_fits<att_lds<S, DB, NW, KS>(32 * A::kFwdNB * KS)>(), st, "attention");
}
template <typename S, int DB, int NW, int KS>
int att_dq_run(const AttArgs& a, hipStream_t st) {
  using A = AttShape<S, DB>;
  constexpr int BM = 32 * NW / KS;
  return att_launch(att_dq_kernel<S, DB, NW, KS, A::kBwdNB, A::kWPE>, a, att_slots(a.n.cu_q != nullptr, a.n.Tq, a.n.B, a.n.Sq, BM),
                    a.n.H, 64 * NW, att_fits<att_lds<S, DB, NW, KS>(32 * A::kBwdNB * KS)>(), st, "attention_backward");
}

template <typename S, int DB>
int att_fwd_width(const AttArgs& a, hipStream_t st) {
  const int cus = device_cu_count();
  const AttSplit p = att_split(a.n, cus);
  if (p.use) return att_split_run<S, DB>(a, p, st);
  const AttBlocks b = att_blocks(a.n, AttShape<S, DB>::kBig, cus);
  if constexpr (AttShape<S, DB>::kBig)
    if (b == kBlocks256) return att_fwd_run<S, DB, 8, 1>(a, st);
  if constexpr (AttShape<S, DB>::kFwdWPE == 2 && DB < 8)
    if (b == kBlocksPairs) return att_fwd_run<S, DB, 8, 2>(a, st);
  return att_fwd_run<S, DB, AttShape<S, DB>::kFwdNW, 1>(a, st);
}

template <typename S, int DB>
int att_dq_width(const AttArgs& a, hipStream_t st) {
  const int cus = device_cu_count();
  const AttSplit p = att_split(a.n, cus);
  if (p.use)
    return att_launch(att_dq_split_kernel<S, DB, AttShape<S, DB>::kBytes <= 128 ? 2 : 1>, a, p.slots, a.n.Hk, 64 * kSplitWaves,
                      att_fits<split_lds<S, DB>()>(), st, "attention_backward");
  const AttBlocks b = att_blocks(a.n, AttShape<S, DB>::kBig, cus);
  if constexpr (AttShape<S, DB>::kBig)
    if (b == kBlocks256) return att_dq_run<S, DB, 8, 1>(a, st);
  if constexpr (AttShape<S, DB>::kWPE == 2)
    if (b == kBlocksPairs) return att_dq_run<S, DB, 8, 2>(a, st);
  return att_dq_run<S, DB, 4, 1>(a, st);
}

template <typename S, int DB, int NW>
int att_dkv_run(const AttArgs& a, const AttBwdPlan& p, hipStream_t st) {
  using A = AttShape<S, DB>;
  constexpr size_t lds = att_fits<att_dkv_lds(sizeof(S), DB, NW, 32 * A::kBwdNB, A::kDkvLds)>();
  return att_launch(att_dkv_kernel<S, DB, NW, A::kBwdNB, A::kWPE, A::kDkvLds>, a, p.slots, (int64_t)a.n.Hk * p.splits, 64 * NW,
                    lds, st, "attention_backward", p.splits);
}

template <typename S, int DB>
int att_bwd_width(const AttArgs& a, hipStream_t st) {
  if (const int rc = att_dq_width<S, DB>(a, st)) return rc;
  if (!a.dk) return MHC_OK;  // (keys' gradients that nobody takes)
  const AttBwdPlan p = att_bwd_plan(a.n, sizeof(S) == 4, AttShape<S, DB>::kBig, device_cu_count());
  int rc;
  if constexpr (AttShape<S, DB>::kBig) rc = p.keys == 256 ? att_dkv_run<S, DB, 8>(a, p, st) : att_dkv_run<S, DB, 4>(a, p, st);
  else rc = att_dkv_run<S, DB, 4>(a, p, st);
  if (rc || p.splits == 1) return rc;
  const int64_t all = a.n.Tk * a.n.Hk * a.n.d, blocks = (2 * all + 1023) / 1024;
  if (blocks > kMaxBlocks256)
    return set_error(MHC_ERR_UNSUPPORTED, "attention_backward: %lld blocks exceed the 2^32 work-items of a dispatch", (long long)blocks);
  hipLaunchKernelGGL(att_dkv_join_kernel<S>, dim3((unsigned)blocks), dim3(256), 0, st, a, all, p.splits);
  return check_launch("attention_backward");
}

template <typename S>
int att_fwd(const AttArgs& a, hipStream_t st) {
  if (a.n.d <= 64) return att_fwd_width<S, 2>(a, st);
  if (a.n.d <= 96) return att_fwd_width<S, 3>(a, st);
  if (a.n.d <= 128) return att_fwd_width<S, 4>(a, st);
  if constexpr (sizeof(S) == 2) return a.n.d <= 192 ? att_fwd_width<S, 6>(a, st) : att_fwd_width<S, 8>(a, st);
  return MHC_ERR_UNSUPPORTED;  // (refused before)
}
template <typename S>
int att_bwd(const AttArgs& a, hipStream_t st) {
  if (a.n.d <= 64) return att_bwd_width<S, 2>(a, st);
  if (a.n.d <= 96) return att_bwd_width<S, 3>(a, st);
  if (a.n.d <= 128) return att_bwd_width<S, 4>(a, st);
  if constexpr (sizeof(S) == 2) return a.n.d <= 192 ? att_bwd_width<S, 6>(a, st) : att_bwd_width<S, 8>(a, st);
  return MHC_ERR_UNSUPPORTED;
}

}  // namespace mhc
