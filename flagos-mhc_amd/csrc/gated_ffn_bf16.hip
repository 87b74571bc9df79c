// The gated feed-forward block's kernels, bf16.
#include "gated_ffn_run.hpp"

namespace mhc {
template int ffn_fwd<bf16_t>(const FfnFwd&, const FfnDims&, char*, hipStream_t);
template int ffn_bwd<bf16_t>(const FfnBwd&, const FfnDims&, char*, hipStream_t);
}  // namespace mhc
