// The gated feed-forward block's kernels, f16.
#include "gated_ffn_run.hpp"

namespace mhc {
template int ffn_fwd<f16_t>(const FfnFwd&, const FfnDims&, char*, hipStream_t);
template int ffn_bwd<f16_t>(const FfnBwd&, const FfnDims&, char*, hipStream_t);
}  // namespace mhc
