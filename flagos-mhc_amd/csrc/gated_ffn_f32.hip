// The gated feed-forward block's kernels, f32.
#include "gated_ffn_run.hpp"

namespace mhc {
template int ffn_fwd<float>(const FfnFwd&, const FfnDims&, char*, hipStream_t);
template int ffn_bwd<float>(const FfnBwd&, const FfnDims&, char*, hipStream_t);
}  // namespace mhc
