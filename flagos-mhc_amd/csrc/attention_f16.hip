#include "attention_run.hpp"

namespace mhc {
template int att_fwd<f16_t>(const AttArgs&, hipStream_t);
template int att_bwd<f16_t>(const AttArgs&, hipStream_t);
}  // namespace mhc
