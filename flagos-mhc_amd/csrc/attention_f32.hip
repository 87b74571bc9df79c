#include "attention_run.hpp"

namespace mhc {
template int att_fwd<float>(const AttArgs&, hipStream_t);
template int att_bwd<float>(const AttArgs&, hipStream_t);
}  // namespace mhc
