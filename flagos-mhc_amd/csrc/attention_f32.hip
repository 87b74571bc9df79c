#include "attention_run.hpp"

namespace mhc {
template int att_fwd<float>(const AttArgs&, void*, hipStream_t);
template int att_bwd<float>(const AttArgs&, void*, hipStream_t);
}  // namespace mhc
