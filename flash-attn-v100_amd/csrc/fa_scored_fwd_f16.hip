// Attention with scored rules, forward, f16 inputs.
#include "fa_scored.hpp"

namespace fa {
template hipError_t launch_scored_fwd<f16>(const ScoredParams&, int, hipStream_t);
}  // namespace fa
