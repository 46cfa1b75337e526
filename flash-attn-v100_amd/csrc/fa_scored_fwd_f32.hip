// Attention with scored rules, forward, f32 inputs.
#include "fa_scored.hpp"

namespace fa {
template hipError_t launch_scored_fwd<float>(const ScoredParams&, int, hipStream_t);
}  // namespace fa
