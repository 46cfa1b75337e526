// Attention with scored rules, backward, f32 inputs.
#include "fa_scored.hpp"

namespace fa {
template hipError_t launch_scored_bwd<float>(const ScoredParams&, int, hipStream_t);
}  // namespace fa
