// Attention with scored rules, forward, bf16 inputs.
#include "fa_scored.hpp"

namespace fa {
template hipError_t launch_scored_fwd<bf16>(const ScoredParams&, int, hipStream_t);
}  // namespace fa
