// Attention with scored rules, backward, bf16 inputs.
#include "fa_scored.hpp"

namespace fa {
template hipError_t launch_scored_bwd<bf16>(const ScoredParams&, int, hipStream_t);
}  // namespace fa
