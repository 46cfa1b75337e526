// New tokens and trees of drafted ones over a cache of pages, float32 inputs.
#include "fa_paged.hpp"

namespace fa {
template hipError_t launch_paged<float>(const PagedParams&, int, hipStream_t);
}  // namespace fa
