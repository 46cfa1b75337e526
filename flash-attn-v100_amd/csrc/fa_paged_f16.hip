// New tokens and trees of drafted ones over a cache of pages, fp16 inputs.
#include "fa_paged.hpp"

namespace fa {
template hipError_t launch_paged<f16>(const PagedParams&, int, hipStream_t);
}  // namespace fa
