// New tokens over caches and a shared prefix, f32 inputs.
#include "fa_rows.hpp"

namespace fa {
template hipError_t launch_rows<float>(const RowsParams&, int, hipStream_t);
}  // namespace fa
