// New tokens over caches and a shared prefix, f16 inputs.
#include "fa_rows.hpp"

namespace fa {
template hipError_t launch_rows<f16>(const RowsParams&, int, hipStream_t);
}  // namespace fa
