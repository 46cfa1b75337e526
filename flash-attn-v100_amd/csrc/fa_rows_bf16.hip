// New tokens over caches and a shared prefix, bf16 inputs.
#include "fa_rows.hpp"

namespace fa {
template hipError_t launch_rows<bf16>(const RowsParams&, int, hipStream_t);
}  // namespace fa
