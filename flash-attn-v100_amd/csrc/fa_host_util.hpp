// What the sources of the host module share: element types, tensor layouts.
#pragma once

#include <Python.h>

#include <ATen/ATen.h>

#include "fa_abi.h"

namespace fa_host {

inline int32_t dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return FA_DTYPE_F16;
        case at::kBFloat16: return FA_DTYPE_BF16;
        case at::kFloat: return FA_DTYPE_F32;
        default: return -1;  // the library refuses it
    }
}

// t, or a contiguous copy where the kernels' 16-byte loads need one: d stride
// 1, other strides non-negative multiples of 16 bytes, base 16-byte aligned
inline at::Tensor prepare(const at::Tensor& t) {
    const int64_t es = t.element_size(), n = t.dim();
    bool ok = n > 0 && t.stride(n - 1) == 1 && ((uintptr_t)t.data_ptr() & 15) == 0;
    for (int64_t d = 0; ok && d + 1 < n; ++d) ok = t.stride(d) >= 0 && (t.stride(d) * es) % 16 == 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

inline void put_strides(int64_t (&dst)[4], const at::Tensor& t) {
    for (int d = 0; d < 4; ++d) dst[d] = t.stride(d);
}

extern PyMethodDef ops_methods[];  // fa_ops_host.cpp

}  // namespace fa_host
