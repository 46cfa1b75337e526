// Checks of sizes, strides and rules that the shims of include/fa_ops.h and
// include/fa_paged.h share (host only).
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "fa_abi.h"
#include "fa_ops.h"

namespace fa_ops_check {

constexpr double kLog2eD = 1.4426950408889634;
constexpr int64_t kMaxStride = (int64_t)1 << 40;  // elements; larger ones are refused before any arithmetic on them
constexpr int32_t kTileRows = 256;                // rows whose byte span a tile copy addresses with 32 bits
constexpr int32_t kMaxLen = 1 << 28;

inline int elem_size(int32_t dtype) { return dtype == FA_DTYPE_F32 ? 4 : 2; }
inline bool aligned(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }
inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
inline int compiled_dim(int32_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

// a (.., s, h, d)-strided tensor of rows of whole 16-byte chunks; n strides, the last that of d
inline int32_t check_tensor(const void* ptr, const int64_t* st, int n, int32_t S, int32_t D, int es) {
    if (!ptr) return FA_ERR_NULL_ARG;
    if (!aligned(ptr, 16)) return FA_ERR_ALIGN;
    if (st[n - 1] != 1) return FA_ERR_STRIDE;
    for (int i = 0; i + 1 < n; ++i) {
        if (st[i] < 0) return FA_ERR_STRIDE;
        if (st[i] > kMaxStride) return FA_ERR_TOO_LARGE;
        if ((st[i] * es) % 16 != 0) return FA_ERR_STRIDE;
    }
    const int64_t span = ((int64_t)(kTileRows - 1) * st[n - 3] + D) * es;
    return S <= 0 || span < (1LL << 31) ? FA_OK : FA_ERR_TOO_LARGE;
}

inline int32_t check_sizes(int32_t B, int32_t Sq, int32_t Sk, int32_t H, int32_t Hkv, int32_t D, int32_t dtype, float scale,
                           float softcap) {
    if (B < 0 || Sq < 0 || Sk < 0 || H < 0 || Hkv < 0) return FA_ERR_SHAPE;
    if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16 && dtype != FA_DTYPE_F32) return FA_ERR_DTYPE;
    if (D <= 0 || D > 128 || (D * elem_size(dtype)) % 16 != 0) return FA_ERR_HEAD_DIM;
    if (H == 0 || Hkv == 0 || H % Hkv != 0) return FA_ERR_HEADS;
    if (!std::isfinite(scale) || !(scale > 0.f)) return FA_ERR_SCALE;
    // outside these the constants of the cap leave float32
    if (!std::isfinite(softcap) || (softcap != 0.f && !(softcap >= 1e-6f && softcap <= 1e30f))) return FA_ERR_RULE;
    if (softcap != 0.f && (double)scale / softcap > 1e37) return FA_ERR_RULE;
    if (Sq >= kMaxLen || Sk >= kMaxLen) return FA_ERR_TOO_LARGE;
    const int64_t tiles = ((int64_t)std::max(Sq, Sk) + 31) / 32;
    if (B > 0 && tiles * (int64_t)H > 0x7fffffffLL / B) return FA_ERR_TOO_LARGE;
    return FA_OK;
}

inline int32_t check_slopes(const float* slopes, int64_t sb, int32_t H) {
    if (!slopes) return FA_OK;
    if (!aligned(slopes, 4)) return FA_ERR_ALIGN;
    return sb == 0 || sb == H ? FA_OK : FA_ERR_RULE;
}

template <typename P>
void put_cap(P& p, float scale, float cap) {
    p.scale_log2 = (float)((double)scale * kLog2eD);
    p.cap = cap;
    p.cap_k1 = cap > 0.f ? (float)((double)scale / cap) : 0.f;
    p.cap_k2 = cap > 0.f ? (float)((double)scale / cap * 2.0 * kLog2eD) : 0.f;
    p.cap_top = (float)((double)cap * kLog2eD);
}

template <typename T>
T ceil_div(T a, T b) { return (a + b - 1) / b; }

}  // namespace fa_ops_check
