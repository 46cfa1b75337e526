// Rotary positions: pairs of columns (a, b) of q and k turned by the angle of
// the token's position,
//   y_a = x_a cos - x_b sin,   y_b = x_b cos + x_a sin,
// pairs (j, j + R / 2) or, interleaved, (2 j, 2 j + 1) of the first R columns; the
// transposed rotation (gradients) has -sin.  Angles are multiplied out and their
// cosines and sines taken in 64 bits once, into a float32 table; the rotation
// itself is a few float32 operations on each value and bound by the bytes of q
// and k, read and written once.
#include "fa_common.hpp"
#include "fa_ops_params.hpp"

namespace fa {

// one thread an angle: row n of the table is cos(n w_j) for the R / 2 pairs, then
// sin(n w_j), both times p.mul
__global__ __launch_bounds__(256) void rotary_table_kernel(const RotaryTableParams p) {
    const int half = p.R / 2;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= p.n * half) return;
    const int64_t n = id / half;
    const int j = (int)(id - n * half);
    double base = p.base;
    // base mode: the slowest pair is stretched by the factor, the fastest keeps its rate
    if (p.mode == 2 && p.R > 2) base *= pow(p.factor, (double)p.R / (double)(p.R - 2));
    double wj = exp(-2.0 * (double)j / (double)p.R * log(base));
    if (p.mode == 1) wj /= p.factor;
    if (p.mode == 3) {
        // ramp: pairs of at least `high` turns over the original length keep
        // their rate, those of at most `low` are stretched, blended in between
        const double turns = p.original * wj / 6.283185307179586476925286766559;
        const double keep = fmin(1.0, fmax(0.0, (turns - p.low) / (p.high - p.low)));
        wj = wj * keep + wj / p.factor * (1.0 - keep);
    }
    double s, c;
    sincos((double)n * wj, &s, &c);
    p.table[n * p.R + j] = (float)(c * p.mul);
    p.table[n * p.R + half + j] = (float)(s * p.mul);
}

hipError_t launch_rotary_table(const RotaryTableParams& p, hipStream_t s) {
    const int64_t nt = p.n * (p.R / 2);
    if (nt <= 0) return hipSuccess;
    if ((nt + 255) / 256 > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL(rotary_table_kernel, dim3((unsigned)((nt + 255) / 256)), dim3(256), 0, s, p);
    return hipGetLastError();
}

namespace {

template <typename T>
__device__ FA_INLINE inline float to_f32(T x) { return (float)x; }

// V values at an address that is a multiple of A bytes
template <typename T, int V, int A = (int)sizeof(T) * V>
struct alignas(A) Pack {
    T e[V];
};

}  // namespace

// A wave takes one token (and one share of its heads): its lanes are items of V
// columns (2 V of a half-layout pair) times the heads that fit, so that a lane
// loads the cosines and sines of its columns once for all the heads it walks.
// A: alignment of the accesses in bytes
template <typename T, int V, bool INTER, int A>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p, const int n_rot, const int n_items,
                                                     const int head_shares) {
    const int lane = threadIdx.x & 63;
    const int64_t wid = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t tok = wid / head_shares;
    const int share = (int)(wid - tok * head_shares);
    if (tok >= (int64_t)p.B * p.S) return;
    const int b = (int)(tok / p.S), t = (int)(tok - (int64_t)b * p.S);
    int64_t pos = t;
    if (p.pos) {
        const int64_t at = b * p.pos_sb + t * p.pos_ss;
        pos = p.pos64 ? ((const int64_t*)p.pos)[at] : (int64_t)((const int*)p.pos)[at];
    }
    const int hq = p.x[0].heads, heads = hq + p.x[1].heads;
    const float nan = __builtin_nanf("");
    for (int i0 = 0; i0 < n_items; i0 += 64) {  // more items than lanes: in turns
        const int n_here = min(64, n_items - i0);
        const int per = 64 / n_here;  // heads side by side
        const int item = i0 + lane % n_here, hl = lane / n_here;
        if (hl >= per) continue;
        const bool rot = item < n_rot;
        constexpr int NP = INTER ? V / 2 : V;  // pairs of an item
        float c[NP > 0 ? NP : 1], s[NP > 0 ? NP : 1];
#pragma unroll
        for (int e = 0; e < NP; ++e) c[e] = s[e] = 0.f;
        if (rot && pos >= 0) {
            const float* row = p.table + (pos < p.n_pos ? pos : 0) * p.R + item * NP;
            const Pack<float, (NP > 4 ? 4 : NP)>* cp = (const Pack<float, (NP > 4 ? 4 : NP)>*)row;
            const Pack<float, (NP > 4 ? 4 : NP)>* sp = (const Pack<float, (NP > 4 ? 4 : NP)>*)(row + p.R / 2);
#pragma unroll
            for (int e = 0; e < NP; ++e) {
                c[e] = cp[e / 4].e[e % 4];
                s[e] = sp[e / 4].e[e % 4] * p.sign;
            }
            if (pos >= p.n_pos) {
#pragma unroll
                for (int e = 0; e < NP; ++e) c[e] = s[e] = nan;
            }
        }
        // U heads at a time, all read before the first is written: the loads of a head
        // cannot pass the stores of the one before (in and out may be one tensor).
        // Rotated and copied columns share the loads and stores, or a wave would do
        // both one after the other.  16 k tokens x 64 heads of 128, rotated: 237 us
        // with U = 1, 198 with 2, 198 with 4 (forward and backward, 5.5 TB/s);
        // 30001 x 20 heads, half of the columns: 62, 62, 71 us (5.0 TB/s)
        constexpr int U = 2;
        const int step = head_shares * per;
        for (int h0 = share * per + hl; h0 < heads; h0 += U * step) {
            const T* in[U];
            T* out[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int hh = min(h0 + u * step, heads - 1);
                const bool second = hh >= hq;
                const RotaryTensor& x = p.x[second ? 1 : 0];
                const int h = second ? hh - hq : hh;
                in[u] = (const T*)x.in + b * x.in_sb + t * x.in_ss + h * x.in_sh;
                out[u] = (T*)x.out + b * x.out_sb + t * x.out_ss + h * x.out_sh;
            }
            const int col = rot ? item * V : p.R + (item - n_rot) * V;
            if (!rot && col + V > p.D) {  // the last columns
                for (int u = 0; u < U && h0 + u * step < heads; ++u)
                    for (int e = col; e < p.D; ++e) out[u][e] = in[u][e];
                continue;
            }
            Pack<T, V, A> a[U], z[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (h0 + u * step >= heads) break;
                a[u] = *(const Pack<T, V, A>*)(in[u] + col);
                if (!INTER && rot) z[u] = *(const Pack<T, V, A>*)(in[u] + p.R / 2 + col);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (h0 + u * step >= heads) break;
                if (rot && pos >= 0) {  // (else copied: times 1 and 0 an infinity would become NaN, -0 a 0)
#pragma unroll
                    for (int e = 0; e < NP; ++e) {
                        T& p0 = INTER ? a[u].e[(2 * e) % V] : a[u].e[e];
                        T& p1 = INTER ? a[u].e[(2 * e + 1) % V] : z[u].e[e];
                        const float x0 = to_f32(p0), x1 = to_f32(p1);
                        p0 = (T)__builtin_fmaf(x0, c[e], -(x1 * s[e]));
                        p1 = (T)__builtin_fmaf(x1, c[e], x0 * s[e]);
                    }
                }
                *(Pack<T, V, A>*)(out[u] + col) = a[u];
                if (!INTER && rot) *(Pack<T, V, A>*)(out[u] + p.R / 2 + col) = z[u];
            }
        }
    }
}

// Columns an access may hold: what divides the rotated half (the rotated
// columns, interleaved), the columns past them, every stride and base address.
template <typename T, int V, bool INTER, int A = (int)sizeof(T) * V>
hipError_t launch_rotary_v(const RotaryParams& p, hipStream_t s) {
    const int n_rot = INTER ? p.R / V : p.R / 2 / V;
    const int n_items = n_rot + (p.copy ? (p.D - p.R + V - 1) / V : 0);
    if (n_items <= 0) return hipSuccess;
    const int64_t tokens = (int64_t)p.B * p.S;
    const int per = n_items >= 64 ? 1 : 64 / n_items;
    const int turns = (p.x[0].heads + p.x[1].heads + per - 1) / per;  // head turns of a token
    // few tokens: a wave a turn, for the latency; many: a wave a token
    const int shares = (int)(tokens >= 2048 ? 1 : tokens * turns <= 2048 ? turns : (2048 + tokens - 1) / tokens);
    const int64_t nb = (tokens * shares + 3) / 4;
    if (nb > 0x7fffffff) return hipErrorInvalidValue;
    if (nb > 0)
        hipLaunchKernelGGL((rotary_kernel<T, V, INTER, A>), dim3((unsigned)nb), dim3(256), 0, s, p, n_rot, n_items, shares);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_rotary(const RotaryParams& p, hipStream_t s) {
    constexpr int MAXV = 16 / (int)sizeof(T);
    int v = p.vec < MAXV ? p.vec : MAXV;
#define FA_CASE(VV)                                                                                \
    if (v == VV) {                                                                                 \
        if (p.interleaved) {                                                                       \
            if constexpr (VV >= 2) return launch_rotary_v<T, VV, true>(p, s);                      \
            return launch_rotary_v<T, 2, true, (int)sizeof(T)>(p, s);                              \
        }                                                                                          \
        return launch_rotary_v<T, VV, false>(p, s);                                                \
    }
    if constexpr (MAXV >= 8) FA_CASE(8)
    FA_CASE(4)
    FA_CASE(2)
    FA_CASE(1)
#undef FA_CASE
    return hipErrorInvalidValue;
}
template hipError_t launch_rotary<bf16>(const RotaryParams&, hipStream_t);
template hipError_t launch_rotary<f16>(const RotaryParams&, hipStream_t);
template hipError_t launch_rotary<float>(const RotaryParams&, hipStream_t);

}  // namespace fa
