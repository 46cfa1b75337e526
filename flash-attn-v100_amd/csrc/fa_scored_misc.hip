// Small kernels around attention with scored rules: document ids in tiles, and
// the sum of the slopes' gradient.
#include <limits.h>

#include "fa_common.hpp"
#include "fa_ops_params.hpp"

namespace fa {

// Document ids as the attention kernels read them: a copy padded to whole
// 64-token tiles (negative ids and padding as -1) and the range of each tile's
// ids (a tile with a negative id has min -1).  One wave a tile; a few bytes a
// token against the 2 D and more of k and v.
__global__ __launch_bounds__(256) void doc_tiles_kernel(const DocParams p) {
    const int lane = threadIdx.x & 63;
    const int t = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= p.n_tiles) return;
    const int per = p.pad / 64, b = t / per, i = (t - b * per) * 64 + lane;
    int id = -1;
    if (i < p.S) id = max(-1, p.ids[b * p.sb + i]);
    p.out[(int64_t)b * p.pad + i] = id;
    // padding past the last token neither widens a range nor marks the tile
    int lo = i < p.S ? id : INT_MAX, hi = i < p.S ? id : -1;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        lo = min(lo, __shfl_xor(lo, x));
        hi = max(hi, __shfl_xor(hi, x));
    }
    if (lane == 0) p.rng[t] = make_int2(lo, hi);
}

hipError_t launch_doc_tiles(const DocParams& p, hipStream_t s) {
    if (p.n_tiles <= 0) return hipSuccess;
    hipLaunchKernelGGL(doc_tiles_kernel, dim3((unsigned)((p.n_tiles + 3) / 4)), dim3(256), 0, s, p);
    return hipGetLastError();
}

// One workgroup a slope: the rows of its (batch and) head summed in a fixed
// order, each thread's share in 64 bits.  Bound by the latency of a thread's loads:
// 16 waves, four rows of a thread in flight (12 heads of 2 x 1777 rows: 5.5 us with 4
// waves and one row, 3.9 us).
constexpr int kSlopeThreads = 1024;
__global__ __launch_bounds__(kSlopeThreads) void slope_sum_kernel(const float* __restrict__ rows, float* __restrict__ dst,
                                                                  int B, int H, int Sq, int per_batch) {
    constexpr int NT = kSlopeThreads;
    __shared__ double part[NT];
    const int h = (int)blockIdx.x % H, b0 = per_batch ? (int)blockIdx.x / H : 0, b1 = per_batch ? b0 + 1 : B;
    double acc = 0.0;
    for (int b = b0; b < b1; ++b) {
        const float* r = rows + ((int64_t)b * H + h) * Sq;
        for (int i = (int)threadIdx.x; i < Sq; i += 4 * NT) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = i + j * NT < Sq ? r[i + j * NT] : 0.f;
            acc += ((double)x[0] + (double)x[1]) + ((double)x[2] + (double)x[3]);
        }
    }
    part[threadIdx.x] = acc;
    __syncthreads();
    for (int n = NT / 2; n > 0; n >>= 1) {
        if ((int)threadIdx.x < n) part[threadIdx.x] += part[threadIdx.x + n];
        __syncthreads();
    }
    if (threadIdx.x == 0) dst[blockIdx.x] = (float)part[0];
}

hipError_t launch_slope_sum(const float* rows, float* dst, int B, int H, int Sq, bool per_batch, hipStream_t s) {
    const int n = per_batch ? B * H : H;
    if (n <= 0) return hipSuccess;
    hipLaunchKernelGGL(slope_sum_kernel, dim3((unsigned)n), dim3(kSlopeThreads), 0, s, rows, dst, B, H, Sq, per_batch ? 1 : 0);
    return hipGetLastError();
}

}  // namespace fa
