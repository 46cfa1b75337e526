// Operators of a cache of pages: rows of new tokens written into it, an accepted path
// of drafted tokens moved together, sequences forked, pages compacted; gfx950.
//
// All of them move rows of a token (every KV head's columns, 16-byte chunks); a wave
// takes 64 chunks of a row, so that a row's place is found by scalar instructions.
// Bound by the bytes read and written; small calls by the launch.
#include <hip/hip_runtime.h>

#include "fa_common.hpp"
#include "fa_ops_params.hpp"

namespace fa {

namespace {

typedef unsigned chunk_t __attribute__((ext_vector_type(4)));

__device__ FA_INLINE inline int filled(const PoolParams& p, int b) { return p.lens ? max(0, min(p.room, p.lens[b])) : p.room; }

// a token's page (-1: none) and row
struct Place {
    int page, row;
};
__device__ FA_INLINE inline Place place_of(const PoolParams& p, int b, int x) {
    if (!p.table) return {b, x};
    const int col = x / p.page_size;
    const int page = p.table[b * p.table_sb + col];
    return {(unsigned)page < (unsigned)p.pages ? page : -1, x - col * p.page_size};
}
__device__ FA_INLINE inline char* row_at(const PoolParams& p, int kv, int layer, Place at) {
    return p.x[kv] + layer * p.sl[kv] + at.page * p.sp[kv] + at.row * p.sr[kv];
}
// chunk c of a row, of the pool and of a tensor with head stride sh (bytes)
struct Chunk {
    int head, col;
    __device__ FA_INLINE inline Chunk(const PoolParams& p, int c) : head(c / p.chunks), col(16 * (c - c / p.chunks * p.chunks)) {}
};

// ---------------------------------------------------------------------------
// R rows a wave, whose loads are in flight together
template <int R>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheWriteParams p) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv = blockIdx.y & 1, layer = blockIdx.y >> 1;
    const int64_t r0 = ((int64_t)blockIdx.x * 4 + w) * R, rows = (int64_t)p.B * p.N;
    const char* from[R];
    char* to[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        from[r] = nullptr;
        to[r] = nullptr;
        if (r0 + r >= rows) continue;
        const int b = (int)((r0 + r) / p.N), i = (int)((r0 + r) % p.N);
        const int x = __builtin_amdgcn_readfirstlane(filled(p, b)) - p.N + i;
        if (x < 0) continue;
        const Place at = place_of(p, b, x);
        if (at.page < 0) continue;
        from[r] = p.in[kv] + layer * p.in_sl[kv] + b * p.in_sb[kv] + i * p.in_ss[kv];
        to[r] = row_at(p, kv, layer, at);
    }
    const int n = p.heads * p.chunks;
    for (int c0 = 0; c0 < n; c0 += 64) {
        if (c0 + lane >= n) break;
        const Chunk c(p, c0 + lane);
        chunk_t v[R];
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (to[r]) v[r] = *reinterpret_cast<const chunk_t*>(from[r] + c.head * p.in_sh[kv] + c.col);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (to[r]) *reinterpret_cast<chunk_t*>(to[r] + c.head * p.sh[kv] + c.col) = v[r];
    }
}

// ---------------------------------------------------------------------------
// A wave takes 64 chunks of all rows of one path.  Its entries ascend, so that row j
// takes from row j or one behind it: rows are read in groups of 8, before any of them is
// written, and nothing that is still to be read has been written before.
__global__ __launch_bounds__(256) void cache_accept_kernel(const CacheAcceptParams p) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = p.heads * p.chunks, blocks = (n + 63) / 64;
    const int64_t item = (int64_t)blockIdx.x * 4 + w;
    const int per_seq = 2 * p.layers * blocks;
    const int b = (int)(item / per_seq), x = (int)(item % per_seq);
    if (b >= p.B) return;
    const int kv = x & 1, layer = (x >> 1) / blocks, c0 = 64 * ((x >> 1) % blocks);
    const int len = __builtin_amdgcn_readfirstlane(filled(p, b)), first = len - p.N;
    const int* path = p.path + b * p.path_sb;
    int count = 0;
    if (first >= 0) {
        for (int last = -1; count < p.path_cols; count += 64) {
            const int j = count + lane;
            const int a = j < p.path_cols ? path[j] : -1;
            int before = __shfl_up(a, 1);
            if (lane == 0) before = last;
            const uint64_t end = __ballot(a <= before || a >= p.N);
            if (end) {
                count += (int)__builtin_ctzll(end);
                break;
            }
            last = __builtin_amdgcn_readlane(a, 63);
        }
        count = min(count, p.path_cols);
    }
    if (x == 0 && lane == 0) p.new_lens[b] = first >= 0 ? first + count : len;
    const bool mine = c0 + lane < n;
    const Chunk c(p, mine ? c0 + lane : 0);
    const int64_t off = c.head * p.sh[kv] + c.col;
    for (int j0 = 0; j0 < count; j0 += 8) {
        chunk_t v[8];
        char* to[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            to[u] = nullptr;
            const int j = j0 + u;
            if (j >= count) continue;
            const int a = __builtin_amdgcn_readfirstlane(path[j]);
            if (a == j) continue;
            const Place src = place_of(p, b, first + a), dst = place_of(p, b, first + j);
            if (src.page < 0 || dst.page < 0) continue;
            to[u] = row_at(p, kv, layer, dst);
            if (mine) v[u] = *reinterpret_cast<const chunk_t*>(row_at(p, kv, layer, src) + off);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (to[u] && mine) *reinterpret_cast<chunk_t*>(to[u] + off) = v[u];
    }
}

// ---------------------------------------------------------------------------
// Pages in use as bits in LDS, by one workgroup: 16 KB for up to 2^17 pages, 128 KB for
// up to 2^20.
constexpr int kPlan = 1024;  // threads

// sum of x over the workgroup's threads before this one, and the total
__device__ FA_INLINE inline int scan(int x, int* sums, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int inc = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(inc, d);
        if (lane >= d) inc += y;
    }
    __syncthreads();  // (the sums of a call before this one have been read)
    if (lane == 63) sums[w] = inc;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < kPlan / 64; ++i) {
        if (i < w) before += sums[i];
        total += sums[i];
    }
    return before + inc - x;
}

__device__ FA_INLINE inline void mark(const PoolParams& p, unsigned* bits, int page) {
    if ((unsigned)page < (unsigned)p.pages) atomicOr(&bits[page >> 5], 1u << (page & 31));
}

// what sequence b of the new batch has of its source
struct Forked {
    int src, len, part, kept, need;  // part: rows of a partly filled page; kept: pages; need: new ones
    bool drop, copy;                 // no room in the table; the part goes to a new page
    __device__ FA_INLINE inline Forked(const CacheForkParams& p, const int* heirs, int b) {
        src = p.sources[b];
        len = part = kept = need = 0;
        drop = copy = false;
        if ((unsigned)src >= (unsigned)p.B) {
            src = -1;
            return;
        }
        const int n = filled(p, src), full = n / p.page_size;
        const int64_t all = (int64_t)n + max(0, p.more ? p.more[b] : p.more_all);
        drop = all > p.room;
        if (drop) return;
        len = (int)all;
        part = n - full * p.page_size;
        kept = full;
        if (part) {
            const int page = p.table[src * p.table_sb + full];
            copy = heirs[src] != b && (unsigned)page < (unsigned)p.pages;
            if (!copy) ++kept;
        }
        need = (len + p.page_size - 1) / p.page_size - kept;
    }
};

// p.copies doubles as the place of (first new page, 1 where dropped) between the passes
template <int WORDS>
__global__ __launch_bounds__(kPlan) void fork_plan_kernel(const CacheForkParams p) {
    __shared__ unsigned bits[WORDS];
    __shared__ int sums[kPlan / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int* heirs = p.free_list + p.pages;  // per source the first that continues it
    for (int i = tid; i < (p.pages + 31) / 32; i += kPlan) bits[i] = 0u;
    for (int i = tid; i < p.B; i += kPlan) heirs[i] = INT_MAX;
    __threadfence_block();
    __syncthreads();
    for (int i = tid; i < p.n_new; i += kPlan) {
        const int s = p.sources[i];
        if ((unsigned)s >= (unsigned)p.B) continue;
        // one without room for its new tokens does not keep the partly filled page
        if ((int64_t)filled(p, s) + max(0, p.more ? p.more[i] : p.more_all) <= p.room) atomicMin(&heirs[s], i);
    }
    __threadfence_block();
    __syncthreads();
    // pages that the new batch shares or keeps
    for (int b = w; b < p.n_new; b += kPlan / 64) {
        const Forked f(p, heirs, b);
        for (int m = lane; m < f.kept; m += 64) mark(p, bits, p.table[f.src * p.table_sb + m]);
    }
    __syncthreads();
    // the free ones, lowest first
    const int words = (p.pages + 31) / 32, per = (words + kPlan - 1) / kPlan, i0 = min(words, tid * per), i1 = min(words, i0 + per);
    auto free_bits = [&](int i) {
        const int n = p.pages - 32 * i;
        return ~bits[i] & (n >= 32 ? ~0u : (1u << n) - 1u);
    };
    int mine = 0, have;
    for (int i = i0; i < i1; ++i) mine += __popc(free_bits(i));
    int rank = scan(mine, sums, have);
    // what each sequence needs, in the batch's order
    int wanted = 0;
    for (int b0 = 0; b0 < p.n_new; b0 += kPlan) {
        const int b = b0 + tid;
        int need = 0, total;
        if (b < p.n_new) need = Forked(p, heirs, b).need;
        // (sums of parts of a batch stay below 2^31: 1024 sequences of up to 2^20 pages that exist)
        const int before = scan(min(need, p.pages + 1), sums, total);
        if (b < p.n_new) {
            const bool out = need > 0 && (int64_t)wanted + before + need > have;
            p.copies[b] = make_int4(wanted + before, out ? 1 : 0, 0, 0);
        }
        wanted = (int)min((int64_t)p.pages + 1, (int64_t)wanted + total);
    }
    for (int i = i0; i < i1 && rank < wanted; ++i)
        for (unsigned x = free_bits(i); x; x &= x - 1) p.free_list[rank++] = 32 * i + __ffs(x) - 1;
    __threadfence_block();
    __syncthreads();
    for (int b = w; b < p.n_new; b += kPlan / 64) {
        const Forked f(p, heirs, b);
        const int4 plan = p.copies[b];
        const bool gone = f.src < 0 || f.drop || plan.y;
        const int pages = gone ? 0 : f.kept + f.need;
        int* row = p.new_table + (int64_t)b * p.cols;
        for (int m = lane; m < p.cols; m += 64) {
            int page = -1;
            if (m < pages) page = m < f.kept ? p.table[f.src * p.table_sb + m] : p.free_list[plan.x + m - f.kept];
            row[m] = (unsigned)page < (unsigned)p.pages ? page : -1;
        }
        if (lane == 0) {
            p.new_lens[b] = gone ? 0 : f.len;
            p.copies[b] = !gone && f.copy ? make_int4(p.table[f.src * p.table_sb + f.kept], p.free_list[plan.x], f.part, 0)
                                          : make_int4(-1, -1, 0, 0);
        }
    }
}

// rows [0, rows) of one page to another, one layer's keys or values
__device__ FA_INLINE inline void copy_rows(const PoolParams& p, int kv, int layer, int from, int to, int rows, int first, int step) {
    const char* src = row_at(p, kv, layer, Place{from, 0});
    char* dst = row_at(p, kv, layer, Place{to, 0});
    const int n = p.heads * p.chunks, all = rows * n;
    for (int x0 = first; x0 < all; x0 += 4 * step) {
        chunk_t v[4];
        int64_t off[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int x = x0 + u * step;
            if (x >= all) break;
            const int r = x / n;
            const Chunk c(p, x - r * n);
            off[u] = r * p.sr[kv] + c.head * p.sh[kv] + c.col;
            v[u] = *reinterpret_cast<const chunk_t*>(src + off[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (x0 + u * step < all) *reinterpret_cast<chunk_t*>(dst + off[u]) = v[u];
    }
}

__global__ __launch_bounds__(256) void fork_copy_kernel(const CacheForkParams p) {
    const int4 c = p.copies[blockIdx.x];
    if (c.z == 0) return;
    copy_rows(p, blockIdx.y & 1, blockIdx.y >> 1, c.x, c.y, c.z, blockIdx.z * 256 + threadIdx.x, 256 * gridDim.z);
}

// ---------------------------------------------------------------------------
template <int WORDS>
__global__ __launch_bounds__(kPlan) void compact_plan_kernel(const CacheCompactParams p) {
    __shared__ unsigned bits[WORDS];
    __shared__ int sums[kPlan / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int words = (p.pages + 31) / 32;
    for (int i = tid; i < words; i += kPlan) bits[i] = 0u;
    __syncthreads();
    for (int b = w; b < p.B; b += kPlan / 64) {
        const int n = (filled(p, b) + p.page_size - 1) / p.page_size;
        for (int m = lane; m < n; m += 64) mark(p, bits, p.table[b * p.table_sb + m]);
    }
    __syncthreads();
    const int per = (words + kPlan - 1) / kPlan, i0 = min(words, tid * per), i1 = min(words, i0 + per);
    int live = 0, used;
    for (int i = i0; i < i1; ++i) live += __popc(bits[i]);
    const int before = scan(live, sums, used);
    // bits of pages below the number of used ones
    auto low = [&](int i) { return used >= 32 * i + 32 ? ~0u : used <= 32 * i ? 0u : (1u << (used - 32 * i)) - 1u; };
    int hole = 0, holes;
    for (int i = i0; i < i1; ++i) hole += __popc(~bits[i] & low(i));
    int at = scan(hole, sums, holes);
    // pages in use from `used` on: as many as holes; those before this thread's words
    int kept = 0, total;
    for (int i = i0; i < i1; ++i) kept += __popc(bits[i] & low(i));
    int from = before - scan(kept, sums, total);
    for (int i = i0; i < i1; ++i) {
        for (unsigned x = ~bits[i] & low(i); x; x &= x - 1) p.moves[at++].y = 32 * i + __ffs(x) - 1;
        for (unsigned x = bits[i] & ~low(i); x; x &= x - 1) p.moves[from++].x = 32 * i + __ffs(x) - 1;
    }
    if (tid == 0) {
        *p.used = used;
        *p.n_moves = holes;
    }
    __threadfence_block();
    __syncthreads();
    for (int k = tid; k < holes; k += kPlan) p.to[p.moves[k].x] = p.moves[k].y;
    __threadfence_block();
    __syncthreads();
    for (int b = w; b < p.B; b += kPlan / 64) {
        const int n = (filled(p, b) + p.page_size - 1) / p.page_size;
        int* row = p.new_table + (int64_t)b * p.cols;
        for (int m = lane; m < p.cols; m += 64) {
            int page = m < n ? p.table[b * p.table_sb + m] : -1;
            if ((unsigned)page >= (unsigned)p.pages) page = -1;
            row[m] = page >= used ? p.to[page] : page;
        }
    }
}

__global__ __launch_bounds__(256) void compact_copy_kernel(const CacheCompactParams p) {
    const int64_t items = (int64_t)*p.n_moves * 2 * p.layers;
    for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const int x = (int)(i % (2 * p.layers));
        const int2 m = p.moves[i / (2 * p.layers)];
        copy_rows(p, x & 1, x >> 1, m.x, m.y, p.page_size, threadIdx.x, 256);
    }
}

constexpr int kSmallWords = 1 << 12, kLargeWords = 1 << 15;

}  // namespace

hipError_t launch_cache_write(const CacheWriteParams& p, hipStream_t s) {
    const int64_t rows = (int64_t)p.B * p.N;
    const unsigned y = 2 * p.layers;
    if (rows * y >= 16384)
        hipLaunchKernelGGL((cache_write_kernel<4>), dim3((unsigned)((rows + 15) / 16), y), dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((cache_write_kernel<1>), dim3((unsigned)((rows + 3) / 4), y), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_cache_accept(const CacheAcceptParams& p, hipStream_t s) {
    const int64_t items = (int64_t)p.B * 2 * p.layers * ((p.heads * p.chunks + 63) / 64);
    hipLaunchKernelGGL(cache_accept_kernel, dim3((unsigned)((items + 3) / 4)), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_cache_fork(const CacheForkParams& p, hipStream_t s) {
    if (p.pages <= 32 * kSmallWords)
        hipLaunchKernelGGL((fork_plan_kernel<kSmallWords>), dim3(1), dim3(kPlan), 0, s, p);
    else
        hipLaunchKernelGGL((fork_plan_kernel<kLargeWords>), dim3(1), dim3(kPlan), 0, s, p);
    const int z = (p.page_size * p.heads * p.chunks + 1023) / 1024;
    hipLaunchKernelGGL(fork_copy_kernel, dim3((unsigned)p.n_new, (unsigned)(2 * p.layers), (unsigned)min(z, 64)), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_cache_compact(const CacheCompactParams& p, hipStream_t s) {
    if (p.pages <= 32 * kSmallWords)
        hipLaunchKernelGGL((compact_plan_kernel<kSmallWords>), dim3(1), dim3(kPlan), 0, s, p);
    else
        hipLaunchKernelGGL((compact_plan_kernel<kLargeWords>), dim3(1), dim3(kPlan), 0, s, p);
    const int64_t most = (int64_t)(p.pages / 2) * 2 * p.layers;
    if (most > 0) hipLaunchKernelGGL(compact_copy_kernel, dim3((unsigned)min(most, (int64_t)2048)), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace fa
