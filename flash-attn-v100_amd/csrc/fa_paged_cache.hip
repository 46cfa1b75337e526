// Operators of a cache of pages: rows of new tokens written into it, an accepted path
// of drafted tokens moved together, sequences forked, pages compacted; gfx950.
//
// All of them move rows of a token (every KV head's columns, 16-byte chunks); a wave
// takes 64 chunks of a row, so that a row's place is found by scalar instructions.
// Bound by the bytes read and written: prompts of 2048 tokens (50 MB in and out) 9.0 us,
// 5.6 TB/s (the writes stay in the last cache); drafts of 64 tokens of 64 sequences in 8
// layers (283 MB with the accepted rows) 53 + 8 us, 4.6 TB/s; a pool of 2520 pages compacted
// (165 MB) 36 us for the rows, 4.6 TB/s, after 8 for its plan.  A small call (one token, a
// fork, a plan) is bound by its launch and a few round trips to memory, 2 to 8 us.
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
// byte offset of chunk c of a row whose heads lie sh bytes apart
__device__ FA_INLINE inline int64_t chunk_at(const PoolParams& p, int64_t sh, int c) {
    if (sh == 16 * p.chunks) return 16 * c;  // (heads in a row: no division)
    const int head = c / p.chunks;
    return head * sh + 16 * (c - head * p.chunks);
}

// ---------------------------------------------------------------------------
// R rows a wave, whose loads are in flight together
template <int R>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheWriteParams p) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv = blockIdx.y & 1, layer = blockIdx.y >> 1;
    const int r0 = (blockIdx.x * 4 + w) * R, rows = p.B * p.N;  // below 2^31
    const char* from[R];
    char* to[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        from[r] = nullptr;
        to[r] = nullptr;
        if (r0 + r >= rows) continue;
        const int b = (r0 + r) / p.N, i = (r0 + r) - b * p.N;
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
        const int64_t in = chunk_at(p, p.in_sh[kv], c0 + lane), out = chunk_at(p, p.sh[kv], c0 + lane);
        chunk_t v[R];
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (to[r]) v[r] = *reinterpret_cast<const chunk_t*>(from[r] + in);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (to[r]) *reinterpret_cast<chunk_t*>(to[r] + out) = v[r];
    }
}

// Rows of at most half a wave's chunks: a wave takes as many rows side by side as fit, R times,
// each lane looking up its own (3120 tokens of each of 59 sequences, one head of 128, 185 MB: 99 us
// with a row a wave, 45 so; 700 of 16, two heads of 64: 9.2 and 5.8)
template <int R>
__global__ __launch_bounds__(256) void cache_write_short_kernel(const CacheWriteParams p) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv = blockIdx.y & 1, layer = blockIdx.y >> 1;
    const int n = p.heads * p.chunks, per = 64 / n, sub = lane / n, c = lane - sub * n, rows = p.B * p.N;
    if (sub >= per) return;
    const int64_t in = chunk_at(p, p.in_sh[kv], c), out = chunk_at(p, p.sh[kv], c);
    const int r0 = (blockIdx.x * 4 + w) * R * per + sub;  // below 2^31: at most 64 R past the rows
    chunk_t v[R];
    char* to[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        to[r] = nullptr;
        const int row = r0 + r * per;
        if (row >= rows) continue;
        const int b = row / p.N, i = row - b * p.N, x = filled(p, b) - p.N + i;
        if (x < 0) continue;
        const Place at = place_of(p, b, x);
        if (at.page < 0) continue;
        to[r] = row_at(p, kv, layer, at) + out;
        v[r] = *reinterpret_cast<const chunk_t*>(p.in[kv] + layer * p.in_sl[kv] + b * p.in_sb[kv] + i * p.in_ss[kv] + in);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (to[r]) *reinterpret_cast<chunk_t*>(to[r]) = v[r];
}

// ---------------------------------------------------------------------------
// A wave takes 64 chunks of all rows of one path.  Its entries ascend, so that row j
// takes from row j or one behind it: rows are read in groups of 8, before any of them is
// written, and nothing that is still to be read has been written before.  Lane j looks up
// the places of entry j: read one after the other, they took 8 of the 15 us of 64 paths of
// up to 9 in 8 layers.
__global__ __launch_bounds__(256) void cache_accept_kernel(const CacheAcceptParams p) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = p.heads * p.chunks, blocks = (n + 63) / 64;
    const int item = blockIdx.x * 4 + w, per_seq = 2 * p.layers * blocks;  // items: below 2^31
    const int b = item / per_seq, x = item - b * per_seq;
    if (b >= p.B) return;
    const int kv = x & 1, layer = (x >> 1) / blocks, c0 = 64 * ((x >> 1) - layer * blocks);
    const int* path = p.path + b * p.path_sb;
    int a = lane < p.path_cols ? path[lane] : -1;
    const int len = __builtin_amdgcn_readfirstlane(filled(p, b)), first = len - p.N;
    const bool mine = c0 + lane < n;
    char* const rows = row_at(p, kv, layer, Place{0, 0}) + (mine ? chunk_at(p, p.sh[kv], c0 + lane) : 0);
    int count = 0;
    for (int j0 = 0, last = -1; first >= 0 && j0 < p.path_cols; j0 += 64) {
        if (j0) a = j0 + lane < p.path_cols ? path[j0 + lane] : -1;
        int before = __shfl_up(a, 1);
        if (lane == 0) before = last;
        const uint64_t end = __ballot(a <= before || a >= p.N);
        const int m = end ? (int)__builtin_ctzll(end) : 64;
        int64_t from = -1, to = -1;
        if (lane < m && a != j0 + lane) {
            const Place src = place_of(p, b, first + a), dst = place_of(p, b, first + j0 + lane);
            if (src.page >= 0 && dst.page >= 0) {
                from = src.page * p.sp[kv] + src.row * p.sr[kv];
                to = dst.page * p.sp[kv] + dst.row * p.sr[kv];
            }
        }
        for (int g = 0; g < m; g += 8) {
            chunk_t v[8];
            int64_t at[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int64_t src = __shfl(from, g + u);
                at[u] = __shfl(to, g + u);
                if (src >= 0 && mine) v[u] = *reinterpret_cast<const chunk_t*>(rows + src);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (at[u] >= 0 && mine) *reinterpret_cast<chunk_t*>(rows + at[u]) = v[u];
        }
        count = j0 + m;
        if (end) break;
        last = __builtin_amdgcn_readlane(a, 63);
    }
    if (x == 0 && lane == 0) p.new_lens[b] = first >= 0 ? first + min(count, p.path_cols) : len;
}

// ---------------------------------------------------------------------------
// Pages in use as bits in LDS, by one workgroup: 16 KB for up to 2^17 pages (and there what
// is known of up to 1024 sequences), 128 KB for up to 2^20.  Bound by the round trips to
// memory, one after the other.
constexpr int kPlan = 1024;  // threads
constexpr int kSmallWords = 1 << 12, kLargeWords = 1 << 15;

// sum of x over the workgroup's threads before this one, and the total
template <typename I>
__device__ FA_INLINE inline I scan(I x, I* sums, I& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    I inc = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const I y = __shfl_up(inc, d);
        if (lane >= d) inc += y;
    }
    __syncthreads();  // (the sums of a call before this one have been read)
    if (lane == 63) sums[w] = inc;
    __syncthreads();
    I before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPlan / 64; ++i) {
        const I y = sums[i];
        if (i < w) before += y;
        total += y;
    }
    return before + inc - x;
}

__device__ FA_INLINE inline void mark(const PoolParams& p, unsigned* bits, int page) {
    if ((unsigned)page < (unsigned)p.pages) atomicOr(&bits[page >> 5], 1u << (page & 31));
}

// f(row, column, page of the table or -1) for every column of every one of `rows` rows, whose
// first kept(row) columns are read of row source(row): four reads of a thread in flight
template <typename K, typename S, typename F>
__device__ FA_INLINE inline void each_column(const PoolParams& p, int rows, K&& kept, S&& source, F&& f) {
    const int64_t all = (int64_t)rows * p.cols;
    for (int64_t x0 = threadIdx.x; x0 < all; x0 += 4 * kPlan) {
        int page[4], row[4], col[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t x = x0 + u * kPlan;
            row[u] = -1;
            if (x >= all) continue;
            row[u] = (int)((unsigned)x / (unsigned)p.cols);  // (rows times columns: below 2^31)
            col[u] = (int)x - row[u] * p.cols;
            page[u] = col[u] < kept(row[u]) ? p.table[source(row[u]) * p.table_sb + col[u]] : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (row[u] >= 0) f(row[u], col[u], page[u]);
    }
}

template <int WORDS>
__global__ __launch_bounds__(kPlan) void fork_plan_kernel(const CacheForkParams p) {
    constexpr bool SMALL = WORDS == kSmallWords;
    constexpr int NEAR = SMALL ? 1024 : 1, LIST = SMALL ? 4096 : 1;
    __shared__ unsigned bits[WORDS];
    __shared__ int sums[kPlan / 64], near_heirs[NEAR], near_list[LIST];
    __shared__ ForkPlan near_plan[NEAR];
    const int tid = threadIdx.x;
    // per source the first that continues it; per sequence what it takes; pages to give
    int* const heirs = SMALL && p.B <= NEAR ? near_heirs : p.heirs;
    ForkPlan* const plan = SMALL && p.n_new <= NEAR ? near_plan : p.plan;
    int* const list = SMALL && p.pages <= LIST ? near_list : p.free_list;
    for (int i = tid; i < (p.pages + 31) / 32; i += kPlan) bits[i] = 0u;
    for (int i = tid; i < p.B; i += kPlan) heirs[i] = INT_MAX;
    __threadfence_block();
    __syncthreads();
    for (int b = tid; b < p.n_new; b += kPlan) {
        ForkPlan f = {};
        f.src = p.sources[b];
        f.len = -1;  // dropped, or no source
        if ((unsigned)f.src < (unsigned)p.B) {
            const int n = filled(p, f.src);
            const int64_t all = (int64_t)n + max(0, p.more ? p.more[b] : p.more_all);
            if (all <= p.room) {
                f.len = (int)all;
                f.kept = n / p.page_size;
                f.part = n - f.kept * p.page_size;
                // the page that the part is in (one that is none stays with all)
                f.page = f.part ? p.table[f.src * p.table_sb + f.kept] : -1;
                atomicMin(&heirs[f.src], b);
            }
        }
        plan[b] = f;
    }
    __threadfence_block();
    __syncthreads();
    // what each needs, in the batch's order: counts that no pool holds stay beyond it
    int wanted = 0;
    for (int b0 = 0; b0 < p.n_new; b0 += kPlan) {
        const int b = b0 + tid;
        int total;
        ForkPlan f = {};
        if (b < p.n_new) {
            f = plan[b];
            if (f.len >= 0) {
                f.copy = f.part && (unsigned)f.page < (unsigned)p.pages &&
                         __hip_atomic_load(&heirs[f.src], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != b;
                if (f.part && !f.copy) ++f.kept;
                f.need = (f.len + p.page_size - 1) / p.page_size - f.kept;
            }
        }
        const int before = scan(min(f.need, p.pages + 1), sums, total);
        f.first = wanted + before;
        if (b < p.n_new) plan[b] = f;
        wanted = (int)min((int64_t)p.pages + 1, (int64_t)wanted + total);
    }
    __threadfence_block();
    __syncthreads();
    // pages that the new batch shares or keeps
    auto kept = [&](int b) { return plan[b].kept; };  // (0 where dropped)
    auto source = [&](int b) { return (int64_t)plan[b].src; };
    each_column(p, p.n_new, kept, source, [&](int, int, int page) { mark(p, bits, page); });
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
    for (int i = i0; i < i1 && rank < wanted; ++i)
        for (unsigned x = free_bits(i); x; x &= x - 1) list[rank++] = 32 * i + __ffs(x) - 1;
    __threadfence_block();
    __syncthreads();
    auto gone = [&](const ForkPlan& f) { return f.len < 0 || (f.need > 0 && (int64_t)f.first + f.need > have); };
    each_column(p, p.n_new, kept, source, [&](int b, int m, int page) {
        const ForkPlan f = plan[b];
        if (m >= f.kept && m < f.kept + f.need) page = gone(f) ? -1 : list[f.first + m - f.kept];
        if (gone(f) || (unsigned)page >= (unsigned)p.pages) page = -1;
        p.new_table[(int64_t)b * p.cols + m] = page;
    });
    for (int b = tid; b < p.n_new; b += kPlan) {
        const ForkPlan f = plan[b];
        p.new_lens[b] = gone(f) ? 0 : f.len;
        p.copies[b] = !gone(f) && f.copy ? make_int4(f.page, list[f.first], f.part, 0) : make_int4(-1, -1, 0, 0);
    }
}

// rows [0, rows) of one page to another, one layer's keys or values: chunks `first` and every
// step-th after it, of `most` from the workgroup's first on
__device__ FA_INLINE inline void copy_rows(const PoolParams& p, int kv, int layer, int from, int to, int rows, int first, int step, int most) {
    const char* src = row_at(p, kv, layer, Place{from, 0});
    char* dst = row_at(p, kv, layer, Place{to, 0});
    const int n = p.heads * p.chunks, all = min(rows * n, first - (int)threadIdx.x + most);
    const bool flat = p.sh[kv] == 16 * p.chunks && p.sr[kv] == 16 * n;  // (rows in a row: no division)
    for (int x0 = first; x0 < all; x0 += 4 * step) {
        chunk_t v[4];
        int64_t off[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int x = x0 + u * step;
            if (x >= all) break;
            if (flat) {
                off[u] = (int64_t)16 * x;
            } else {
                const int r = x / n;
                off[u] = r * p.sr[kv] + chunk_at(p, p.sh[kv], x - r * n);
            }
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
    for (int x = blockIdx.z * 1024; x < c.z * p.heads * p.chunks; x += gridDim.z * 1024)
        copy_rows(p, blockIdx.y & 1, blockIdx.y >> 1, c.x, c.y, c.z, x + threadIdx.x, 256, 1024);
}

// ---------------------------------------------------------------------------
template <int WORDS>
__global__ __launch_bounds__(kPlan) void compact_plan_kernel(const CacheCompactParams p) {
    __shared__ unsigned bits[WORDS];
    __shared__ int sums[kPlan / 64], live_before[kPlan];
    __shared__ unsigned long long sums2[kPlan / 64];
    __shared__ int near_kept[kPlan];
    const int tid = threadIdx.x;
    const int words = (p.pages + 31) / 32;
    auto pages_of = [&](int b) { return (filled(p, b) + p.page_size - 1) / p.page_size; };
    if (tid < p.B) near_kept[tid] = pages_of(tid);
    for (int i = tid; i < words; i += kPlan) bits[i] = 0u;
    __syncthreads();
    auto kept_of = [&](int b) { return b < kPlan ? near_kept[b] : pages_of(b); };
    auto source = [](int b) { return (int64_t)b; };
    each_column(p, p.B, kept_of, source, [&](int, int, int page) { mark(p, bits, page); });
    __syncthreads();
    const int per = (words + kPlan - 1) / kPlan, i0 = min(words, tid * per), i1 = min(words, i0 + per);
    int live = 0, used;
    for (int i = i0; i < i1; ++i) live += __popc(bits[i]);
    live_before[tid] = scan(live, sums, used);
    // bits of pages below the number of used ones
    auto low = [&](int i) { return used >= 32 * i + 32 ? ~0u : used <= 32 * i ? 0u : (1u << (used - 32 * i)) - 1u; };
    // free ones and used ones among them: as many are free as are used from there on
    unsigned hole = 0, kept = 0;
    for (int i = i0; i < i1; ++i) {
        hole += __popc(~bits[i] & low(i));
        kept += __popc(bits[i] & low(i));
    }
    unsigned long long totals;
    const unsigned long long before = scan((unsigned long long)hole << 32 | kept, sums2, totals);
    const int holes = (int)(totals >> 32), stay = (int)(unsigned)totals;
    int at = (int)(before >> 32), from = live_before[tid] - (int)(unsigned)before;
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
    // a page that moves is the k-th used one from there on
    auto moved = [&](int page) {
        const int i = page >> 5, t = i / per;
        int k = live_before[t] - stay + __popc(bits[i] & ((1u << (page & 31)) - 1u));
        for (int j = t * per; j < i; ++j) k += __popc(bits[j]);
        return p.moves[k].y;
    };
    each_column(p, p.B, kept_of, source, [&](int b, int m, int page) {
        if ((unsigned)page >= (unsigned)p.pages) page = -1;
        p.new_table[(int64_t)b * p.cols + m] = page >= used ? moved(page) : page;
    });
}

// 16 KB of a page at a time
__global__ __launch_bounds__(256) void compact_copy_kernel(const CacheCompactParams p, const int pieces) {
    const int per_move = 2 * p.layers * pieces;
    const int64_t items = (int64_t)*p.n_moves * per_move;
    for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const int k = (int)(i / per_move), x = (int)(i - (int64_t)k * per_move), side = x / pieces;
        const int2 m = p.moves[k];
        copy_rows(p, side & 1, side >> 1, m.x, m.y, p.page_size, (x - side * pieces) * 1024 + threadIdx.x, 256, 1024);
    }
}

}  // namespace

hipError_t launch_cache_write(const CacheWriteParams& p, hipStream_t s) {
    const int64_t rows = (int64_t)p.B * p.N;
    const unsigned y = 2 * p.layers;
    const int per = 64 / (p.heads * p.chunks);  // rows that fit a wave
    if (per >= 2) {
        if (rows * y >= 65536)
            hipLaunchKernelGGL((cache_write_short_kernel<4>), dim3((unsigned)((rows + 16 * per - 1) / (16 * per)), y), dim3(256), 0, s, p);
        else
            hipLaunchKernelGGL((cache_write_short_kernel<1>), dim3((unsigned)((rows + 4 * per - 1) / (4 * per)), y), dim3(256), 0, s, p);
    } else if (rows * y >= 65536)
        hipLaunchKernelGGL((cache_write_kernel<4>), dim3((unsigned)((rows + 15) / 16), y), dim3(256), 0, s, p);
    else if (rows * y >= 8192)
        hipLaunchKernelGGL((cache_write_kernel<2>), dim3((unsigned)((rows + 7) / 8), y), dim3(256), 0, s, p);
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
    hipLaunchKernelGGL(fork_copy_kernel, dim3((unsigned)p.n_new, (unsigned)(2 * p.layers), (unsigned)min(z, 1024)), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_cache_compact(const CacheCompactParams& p, hipStream_t s) {
    if (p.pages <= 32 * kSmallWords)
        hipLaunchKernelGGL((compact_plan_kernel<kSmallWords>), dim3(1), dim3(kPlan), 0, s, p);
    else
        hipLaunchKernelGGL((compact_plan_kernel<kLargeWords>), dim3(1), dim3(kPlan), 0, s, p);
    const int pieces = (p.page_size * p.heads * p.chunks + 1023) / 1024;
    const int64_t most = (int64_t)(p.pages / 2) * 2 * p.layers * pieces;
    if (most > 0) hipLaunchKernelGGL(compact_copy_kernel, dim3((unsigned)min(most, (int64_t)8192)), dim3(256), 0, s, p, pieces);
    return hipGetLastError();
}

}  // namespace fa
