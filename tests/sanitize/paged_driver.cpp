// Drives the C ABI of the paged key/value cache (csrc/fa_paged_abi.cpp), built with
// host AddressSanitizer and UndefinedBehaviorSanitizer, over random and extreme
// sizes, strides and options.  The stub launchers below check that grids fit a launch,
// that what a kernel is given stays inside the workspace that was asked for, and,
// with the kernels' own arithmetic over lengths drawn anew, that workgroups and
// parts do.  Addresses are never read.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <random>

#include "fa_paged.h"
#include "fa_common.hpp"
#include "fa_ops_params.hpp"

static long g_cases = 0, g_fails = 0, g_launches = 0;
#define CHECK(cond)                                                         \
    do {                                                                    \
        ++g_cases;                                                          \
        if (!(cond)) {                                                      \
            if (++g_fails < 20) std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
        }                                                                   \
    } while (0)

static std::mt19937_64 rng(11);
static int64_t pick(std::initializer_list<int64_t> v) { return v.begin()[rng() % v.size()]; }

static uintptr_t g_ws = 0, g_end = 0;  // the workspace of the call in progress
static bool inside(const void* p, double bytes) {
    return (uintptr_t)p >= g_ws && (double)((uintptr_t)p - g_ws) + bytes <= (double)(g_end - g_ws);
}
static bool grid(double x, double threads, double y = 1, double z = 1) {
    return x >= 1 && x < 2147483648.0 && x * threads < 4294967296.0 && y < 65536 && z < 65536;
}

namespace fa {
template <typename T>
hipError_t launch_paged(const PagedParams& p, int D, hipStream_t) {
    ++g_launches;
    CHECK(D >= p.cols && (D == 32 || D == 64 || D == 128) && p.H == p.Hkv * p.group);
    CHECK(p.wide == 1 || ((p.wide == 4 || (p.wide == 8 && D == 128)) && sizeof(T) == 2));
    const int64_t rows = (int64_t)p.Sq * p.group, unit = 32 * p.wide, units = (int64_t)p.Hkv * p.unit_tiles;
    const int step = p.wide == 1 ? 128 : 64;
    CHECK(p.unit_tiles * unit >= rows && (p.unit_tiles - 1) * unit < rows && rows < (1LL << 31));
    CHECK(grid((double)p.o_wgs, p.wide == 8 ? 512 : 256) && p.groups >= 1 && p.least >= 1);
    CHECK(p.table ? p.page_blocks >= 1 : p.page_magic == 0);
    if (p.table) {  // the column of every block
        const int64_t last = ((int64_t)p.table_cols * p.page_blocks) - 1;
        for (int64_t blk : {last, last / 2, last - last % p.page_blocks, (int64_t)p.page_blocks - 1, std::min<int64_t>(last, p.page_blocks)})
            CHECK((p.page_blocks == 1 ? blk : (int64_t)(((uint64_t)blk * p.page_magic) >> 32)) == blk / p.page_blocks);
    }
    // the list of steps of lengths drawn anew
    for (int rep = 0; rep < (p.lens ? 4 : 1); ++rep) {
        int64_t steps = 0, most = 0;
        const int mode = (int)(rng() % 4);
        for (int b = 0; b < p.B; ++b) {
            const int64_t n = !p.lens || mode == 0 ? p.Sk : mode == 1 ? (b ? 0 : p.Sk) : (int64_t)(rng() % ((uint64_t)p.Sk + 1));
            const int64_t st = std::max<int64_t>(1, (n + step - 1) / step) + p.extra;
            steps += st;
            most = std::max(most, st);
        }
        CHECK(steps < (1LL << 31));
        int64_t W = std::min<int64_t>(p.groups, (steps + p.least - 1) / p.least);
        const bool whole = !p.part || W <= 1 || most - p.extra <= std::max<int64_t>(p.alone, (steps + W - 1) / W);
        if (whole) W = p.B;
        CHECK(W * units <= p.o_wgs);
        if (!whole) {
            CHECK(p.part && p.stat);
            const double parts = 2.0 * W * units * unit;
            CHECK(inside(p.stat, 8 * parts) && inside(p.part, 4 * parts * D));
            CHECK((double)((char*)p.spans - (char*)p.stat) >= 8 * parts && (char*)p.part - (char*)p.spans >= 8LL * p.B);
            CHECK(grid((double)units * p.wide, 512, 4, p.B));
        }
    }
    return hipSuccess;
}
template hipError_t launch_paged<float>(const PagedParams&, int, hipStream_t);
template hipError_t launch_paged<bf16>(const PagedParams&, int, hipStream_t);
template hipError_t launch_paged<f16>(const PagedParams&, int, hipStream_t);

hipError_t launch_cache_write(const CacheWriteParams& p, hipStream_t) {
    ++g_launches;
    const double rows = (double)p.B * p.N;
    CHECK(rows < 2147483648.0 && grid((rows + 15) / 16, 256, 2.0 * p.layers) && p.page_size > 0);
    return hipSuccess;
}
hipError_t launch_cache_accept(const CacheAcceptParams& p, hipStream_t) {
    ++g_launches;
    CHECK(grid((double)p.B * 2 * p.layers * ((p.heads * p.chunks + 63) / 64) / 4 + 1, 256));
    return hipSuccess;
}
hipError_t launch_cache_fork(const CacheForkParams& p, hipStream_t) {
    ++g_launches;
    CHECK(inside(p.copies, 16.0 * p.n_new) && inside(p.plan, (double)sizeof(ForkPlan) * p.n_new));
    CHECK(inside(p.free_list, 4.0 * p.pages) && inside(p.heirs, 4.0 * p.B));
    CHECK((char*)p.plan >= (char*)p.copies + 16LL * p.n_new && (char*)p.free_list >= (char*)(p.plan + p.n_new) && p.heirs == p.free_list + p.pages);
    CHECK(grid(p.n_new, 256, 2.0 * p.layers, 1024) && (double)p.page_size * p.heads * p.chunks < 2147483648.0);
    CHECK((double)p.n_new * p.cols < 2147483648.0 && p.pages <= FA_MAX_POOL_PAGES);
    return hipSuccess;
}
hipError_t launch_cache_compact(const CacheCompactParams& p, hipStream_t) {
    ++g_launches;
    CHECK(inside(p.n_moves, 4) && inside(p.moves, 8.0 * p.pages) && (char*)p.moves >= (char*)p.n_moves + 4);
    const int64_t pieces = ((int64_t)p.page_size * p.heads * p.chunks + 1023) / 1024;
    CHECK(2.0 * p.layers * pieces < 2147483648.0 && p.pages <= FA_MAX_POOL_PAGES);
    return hipSuccess;
}
}  // namespace fa

static int32_t size() {
    return (int32_t)pick({0, 1, 2, 15, 16, 33, 100, 128, 1000, 4096, 65537, 1 << 20, (1 << 28) - 1, 1 << 28, INT32_MAX, -1});
}
static int64_t stride() { return pick({8, 64, 128, 4096, 1 << 20, 1LL << 33, 1LL << 40, INT64_MAX, 0, -8, 7, 16, 1024}); }
static void* addr() { return (void*)(uintptr_t)pick({1 << 20, 1 << 20, 1 << 20, 1 << 20, 0, (1 << 20) + 8, (1 << 20) + 2}); }
static void* good() { return (void*)(uintptr_t)(1 << 20); }
static void* opt() { return (rng() & 1) ? good() : nullptr; }
static void* use(size_t need) {  // a workspace of just that size, somewhere
    g_ws = (uintptr_t)1 << 40;
    g_end = g_ws + need;
    return (void*)g_ws;
}
static int64_t mul(int64_t a, int64_t b) { return (int64_t)((uint64_t)a * (uint64_t)b); }  // (extreme sizes wrap)

static void pool(fa_page_pool& c, bool wild, bool table, bool layers) {
    std::memset(&c, 0, sizeof(c));
    c.layers = layers ? (int32_t)(wild ? size() : pick({1, 2, 8})) : 1;
    c.num_heads_kv = (int32_t)(wild ? pick({1, 2, 8, 1 << 16, 0, 1 << 17}) : pick({1, 2, 8}));
    c.dtype = (int32_t)(rng() % (wild ? 4 : 3));
    c.head_dim = (int32_t)(wild ? pick({8, 64, 80, 128, 136, 0, 60}) : pick({8, 32, 64, 80, 128}));
    c.batch = wild ? size() : (int32_t)pick({0, 1, 2, 3, 16, 65, 200});
    table = table || (rng() & 1);
    if (table) {
        c.page_size = wild ? size() : (int32_t)pick({16, 32, 48, 64, 256, 1024});
        c.table_cols = wild ? size() : (int32_t)pick({1, 2, 7, 64, 513});
        c.pages = wild ? size() : (int32_t)pick({1, 40, 5000, 1 << 20});
        c.page_table = (const int32_t*)(wild ? addr() : good());
        c.table_stride = wild ? stride() : c.table_cols;
    } else {
        c.page_size = wild ? size() : (int32_t)pick({1, 5, 512, 1003, 70000, (1 << 21) + 16});
        c.table_cols = wild ? (int32_t)pick({1, 1, 2, 0}) : 1;
        c.pages = wild ? size() : c.batch;
    }
    c.key_lengths = (const int32_t*)(uintptr_t)((rng() & 1) ? 1 << 21 : 0);
    c.k = wild ? addr() : good();
    c.v = wild ? addr() : (void*)(uintptr_t)(1 << 22);
    for (auto st : {&c.k_stride, &c.v_stride}) {
        if (wild) {
            for (int d = 0; d < 5; ++d) (*st)[d] = d == 4 ? 1 : stride();
        } else {
            const int64_t row = (int64_t)c.num_heads_kv * c.head_dim;
            const int64_t all[5] = {mul(mul(row, c.page_size), c.pages), row * c.page_size, row, c.head_dim, 1};
            std::memcpy(*st, all, sizeof(all));
        }
    }
}

static void paged(bool wild) {
    fa_paged_args a;
    std::memset(&a, 0, sizeof(a));
    pool(a.pool, wild, false, false);
    a.seqlen_q = wild ? size() : (int32_t)pick({0, 1, 2, 12, 64, 100, 256, 2000});
    a.num_heads = (int32_t)(wild ? pick({1, 2, 8, 64, 0, 3, 1 << 20}) : a.pool.num_heads_kv * pick({1, 2, 4, 64}));
    a.scale = wild ? (float)pick({0, 1, -1}) : 0.1f;
    a.softcap = (rng() & 1) ? 30.f : 0.f;
    a.q = wild ? addr() : good();
    a.o = wild ? addr() : good();
    for (auto st : {&a.q_stride, &a.o_stride}) {
        const int64_t row = mul(a.num_heads, a.pool.head_dim), plain[4] = {mul(row, a.seqlen_q), row, a.pool.head_dim, 1};
        for (int d = 0; d < 4; ++d) (*st)[d] = wild && d < 3 ? stride() : plain[d];
    }
    a.lse = (float*)opt();
    a.slopes = (const float*)opt();
    a.slopes_batch_stride = (rng() & 1) ? a.num_heads : 0;
    if (wild || a.seqlen_q <= FA_MAX_TREE_NODES) a.parents = (const int32_t*)opt();
    a.parents_stride = wild ? stride() : pick({0, a.seqlen_q});
    const int32_t st = fa_paged_check(&a);
    const double tiles = std::max(a.seqlen_q, a.pool.table_cols * (wild ? 0 : a.pool.page_size)) / 32.0 + 1;
    CHECK(wild || st == FA_OK || (st == FA_ERR_TOO_LARGE && tiles * a.num_heads * a.pool.batch > 2e9));
    const size_t n = fa_paged_workspace_size(&a);
    CHECK(st == FA_OK || n == 0);
    CHECK(fa_paged_fwd(&a, use(n), n, nullptr) == st);
    if (n) CHECK(fa_paged_fwd(&a, use(n), n - 1, nullptr) == FA_ERR_WORKSPACE);
}

static void cache(bool wild) {
    fa_cache_write_args w;
    std::memset(&w, 0, sizeof(w));
    pool(w.pool, wild, false, true);
    w.tokens = wild ? size() : (int32_t)pick({0, 1, 64, 5000});
    w.k = wild ? addr() : good();
    w.v = good();
    for (auto st : {&w.k_stride, &w.v_stride}) {
        const int64_t row = mul(w.pool.num_heads_kv, w.pool.head_dim);
        const int64_t plain[5] = {mul(mul(row, w.tokens), w.pool.batch), mul(row, w.tokens), row, w.pool.head_dim, 1};
        for (int d = 0; d < 5; ++d) (*st)[d] = wild && d < 4 ? stride() : plain[d];
    }
    int32_t st = fa_cache_write_check(&w);
    CHECK(wild || st == FA_OK);
    CHECK(fa_cache_write(&w, nullptr) == st);

    fa_cache_accept_args a;
    std::memset(&a, 0, sizeof(a));
    pool(a.pool, wild, false, true);
    a.path = (const int32_t*)(wild ? addr() : good());
    a.path_cols = wild ? size() : (int32_t)pick({0, 1, 9, 200});
    a.path_stride = wild ? stride() : a.path_cols;
    a.tokens = wild ? size() : 64;
    a.new_lengths = (int32_t*)(wild ? addr() : good());
    st = fa_cache_accept_check(&a);
    CHECK(wild || st == FA_OK);
    CHECK(fa_cache_accept(&a, nullptr) == st);

    fa_cache_fork_args f;
    std::memset(&f, 0, sizeof(f));
    pool(f.pool, wild, true, true);
    f.sources = (const int32_t*)(wild ? addr() : good());
    f.more = (const int32_t*)opt();
    f.more_all = (int32_t)pick({0, 1, -1, INT32_MAX});
    f.new_batch = wild ? size() : (int32_t)pick({0, 1, 7, 1500});
    f.new_table = (int32_t*)(uintptr_t)(1 << 23);
    f.new_lengths = (int32_t*)(wild ? addr() : good());
    st = fa_cache_fork_check(&f);
    CHECK(wild || st == FA_OK);
    size_t n = fa_cache_fork_workspace_size(&f);
    CHECK(st == FA_OK || n == 0);
    CHECK(fa_cache_fork(&f, use(n), n, nullptr) == st);
    if (n) CHECK(fa_cache_fork(&f, use(n), n - 1, nullptr) == FA_ERR_WORKSPACE);

    fa_cache_compact_args c;
    std::memset(&c, 0, sizeof(c));
    pool(c.pool, wild, true, true);
    c.new_table = (int32_t*)(uintptr_t)(1 << 23);
    c.used = (int32_t*)(wild ? addr() : good());
    st = fa_cache_compact_check(&c);
    CHECK(wild || st == FA_OK);
    n = fa_cache_compact_workspace_size(&c);
    CHECK(st == FA_OK || n == 0);
    CHECK(fa_cache_compact(&c, use(n), n, nullptr) == st);
    if (n) CHECK(fa_cache_compact(&c, use(n), n - 1, nullptr) == FA_ERR_WORKSPACE);
}

int main() {
    for (int i = 0; i < 20000; ++i) {
        paged(i & 1);
        cache(i & 1);
    }
    CHECK(g_launches > 20000);
    CHECK(fa_paged_check(nullptr) == FA_ERR_NULL_ARG && fa_cache_write_check(nullptr) == FA_ERR_NULL_ARG);
    CHECK(fa_cache_accept_check(nullptr) == FA_ERR_NULL_ARG && fa_cache_fork_check(nullptr) == FA_ERR_NULL_ARG);
    CHECK(fa_cache_compact_check(nullptr) == FA_ERR_NULL_ARG);
    std::printf("%ld checks, %ld launches, %ld failed\n", g_cases, g_launches, g_fails);
    return g_fails != 0;
}
