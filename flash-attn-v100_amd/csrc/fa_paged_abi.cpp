// Host side of the C ABI declared in include/fa_paged.h: argument validation (no
// HIP call before it passes), workspace layout and the choice of kernels.
// Stateless; launches on the caller's stream and never synchronises.
#include "fa_paged.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fa_common.hpp"
#include "fa_ops_check.hpp"
#include "fa_ops_params.hpp"

namespace {

using namespace fa_ops_check;
using fa::PagedParams;
using fa::PoolParams;

// tokens a sequence has room for, held below 2^28
int64_t room_of(const fa_page_pool& c) { return (int64_t)c.table_cols * c.page_size; }

int32_t check_pool(const fa_page_pool& c, bool table) {
    if (c.layers < 1 || c.pages < 0 || c.page_size < 0 || c.num_heads_kv < 0 || c.batch < 0 || c.table_cols < 0)
        return FA_ERR_SHAPE;
    if (c.dtype != FA_DTYPE_F16 && c.dtype != FA_DTYPE_BF16 && c.dtype != FA_DTYPE_F32) return FA_ERR_DTYPE;
    const int es = elem_size(c.dtype);
    if (c.head_dim <= 0 || c.head_dim > 128 || (c.head_dim * es) % 16 != 0) return FA_ERR_HEAD_DIM;
    if (c.num_heads_kv == 0) return FA_ERR_HEADS;
    if (c.num_heads_kv > (1 << 16) || c.layers > (1 << 14)) return FA_ERR_TOO_LARGE;
    const bool work = c.batch > 0 && c.table_cols > 0;
    if (c.page_table || table) {
        if (c.page_size == 0 || c.page_size % 16 != 0) return FA_ERR_PAGES;
        if (work && !c.page_table) return FA_ERR_NULL_ARG;
        if (!aligned(c.page_table, 4)) return FA_ERR_ALIGN;
        if (c.table_stride < 0 || c.table_stride > kMaxStride) return FA_ERR_PAGES;
    } else if (work && (c.table_cols != 1 || c.pages < c.batch)) {
        return FA_ERR_PAGES;
    }
    if (room_of(c) >= kMaxLen || c.page_size >= kMaxLen) return FA_ERR_TOO_LARGE;
    // blocks of 16 tokens are divided by those of a page with a product of 32 bits, exact up to here
    if (c.page_table && room_of(c) / 16 * (c.page_size / 16) >= (1LL << 32)) return FA_ERR_TOO_LARGE;
    if (!aligned(c.key_lengths, 4)) return FA_ERR_ALIGN;
    if (c.pages == 0 || c.page_size == 0) return FA_OK;
    for (int x = 0; x < 2; ++x) {
        const int64_t* st = x ? c.v_stride : c.k_stride;
        const int32_t e = check_tensor(x ? c.v : c.k, st, 5, c.page_size, c.head_dim, es);
        if (e) return e;
    }
    return FA_OK;
}
// whether there is anything that a sequence may hold
bool empty_pool(const fa_page_pool& c) { return c.pages == 0 || room_of(c) == 0; }

void put_pool(const fa_page_pool& c, PoolParams& p) {
    const int64_t es = elem_size(c.dtype);
    p.x[0] = (char*)c.k;
    p.x[1] = (char*)c.v;
    for (int x = 0; x < 2 && c.pages && c.page_size; ++x) {  // (strides of nothing have not been checked)
        const int64_t* st = x ? c.v_stride : c.k_stride;
        p.sl[x] = st[0] * es;
        p.sp[x] = st[1] * es;
        p.sr[x] = st[2] * es;
        p.sh[x] = st[3] * es;
    }
    p.layers = c.layers;
    p.pages = c.pages;
    p.page_size = c.page_size;
    p.heads = c.num_heads_kv;
    p.chunks = (int)(c.head_dim * es / 16);
    p.B = c.batch;
    p.cols = c.table_cols;
    p.table = c.page_table;
    p.table_sb = c.table_stride;
    p.lens = c.key_lengths;
    p.room = empty_pool(c) ? 0 : (int)room_of(c);
}

// ---------------------------------------------------------------------------
// attention: units of rows of one (sequence, KV head), and their steps
int unit_rows(const PagedParams& p) { return 32 * p.wide; }
void plan(const fa_paged_args* a, PagedParams& p, int64_t& grid, int64_t& shared) {
    const fa_page_pool& c = a->pool;
    const bool f32 = c.dtype == FA_DTYPE_F32, d128 = compiled_dim(c.head_dim) == 128;
    const int64_t rows = (int64_t)a->seqlen_q * (a->num_heads / c.num_heads_kv);
    // Waves that share tiles read K and V once for 128 or 256 rows, but leave larger parts and
    // fewer units: worth it where a workgroup gets enough steps of units that are full enough.
    // us of trees of N on 32 and 8 heads of 128 in units of 32, 128 and 256 rows, pages of 64
    // (sequences x room, N): 16 x 8192, 64: 263, 143, 132; 24 x 4096, 64: 176, 117, 111; 16 x 4000, 64: 125,
    // 82, 80; 2 x 16000, 48: 52, 48, 47; 8 x 4000, 24: 36, 34, 42; the other way 2 x 1000, 64: 17, 23,
    // 26; 16 x 4000, 12: 53, 53, 66; 4 x 16000, 12: 43, 46, 54.  Pages of 16 (which cost wide units more:
    // PageTable::holes): 16 x 8192, 64: 304, 187, 190; 16 x 4000, 64: 142, 101, 106; 16 x 4000, 12: 55, 60, 86.
    // Head dims up to 64 have three workgroups of 128 rows a CU, in units of 32 and 128: 16 x 8192, 64:
    // 161, 86 (64 on 8 heads 287, 148); chunks of 189 in 28 x 546, 96 on 12 heads, pages of 48: 237, 108
    auto busy = [&](int64_t unit, int64_t keys, int64_t workgroups) {
        const int64_t tiles = ceil_div<int64_t>(rows, unit);
        return (double)c.batch * c.num_heads_kv * ceil_div<int64_t>(p.Sk, keys) * tiles / workgroups;
    };
    auto full = [&](int64_t unit) { return (double)rows / (double)(unit * ceil_div<int64_t>(rows, unit)); };
    // Short sequences, whose units cost their beginnings and ends (trees of 64 over up to 300, in
    // units of 32 and 128 rows: 32 sequences 51 and 27, 16 29 and 22, the other way 8 16 and 19; of 12: 32
    // sequences 16 and 20): where units alone fill the device and are filled by their rows.
    const double units128 = (double)c.batch * c.num_heads_kv * ceil_div<int64_t>(rows, 128);
    if (f32 || rows <= 32 || (busy(32, 128, 512) * full(128) < 8 && units128 * full(128) * full(128) < 140))
        p.wide = 1;
    else
        p.wide = !d128 || rows <= 128 || busy(256, 64, 256) * full(256) < 40 ? 4 : 8;
    const int step = p.wide == 1 ? 128 : 64;
    p.unit_tiles = (int)ceil_div<int64_t>(rows, unit_rows(p));
    // workgroups that run at once
    const int64_t slots = p.wide == 1 ? (f32 && d128 ? 256 : 512) : p.wide == 8 ? 256 : d128 ? 512 : 768;
    const int64_t units = (int64_t)c.num_heads_kv * p.unit_tiles;  // of a sequence
    const int64_t most = std::max<int64_t>(1, ceil_div<int64_t>(p.Sk, step));  // steps of a unit
    // groups of a workgroup for each unit that fill the device once, or (more than 1 in 7 of it
    // would stay empty) twice
    int64_t groups = slots / units;
    if (groups * units * 7 < slots * 6) groups = 2 * slots / units;
    p.groups = (int)std::max<int64_t>(groups, 1);
    // Units are shared where a sequence has room for more than join_from steps: below, the join
    // costs more than it saves, the more so the more units there are beside it.  us of one token
    // of each of B sequences on 8 and 4 heads of 128, shared / whole: B x up to 600 keys (5 steps), 16 x
    // 8 heads 16.6 / 14.9, 64 x 8 29 / 26; 1000 keys (8 steps), 64 x 4 25.5 / 22.7, 16 x 8 23.8 / 18.0, the
    // other way 16 x 4 16.5 / 17.5; 2000 (16 steps), 64 x 8 77 / 74, the other way 16 x 4 23.4 / 26.8,
    // 128 with one head 28.5 / 31.4.
    // Where the join is launched all the same (tables with room for more than the sequences hold),
    // what is found to be of `alone` steps at most stays whole: 64 sequences of 150 to 600 of 4096
    // keys, 8 heads, 35 us shared, 30 whole.  Others are shared down to `least` a workgroup: 4 trees of
    // 12 over up to 1000, us with 1, 2 and 4: 15.5, 21.4, 23.3 (16.6 whole); 2 of 24 over up to 4000 23.3,
    // 23.4, 26.2; one token over 8192 16.9, 15.8, 16.8.
    // float32, whose steps take longer, from the third step on (one token of each of 64 sequences
    // over up to 250 keys, 16 on 8 heads of 128: 43 us shared from the second on, 39 so); wide units, whose
    // parts are large, from the ninth (16 trees of 64 over up to 300 keys 26 us shared, 24 whole; 16
    // trees of 48 over up to 600, head dim 64, 28 and, were they whole, 32; 4 chunks of 500 of 600, head
    // dim 64, 35 / 32).
    const int64_t all = units * c.batch;
    const int64_t join_from = f32 ? 2 : p.wide == 1 ? 5 + all / 32 : std::max<int64_t>(8, 4 + all / 64);
    p.alone = (int)std::min<int64_t>(p.wide == 1 ? std::max<int64_t>(all / 32, 1) : join_from, INT32_MAX);
    p.least = f32 || (p.wide == 1 && most <= 16) ? 1 : p.wide == 1 ? 2 : 4;
    // a wide unit's tree, rows and parts take about as long as 3 of its steps: 16 x 8192, trees of
    // 64: 136 us without, 131 to 135 with 1 to 6 of them in the balance
    p.extra = p.wide == 1 ? 0 : 3;
    // workgroups that may share sequences: none where none is that long or, with all of them
    // full, longer than an even share
    const int64_t T = c.batch * (most + p.extra), w = std::min<int64_t>(p.groups, ceil_div<int64_t>(T, p.least));
    shared = w > 1 && most > join_from && (c.key_lengths || most > ceil_div<int64_t>(T, w)) ? w * units : 0;
    p.many = w > 40 * (int64_t)c.batch;
    grid = std::max(units * c.batch, shared);
}
size_t part_rows(const PagedParams& p, int64_t shared) { return (size_t)(2 * shared * unit_rows(p)); }
size_t paged_bytes(const PagedParams& p, int64_t shared) {
    if (!shared) return 0;
    return up256(part_rows(p, shared) * sizeof(float2)) + up256(p.B * sizeof(int2)) +
           up256(part_rows(p, shared) * compiled_dim(p.cols) * sizeof(float));
}

void put_paged(const fa_paged_args* a, PagedParams& p, int64_t& grid, int64_t& shared) {
    const fa_page_pool& c = a->pool;
    p = PagedParams{};
    p.q = a->q; p.k = c.k; p.v = c.v; p.o = a->o; p.lse = a->lse;
    p.q_sb = a->q_stride[0]; p.q_ss = a->q_stride[1]; p.q_sh = a->q_stride[2];
    p.o_sb = a->o_stride[0]; p.o_ss = a->o_stride[1]; p.o_sh = a->o_stride[2];
    p.k_sp = c.k_stride[1]; p.k_ss = c.k_stride[2]; p.k_sh = c.k_stride[3];
    p.v_sp = c.v_stride[1]; p.v_ss = c.v_stride[2]; p.v_sh = c.v_stride[3];
    p.B = c.batch; p.Sq = a->seqlen_q;
    p.Sk = empty_pool(c) ? 0 : (int)room_of(c);
    p.H = a->num_heads; p.Hkv = c.num_heads_kv; p.group = a->num_heads / c.num_heads_kv;
    p.cols = c.head_dim;
    put_cap(p, a->scale, a->softcap);
    p.slopes = a->slopes; p.slopes_sb = a->slopes_batch_stride;
    p.lens = c.key_lengths;
    p.table = p.Sk ? c.page_table : nullptr;
    p.table_sb = c.table_stride;
    p.table_cols = c.table_cols;
    p.pages = c.pages;
    // (a row of tokens: every block is in the first column; rows may be longer than pages that
    // the product divides by exactly)
    p.page_blocks = p.table ? c.page_size / 16 : 2;
    p.page_magic = p.table ? (unsigned)(((1ull << 32) + p.page_blocks - 1) / p.page_blocks) : 0u;
    p.parents = a->parents;
    p.parents_sb = a->parents_stride;
    plan(a, p, grid, shared);
    p.o_wgs = grid;
}

}  // namespace

extern "C" {

int32_t fa_paged_version(void) { return FA_PAGED_VERSION; }

int32_t fa_paged_check(const fa_paged_args* a) {
    if (!a) return FA_ERR_NULL_ARG;
    const fa_page_pool& c = a->pool;
    int32_t st = check_pool(c, false);
    if (st) return st;
    if (c.layers != 1) return FA_ERR_SHAPE;
    if ((st = check_sizes(c.batch, a->seqlen_q, (int32_t)room_of(c), a->num_heads, c.num_heads_kv, c.head_dim, c.dtype,
                          a->scale, a->softcap)))
        return st;
    if ((st = check_slopes(a->slopes, a->slopes_batch_stride, a->num_heads))) return st;
    if (!aligned(a->lse, 4) || !aligned(a->parents, 4)) return FA_ERR_ALIGN;
    if (a->parents && (a->seqlen_q > FA_MAX_TREE_NODES || a->parents_stride < 0 || a->parents_stride > kMaxStride))
        return FA_ERR_PAGES;
    if (c.batch == 0 || a->seqlen_q == 0) return FA_OK;
    const int es = elem_size(c.dtype);
    if ((st = check_tensor(a->q, a->q_stride, 4, a->seqlen_q, c.head_dim, es)) ||
        (st = check_tensor(a->o, a->o_stride, 4, a->seqlen_q, c.head_dim, es)))
        return st;
    // the steps of all sequences in 32 bits, a grid's threads too
    const int64_t rows = (int64_t)a->seqlen_q * (a->num_heads / c.num_heads_kv);
    const double steps = (double)c.batch * (double)(ceil_div<int64_t>(room_of(c), 64) + 4);
    if (steps >= 2e9 || c.batch > 65535 || (double)c.batch * c.num_heads_kv * (double)ceil_div<int64_t>(rows, 32) >= 1 << 24)
        return FA_ERR_TOO_LARGE;
    return FA_OK;
}

size_t fa_paged_workspace_size(const fa_paged_args* a) {
    if (fa_paged_check(a) || a->pool.batch == 0 || a->seqlen_q == 0) return 0;
    PagedParams p;
    int64_t grid, shared;
    put_paged(a, p, grid, shared);
    return paged_bytes(p, shared);
}

int32_t fa_paged_fwd(const fa_paged_args* a, void* workspace, size_t bytes, void* stream) {
    const int32_t st = fa_paged_check(a);
    if (st) return st;
    if (a->pool.batch == 0 || a->seqlen_q == 0) return FA_OK;
    PagedParams p;
    int64_t grid, shared;
    put_paged(a, p, grid, shared);
    const size_t need = paged_bytes(p, shared);
    if (need && (!workspace || bytes < need || !aligned(workspace, 16))) return FA_ERR_WORKSPACE;
    if (need) {
        p.stat = (float2*)workspace;
        p.spans = (int2*)((char*)workspace + up256(part_rows(p, shared) * sizeof(float2)));
        p.part = (float*)((char*)p.spans + up256(p.B * sizeof(int2)));
    }
    const int D = compiled_dim(p.cols);
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a->pool.dtype == FA_DTYPE_F32    ? fa::launch_paged<float>(p, D, s)
                         : a->pool.dtype == FA_DTYPE_BF16 ? fa::launch_paged<fa::bf16>(p, D, s)
                                                          : fa::launch_paged<fa::f16>(p, D, s);
    return e == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------
int32_t fa_cache_write_check(const fa_cache_write_args* a) {
    if (!a) return FA_ERR_NULL_ARG;
    const fa_page_pool& c = a->pool;
    int32_t st = check_pool(c, false);
    if (st) return st;
    if (a->tokens < 0) return FA_ERR_SHAPE;
    // 16 rows a workgroup of 256 threads, which are fewer than 2^32 in a grid
    if ((int64_t)c.batch * a->tokens > (1LL << 28) - 16) return FA_ERR_TOO_LARGE;
    if (c.batch == 0 || a->tokens == 0 || empty_pool(c)) return FA_OK;
    const int es = elem_size(c.dtype);
    if ((st = check_tensor(a->k, a->k_stride, 5, a->tokens, c.head_dim, es)) ||
        (st = check_tensor(a->v, a->v_stride, 5, a->tokens, c.head_dim, es)))
        return st;
    return FA_OK;
}

int32_t fa_cache_write(const fa_cache_write_args* a, void* stream) {
    const int32_t st = fa_cache_write_check(a);
    if (st) return st;
    if (a->pool.batch == 0 || a->tokens == 0 || empty_pool(a->pool)) return FA_OK;
    fa::CacheWriteParams p = {};
    put_pool(a->pool, p);
    const int64_t es = elem_size(a->pool.dtype);
    for (int x = 0; x < 2; ++x) {
        const int64_t* s = x ? a->v_stride : a->k_stride;
        p.in[x] = (const char*)(x ? a->v : a->k);
        p.in_sl[x] = s[0] * es;
        p.in_sb[x] = s[1] * es;
        p.in_ss[x] = s[2] * es;
        p.in_sh[x] = s[3] * es;
    }
    p.N = a->tokens;
    return fa::launch_cache_write(p, (hipStream_t)stream) == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------
int32_t fa_cache_accept_check(const fa_cache_accept_args* a) {
    if (!a) return FA_ERR_NULL_ARG;
    const fa_page_pool& c = a->pool;
    const int32_t st = check_pool(c, false);
    if (st) return st;
    if (a->tokens < 0 || a->path_cols < 0) return FA_ERR_SHAPE;
    if (a->path_stride < 0 || a->path_stride > kMaxStride) return FA_ERR_PAGES;
    if ((double)c.batch * 2 * c.layers * c.num_heads_kv * 32 >= 2e9) return FA_ERR_TOO_LARGE;
    if (c.batch == 0) return FA_OK;
    if (!a->new_lengths || (a->path_cols > 0 && !a->path)) return FA_ERR_NULL_ARG;
    if (!aligned(a->path, 4) || !aligned(a->new_lengths, 4)) return FA_ERR_ALIGN;
    return a->new_lengths == c.key_lengths ? FA_ERR_PAGES : FA_OK;
}

int32_t fa_cache_accept(const fa_cache_accept_args* a, void* stream) {
    const int32_t st = fa_cache_accept_check(a);
    if (st) return st;
    if (a->pool.batch == 0) return FA_OK;
    fa::CacheAcceptParams p = {};
    put_pool(a->pool, p);
    p.path = a->path;
    p.path_sb = a->path_stride;
    p.path_cols = a->path_cols;
    p.N = a->tokens;
    p.new_lens = a->new_lengths;
    return fa::launch_cache_accept(p, (hipStream_t)stream) == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------
int32_t fa_cache_fork_check(const fa_cache_fork_args* a) {
    if (!a) return FA_ERR_NULL_ARG;
    const fa_page_pool& c = a->pool;
    const int32_t st = check_pool(c, true);
    if (st) return st;
    if (a->new_batch < 0) return FA_ERR_SHAPE;
    if (c.pages > FA_MAX_POOL_PAGES) return FA_ERR_PAGES;
    if ((int64_t)a->new_batch * c.table_cols >= (1LL << 31) || a->new_batch >= 1 << 24 ||
        (int64_t)c.page_size * c.num_heads_kv * 32 >= (1LL << 30))
        return FA_ERR_TOO_LARGE;
    if (a->new_batch == 0) return FA_OK;
    if (!a->sources || !a->new_lengths || (c.table_cols > 0 && !a->new_table)) return FA_ERR_NULL_ARG;
    for (const void* x : {(const void*)a->sources, (const void*)a->more, (const void*)a->new_table, (const void*)a->new_lengths})
        if (!aligned(x, 4)) return FA_ERR_ALIGN;
    return a->new_lengths == c.key_lengths || (c.table_cols > 0 && a->new_table == c.page_table) ? FA_ERR_PAGES : FA_OK;
}

size_t fa_cache_fork_workspace_size(const fa_cache_fork_args* a) {
    if (fa_cache_fork_check(a) || a->new_batch == 0) return 0;
    return up256((size_t)a->new_batch * sizeof(int4)) + up256((size_t)a->new_batch * sizeof(fa::ForkPlan)) +
           up256(((size_t)a->pool.pages + a->pool.batch) * 4);
}

int32_t fa_cache_fork(const fa_cache_fork_args* a, void* workspace, size_t bytes, void* stream) {
    const int32_t st = fa_cache_fork_check(a);
    if (st) return st;
    if (a->new_batch == 0) return FA_OK;
    const size_t need = fa_cache_fork_workspace_size(a);
    if (!workspace || bytes < need || !aligned(workspace, 16)) return FA_ERR_WORKSPACE;
    fa::CacheForkParams p = {};
    put_pool(a->pool, p);
    p.sources = a->sources;
    p.more = a->more;
    p.more_all = a->more_all;
    p.n_new = a->new_batch;
    p.new_table = a->new_table;
    p.new_lens = a->new_lengths;
    char* ws = (char*)workspace;
    p.copies = (int4*)ws;
    ws += up256((size_t)a->new_batch * sizeof(int4));
    p.plan = (fa::ForkPlan*)ws;
    ws += up256((size_t)a->new_batch * sizeof(fa::ForkPlan));
    p.free_list = (int*)ws;
    p.heirs = p.free_list + a->pool.pages;
    return fa::launch_cache_fork(p, (hipStream_t)stream) == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------
int32_t fa_cache_compact_check(const fa_cache_compact_args* a) {
    if (!a) return FA_ERR_NULL_ARG;
    const fa_page_pool& c = a->pool;
    const int32_t st = check_pool(c, true);
    if (st) return st;
    if (c.pages > FA_MAX_POOL_PAGES) return FA_ERR_PAGES;
    const int64_t chunks = (int64_t)c.page_size * c.num_heads_kv * 32;
    if ((int64_t)c.batch * c.table_cols >= (1LL << 31) || chunks >= (1LL << 30) || c.layers * (chunks / 512 + 2) >= (1LL << 31))
        return FA_ERR_TOO_LARGE;
    if (!a->used || (c.batch > 0 && c.table_cols > 0 && !a->new_table)) return FA_ERR_NULL_ARG;
    if (!aligned(a->used, 4) || !aligned(a->new_table, 4)) return FA_ERR_ALIGN;
    return c.table_cols > 0 && c.batch > 0 && a->new_table == c.page_table ? FA_ERR_PAGES : FA_OK;
}

size_t fa_cache_compact_workspace_size(const fa_cache_compact_args* a) {
    if (fa_cache_compact_check(a)) return 0;
    return up256((size_t)a->pool.pages * sizeof(int2)) + 256;
}

int32_t fa_cache_compact(const fa_cache_compact_args* a, void* workspace, size_t bytes, void* stream) {
    const int32_t st = fa_cache_compact_check(a);
    if (st) return st;
    const size_t need = fa_cache_compact_workspace_size(a);
    if (!workspace || bytes < need || !aligned(workspace, 16)) return FA_ERR_WORKSPACE;
    fa::CacheCompactParams p = {};
    put_pool(a->pool, p);
    p.new_table = a->new_table;
    p.used = a->used;
    char* ws = (char*)workspace;
    p.n_moves = (int*)ws;
    p.moves = (int2*)(ws + 256);
    return fa::launch_cache_compact(p, (hipStream_t)stream) == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

}  // extern "C"
