// Drives the C ABI of the operators around attention (csrc/fa_ops_abi.cpp), built
// with host AddressSanitizer and UndefinedBehaviorSanitizer, over random and
// extreme sizes, strides and options.  The stub launchers below check that what a
// kernel would be given stays inside the workspace that was asked for, and that
// units and parts cover every row.  Addresses are never read.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "fa_ops.h"
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

static uintptr_t g_ws = 0, g_end = 0;  // the workspace of the call in progress
static bool inside(const void* p, double bytes) {
    return (uintptr_t)p >= g_ws && (double)((uintptr_t)p - g_ws) + bytes <= (double)(g_end - g_ws);
}
static int dim(int cols) { return cols <= 32 ? 32 : cols <= 64 ? 64 : 128; }

namespace fa {
hipError_t launch_doc_tiles(const DocParams& p, hipStream_t) {
    ++g_launches;
    CHECK(p.pad % 64 == 0 && p.pad >= p.S && p.n_tiles >= 0);
    CHECK(inside(p.out, 64.0 * p.n_tiles * 4) && inside(p.rng, 8.0 * p.n_tiles));
    CHECK((const char*)p.rng >= (const char*)p.out + 256LL * p.n_tiles);
    return hipSuccess;
}
hipError_t launch_slope_sum(const float* rows, float* dst, int B, int H, int Sq, bool, hipStream_t) {
    ++g_launches;
    CHECK(dst && inside(rows, 4.0 * B * H * Sq));
    return hipSuccess;
}
static void docs(const ScoredParams& p) {
    if (!p.q_docs) return;
    CHECK(p.q_docs_pad >= p.Sq && p.k_docs_pad >= p.Sk);
    CHECK(inside(p.q_docs, 4.0 * p.B * p.q_docs_pad) && inside(p.k_docs, 4.0 * p.B * p.k_docs_pad));
    CHECK(inside(p.q_rng, 8.0 * p.B * (p.q_docs_pad / 64)) && inside(p.k_rng, 8.0 * p.B * (p.k_docs_pad / 64)));
}
template <typename T>
hipError_t launch_scored_fwd(const ScoredParams& p, int D, hipStream_t) {
    ++g_launches;
    CHECK(D == dim(p.cols) && p.H == p.Hkv * p.group);
    docs(p);
    return hipSuccess;
}
template <typename T>
hipError_t launch_scored_bwd(const ScoredParams& p, int D, hipStream_t) {
    ++g_launches;
    CHECK(D == dim(p.cols) && p.sq_pad % 128 == 0 && p.sq_pad >= p.Sq && p.ws_stride == 2 * p.sq_pad);
    const double rows = 4.0 * p.B * p.H * p.ws_stride;
    CHECK(inside(p.lse2, rows));
    if (p.dslope_rows) CHECK(inside(p.dslope_rows, 4.0 * p.B * p.H * p.Sq) && (double)((char*)p.dslope_rows - (char*)p.lse2) >= rows);
    CHECK(p.kv_parts == 1 || p.kv_parts == 2 || p.kv_parts == 4 || p.kv_parts == 8);
    if (p.kv_parts > 1) CHECK(inside(p.kv_part, 4.0 * p.kv_parts * p.B * p.Hkv * 2 * p.Sk * D));
    CHECK((double)p.kv_parts * ((p.Sk + 127) / 128) * p.Hkv * p.B < 2147483648.0);
    docs(p);
    return hipSuccess;
}
template <typename T>
hipError_t launch_rows(const RowsParams& p, int D, hipStream_t) {
    ++g_launches;
    const int64_t rows = (int64_t)p.Sq * p.group;
    CHECK(D == dim(p.cols) && p.H == p.Hkv * p.group);
    CHECK(p.o_rt * 32LL >= rows && p.o_splits >= 1 && p.o_splits <= 64);
    CHECK(p.o_wgs == (int64_t)p.B * p.Hkv * p.o_rt * p.o_splits && p.p_wgs + p.o_wgs < (1LL << 31));
    const bool prefix = p.P > 0 && !p.joined;
    CHECK(prefix ? p.p_splits >= 1 && p.p_splits <= 64 : p.p_splits == 0 && p.p_wgs == 0);
    if (prefix) {
        CHECK((p.p_unit == 32 || p.p_unit == 128) && (int64_t)p.p_rt * p.p_unit >= rows * p.B);
        CHECK(p.p_wgs == (int64_t)p.Hkv * p.p_rt * p.p_splits);
    }
    CHECK(p.p_rows == p.p_wgs * p.p_unit || !prefix);
    if (p.joined) CHECK(p.o_splits == 1 && p.P > 0);
    const double n = (double)p.p_rows + 32.0 * p.o_wgs;
    if (p.p_splits + p.o_splits > 1)
        CHECK(inside(p.stat, 8.0 * n) && inside(p.part, 4.0 * n * D) && (char*)p.part >= (char*)p.stat + (int64_t)(8.0 * n));
    return hipSuccess;
}
hipError_t launch_rotary_table(const RotaryTableParams& p, hipStream_t) {
    ++g_launches;
    CHECK(p.n >= 0 && p.R % 2 == 0 && p.table);
    return hipSuccess;
}
template <typename T>
hipError_t launch_rotary(const RotaryParams& p, hipStream_t) {
    ++g_launches;
    CHECK(p.R <= p.D && p.vec >= 1);
    return hipSuccess;
}
#define INST(T)                                                                  \
    template hipError_t launch_scored_fwd<T>(const ScoredParams&, int, hipStream_t); \
    template hipError_t launch_scored_bwd<T>(const ScoredParams&, int, hipStream_t); \
    template hipError_t launch_rows<T>(const RowsParams&, int, hipStream_t);     \
    template hipError_t launch_rotary<T>(const RotaryParams&, hipStream_t);
INST(float)
INST(bf16)
INST(f16)
}  // namespace fa

static std::mt19937_64 rng(7);
static int64_t pick(std::initializer_list<int64_t> v) { return v.begin()[rng() % v.size()]; }
static int32_t size() {
    return (int32_t)pick({0, 1, 2, 31, 32, 33, 100, 128, 129, 1000, 4096, 65537, 1 << 20, (1 << 28) - 1, 1 << 28, INT32_MAX, -1});
}
static int32_t small() { return (int32_t)pick({1, 1, 2, 3, 8, 40, 128}); }
static int32_t heads() { return (int32_t)pick({1, 2, 4, 8, 32, 0, 3}); }
static int64_t stride() {
    return pick({8, 64, 128, 4096, 1 << 20, 1LL << 33, 1LL << 40, INT64_MAX, 0, -8, 7, 16, 1024});
}
static void* addr() { return (void*)(uintptr_t)pick({1 << 20, 1 << 20, 1 << 20, 1 << 20, 0, (1 << 20) + 8, (1 << 20) + 2}); }
static void* good() { return (void*)(uintptr_t)(1 << 20); }
static void* opt() { return (rng() & 1) ? good() : nullptr; }

template <size_t N>
static void plain(int64_t (&st)[N], int S, int H, int D) {
    const int64_t row = (int64_t)H * D;
    if (N == 4) {
        st[0] = (int64_t)((uint64_t)S * (uint64_t)row);  // (extreme sizes wrap)
        st[N - 3] = row;
    } else {
        st[0] = row;
    }
    st[N - 2] = D;
    st[N - 1] = 1;
}

static void* use(size_t need) {  // a workspace of just that size, somewhere
    g_ws = (uintptr_t)1 << 40;
    g_end = g_ws + need;
    return (void*)g_ws;
}

static void scored(bool wild) {
    fa_scored_args a;
    std::memset(&a, 0, sizeof(a));
    a.batch = wild ? size() : small();
    a.seqlen_q = wild ? size() : (int32_t)pick({0, 1, 2, 16, 33, 100, 700, 4096, 9000});
    a.seqlen_k = wild ? size() : (int32_t)pick({0, 1, 65, 700, 4096, 70000, a.seqlen_q});
    a.num_heads_kv = wild ? heads() : (int32_t)pick({1, 2, 8});
    a.num_heads = wild ? heads() : a.num_heads_kv * (int32_t)pick({1, 2, 5});
    a.dtype = (int32_t)(rng() % (wild ? 4 : 3));
    a.head_dim = (int32_t)(wild ? pick({8, 64, 80, 128, 136, 0, 60}) : pick({8, 32, 64, 80, 128}));
    a.causal = (int)(rng() & 1);
    a.scale = wild ? (float)pick({0, 1, -1}) : 0.1f;
    a.softcap = (rng() & 1) ? 30.f : 0.f;
    const void** in[] = {&a.q, &a.k, &a.v, &a.dout};
    for (auto p : in) *p = wild ? addr() : good();
    a.o = a.dq = a.dk = a.dv = wild ? addr() : good();
    a.lse = (float*)good();
    int64_t(*st[8])[4] = {&a.q_stride, &a.o_stride, &a.do_stride, &a.dq_stride, &a.k_stride, &a.v_stride, &a.dk_stride, &a.dv_stride};
    for (int i = 0; i < 8; ++i) {
        if (wild)
            for (int d = 0; d < 4; ++d) (*st[i])[d] = d == 3 ? 1 : stride();
        else
            plain(*st[i], i < 4 ? a.seqlen_q : a.seqlen_k, i < 4 ? a.num_heads : a.num_heads_kv, a.head_dim);
    }
    a.slopes = (const float*)opt();
    a.dslopes = a.slopes ? (float*)opt() : nullptr;
    a.slopes_batch_stride = (rng() & 1) ? a.num_heads : 0;
    a.key_lengths = (const int32_t*)opt();
    a.prefix_lengths = (const int32_t*)opt();
    a.query_offset = (int32_t)pick({0, INT32_MAX, INT32_MIN, 5});
    if (rng() & 1) {
        a.q_documents = (const int32_t*)good();
        a.k_documents = (rng() & 1) ? a.q_documents : (const int32_t*)(uintptr_t)(1 << 21);
        a.q_documents_stride = wild ? stride() : a.seqlen_q;
        a.k_documents_stride = wild ? stride() : a.seqlen_k;
    }
    const int32_t f = fa_scored_check(&a, 0), b = fa_scored_check(&a, 1);
    CHECK(wild || (f == FA_OK && b == FA_OK));
    const size_t nf = fa_scored_fwd_workspace_size(&a);
    CHECK(f == FA_OK || nf == 0);
    const int32_t rf = fa_scored_fwd(&a, use(nf), nf, nullptr);
    CHECK(rf == f);
    if (nf) CHECK(fa_scored_fwd(&a, use(nf), nf - 1, nullptr) == FA_ERR_WORKSPACE || a.batch == 0 || a.seqlen_q == 0);
    const size_t nb = fa_scored_bwd_workspace_size(&a);
    CHECK(fa_scored_bwd(&a, use(nb), nb, nullptr) == b);
    if (b == FA_OK && nb) CHECK(fa_scored_bwd(&a, use(nb), nb - 1, nullptr) == FA_ERR_WORKSPACE);
}

static void prefix(bool wild) {
    fa_prefix_args a;
    std::memset(&a, 0, sizeof(a));
    a.batch = wild ? size() : small();
    a.seqlen_q = wild ? size() : (int32_t)pick({0, 1, 3, 7, 100});
    a.seqlen_k = wild ? size() : (int32_t)pick({0, 1, 65, 700, 9000});
    a.prefix_len = wild ? size() : (int32_t)pick({0, 1, 300, 640, 8192, 1000000});
    a.num_heads_kv = wild ? heads() : (int32_t)pick({1, 2, 8});
    a.num_heads = wild ? heads() : a.num_heads_kv * (int32_t)pick({1, 2, 5});
    a.dtype = (int32_t)(rng() % (wild ? 4 : 3));
    a.head_dim = (int32_t)(wild ? pick({8, 64, 80, 128, 136, 0, 60}) : pick({8, 32, 64, 80, 128}));
    a.scale = 0.1f;
    const void** in[] = {&a.q, &a.k, &a.v, &a.k_prefix, &a.v_prefix};
    for (auto p : in) *p = wild ? addr() : good();
    a.o = wild ? addr() : good();
    a.lse = (float*)opt();
    plain(a.q_stride, a.seqlen_q, a.num_heads, a.head_dim);
    plain(a.o_stride, a.seqlen_q, a.num_heads, a.head_dim);
    plain(a.k_stride, a.seqlen_k, a.num_heads_kv, a.head_dim);
    plain(a.v_stride, a.seqlen_k, a.num_heads_kv, a.head_dim);
    plain(a.kp_stride, a.prefix_len, a.num_heads_kv, a.head_dim);
    plain(a.vp_stride, a.prefix_len, a.num_heads_kv, a.head_dim);
    if (wild)
        for (int d = 0; d < 3; ++d) a.k_stride[d] = stride();
    a.slopes = (const float*)opt();
    a.slopes_batch_stride = (rng() & 1) ? a.num_heads : 0;
    a.key_lengths = (const int32_t*)opt();
    const int32_t st = fa_prefix_check(&a);
    CHECK(wild || st == FA_OK);
    const size_t n = fa_prefix_workspace_size(&a);
    const int32_t r = fa_prefix_fwd(&a, use(n), n, nullptr);
    CHECK(r == st || r == FA_ERR_TOO_LARGE);
    if (st == FA_OK && r == FA_OK && n) CHECK(fa_prefix_fwd(&a, use(n), n - 1, nullptr) == FA_ERR_WORKSPACE);
}

static void rotary(bool wild) {
    fa_rotary_args a;
    std::memset(&a, 0, sizeof(a));
    a.q = a.k = wild ? addr() : good();
    a.q_out = a.k_out = wild ? addr() : good();
    a.batch = wild ? size() : small();
    a.seqlen = wild ? size() : (int32_t)pick({0, 1, 100, 70000});
    a.num_heads = wild ? size() : (int32_t)pick({1, 8, 33});
    a.num_heads_k = wild ? size() : (int32_t)pick({0, 1, 8});
    a.head_dim = (int32_t)(wild ? pick({0, 33, 256, 257, 64}) : pick({33, 64, 80, 256}));
    a.rotary_dim = (int32_t)(wild ? pick({0, 2, 3, 64, 300}) : pick({2, 20, 32}));
    a.dtype = (int32_t)(rng() % (wild ? 4 : 3));
    a.interleaved = (int)(rng() & 1);
    a.inverse = (int)(rng() & 1);
    int64_t(*st[4])[4] = {&a.q_stride, &a.q_out_stride, &a.k_stride, &a.k_out_stride};
    for (int i = 0; i < 4; ++i) {
        plain(*st[i], a.seqlen, i < 2 ? a.num_heads : a.num_heads_k, a.head_dim);
        if (wild) (*st[i])[rng() % 4] = stride();
    }
    a.table = (const float*)(wild ? addr() : good());
    a.table_positions = wild ? pick({0, 1, 1LL << 40, -1}) : 4096;
    a.positions = opt();
    a.positions_64 = (int)(rng() & 1);
    a.positions_stride[0] = wild ? stride() : a.seqlen;
    a.positions_stride[1] = 1;
    const int32_t c = fa_rotary_check(&a);
    CHECK(wild || c == FA_OK);
    CHECK(fa_rotary(&a, nullptr) == c);
}

int main() {
    for (int i = 0; i < 20000; ++i) {
        scored(i & 1);
        prefix(i & 1);
        rotary(i & 1);
    }
    std::printf("%ld launches, %ld checks, %ld failed\n", g_launches, g_cases, g_fails);
    std::printf(", %ld failed\n", g_fails);
    return g_fails ? 1 : g_launches > 10000 ? 0 : 2;
}
