// Host side of the C ABI declared in include/fa_ops.h: argument validation (no
// HIP call before it passes), workspace layout and the choice of kernels.
// Stateless; launches on the caller's stream and never synchronises.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "fa_common.hpp"
#include "fa_ops.h"
#include "fa_ops_params.hpp"

namespace {

using fa::RotaryParams;
using fa::RowsParams;
using fa::ScoredParams;

constexpr double kLog2eD = 1.4426950408889634;
constexpr int64_t kMaxStride = (int64_t)1 << 40;  // elements; larger ones are refused before any arithmetic on them
constexpr int32_t kTileRows = 256;                // rows whose byte span a tile copy addresses with 32 bits
constexpr int32_t kMaxLen = 1 << 28;

int elem_size(int32_t dtype) { return dtype == FA_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
int compiled_dim(int32_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

// a (.., s, h, d)-strided tensor of rows of whole 16-byte chunks; n strides, the last that of d
int32_t check_tensor(const void* ptr, const int64_t* st, int n, int32_t S, int32_t D, int es) {
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

int32_t check_sizes(int32_t B, int32_t Sq, int32_t Sk, int32_t H, int32_t Hkv, int32_t D, int32_t dtype, float scale,
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

int32_t check_slopes(const float* slopes, int64_t sb, int32_t H) {
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

// ---------------------------------------------------------------------------
// document ids in the workspace: padded ids, then the tiles' ranges
int32_t doc_pad(int32_t S) { return (S + 63) / 64 * 64; }
size_t doc_bytes(int32_t B, int32_t S) {
    const size_t n = (size_t)B * doc_pad(S);
    return up256(n * 4) + up256(n / 64 * sizeof(int2));
}
// (an empty side's array may be null: with no token there the documents rule nothing)
bool has_docs(const fa_scored_args* a) { return a->q_documents && a->k_documents; }
bool one_doc_array(const fa_scored_args* a) {
    return a->q_documents == a->k_documents && a->seqlen_q == a->seqlen_k &&
           a->q_documents_stride == a->k_documents_stride;
}
size_t docs_bytes(const fa_scored_args* a) {
    if (!has_docs(a)) return 0;
    return doc_bytes(a->batch, a->seqlen_k) + (one_doc_array(a) ? 0 : doc_bytes(a->batch, a->seqlen_q));
}
hipError_t make_docs(const int32_t* ids, int64_t sb, int32_t B, int32_t S, char*& ws, const int*& out, const int2*& rng,
                     int& pad, hipStream_t s) {
    fa::DocParams d;
    d.ids = ids;
    d.sb = sb;
    d.S = S;
    d.pad = pad = doc_pad(S);
    d.n_tiles = (int)((int64_t)B * d.pad / 64);
    const size_t n = (size_t)B * d.pad;
    d.out = (int*)ws;
    d.rng = (int2*)(ws + up256(n * 4));
    ws += doc_bytes(B, S);
    out = d.out;
    rng = d.rng;
    return fa::launch_doc_tiles(d, s);
}
hipError_t put_docs(const fa_scored_args* a, ScoredParams& p, char*& ws, hipStream_t s) {
    p.q_docs = p.k_docs = nullptr;
    p.q_rng = p.k_rng = nullptr;
    p.q_docs_pad = p.k_docs_pad = 0;
    if (!has_docs(a)) return hipSuccess;
    hipError_t e = make_docs(a->k_documents, a->k_documents_stride, a->batch, a->seqlen_k, ws, p.k_docs, p.k_rng,
                             p.k_docs_pad, s);
    if (e != hipSuccess) return e;
    if (one_doc_array(a)) {
        p.q_docs = p.k_docs;
        p.q_rng = p.k_rng;
        p.q_docs_pad = p.k_docs_pad;
        return hipSuccess;
    }
    return make_docs(a->q_documents, a->q_documents_stride, a->batch, a->seqlen_q, ws, p.q_docs, p.q_rng, p.q_docs_pad, s);
}

void put_scored(const fa_scored_args* a, ScoredParams& p) {
    p = ScoredParams{};
    p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o; p.lse = a->lse; p.lse_near = a->lse_near;
    p.dout = a->dout; p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
    auto put = [](const int64_t st[4], int64_t& sb, int64_t& ss, int64_t& sh) {
        sb = st[0];
        ss = st[1];
        sh = st[2];
    };
    put(a->q_stride, p.q_sb, p.q_ss, p.q_sh);
    put(a->k_stride, p.k_sb, p.k_ss, p.k_sh);
    put(a->v_stride, p.v_sb, p.v_ss, p.v_sh);
    put(a->o_stride, p.o_sb, p.o_ss, p.o_sh);
    put(a->do_stride, p.do_sb, p.do_ss, p.do_sh);
    put(a->dq_stride, p.dq_sb, p.dq_ss, p.dq_sh);
    put(a->dk_stride, p.dk_sb, p.dk_ss, p.dk_sh);
    put(a->dv_stride, p.dv_sb, p.dv_ss, p.dv_sh);
    p.B = a->batch;
    p.Sq = a->seqlen_q;
    p.Sk = a->seqlen_k;
    p.H = a->num_heads;
    p.Hkv = a->num_heads_kv;
    p.group = a->num_heads / a->num_heads_kv;
    p.cols = a->head_dim;
    p.causal = a->causal != 0;
    p.scale = a->scale;
    put_cap(p, a->scale, a->softcap);
    p.slopes = a->slopes;
    p.slopes_sb = a->slopes_batch_stride;
    p.prefix = a->prefix_lengths;
    p.lens = a->key_lengths;
    p.offsets = a->query_offsets;
    p.offset0 = a->query_offset;
}

// ---------------------------------------------------------------------------
// few rows: splits of the keys.  Units are 32-row tiles of one KV head (over the
// prefix) or of one (sequence, KV head).
template <typename T>
T ceil_div(T a, T b) { return (a + b - 1) / b; }

void plan_rows(RowsParams& p, int32_t dtype) {
    const int D = compiled_dim(p.cols);
    const int64_t slots = dtype == FA_DTYPE_F32 && D == 128 ? 256 : 512;  // workgroups that run at once
    const int64_t rows = (int64_t)p.Sq * p.group;
    p.p_unit = rows * p.B > 64 ? 128 : 32;
    p.o_rt = (int)ceil_div<int64_t>(rows, 32);
    const int64_t ou = (int64_t)p.B * p.Hkv * p.o_rt;
    // A short prefix before short sequences: one walk over both costs less than a
    // second launch to join two.  (sequences, KV heads, prefix + own keys), one walk
    // against two in us: (4, 8, 300 + 40) 7.7 / 11.2; (32, 8, 500 + 100) 12.8 / 17.2;
    // (64, 8, 400 + 100) 17.6 / 22.0; (4, 8, 900 + 100) 16.2 / 15.3; (16, 8, 1900 +
    // 100) 24.4 / 16.2
    p.joined = p.P > 0 && ou <= 512 && (int64_t)p.P + p.Sk <= 640;
    p.p_rt = p.P > 0 && !p.joined ? (int)ceil_div<int64_t>(rows * p.B, p.p_unit) : 0;
    const int64_t pu = (int64_t)p.Hkv * p.p_rt;
    const int64_t ont = ceil_div<int64_t>(p.Sk, 64), pnt = ceil_div<int64_t>(p.P, 64);
    // As many splits as fill the device once, but none below 4 steps of a workgroup
    // (a step is 128 keys in a unit of 32 rows, 64 keys in one of 128), whose part
    // would cost more to write and join than its keys: one token of 8 heads
    // over 512 keys takes 13.1 us in one split a unit and 15.6 us in two.
    const int64_t chunk = ceil_div<int64_t>(ou * ont + pu * pnt, slots);
    auto splits = [&](int64_t nt, int64_t least) {
        return (int)std::max<int64_t>(1, std::min<int64_t>(64, ceil_div(nt, std::max<int64_t>(chunk, least))));
    };
    // A cache alone is joined for its own parts only: one part under 16 tiles, and where
    // the device is full, whole parts that fit it once (sequences, queries, keys, query
    // heads on KV heads of a size; us with the parts of the rule above / with these):
    // (1, 1, 600, 8 of 64) 11.0 / 9.5; (2, 128, 600, 32 on 4 of 128) 21.1 / 12.9, 1600
    // keys 26.6 / 20.9; (1, 400, 1600, 32 on 4 of 128) 41.8 / 26.7; (16, 1, 1600, 32 on 8
    // of 128) 25.8 / 26.4
    if (p.P == 0)
        p.o_splits = ont < 16 ? 1 : chunk > 8 ? (int)std::max<int64_t>(1, std::min<int64_t>(64, ont / chunk)) : splits(ont, 8);
    else
        p.o_splits = p.joined ? 1 : splits(ont, 8);
    p.p_splits = pu ? splits(pnt, p.p_unit == 128 ? 4 : 8) : 0;
    p.p_wgs = pu * p.p_splits;
    p.o_wgs = ou * p.o_splits;
    p.p_rows = p.p_wgs * p.p_unit;
}
bool rows_need_parts(const RowsParams& p) { return p.p_splits + p.o_splits > 1; }
size_t part_rows(const RowsParams& p) { return (size_t)(p.p_rows + p.o_wgs * 32); }
size_t rows_bytes(const RowsParams& p) {
    if (!rows_need_parts(p)) return 0;
    const size_t n = part_rows(p);
    return up256(n * sizeof(float2)) + up256(n * compiled_dim(p.cols) * sizeof(float));
}
void put_parts(RowsParams& p, void* ws) {
    p.stat = nullptr;
    p.part = nullptr;
    if (!rows_need_parts(p)) return;
    p.stat = (float2*)ws;
    p.part = (float*)((char*)ws + up256(part_rows(p) * sizeof(float2)));
}
hipError_t run_rows(const RowsParams& p, int32_t dtype, hipStream_t s) {
    const int D = compiled_dim(p.cols);
    if (dtype == FA_DTYPE_F32) return fa::launch_rows<float>(p, D, s);
    return dtype == FA_DTYPE_BF16 ? fa::launch_rows<fa::bf16>(p, D, s) : fa::launch_rows<fa::f16>(p, D, s);
}

// Whether a forward runs on the few-row kernel, which splits the keys over
// workgroups but reads them again for each 32 rows: few queries, or a grid of the
// other one that is half of the device, over keys of at least four times their
// number.  us, the 128-query kernel against this one (sequences, queries, keys, query
// heads on KV heads of a size; bf16, causal at the end of the keys):
//   (16, 1, 8192, 32 on 8 of 128) 291 / 108; (1, 1, 600, 8 of 64) 13.7 / 9.5; (64, 16, 700,
//   16 of 64) 41 / 34; (64, 32, 1000, 32 on 8 of 128) 141 / 95; (128, 8, 64, 16 of 64)
//   18.9 / 19.2; (2, 128, 600, 32 on 4 of 128) 19.1 / 13.1; (1, 1024, 4096, 8 of 128) 67 /
//   40; (1, 400, 2500, 32 on 8 of 128) 48 / 37; (4, 128, 512, 32 on 8 of 128) 17.6 / 16.7
//   outside the rule: (16, 64, 8192, 32 on 8 of 128) 303 / 274; (64, 64, 700, 16 of 64)
//   42 / 43; (128, 128, 512, 16 of 128) 149 / 243; (64, 128, 128, 16 of 64) 21 / 41; (64,
//   16, 16, 16 of 64) 11.7 / 12.2
bool few_rows(const fa_scored_args* a, RowsParams& r) {
    if (has_docs(a) || a->prefix_lengths || a->seqlen_k == 0) return false;
    if (a->seqlen_k < 4 * (int64_t)a->seqlen_q) return false;
    const int64_t blocks = ceil_div<int64_t>(a->seqlen_q, 128) * a->num_heads * a->batch;
    if (a->seqlen_q > 32 && blocks > 128) return false;
    r = RowsParams{};
    r.q = a->q; r.k = a->k; r.v = a->v; r.o = a->o; r.lse = a->lse; r.lse_near = a->lse_near;
    r.q_sb = a->q_stride[0]; r.q_ss = a->q_stride[1]; r.q_sh = a->q_stride[2];
    r.k_sb = a->k_stride[0]; r.k_ss = a->k_stride[1]; r.k_sh = a->k_stride[2];
    r.v_sb = a->v_stride[0]; r.v_ss = a->v_stride[1]; r.v_sh = a->v_stride[2];
    r.o_sb = a->o_stride[0]; r.o_ss = a->o_stride[1]; r.o_sh = a->o_stride[2];
    r.B = a->batch; r.Sq = a->seqlen_q; r.P = 0; r.Sk = a->seqlen_k;
    r.H = a->num_heads; r.Hkv = a->num_heads_kv; r.group = a->num_heads / a->num_heads_kv;
    r.cols = a->head_dim;
    put_cap(r, a->scale, a->softcap);
    r.slopes = a->slopes; r.slopes_sb = a->slopes_batch_stride;
    r.lens = a->key_lengths;
    r.offsets = a->query_offsets; r.offset0 = a->query_offset; r.tail = 0;
    r.causal = a->causal != 0; r.masked_neg = 0;
    plan_rows(r, a->dtype);
    return r.o_wgs < (1LL << 31);
}

// Parts of the dK / dV pass.  A workgroup (128 keys of a KV head) walks the
// queries of every head of the group, and under a causal mask the first keys'
// walk all of them, so a grid of few workgroups runs for its longest: it is cut
// into parts of every n-th query tile, whose float32 sums meet in a pass after
// it.  Worth it while the grid is short of the device (with no causal mask, of
// half of it) and each part is long; backward in 1, 2, 4 and 8 parts of
//   1 x 2048, 8 on 2 heads of 128, cap: 521, 304, 195, 143 us
//   1 x 1024, 8 heads of 128, cap: 105, 89, 78, 80
//   2 x 1777, 12 heads of 64, cap: 123, 113, 130, 159; 3 documents 61, 72, 85, 113
//   4 x 700, 12 heads of 128 in float32, cap: 394, 398, 443, 526
//   2 x 4096, 32 on 8 heads of 128, cap: 1419, 1143, 1187, 1292
//   2 x 8192, 16 heads of 128, cap: 2168, 2343, 2574, 3143
//   2 x 2048, 16 heads of 64, cap, not causal: 185, 207
// and over documents of lengths up to
//   558: 2 x 1464, 12 on 6 heads of 128, cap: 178, 147, 136
//   1354: 3 x 3718, 4 heads of 80: 196, 182, 198
//   1286: 1 x 4096, 8 heads of 128: 169, 170, 185
//   2911: 2 x 8192, 4 on 2 heads of 128: 596, 386, 340, 458
//   488: 4 x 1000, 16 heads of 64: 64, 84, 108, 165
int kv_parts(const fa_scored_args* a) {
    const int64_t n = ceil_div<int64_t>(a->seqlen_k, 128) * a->num_heads_kv * a->batch;
    // queries of a walk (with documents, those of its own: half of all are taken)
    const int64_t walk = (int64_t)(a->num_heads / a->num_heads_kv) * a->seqlen_q / (has_docs(a) ? 2 : 1);
    int parts = 1;
    const int64_t most = a->causal ? 512 : 256;
    while (parts < 8 && n * parts <= most && walk >= (n * parts <= 128 ? 512 * parts : 1024 * parts + 1)) parts *= 2;
    return parts;
}
size_t part_bytes(const fa_scored_args* a) {
    const int n = kv_parts(a);
    if (n == 1) return 0;
    return up256((size_t)n * a->batch * a->num_heads_kv * 2 * a->seqlen_k * compiled_dim(a->head_dim) * sizeof(float));
}
size_t bwd_rows_bytes(const fa_scored_args* a, int32_t& sq_pad) {
    sq_pad = (a->seqlen_q + 127) / 128 * 128;
    return up256((size_t)a->batch * a->num_heads * 2 * sq_pad * sizeof(float));
}

}  // namespace

extern "C" {

int32_t fa_ops_version(void) { return FA_OPS_VERSION; }

int32_t fa_scored_check(const fa_scored_args* a, int32_t backward) {
    if (!a) return FA_ERR_NULL_ARG;
    int32_t st = check_sizes(a->batch, a->seqlen_q, a->seqlen_k, a->num_heads, a->num_heads_kv, a->head_dim, a->dtype,
                             a->scale, a->softcap);
    if (st) return st;
    if ((st = check_slopes(a->slopes, a->slopes_batch_stride, a->num_heads))) return st;
    const bool any = a->batch > 0 && a->seqlen_q > 0 && a->seqlen_k > 0;
    if (any && !a->q_documents != !a->k_documents) return FA_ERR_RULE;
    for (const int32_t* x : {a->prefix_lengths, a->key_lengths, a->query_offsets, a->q_documents, a->k_documents})
        if (!aligned(x, 4)) return FA_ERR_ALIGN;
    if (has_docs(a)) {
        for (int64_t x : {a->q_documents_stride, a->k_documents_stride})
            if (x < 0 || x > kMaxStride) return FA_ERR_RULE;
        if ((int64_t)a->batch * (doc_pad(std::max(a->seqlen_q, a->seqlen_k)) / 64) >= (1LL << 31)) return FA_ERR_TOO_LARGE;
    }
    const int es = elem_size(a->dtype);
    const int32_t B = a->batch, Sq = a->seqlen_q, Sk = a->seqlen_k, D = a->head_dim;
    const bool q = B > 0 && Sq > 0, k = B > 0 && Sk > 0;
    if (q) {
        if ((st = check_tensor(a->q, a->q_stride, 4, Sq, D, es)) || (st = check_tensor(a->o, a->o_stride, 4, Sq, D, es)))
            return st;
        if (backward && !a->lse) return FA_ERR_NULL_ARG;
        if (!aligned(a->lse, 4) || !aligned(a->lse_near, 4)) return FA_ERR_ALIGN;
    }
    if (k && ((st = check_tensor(a->k, a->k_stride, 4, Sk, D, es)) || (st = check_tensor(a->v, a->v_stride, 4, Sk, D, es))))
        return st;
    if (!backward) return FA_OK;
    if (q && ((st = check_tensor(a->dout, a->do_stride, 4, Sq, D, es)) ||
              (st = check_tensor(a->dq, a->dq_stride, 4, Sq, D, es))))
        return st;
    if (k && ((st = check_tensor(a->dk, a->dk_stride, 4, Sk, D, es)) ||
              (st = check_tensor(a->dv, a->dv_stride, 4, Sk, D, es))))
        return st;
    if (a->dslopes && !a->slopes) return FA_ERR_RULE;
    return aligned(a->dslopes, 4) ? FA_OK : FA_ERR_ALIGN;
}

size_t fa_scored_fwd_workspace_size(const fa_scored_args* a) {
    if (fa_scored_check(a, 0)) return 0;
    RowsParams r;
    if (few_rows(a, r)) return rows_bytes(r);
    return docs_bytes(a);
}

int32_t fa_scored_fwd(const fa_scored_args* a, void* workspace, size_t bytes, void* stream) {
    const int32_t st = fa_scored_check(a, 0);
    if (st) return st;
    if (a->batch == 0 || a->seqlen_q == 0) return FA_OK;
    const size_t need = fa_scored_fwd_workspace_size(a);
    if (need && (!workspace || bytes < need || !aligned(workspace, 16))) return FA_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    RowsParams r;
    if (few_rows(a, r)) {
        put_parts(r, workspace);
        return run_rows(r, a->dtype, s) == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
    }
    ScoredParams p;
    put_scored(a, p);
    char* ws = (char*)workspace;
    if (put_docs(a, p, ws, s) != hipSuccess) return FA_ERR_LAUNCH;
    const int D = compiled_dim(a->head_dim);
    const hipError_t e = a->dtype == FA_DTYPE_F32    ? fa::launch_scored_fwd<float>(p, D, s)
                         : a->dtype == FA_DTYPE_BF16 ? fa::launch_scored_fwd<fa::bf16>(p, D, s)
                                                     : fa::launch_scored_fwd<fa::f16>(p, D, s);
    return e == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

size_t fa_scored_bwd_workspace_size(const fa_scored_args* a) {
    if (fa_scored_check(a, 1)) return 0;
    int32_t pad;
    size_t n = bwd_rows_bytes(a, pad) + docs_bytes(a) + part_bytes(a);
    if (a->dslopes) n += up256((size_t)a->batch * a->num_heads * a->seqlen_q * sizeof(float));
    return n;
}

int32_t fa_scored_bwd(const fa_scored_args* a, void* workspace, size_t bytes, void* stream) {
    const int32_t st = fa_scored_check(a, 1);
    if (st) return st;
    const size_t need = fa_scored_bwd_workspace_size(a);
    if (need && (!workspace || bytes < need || !aligned(workspace, 256))) return FA_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    ScoredParams p;
    put_scored(a, p);
    char* ws = (char*)workspace;
    const size_t rows = bwd_rows_bytes(a, p.sq_pad);
    p.ws_stride = 2 * p.sq_pad;
    p.lse2 = (float*)ws;
    ws += rows;
    if (a->dslopes) {
        p.dslope_rows = (float*)ws;
        ws += up256((size_t)a->batch * a->num_heads * a->seqlen_q * sizeof(float));
    }
    p.kv_parts = kv_parts(a);
    p.kv_part = (float*)ws;
    ws += part_bytes(a);
    if (put_docs(a, p, ws, s) != hipSuccess) return FA_ERR_LAUNCH;
    const int D = compiled_dim(a->head_dim);
    hipError_t e = a->dtype == FA_DTYPE_F32    ? fa::launch_scored_bwd<float>(p, D, s)
                   : a->dtype == FA_DTYPE_BF16 ? fa::launch_scored_bwd<fa::bf16>(p, D, s)
                                               : fa::launch_scored_bwd<fa::f16>(p, D, s);
    if (e == hipSuccess && a->dslopes)
        e = fa::launch_slope_sum(p.dslope_rows, a->dslopes, a->batch, a->num_heads, a->seqlen_q,
                                 a->slopes_batch_stride != 0, s);
    return e == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------
int32_t fa_prefix_check(const fa_prefix_args* a) {
    if (!a) return FA_ERR_NULL_ARG;
    if (a->prefix_len < 0) return FA_ERR_SHAPE;
    int32_t st = check_sizes(a->batch, a->seqlen_q, std::max(a->seqlen_k, a->prefix_len), a->num_heads, a->num_heads_kv,
                             a->head_dim, a->dtype, a->scale, a->softcap);
    if (st) return st;
    if (a->seqlen_k < 0) return FA_ERR_SHAPE;
    if ((st = check_slopes(a->slopes, a->slopes_batch_stride, a->num_heads))) return st;
    if (!aligned(a->key_lengths, 4) || !aligned(a->lse, 4)) return FA_ERR_ALIGN;
    if (a->batch == 0 || a->seqlen_q == 0) return FA_OK;
    const int es = elem_size(a->dtype);
    if ((st = check_tensor(a->q, a->q_stride, 4, a->seqlen_q, a->head_dim, es)) ||
        (st = check_tensor(a->o, a->o_stride, 4, a->seqlen_q, a->head_dim, es)))
        return st;
    if (a->prefix_len > 0 && ((st = check_tensor(a->k_prefix, a->kp_stride, 3, a->prefix_len, a->head_dim, es)) ||
                              (st = check_tensor(a->v_prefix, a->vp_stride, 3, a->prefix_len, a->head_dim, es))))
        return st;
    if (a->seqlen_k > 0 && ((st = check_tensor(a->k, a->k_stride, 4, a->seqlen_k, a->head_dim, es)) ||
                            (st = check_tensor(a->v, a->v_stride, 4, a->seqlen_k, a->head_dim, es))))
        return st;
    // rows of all sequences, and parts of them, in 32-bit tile counts
    const int64_t rows = (int64_t)a->batch * a->seqlen_q * a->num_heads;
    return rows < (1LL << 26) ? FA_OK : FA_ERR_TOO_LARGE;
}

static void put_prefix(const fa_prefix_args* a, RowsParams& r) {
    r = RowsParams{};
    r.q = a->q; r.kp = a->k_prefix; r.vp = a->v_prefix; r.k = a->k; r.v = a->v; r.o = a->o; r.lse = a->lse;
    r.q_sb = a->q_stride[0]; r.q_ss = a->q_stride[1]; r.q_sh = a->q_stride[2];
    r.kp_ss = a->kp_stride[0]; r.kp_sh = a->kp_stride[1];
    r.vp_ss = a->vp_stride[0]; r.vp_sh = a->vp_stride[1];
    r.k_sb = a->k_stride[0]; r.k_ss = a->k_stride[1]; r.k_sh = a->k_stride[2];
    r.v_sb = a->v_stride[0]; r.v_ss = a->v_stride[1]; r.v_sh = a->v_stride[2];
    r.o_sb = a->o_stride[0]; r.o_ss = a->o_stride[1]; r.o_sh = a->o_stride[2];
    r.B = a->batch; r.Sq = a->seqlen_q; r.P = a->prefix_len; r.Sk = a->seqlen_k;
    r.H = a->num_heads; r.Hkv = a->num_heads_kv; r.group = a->num_heads / a->num_heads_kv;
    r.cols = a->head_dim;
    put_cap(r, a->scale, a->softcap);
    r.slopes = a->slopes; r.slopes_sb = a->slopes_batch_stride;
    r.lens = a->key_lengths;
    r.offsets = nullptr; r.offset0 = 0; r.tail = 1;
    r.causal = 1; r.masked_neg = 1;
    plan_rows(r, a->dtype);
}

size_t fa_prefix_workspace_size(const fa_prefix_args* a) {
    if (fa_prefix_check(a) || a->batch == 0 || a->seqlen_q == 0) return 0;
    RowsParams r;
    put_prefix(a, r);
    return rows_bytes(r);
}

int32_t fa_prefix_fwd(const fa_prefix_args* a, void* workspace, size_t bytes, void* stream) {
    const int32_t st = fa_prefix_check(a);
    if (st) return st;
    if (a->batch == 0 || a->seqlen_q == 0) return FA_OK;
    RowsParams r;
    put_prefix(a, r);
    if (r.p_wgs + r.o_wgs >= (1LL << 31)) return FA_ERR_TOO_LARGE;
    const size_t need = rows_bytes(r);
    if (need && (!workspace || bytes < need || !aligned(workspace, 16))) return FA_ERR_WORKSPACE;
    put_parts(r, workspace);
    return run_rows(r, a->dtype, (hipStream_t)stream) == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------
int32_t fa_rotary_table(float* table, int64_t positions, int32_t rotary_dim, int32_t scaling, double base, double factor,
                        double original, double low, double high, double mul, void* stream) {
    if (positions < 0 || positions > ((int64_t)1 << 31)) return FA_ERR_SHAPE;
    if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > 256) return FA_ERR_ROTARY;
    if (scaling < FA_ROTARY_NONE || scaling > FA_ROTARY_RAMP) return FA_ERR_ROTARY;
    if (!std::isfinite(base) || !(base > 0.0) || !std::isfinite(factor) || !(factor > 0.0) || !std::isfinite(mul))
        return FA_ERR_ROTARY;
    if (scaling == FA_ROTARY_RAMP &&
        (!std::isfinite(original) || !(original > 0.0) || !std::isfinite(low) || !std::isfinite(high) || !(high > low)))
        return FA_ERR_ROTARY;
    if (positions == 0) return FA_OK;
    if (!table) return FA_ERR_NULL_ARG;
    if (!aligned(table, 4)) return FA_ERR_ALIGN;
    fa::RotaryTableParams p{table, positions, rotary_dim, scaling, base, factor, original, low, high, mul};
    return fa::launch_rotary_table(p, (hipStream_t)stream) == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

int32_t fa_rotary_check(const fa_rotary_args* a) {
    if (!a) return FA_ERR_NULL_ARG;
    if (a->batch < 0 || a->seqlen < 0 || a->num_heads < 0 || a->num_heads_k < 0 || a->table_positions < 0) return FA_ERR_SHAPE;
    if (a->dtype != FA_DTYPE_F16 && a->dtype != FA_DTYPE_BF16 && a->dtype != FA_DTYPE_F32) return FA_ERR_DTYPE;
    if (a->head_dim <= 0 || a->head_dim > 256) return FA_ERR_HEAD_DIM;
    if (a->rotary_dim < 2 || a->rotary_dim % 2 != 0 || a->rotary_dim > a->head_dim) return FA_ERR_ROTARY;
    if ((int64_t)a->num_heads + a->num_heads_k == 0) return FA_ERR_HEADS;
    if ((int64_t)a->num_heads + a->num_heads_k > (1 << 20)) return FA_ERR_TOO_LARGE;
    if ((int64_t)a->batch * a->seqlen >= (1LL << 31)) return FA_ERR_TOO_LARGE;
    if (a->batch == 0 || a->seqlen == 0) return FA_OK;
    if (!a->table || a->table_positions == 0) return FA_ERR_ROTARY;
    const unsigned es = (unsigned)elem_size(a->dtype);
    auto tensor = [&](const void* in, const void* out, const int64_t* si, const int64_t* so) -> int32_t {
        if (!in || !out) return FA_ERR_NULL_ARG;
        if (!aligned(in, es) || !aligned(out, es)) return FA_ERR_ALIGN;
        for (int i = 0; i < 3; ++i) {
            if (si[i] < 0 || so[i] < 0) return FA_ERR_STRIDE;
            if (si[i] > kMaxStride || so[i] > kMaxStride) return FA_ERR_TOO_LARGE;
            if (in == out && si[i] != so[i]) return FA_ERR_STRIDE;  // an element would be written before it is read
        }
        return si[3] == 1 && so[3] == 1 ? FA_OK : FA_ERR_STRIDE;
    };
    int32_t st;
    if (a->num_heads && (st = tensor(a->q, a->q_out, a->q_stride, a->q_out_stride))) return st;
    if (a->num_heads_k && (st = tensor(a->k, a->k_out, a->k_stride, a->k_out_stride))) return st;
    if (!aligned(a->table, 4) || !aligned(a->positions, a->positions_64 ? 8 : 4)) return FA_ERR_ALIGN;
    for (int i = 0; i < 2; ++i)
        if (a->positions && (a->positions_stride[i] < 0 || a->positions_stride[i] > kMaxStride)) return FA_ERR_STRIDE;
    return FA_OK;
}

int32_t fa_rotary(const fa_rotary_args* a, void* stream) {
    const int32_t st = fa_rotary_check(a);
    if (st) return st;
    if (a->batch == 0 || a->seqlen == 0) return FA_OK;
    RotaryParams p = {};
    const int64_t* si[2] = {a->q_stride, a->k_stride};
    const int64_t* so[2] = {a->q_out_stride, a->k_out_stride};
    const void* in[2] = {a->q, a->k};
    void* out[2] = {a->q_out, a->k_out};
    const int heads[2] = {a->num_heads, a->num_heads_k};
    const int es = elem_size(a->dtype);
    // elements an access may hold: what divides the widths, strides and addresses
    int64_t bits = 16 / es;
    bits |= a->interleaved ? a->rotary_dim : a->rotary_dim / 2;
    bool copy = false;
    for (int i = 0; i < 2; ++i) {
        p.x[i] = fa::RotaryTensor{in[i], out[i], si[i][0], si[i][1], si[i][2], so[i][0], so[i][1], so[i][2], heads[i]};
        if (!heads[i]) continue;
        copy |= in[i] != out[i];
        for (int d = 0; d < 3; ++d) bits |= si[i][d] | so[i][d];
        bits |= (int64_t)((uintptr_t)in[i] / es) | (int64_t)((uintptr_t)out[i] / es);
    }
    if (copy) bits |= a->head_dim - a->rotary_dim;
    // the table's rows of float32: half of them for cosines, half for sines
    const int64_t tb = (a->rotary_dim / 2) | (int64_t)((uintptr_t)a->table / 4) | 4;
    p.vec = (int)(bits & -bits);
    const int tv = (int)(tb & -tb);  // floats a table access may hold
    const int pairs = a->interleaved ? p.vec / 2 : p.vec;
    if (std::min(pairs, 4) > tv) p.vec = a->interleaved ? 2 * tv : tv;
    p.table = a->table;
    p.pos = a->positions;
    p.pos_sb = a->positions_stride[0];
    p.pos_ss = a->positions_stride[1];
    p.pos64 = a->positions_64 != 0;
    p.n_pos = a->table_positions;
    p.B = a->batch;
    p.S = a->seqlen;
    p.D = a->head_dim;
    p.R = a->rotary_dim;
    p.interleaved = a->interleaved != 0;
    p.copy = copy && a->head_dim > a->rotary_dim;
    p.sign = a->inverse ? -1.f : 1.f;
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a->dtype == FA_DTYPE_F32    ? fa::launch_rotary<float>(p, s)
                         : a->dtype == FA_DTYPE_BF16 ? fa::launch_rotary<fa::bf16>(p, s)
                                                     : fa::launch_rotary<fa::f16>(p, s);
    return e == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

}  // extern "C"
