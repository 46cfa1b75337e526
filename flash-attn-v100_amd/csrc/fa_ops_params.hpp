// Kernel parameter blocks and launchers of the operators around attention
// (include/fa_ops.h), shared by their host shim and the kernel translation units.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fa {

constexpr int kMaxOffset = 1 << 30;  // query offsets are held within +-this

// Attention with scored rules (fa_scored.hpp).  Strides in elements, d stride 1.
struct ScoredParams {
    const void* q;
    const void* k;
    const void* v;
    const void* o;  // written by the forward
    float* lse;
    float* lse_near;  // optional: the LSE over distances from the nearest key
    const void* dout;
    void* dq;
    void* dk;
    void* dv;
    int64_t q_sb, q_ss, q_sh;
    int64_t k_sb, k_ss, k_sh;
    int64_t v_sb, v_ss, v_sh;
    int64_t o_sb, o_ss, o_sh;
    int64_t do_sb, do_ss, do_sh;
    int64_t dq_sb, dq_ss, dq_sh;
    int64_t dk_sb, dk_ss, dk_sh;
    int64_t dv_sb, dv_ss, dv_sh;
    int B, Sq, Sk, H, Hkv, group;
    int cols;     // columns that exist, whole 16-byte chunks
    int n_tiles;  // blocks of 128 queries (keys) a slice
    int causal;
    float scale, scale_log2;         // softmax scale; times log2 e
    float cap, cap_k1, cap_k2, cap_top;  // 0: none; scale / cap; 2 log2 e of that; cap log2 e
    const float* slopes;             // optional (H) or (B, H)
    int64_t slopes_sb;               // its batch stride, 0 where shared
    const int* prefix;               // optional (B)
    const int* lens;                 // optional (B)
    const int* offsets;              // optional (B), else offset0
    int offset0;
    // document ids in tiles (doc_tiles_kernel), null where there are none
    const int* q_docs;   // (B, q_docs_pad)
    const int* k_docs;   // (B, k_docs_pad)
    const int2* q_rng;   // (B, q_docs_pad / 64)
    const int2* k_rng;
    int q_docs_pad, k_docs_pad;
    // backward workspace: per (batch, head) ws_stride = 2 sq_pad floats, LSE *
    // log2 e then rowsum(dO O); and optional (B, H, Sq) parts of the slopes' gradient
    float* lse2;
    int sq_pad, ws_stride;
    float* dslope_rows;
    // dK / dV in 1, 2, 4 or 8 parts by query tiles (1: no sums to join): float32
    // (part, B, Hkv, 2, Sk, D)
    int kv_parts;
    float* kv_part;
};

struct DocParams {
    const int* ids;      // (B, S), batch stride sb
    int64_t sb;
    int S, pad, n_tiles;  // pad: S rounded up to whole 64-token tiles; n_tiles = B pad / 64
    int* out;            // (B, pad)
    int2* rng;           // (B, pad / 64)
};
hipError_t launch_doc_tiles(const DocParams& p, hipStream_t s);
// sum of rows (B, H, Sq) to dst[b * dst_sb + h] (dst_sb 0: over the batches too)
hipError_t launch_slope_sum(const float* rows, float* dst, int B, int H, int Sq, bool per_batch, hipStream_t s);

template <typename T>
hipError_t launch_scored_fwd(const ScoredParams& p, int D, hipStream_t s);
template <typename T>
hipError_t launch_scored_bwd(const ScoredParams& p, int D, hipStream_t s);

// New tokens over caches and a prefix that their batch shares (fa_rows.hpp)
struct RowsParams {
    const void* q;   // (B, Sq, H, D)
    const void* kp;  // (P, Hkv, D), P may be 0
    const void* vp;
    const void* k;   // (B, Sk, Hkv, D)
    const void* v;
    void* o;
    float* lse;      // optional (B, H, Sq)
    float* lse_near; // optional, as ScoredParams::lse_near
    int64_t q_sb, q_ss, q_sh;
    int64_t kp_ss, kp_sh, vp_ss, vp_sh;
    int64_t k_sb, k_ss, k_sh;
    int64_t v_sb, v_ss, v_sh;
    int64_t o_sb, o_ss, o_sh;
    int B, Sq, P, Sk, H, Hkv, group;
    int cols;
    float scale_log2, cap, cap_k1, cap_k2, cap_top;
    const float* slopes;
    int64_t slopes_sb;
    const int* lens;     // optional (B): filled keys, the new tokens among them
    const int* offsets;  // optional (B): own position of query 0, else offset0
    int offset0;
    int tail;            // 1: own position of query 0 is len - Sq
    int causal;          // 0: every filled key is seen
    int masked_neg;      // queries at positions below 0 see nothing, the prefix neither
    // parts: the prefix keys go to p_splits workgroups for each unit of p_unit rows
    // (p_rt units a KV head), a sequence's own to o_splits (o_rt units of 32)
    int p_splits, p_rt, p_unit, o_splits, o_rt;
    // the units of a sequence's own keys walk the prefix too, and nothing is joined
    // (p_splits = 0)
    int joined;
    int64_t p_wgs, o_wgs;
    int64_t p_rows;      // part rows of the prefix, p_wgs p_unit
    float2* stat;        // per part row: maximum (log2 units), sum
    float* part;         // per part row: D floats
};
template <typename T>
hipError_t launch_rows(const RowsParams& p, int D, hipStream_t s);

// Tokens, or trees of drafted tokens, over a cache of pages (fa_paged.hpp): k and v a pool
// of pages; nothing of a prefix, offsets or their plans is read
struct PagedParams : RowsParams {
    const int* table;      // (B, table_cols) pages, null: sequence b is page b
    int64_t table_sb;
    int table_cols, pages;
    int page_blocks;       // blocks of 16 tokens in a page
    unsigned page_magic;   // 2^32 / page_blocks, rounded up
    int64_t k_sp, v_sp;    // page strides
    const int* parents;    // optional (B, Sq), batch stride parents_sb
    int64_t parents_sb;
    // work (PagedWork): units of rows of one (sequence, KV head), unit_tiles a KV head, over
    // steps of keys, shared out to at most `groups` workgroups a unit
    int unit_tiles, groups;
    int alone, least;      // steps of sequences that are not shared; those of a group, at least
    int many;              // a sequence may be in many parts
    int2* spans;           // (B) for the join: first and last group
    int extra;             // steps that a unit counts beside its keys'
    int wide;              // waves of a unit of 32 rows each that share its tiles; 1: of 32 rows, whose waves share its keys
};
template <typename T>
hipError_t launch_paged(const PagedParams& p, int D, hipStream_t s);

// A pool of pages, as its operators read it (fa_paged_cache.hip); strides in bytes
struct PoolParams {
    char* x[2];            // k, v
    int64_t sl[2], sp[2], sr[2], sh[2];  // layer, page, row, head
    int layers, pages, page_size, heads, chunks;  // chunks: 16-byte chunks of a head's row
    int B, cols;
    const int* table;
    int64_t table_sb;
    const int* lens;
    int room;              // tokens a sequence has room for
};
struct CacheWriteParams : PoolParams {
    const char* in[2];     // (layers, B, N, heads, D)
    int64_t in_sl[2], in_sb[2], in_ss[2], in_sh[2];
    int N;
};
hipError_t launch_cache_write(const CacheWriteParams& p, hipStream_t s);
struct CacheAcceptParams : PoolParams {
    const int* path;
    int64_t path_sb;
    int path_cols, N;
    int* new_lens;
};
hipError_t launch_cache_accept(const CacheAcceptParams& p, hipStream_t s);
// what a sequence of the new batch takes of its source
struct ForkPlan {
    int src, len, kept, part;  // len below 0: dropped; kept: pages; part: rows of a partly filled page
    int page, copy, need, first;  // its number; whether it goes to a new page; new ones, from `first` of the free on
};
struct CacheForkParams : PoolParams {
    const int* sources;
    const int* more;
    int more_all, n_new;
    int* new_table;
    int* new_lens;
    int* free_list;        // workspace: pages to give
    int* heirs;            // workspace, per source
    ForkPlan* plan;        // workspace, per new sequence
    int4* copies;          // workspace: per new sequence (page from, page to, rows)
};
hipError_t launch_cache_fork(const CacheForkParams& p, hipStream_t s);
struct CacheCompactParams : PoolParams {
    int* new_table;
    int* used;
    int2* moves;           // workspace: (from, to)
    int* n_moves;
};
hipError_t launch_cache_compact(const CacheCompactParams& p, hipStream_t s);

// Rotary positions (fa_rotary.hip)
struct RotaryTableParams {
    float* table;  // (n, R)
    int64_t n;
    int R;
    int mode;      // 0 none, 1 linear, 2 base, 3 ramp
    double base, factor, original, low, high, mul;
};
hipError_t launch_rotary_table(const RotaryTableParams& p, hipStream_t s);

struct RotaryTensor {
    const void* in;
    void* out;
    int64_t in_sb, in_ss, in_sh, out_sb, out_ss, out_sh;
    int heads;
};
struct RotaryParams {
    RotaryTensor x[2];     // q and, with heads > 0, k
    const float* table;    // (n_pos, R): cos then sin of the R / 2 pairs
    const void* pos;       // optional (B, S) int32 or int64, strides; null: 0 .. S - 1
    int64_t pos_sb, pos_ss;
    int pos64;
    int64_t n_pos;
    int B, S, D, R;
    int interleaved, copy; // copy: the columns past R too (out of place)
    float sign;            // -1: the transposed rotation (gradients)
    int vec;               // rows, strides and R allow 16-byte accesses
};
template <typename T>
hipError_t launch_rotary(const RotaryParams& p, hipStream_t s);

}  // namespace fa
