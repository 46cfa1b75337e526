/* C ABI of the paged key/value cache of the MI355X (gfx950) library: attention
 * of new tokens, or of a tree of drafted tokens, over a cache of pages, and the
 * cache's own operators: write, accept, fork, compact.  The library, its status
 * codes, element types and the rules of memory, streams and capture are those of
 * fa_abi.h: plain C types, device memory allocated by the caller, work enqueued
 * on the caller's HIP stream, no call synchronises the host or keeps state.  The
 * mini-kio/flash-attn-v100 reference has no counterpart of these functions.
 *
 * A cache is a pool of pages of page_size tokens, (pages, page_size, Hkv, D), of
 * one layer or of several (a leading layer stride).  Token x of sequence b lies in
 * row x % page_size of page page_table[b, x / page_size].  Without a page table
 * sequence b is page b, whole.  Tables, lengths, trees, paths and sources are
 * device memory, read by the kernels only.  A page outside 0 .. pages - 1 holds
 * nothing: its keys are not seen and its tokens are not written or moved; lengths
 * are clamped to what the table has room for.  So no value makes a kernel read or
 * write out of range.
 */
#ifndef FA_PAGED_H
#define FA_PAGED_H

#include "fa_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FA_PAGED_VERSION 1

#define FA_ERR_PAGES -17 /* page size not a multiple of 16 (with a table), too many pages or tree nodes, or an invalid table, tree or path array */

#define FA_MAX_TREE_NODES 256  /* drafted tokens of a tree, a sequence */
#define FA_MAX_POOL_PAGES (1 << 20) /* pages of a pool that is forked or compacted */

/* Rows of head_dim elements, whole 16-byte chunks, up to 128 columns; strides in
 * elements in the order (layer, page, row, head, d), the d stride 1, the others
 * multiples of 16 bytes.  k and v of a pool that is written share no memory. */
typedef struct fa_page_pool {
    void* k;
    void* v;
    int64_t k_stride[5];
    int64_t v_stride[5];
    int32_t layers;
    int32_t pages;
    int32_t page_size;
    int32_t num_heads_kv;
    int32_t head_dim;
    int32_t dtype;
    int32_t batch;
    int32_t table_cols;        /* pages a sequence may hold; 1 without a table */
    const int32_t* page_table; /* (batch, table_cols), column stride 1; NULL: sequence b is page b */
    int64_t table_stride;
    const int32_t* key_lengths; /* (batch) filled tokens; NULL: all there is room for */
} fa_page_pool;

int32_t fa_paged_version(void);

/* Attention of the newest N = seqlen_q tokens of each sequence, which are the last
 * of its n = key_lengths[b] filled ones: token i lies at place n - N + i.
 * Without parents it sees every key up to its own place.  With parents the N
 * tokens are a tree behind the n - N tokens before them (the context): parents[b, i]
 * is the index, below i, of the token that i follows, or -1 where it follows the
 * context; it sees the context, the tokens on its way there and itself.  Any
 * other value, or a parent that is no token, makes i none: it sees nothing and is seen by none.  A
 * token at a negative place, or none, has o = 0 and lse = -inf.
 *   x = scale q.k, s = softcap tanh(x / softcap) - slopes[b, h] (tokens from the key
 *   to the query on its way)
 * O = softmax over the keys seen, times V.  What a key that a token does not see
 * holds does not reach it (infinities and NaN neither).  Forward only. */
typedef struct fa_paged_args {
    fa_page_pool pool;     /* one layer; k, v are read only */
    const void* q;         /* (B, N, H, D) */
    void* o;
    float* lse;            /* optional (B, H, N) */
    int64_t q_stride[4];
    int64_t o_stride[4];
    int32_t seqlen_q;
    int32_t num_heads;
    float scale;
    float softcap;
    const float* slopes;   /* optional (H), or (B, H) with slopes_batch_stride = H */
    int64_t slopes_batch_stride;
    const int32_t* parents; /* optional (N), or (B, N) with parents_stride */
    int64_t parents_stride;
} fa_paged_args;

int32_t fa_paged_check(const fa_paged_args* args);
size_t fa_paged_workspace_size(const fa_paged_args* args); /* bytes, 16-byte aligned */
int32_t fa_paged_fwd(const fa_paged_args* args, void* workspace, size_t workspace_bytes, void* hip_stream);

/* Writes the rows of N = tokens new tokens: row i of sequence b to place
 * key_lengths[b] - N + i of every layer (a negative place is not written).  Two
 * sequences that share a page may not write the same row of it; k and v do not overlap
 * the pool. */
typedef struct fa_cache_write_args {
    fa_page_pool pool;
    const void* k;          /* (layers, B, N, Hkv, D): strides in that order */
    const void* v;
    int64_t k_stride[5];
    int64_t v_stride[5];
    int32_t tokens;
} fa_cache_write_args;

int32_t fa_cache_write_check(const fa_cache_write_args* args);
int32_t fa_cache_write(const fa_cache_write_args* args, void* hip_stream);

/* Keeps, of the N = tokens drafted ones at the end of each sequence, those of its
 * path: path[b, j], ascending indices, ended by the first entry that is not above
 * the one before it or not in 0 .. N - 1.  Row path[b, j] of the drafted ones moves
 * to row j, in every layer, and new_lengths[b] = key_lengths[b] - N + their number.
 * A sequence of fewer than N tokens stays as it is.  new_lengths is not key_lengths. */
typedef struct fa_cache_accept_args {
    fa_page_pool pool;
    const int32_t* path;    /* (B, path_cols) */
    int64_t path_stride;
    int32_t path_cols;
    int32_t tokens;
    int32_t* new_lengths;   /* (B) */
} fa_cache_accept_args;

int32_t fa_cache_accept_check(const fa_cache_accept_args* args);
int32_t fa_cache_accept(const fa_cache_accept_args* args, void* hip_stream);

/* Sequence b of the new batch continues sequence sources[b] (none: empty) with
 * room for more[b] new tokens: new_lengths[b] = key_lengths[sources[b]] + more[b].
 * Whole pages are shared.  A partly filled last page stays with the first that
 * continues its sequence, and its filled rows are copied, in every layer, to a
 * page of its own for each other one.  New pages are the lowest ones that the new
 * batch neither shares nor keeps, given in its order.  A sequence that has no room in
 * the table is dropped (length 0, no pages), and so are the first one that the free
 * pages do not suffice for and those after it that need any; what they would have kept
 * is free after this call.  Columns without a page hold -1.  The outputs do not overlap
 * the inputs. */
typedef struct fa_cache_fork_args {
    fa_page_pool pool;          /* with a table */
    const int32_t* sources;     /* (new_batch) */
    const int32_t* more;        /* optional (new_batch), else more_all */
    int32_t more_all;
    int32_t new_batch;
    int32_t* new_table;         /* (new_batch, table_cols) contiguous */
    int32_t* new_lengths;       /* (new_batch) */
} fa_cache_fork_args;

int32_t fa_cache_fork_check(const fa_cache_fork_args* args);
size_t fa_cache_fork_workspace_size(const fa_cache_fork_args* args); /* 16-byte aligned */
int32_t fa_cache_fork(const fa_cache_fork_args* args, void* workspace, size_t workspace_bytes, void* hip_stream);

/* Moves the pages in use to the front of the pool: with U of them, the k-th lowest
 * one from U on goes to the k-th lowest free one below U, in every layer.
 * new_table holds their new numbers (-1 in columns that no token needs), used[0] = U. */
typedef struct fa_cache_compact_args {
    fa_page_pool pool;          /* with a table */
    int32_t* new_table;         /* (batch, table_cols) contiguous; not page_table */
    int32_t* used;              /* (1) */
} fa_cache_compact_args;

int32_t fa_cache_compact_check(const fa_cache_compact_args* args);
size_t fa_cache_compact_workspace_size(const fa_cache_compact_args* args); /* 16-byte aligned */
int32_t fa_cache_compact(const fa_cache_compact_args* args, void* workspace, size_t workspace_bytes, void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif /* FA_PAGED_H */
