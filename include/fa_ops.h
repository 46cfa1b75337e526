/* C ABI of the operators around attention of the MI355X (gfx950) library:
 * attention with scored rules, new tokens after a shared prefix, rotary
 * positions.  The library, its status codes, element types and the rules of
 * memory, streams and capture are those of fa_abi.h: plain C types, device
 * memory allocated by the caller, work enqueued on the caller's HIP stream, no
 * call synchronises the host or keeps state.  The mini-kio/flash-attn-v100
 * reference has no counterpart of these functions.
 *
 * Tensors are (B, S, H, D) with element strides in the order (b, s, h, d); the d
 * stride is 1, base pointers 16-byte aligned, the other strides multiples of 16
 * bytes.  head_dim is any size up to 128 whose rows are whole 16-byte chunks
 * (FA_ERR_HEAD_DIM).  Lengths, offsets, positions and document ids are device
 * memory, read by the kernels only: their values are clamped to what exists, so
 * no value makes a kernel read or write out of range.
 */
#ifndef FA_OPS_H
#define FA_OPS_H

#include "fa_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FA_OPS_VERSION 2

#define FA_ERR_RULE -15   /* softcap neither 0 nor within [1e-6, 1e30], scale over 1e37 softcap, or an id / length array or its stride invalid */
#define FA_ERR_ROTARY -16 /* rotary columns not even, more than the head dim, or an invalid base, factor or table */

/* Attention with scored rules.  For query i and key j of sequence b, head h:
 *   x = scale q.k,  s = softcap tanh(x / softcap) (softcap > 0; x for 0)
 *       - slopes[b, h] |i + offset_b - j| (slopes non-NULL)
 *   seen: j < key_lengths[b]
 *         and (not causal or j <= i + offset_b or j < prefix_lengths[b])
 *         and (no documents or q_documents[b, i] == k_documents[b, j] >= 0)
 * O = softmax over the keys seen, times V; a query that sees no key gets O = 0
 * and lse = -inf (and no gradient).  lse is the natural-log sum of exp(s).
 * Of a query that stands off the keys (i + offset_b not in 0 .. key_lengths[b] - 1),
 * lse holds slope times the distance to the nearest key, a number that may leave it
 * few digits; lse_near is lse without it.
 * Keys from key_lengths[b] on and tokens of a negative document reach no
 * result, whatever their values are. */
typedef struct fa_scored_args {
    const void* q;
    const void* k;
    const void* v;
    void* o;
    float* lse;                    /* (B, H, Sq) contiguous; optional in the forward, read by the backward */
    const void* dout;              /* backward only, as the five below */
    void* dq;
    void* dk;
    void* dv;
    float* dslopes;                /* optional gradient of slopes, in their shape, float32 contiguous */
    int64_t q_stride[4];
    int64_t k_stride[4];
    int64_t v_stride[4];
    int64_t o_stride[4];
    int64_t do_stride[4];
    int64_t dq_stride[4];
    int64_t dk_stride[4];
    int64_t dv_stride[4];
    int32_t batch;
    int32_t seqlen_q;
    int32_t seqlen_k;
    int32_t num_heads;
    int32_t num_heads_kv;
    int32_t head_dim;
    int32_t dtype;
    int32_t causal;
    float scale;
    float softcap;                 /* 0: none */
    const float* slopes;           /* optional (H), or (B, H) with slopes_batch_stride = H */
    int64_t slopes_batch_stride;
    const int32_t* prefix_lengths; /* optional (B) */
    const int32_t* key_lengths;    /* optional (B) */
    const int32_t* query_offsets;  /* optional (B), else query_offset; held within +-2^30 */
    int32_t query_offset;
    const int32_t* q_documents;    /* optional (B, Sq), both or none (any, where one side is empty); token stride 1 */
    const int32_t* k_documents;    /* optional (B, Sk); may be q_documents */
    int64_t q_documents_stride;    /* batch strides in elements */
    int64_t k_documents_stride;
    float* lse_near;               /* optional, beside lse: written by the forward, read by the backward in its place */
} fa_scored_args;

int32_t fa_ops_version(void);

/* Validate-only (host): the status fa_scored_fwd (backward == 0) or
 * fa_scored_bwd would return for these arguments. */
int32_t fa_scored_check(const fa_scored_args* args, int32_t backward);

/* Bytes of device workspace; 0 where none is needed and on invalid arguments.
 * Aligned to 16 bytes for the forwards, to 256 for the backward; used until the
 * call's kernels have run, so calls at once need one each. */
size_t fa_scored_fwd_workspace_size(const fa_scored_args* args);
size_t fa_scored_bwd_workspace_size(const fa_scored_args* args);

/* Forward: o and lse.  Few queries (single tokens and chunks over a longer cache)
 * run with their keys split over workgroups; results differ by the order of
 * float32 sums. */
int32_t fa_scored_fwd(const fa_scored_args* args, void* workspace, size_t workspace_bytes, void* hip_stream);

/* Backward: dq, dk, dv (and dslopes), fully written; deterministic.  P is exp(s - lse)
 * of the lse given (and delta is of the o given), so that dq, dk and dv may be of a part
 * of the keys of a row whose lse and o are of all; dslopes takes the keys seen for all.
 * lse_near, of the same keys as lse, keeps the digits of queries far off the keys. */
int32_t fa_scored_bwd(const fa_scored_args* args, void* workspace, size_t workspace_bytes, void* hip_stream);

/* New tokens of B sequences after a prefix that all of them share.  Query i of
 * a sequence with n = key_lengths[b] keys of its own (the new tokens' among
 * them; seqlen_k where NULL) stands at own position n - Sq + i: it sees the
 * whole prefix and its own keys up to that position; at a negative own position
 * it sees nothing (o = 0, lse = -inf).  Distances (slopes) count the prefix
 * before the own keys.  Forward only. */
typedef struct fa_prefix_args {
    const void* q;                /* (B, Sq, H, D) */
    const void* k_prefix;         /* (P, Hkv, D): strides (s, h, d) */
    const void* v_prefix;
    const void* k;                /* (B, Sk, Hkv, D) */
    const void* v;
    void* o;
    float* lse;                   /* optional (B, H, Sq) */
    int64_t q_stride[4];
    int64_t kp_stride[3];
    int64_t vp_stride[3];
    int64_t k_stride[4];
    int64_t v_stride[4];
    int64_t o_stride[4];
    int32_t batch;
    int32_t seqlen_q;
    int32_t prefix_len;
    int32_t seqlen_k;
    int32_t num_heads;
    int32_t num_heads_kv;
    int32_t head_dim;
    int32_t dtype;
    float scale;
    float softcap;
    const float* slopes;
    int64_t slopes_batch_stride;
    const int32_t* key_lengths;   /* optional (B) */
} fa_prefix_args;

int32_t fa_prefix_check(const fa_prefix_args* args);
size_t fa_prefix_workspace_size(const fa_prefix_args* args);
int32_t fa_prefix_fwd(const fa_prefix_args* args, void* workspace, size_t workspace_bytes, void* hip_stream);

/* Rotary table: (positions, rotary_dim) float32, row n the cosines of the
 * rotary_dim / 2 pairs' angles n w_j, then their sines, each times `mul`; angles
 * in 64 bits.  w_j = base^(-2 j / rotary_dim), with scaling
 *   FA_ROTARY_NONE
 *   FA_ROTARY_LINEAR: w_j / factor
 *   FA_ROTARY_BASE:   base times factor^(R / (R - 2))
 *   FA_ROTARY_RAMP:   w_j (g + (1 - g) / factor), g = clamp((original w_j / 2 pi - low) / (high - low), 0, 1) */
#define FA_ROTARY_NONE 0
#define FA_ROTARY_LINEAR 1
#define FA_ROTARY_BASE 2
#define FA_ROTARY_RAMP 3
int32_t fa_rotary_table(float* table, int64_t positions, int32_t rotary_dim, int32_t scaling, double base,
                        double factor, double original, double low, double high, double mul, void* hip_stream);

/* Rotates the first rotary_dim columns of q (and k): pairs (j, j + rotary_dim / 2),
 * interleaved: (2 j, 2 j + 1).  inverse: the transposed rotation (the gradient of
 * the rotation).  Outputs may be the inputs themselves, with equal strides (the
 * columns past rotary_dim are then left alone, else copied); they may not overlap
 * in any other way.  A negative position leaves its token as it
 * is, a position past the table makes it NaN.  No alignment beyond the element's
 * is needed; the d stride is 1. */
typedef struct fa_rotary_args {
    const void* q;
    void* q_out;
    const void* k;                /* optional */
    void* k_out;
    int64_t q_stride[4];
    int64_t q_out_stride[4];
    int64_t k_stride[4];
    int64_t k_out_stride[4];
    const float* table;
    const void* positions;        /* optional (B, S) int32, or int64 with positions_64; NULL: 0 .. S - 1 */
    int64_t positions_stride[2];
    int64_t table_positions;
    int32_t positions_64;
    int32_t batch;
    int32_t seqlen;
    int32_t num_heads;
    int32_t num_heads_k;          /* 0 without k */
    int32_t head_dim;
    int32_t rotary_dim;
    int32_t dtype;
    int32_t interleaved;
    int32_t inverse;
} fa_rotary_args;

int32_t fa_rotary_check(const fa_rotary_args* args);
int32_t fa_rotary(const fa_rotary_args* args, void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif /* FA_OPS_H */
