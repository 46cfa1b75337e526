// Attention with scored rules for gfx950: scores capped by a tanh, a bias that
// falls with the distance of query and key, and masks by documents, prefixes
// and key lengths, none of them held as a (query, key) matrix.
//
//   x = scale q.k                       t = cap tanh(x / cap)  (or x)
//   s = t - slope |i + off - j|         P = softmax over the keys seen
//   seen: j < lim(i), lim(i) = min(len, causal ? max(i + off + 1, prefix) : len)
//         and the documents of query and key are equal and not negative
//
// off, prefix, len are per sequence.  lim never falls with i, so without
// documents a block of queries sees one run of keys; with documents a block
// visits the key tiles whose range of document ids (doc_tiles_kernel) meets its
// own: 64 tiles are tested at a time, one a lane, and a ballot gives the bit
// mask that the tile loop walks.  A second ballot marks the tiles that every
// query of the wave sees whole: only the others run the masking step.
// tanh x = 1 - 2 r, r = 1 / (1 + e^(2x)): one exp2 and one reciprocal a score,
// and its derivative 1 - tanh^2 = 4 (r - r^2) comes with two more operations; by a
// series under caps far above the scores (Cap).
// Distances are taken from the key nearest to the query (SeqRule::near).
//
// Roundings of 16-bit inputs: P and dS where they enter a product (the matrix
// instructions take 16 bits), and delta from the rounded O that the caller keeps;
// sums, statistics and parts are float32.  bf16, cap: the 2-norm of dQ is off by
// 2.6e-3, of which its own rounding is 1.7e-3 and dS up to 2.4e-3; dS in two pieces
// would cost another product, an unrounded O another saved tensor.
//
// Tiles, operand layouts and pipelines are those of fa_fwd.hpp and fa_bwd.hpp:
// one workgroup has 4 waves of 32 queries (forward, dQ) or 32 keys (dK/dV).
// The forward with a cap is bound by the vector arithmetic of the scores beside the
// products: 11 vector instructions for each, two of a quarter of the rate, leave the
// matrix unit half of the time at most (it has 37%).  The other passes (5 to 8 for
// each, 30 to 39%) wait: one barrier a tile with two workgroups a CU, and in dQ and
// dK/dV nothing of a wave between the products of the scores and their arithmetic.
// The clock is 2.0 to 2.3 GHz under them, of 2.4.  2 x 4096, 32 on 8 heads of 128,
// bf16, causal: forward 286 us and backward 971 us with no rule but the mask (the dense
// kernels 255 and 1020), 333 and 1137 with the cap, 311 and 1033 with slopes (1082 with
// their gradient), 92 and 333 over documents of 700 tokens.
#pragma once

#include <limits.h>

#include <type_traits>

#include "fa_bwd.hpp"
#include "fa_common.hpp"
#include "fa_fwd.hpp"
#include "fa_ops_params.hpp"

namespace fa {

// ---------------------------------------------------------------------------
// per-sequence rules
struct SeqRule {
    int off, prefix, len;
    bool causal;
    __device__ FA_INLINE inline SeqRule(const ScoredParams& p, int b) {
        const int o = p.offsets ? p.offsets[b] : p.offset0;
        off = max(-kMaxOffset, min(kMaxOffset, o));
        len = p.lens ? max(0, min(p.Sk, p.lens[b])) : p.Sk;
        prefix = p.prefix ? max(0, min(p.Sk, p.prefix[b])) : 0;
        causal = p.causal != 0;
    }
    // keys [0, lim(i)) may be seen by query i
    __device__ FA_INLINE inline int lim(int i) const { return causal ? min(len, max(i + off + 1, prefix)) : len; }
    // The key nearest to query i.  A row's softmax does not change when all of its
    // distances lose the one to that key, and |i + off - j| less it is
    // |near(i) - j|: the kernels take distances from there, so that the scores of a
    // query far from the keys keep their digits, and only the LSE holds
    // slope far(i).
    __device__ FA_INLINE inline int near(int i) const { return max(0, min(len - 1, i + off)); }
    __device__ FA_INLINE inline float far(int i) const { return (float)abs(i + off - near(i)); }
    // queries from first(j) on may see key j
    __device__ FA_INLINE inline int first(int j) const {
        return j >= len ? INT_MAX : (!causal || j < prefix) ? 0 : max(0, j - off);
    }
};

// tanh cap.  value(): cap tanh(x / cap) log2 e of a raw score s (x = scale s);
// slope(): the derivative / 4.
// Two forms.  Quick: 1 - 2 r, whose cancellation near 0 leaves an error of about
// 2^-22 of the cap in the score.  EXACT: a series there (through x^13: 2e-8 of the
// value below 0.45), so that small scores keep their digits under any cap.  16-bit
// inputs take the quick form up to kWideCap, where its error in a score, and so in a
// probability, is at most 2^-14, below the 2^-12 and 2^-9 to which fp16 and bf16
// round the probabilities; float32 always the series.  2 x 4096, 32 on 8 heads of 128,
// bf16, causal, quick / series: forward 344 / 461 us, training step 1500 / 1830; single
// tokens over 16 caches of 8192: 108 / 110.
constexpr float kWideCap = 256.f;
template <bool EXACT>
struct Cap {
    float k1, k2, top;  // scale / cap; that times 2 log2 e; cap log2 e
    float r, t;         // of the last score
    template <typename P>
    __device__ FA_INLINE inline explicit Cap(const P& p) : k1(p.cap_k1), k2(p.cap_k2), top(p.cap_top) {}
    __device__ FA_INLINE inline float rcp(float s) { return __builtin_amdgcn_rcpf(1.f + fast_exp2(s * k2)); }
    __device__ FA_INLINE inline float value(float s) {
        r = rcp(s);
        if constexpr (!EXACT) {
            return __builtin_fmaf(-2.f * top, r, top);
        } else {
            const float x = s * k1, u = x * x;
            float q = 21844.f / 6081075.f;
            q = __builtin_fmaf(q, u, -1382.f / 155925.f);
            q = __builtin_fmaf(q, u, 62.f / 2835.f);
            q = __builtin_fmaf(q, u, -17.f / 315.f);
            q = __builtin_fmaf(q, u, 2.f / 15.f);
            q = __builtin_fmaf(q, u, -1.f / 3.f);
            q = __builtin_fmaf(q * u, x, x);
            t = __builtin_fabsf(x) < 0.45f ? q : __builtin_fmaf(-2.f, r, 1.f);
            return top * t;
        }
    }
    __device__ FA_INLINE inline float slope() const {
        if constexpr (!EXACT)
            return __builtin_fmaf(-r, r, r);
        else
            return __builtin_fmaf(-0.25f * t, t, 0.25f);
    }
};

// CAP of the kernels.  kCapWide (16-bit inputs) is compiled with SLOPE only, whose
// kernels hold scores as values; a call without slopes has a slope of 0 there.
constexpr int kCapNone = 0, kCapQuick = 1, kCapWide = 2;
template <int CAP, bool SLOPE>
__device__ FA_INLINE inline bool has_slope(const ScoredParams& p) {
    return SLOPE && (CAP != kCapWide || p.slopes != nullptr);
}

// ---------------------------------------------------------------------------
// whether the id ranges of two blocks meet in an id that is not negative
__device__ FA_INLINE inline bool docs_meet(int2 a, int2 b) {
    return a.y >= max(b.x, 0) && b.y >= max(a.x, 0);
}
__device__ FA_INLINE inline bool docs_one(int2 a, int2 b) { return a.x == a.y && b.x == b.y && a.x == b.x && a.x >= 0; }
__device__ FA_INLINE inline int2 docs_join(int2 a, int2 b) { return make_int2(min(a.x, b.x), max(a.y, b.y)); }
__device__ FA_INLINE inline int2 uniform2(int2 a) {
    return make_int2(__builtin_amdgcn_readfirstlane(a.x), __builtin_amdgcn_readfirstlane(a.y));
}

// A tile of a walk: its index (-1 past the last) and flags, wave-uniform.
// kAct: some row of this wave may see it; kLim: the causal mask and the lengths
// leave it whole to every row, kDoc: so do the documents; kNeg: it holds tokens of
// no document; kMore: the walk has not ended.
struct TileRef {
    int t;
    unsigned fl;
};
constexpr unsigned kAct = 1, kLim = 2, kDoc = 4, kNeg = 8, kMore = 16, kFull = kLim | kDoc;

// 64 tiles of a walk, a bit each: those that some row of the workgroup sees, and
// the flags above.
struct TileChunk {
    uint64_t vis, act, lim, doc, neg;
    __device__ FA_INLINE inline TileRef ref(int base, int i) const {
        return TileRef{base + i, kMore | ((act >> i) & 1 ? kAct : 0u) | ((lim >> i) & 1 ? kLim : 0u) |
                                     ((doc >> i) & 1 ? kDoc : 0u) | ((neg >> i) & 1 ? kNeg : 0u)};
    }
};

// zeros into the rows of a tile that belong to no document (their values may be
// anything, and 0 times a NaN is none).  All threads of the NT; a barrier follows.
template <typename T, int R, int D, int W, int NT>
__device__ FA_INLINE inline void clear_rows(T* tile, const int* docs, int tid) {
    constexpr int EPC = 16 / (int)sizeof(T), CPR = D / EPC;
#pragma unroll 1
    for (int c = tid; c < R * CPR; c += NT) {
        const int row = c / CPR, col = c % CPR;
        if (docs[row] < 0) *reinterpret_cast<uint4*>(tile + row * W + col * EPC) = make_uint4(0u, 0u, 0u, 0u);
    }
}

// float32 products over columns that the inputs do not have (head dim 80 in tiles
// of 128) are left out, 32 columns at a time: an instruction takes 64 cycles, many
// times the test (4 x 700 x 12 heads of 80: 491 -> 407 us a step)
template <int D>
__device__ FA_INLINE inline int live_cols(const ScoredParams& p) {
    return D == 32 ? D : p.cols;
}

// At the head of a rarely taken branch: the compiler would otherwise compute it
// every time and select (the masks of the forward: 60 of 370 vector instructions
// a tile)
__device__ FA_INLINE inline void stay_branch() { asm volatile(""); }

template <int N>
using template_int = std::integral_constant<int, N>;

// The kernel's arguments, to be read where they are used: what only the epilogue
// needs would otherwise be read first and take scalar registers from the loop
// (kept in lanes of vector registers, a read of a lane for each use).
template <typename P = ScoredParams>
__device__ FA_INLINE inline const P& late_args() {
    uint64_t a = (uint64_t)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return *(const P*)(uintptr_t)a;
}

// -x for four floats
__device__ FA_INLINE inline uint4 neg32x4(uint4 v) {
    return make_uint4(v.x ^ 0x80000000u, v.y ^ 0x80000000u, v.z ^ 0x80000000u, v.w ^ 0x80000000u);
}

// The rows of a wave's 32-row block (lane l holds row l % 32, 16 columns of each
// 32 in accumulator order), times mul, through LDS as rows of T and to global
// memory in 16-byte chunks.  Holds a barrier; waves that are not `mine` only pass it.
template <typename T, int D>
__device__ FA_INLINE inline void store_rows(T* Os, int OW, const f32x16 (&acc)[D / 32], float mul, T* base, int64_t stride,
                                           int row0, int n_rows, int cols, int lane, bool mine) {
    const int l32 = lane & 31, hi = lane >> 5;
    if (mine) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * i + 8 * g + 4 * hi;
                if constexpr (Elem<T>::kF32) {
                    f32x4 v4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v4[e] = acc[i][4 * g + e] * mul;
                    *reinterpret_cast<f32x4*>(Os + l32 * OW + d) = v4;
                } else {
                    s16x4 v4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v4[e] = Elem<T>::pack1(acc[i][4 * g + e] * mul);
                    *reinterpret_cast<s16x4*>(Os + l32 * OW + d) = v4;
                }
            }
    }
    lds_barrier();
    if (mine) {
        constexpr int EPC = 16 / (int)sizeof(T), CPR = D / EPC;
#pragma unroll
        for (int i = 0; i < 32 * CPR / 64; ++i) {
            const int cidx = lane + 64 * i, row = cidx / CPR, col = cidx % CPR;
            if (row0 + row < n_rows && col * EPC < cols)
                *reinterpret_cast<uint4*>(base + (int64_t)(row0 + row) * stride + col * EPC) =
                    *reinterpret_cast<const uint4*>(Os + row * OW + col * EPC);
        }
    }
}

// Which (batch, head) and which block of it, from the longest walk on, a workgroup
// takes.  With documents the walks are short and of any length, and a sequence of
// long documents would keep its XCDs busy after the others have drained: there
// the heads of a group come from all sequences in turn, and the groups are twice
// as large (2 x 8192 x 16 heads of 128, documents of 153 to 3355 tokens:
// 1100 -> 962 us a step)
struct BlockOrder {
    int b, head, rank;
};
template <int SLOTS>
__device__ FA_INLINE inline BlockOrder block_order(const ScoredParams& p, int heads) {
    if (p.q_docs) {
        const int2 t = tile_order<2 * SLOTS, true>(p.n_tiles);
        return BlockOrder{t.x % p.B, t.x / p.B, t.y};
    }
    const int2 t = tile_order<SLOTS, true>(p.n_tiles);
    return BlockOrder{t.x / heads, t.x % heads, t.y};
}

// ---------------------------------------------------------------------------
// Forward, over the tiles of a walk.  KS = 2: two groups of 4 waves on the same
// queries, taking the walk's tiles in turn, for grids that leave CUs idle.
template <typename T, int D, int CAP, bool SLOPE, int KS>
__global__ __launch_bounds__(256 * KS, (KS == 1 && !(Elem<T>::kF32 && D == 128) ? 2 : 1)) void scored_fwd_kernel(
    const ScoredParams p) {
    using C = FwdCfg<T, D>;
    constexpr int BN = C::BN, NB = C::NB, KW = C::KW, VW = C::VW, NW = C::NW;
    constexpr int TPD = 64 / BN;  // tiles per range of document ids
    __shared__ __attribute__((aligned(16))) T smem[C::SMEM_ELEMS * KS];
    __shared__ __attribute__((aligned(16))) int ids[KS][2][64];  // document ids of the tiles

    const int tid = threadIdx.x;
    const int lane = tid & 63, wg = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, hi = lane >> 5;
    const int w = wg & 3, sp = KS == 1 ? 0 : wg >> 2;  // (& 3: its range decides copies at compile time)
    const BlockOrder ord = block_order<32 * (KS == 1 ? 2 : 1)>(p, p.H);
    const int qt = p.n_tiles - 1 - ord.rank;  // longest causal rows first
    const int h = ord.head, b = ord.b;
    const int hk = h / p.group;
    const int q0 = qt * C::BM, qw0 = q0 + 32 * w, qi = qw0 + l32;
    const SeqRule rule(p, b);

    const T* __restrict__ kbase = (const T*)p.k + b * p.k_sb + hk * p.k_sh;
    const T* __restrict__ vbase = (const T*)p.v + b * p.v_sb + hk * p.v_sh;

    // ---- Q into registers (MFMA B operand) ----
    constexpr int QR = C::F32 ? D / 8 : D / 16;
    uint4 qreg[QR];
    {
        const T* qrow = (const T*)p.q + b * p.q_sb + (int64_t)qi * p.q_ss + h * p.q_sh;
#pragma unroll
        for (int i = 0; i < QR; ++i) {
            const int d0 = C::F32 ? 8 * i + 4 * hi : 16 * i + 8 * hi;
            qreg[i] = qi < p.Sq && d0 < p.cols ? *reinterpret_cast<const uint4*>(qrow + d0) : make_uint4(0u, 0u, 0u, 0u);
        }
    }

    // ---- the walk over key tiles ----
    const int lim_hi = rule.lim(min(q0 + C::BM, p.Sq) - 1);
    const int n_kt = (max(lim_hi, 0) + BN - 1) / BN;
    const int wlim_lo = rule.lim(qw0), wlim_hi = qw0 < p.Sq ? rule.lim(min(qw0 + 31, p.Sq - 1)) : 0;
    const int lim_l = rule.lim(qi);
    const bool docs = p.q_docs != nullptr;
    const int* kdoc = p.k_docs + (docs ? (int64_t)b * p.k_docs_pad : 0);
    const int2* krng = p.k_rng + (docs ? (int64_t)b * (p.k_docs_pad / 64) : 0);
    int2 qr = {0, 0}, wr = {0, 0};
    int qd = -2;  // no key's id
    if (docs) {
        const int2* qrng = p.q_rng + (int64_t)b * (p.q_docs_pad / 64) + q0 / 64;
        const int2 a = uniform2(qrng[0]), c = q0 + 64 < p.q_docs_pad ? uniform2(qrng[1]) : a;
        qr = docs_join(a, c);
        // a wave past the last query may lie past the ranges: it is never active
        wr = w < 2 ? a : c;
        const int id = qi < p.Sq ? p.q_docs[(int64_t)b * p.q_docs_pad + qi] : -1;
        if (id >= 0) qd = id;
    }
    // key tiles [base, base + 64)
    auto chunk_at = [&](int base) FA_INLINE -> TileChunk {
        const int t = base + lane, k0 = t * BN;
        bool v = t < n_kt, a = v && k0 < wlim_hi;
        TileChunk c;
        c.lim = __ballot(k0 + BN <= wlim_lo);
        c.doc = ~0ull;
        c.neg = 0;
        if (docs) {
            const int2 r = v ? krng[t / TPD] : make_int2(-1, -1);
            v = v && docs_meet(r, qr);
            a = a && v && docs_meet(r, wr);
            c.doc = __ballot(docs_one(r, wr));
            c.neg = __ballot(r.x < 0);
        }
        c.vis = __ballot(v);
        c.act = __ballot(a);
        return c;
    };
    // the next tile of a chunk.  KS = 2: of this group, with kMore and kNeg of the
    // groups together (they share the barriers)
    auto next = [&](TileChunk& c, int base) FA_INLINE -> TileRef {
        auto one = [&]() FA_INLINE -> TileRef {
            if (c.vis == 0) return TileRef{-1, 0u};
            const int i = (int)__builtin_ctzll(c.vis);
            c.vis &= c.vis - 1;
            return c.ref(base, i);
        };
        TileRef r = one();
        if constexpr (KS == 2) {
            const TileRef r2 = one();
            const unsigned both = (r.fl | r2.fl) & (kMore | kNeg);
            if (sp) r = r2;
            r.fl |= both;
        }
        return r;
    };

    f32x16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = f32x16{};
    float m_run = -1e30f;  // running max in log2 units
    float l_run = 0.f;     // lane-partial row sum
    const float c = p.scale_log2;
    Cap<(C::F32 || CAP == kCapWide)> cap(p);
    const float slope2 = has_slope<CAP, SLOPE>(p) ? p.slopes[b * p.slopes_sb + h] * kLog2e : 0.f;
    const int qpos = rule.near(qi);

    T* Ks0 = smem + sp * C::SMEM_ELEMS;
    T* Vs0 = Ks0 + 2 * C::KTILE;
    DmaTile<T, BN, D, KW, NW> kdma;
    kdma.init(p.k_ss, lane, w, p.cols);
    DmaTile<T, BN, D, VW, NW> vdma;
    vdma.init(p.v_ss, lane, w, p.cols);
    // keys past the sequence's length land as zeros; no tile: nothing is read
    auto load_k = [&](const TileRef& r, int slot) FA_INLINE {
        const int k0 = max(r.t, 0) * BN, nv = r.t < 0 ? 0 : rule.len - k0;
        if constexpr (C::F32)
            kdma.load(kbase + (int64_t)k0 * p.k_ss, p.k_ss, nv, Ks0 + slot * C::KTILE, lane);
        else
            kdma.load_untracked(kbase + (int64_t)k0 * p.k_ss, p.k_ss, nv, Ks0 + slot * C::KTILE, lane);
    };
    auto load_v = [&](const TileRef& r, int slot) FA_INLINE {
        const int k0 = max(r.t, 0) * BN, nv = r.t < 0 ? 0 : rule.len - k0;
        if constexpr (C::F32)
            vdma.load(vbase + (int64_t)k0 * p.v_ss, p.v_ss, nv, Vs0 + slot * C::VTILE, lane);
        else
            vdma.load_untracked(vbase + (int64_t)k0 * p.v_ss, p.v_ss, nv, Vs0 + slot * C::VTILE, lane);
    };

    // (the ids of a 64-token range, of which a float32 tile is one half)
    auto load_ids = [&](const TileRef& r, int slot) FA_INLINE {
        if (docs && w == 0 && r.t >= 0)
            dma_load4_untracked(buffer_words(kdoc + r.t / TPD * 64, 256), lds_addr(ids[sp][slot]), 4 * lane);
    };

    // ---- S^T = K Q^T of a tile ----
    auto qk = [&](const T* Ks, f32x16 (&s)[NB]) FA_INLINE {
#pragma unroll
        for (int blk = 0; blk < NB; ++blk) {
            s[blk] = f32x16{};
            const T* krow = Ks + (32 * blk + l32) * KW;
#pragma unroll
            for (int i = 0; i < QR; ++i) {
                if constexpr (C::F32) {
                    if (i % 4 == 0 && 8 * i >= live_cols<D>(p)) break;
                    const f32x4 a = *reinterpret_cast<const f32x4*>(krow + 8 * i + 4 * hi);
                    const f32x4 bq = __builtin_bit_cast(f32x4, qreg[i]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[blk] = mfma_f32(a[e], bq[e], s[blk]);
                } else {
                    const s16x8 a = *reinterpret_cast<const s16x8*>(krow + 16 * i + 8 * hi);
                    s[blk] = Elem<T>::mfma(a, __builtin_bit_cast(s16x8, qreg[i]), s[blk]);
                }
            }
        }
    };
    // ---- rules, then mask and running max.  A score is held as u, its value in log2
    // units is ua u + ub: u the raw product, or r of the cap (which falls with
    // the score), or the value itself ----
    constexpr bool RCP = CAP == kCapQuick && !SLOPE && !C::F32, VALUE = SLOPE || (CAP && C::F32);
    const float ua = VALUE ? 1.f : RCP ? -2.f * cap.top : c, ub = RCP ? cap.top : 0.f;
    constexpr float kHidden = RCP ? INFINITY : -INFINITY;
    auto rules = [&](f32x16 (&s)[NB], int k0) FA_INLINE {
        if constexpr (RCP) {
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[blk][e] = cap.rcp(s[blk][e]);
        } else if constexpr (VALUE) {
            const float d0 = (float)(qpos - k0 - 4 * hi);
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float t = CAP ? cap.value(s[blk][e]) : s[blk][e] * c;
                    const float d = d0 - (float)(32 * blk + 8 * (e >> 2) + (e & 3));
                    s[blk][e] = SLOPE ? __builtin_fmaf(-slope2, __builtin_fabsf(d), t) : t;
                }
        }
    };
    auto mask_max = [&](f32x16 (&s)[NB], const TileRef& r, const int* id) FA_INLINE {
        const int k0 = r.t * BN;
        if (!(r.fl & kLim)) {
            stay_branch();
            const int lim = lim_l - k0 - 4 * hi;
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (32 * blk + 8 * (e >> 2) + (e & 3) >= lim) s[blk][e] = kHidden;
        }
        if (!(r.fl & kDoc)) {
            stay_branch();
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int4 kd = *reinterpret_cast<const int4*>(id + 32 * blk + 8 * g + 4 * hi);
                    if (kd.x != qd) s[blk][4 * g] = kHidden;
                    if (kd.y != qd) s[blk][4 * g + 1] = kHidden;
                    if (kd.z != qd) s[blk][4 * g + 2] = kHidden;
                    if (kd.w != qd) s[blk][4 * g + 3] = kHidden;
                }
        }
        // (four chains: the wave waits out each step of one)
        float m4[4] = {kHidden, kHidden, kHidden, kHidden};
#pragma unroll
        for (int blk = 0; blk < NB; ++blk)
#pragma unroll
            for (int e = 0; e < 16; ++e) m4[e & 3] = RCP ? fminf(m4[e & 3], s[blk][e]) : fmaxf(m4[e & 3], s[blk][e]);
        float mx = RCP ? fminf(fminf(m4[0], m4[1]), fminf(m4[2], m4[3])) : fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        mx = pair_max(__builtin_fmaf(mx, ua, ub));
        const float m_new = fmaxf(m_run, mx);
        if (__ballot(m_new > m_run + 8.0f) != 0ull) {
            const float alpha = fast_exp2(m_run - m_new);
            l_run *= alpha;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
            m_run = m_new;
        }
    };
    constexpr int NPK = C::F32 ? 1 : BN / 16;
    auto softmax = [&](f32x16 (&s)[NB], s16x8 (&pk)[NPK]) FA_INLINE {
        const float um = ub - m_run;
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int blk = 0; blk < NB; ++blk)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[blk][e] = fast_exp2(VALUE ? s[blk][e] + um : __builtin_fmaf(s[blk][e], ua, um));
                ps[e & 3] += s[blk][e];
            }
        l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        asm volatile("" : "+v"(l_run));  // summed here, beside the products
        if constexpr (!C::F32) {
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks) {
                float tmp[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) tmp[e] = s[ks >> 1][8 * (ks & 1) + e];
                pk[ks] = pack8<T>(tmp);
            }
        }
    };
    // ---- O^T += V^T P^T ----
    auto pv = [&](const T* Vs, const f32x16 (&s)[NB], const s16x8 (&pk)[NPK]) FA_INLINE {
        if constexpr (C::F32) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                if (32 * i >= live_cols<D>(p)) break;
#pragma unroll
                for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                    for (int t = 0; t < 16; ++t)
                        o[i] = mfma_f32(Vs[(32 * blk + 8 * (t >> 2) + 4 * hi + (t & 3)) * VW + l32 + 32 * i], s[blk][t], o[i]);
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const T* vp = Vs + (16 * ks + 4 * hi + ((lane & 15) >> 2)) * VW + 32 * i + 16 * ((lane >> 4) & 1) +
                                  4 * (lane & 3);
                    const s16x8 a = cat4(lds_read_tr16(vp), lds_read_tr16(vp + 8 * VW));
                    o[i] = Elem<T>::mfma(a, pk[ks], o[i]);
                }
        }
    };
    auto sync_tiles = [&]() FA_INLINE {
        wait_vmem();
        lds_barrier();
    };

    // Software pipeline: the products S(j + 1) run beside the probabilities of tile
    // j, then P(j) V(j) beside the rules of tile j + 1 (a matrix product takes the
    // matrix unit for 32 cycles and the wave for few of them; two waves on a SIMD
    // fall into step and overlap nothing by themselves).  K is copied two tiles
    // ahead and V one: both slots were last read before the barrier that opens the
    // iteration.  Every wave computes every tile of the workgroup, seen or not
    // (P = 0): the loop has no branch but the masks'.
    auto sched = [&](auto n_tag, auto reads_tag, auto valu_tag) FA_INLINE {
        constexpr int N = decltype(n_tag)::value, RD = decltype(reads_tag)::value, VA = decltype(valu_tag)::value;
        if constexpr (!C::F32) {
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * RD, 0);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, VA, 0);
                if (n + 2 < N) __builtin_amdgcn_sched_group_barrier(0x100, RD, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    template_int<NB * QR> n_qk;
    template_int<(BN / 16) * (D / 32)> n_pv;
    template_int<1> one_read;
    template_int<2> two_reads;
    // vector instructions beside a product
    template_int<(32 * 9 / 2 + NB * QR - 1) / (NB * QR)> va_b;
    template_int<(32 * (RCP ? 4 : VALUE ? (CAP ? 7 : 3) : 1) + NB * QR - 1) / (NB * QR)> va_a;
    f32x16 sa[NB], sb[NB];
    s16x8 pk[NPK];
    auto iter = [&](int slot, TileRef& cur, TileRef& nxt, const TileRef& nn, f32x16 (&sc)[NB], f32x16 (&sn)[NB]) FA_INLINE {
        sync_tiles();
        load_k(nn, slot);
        load_ids(nn, slot);
        load_v(nxt, slot ^ 1);
        T* const Vs = Vs0 + slot * C::VTILE;
        if (cur.fl & kNeg) {  // the groups together
            // (the ids of tile j are overwritten by those of tile j + 2: read its rows' ones from memory)
            if (cur.t >= 0) clear_rows<T, BN, D, VW, 256>(Vs, kdoc + cur.t * BN, tid & 255);
            lds_barrier();
        }
        if constexpr (!C::F32) __builtin_amdgcn_sched_barrier(0);
        qk(Ks0 + (slot ^ 1) * C::KTILE, sn);
        softmax(sc, pk);
        sched(n_qk, one_read, va_b);
        pv(Vs, sc, pk);
        rules(sn, nxt.t * BN);
        // (pinned here: their use below is conditional, and they would move there)
        if constexpr (RCP || VALUE) {
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) asm volatile("" : "+v"(sn[blk]));
        }
        sched(n_pv, two_reads, va_a);
        if (nxt.t >= 0) {
            mask_max(sn, nxt, ids[sp][slot ^ 1] + nxt.t % TPD * BN);
        } else {  // no tile for this group: P = 0 beside the other's
            stay_branch();
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                for (int e = 0; e < 16; ++e) sn[blk][e] = kHidden;
        }
        cur = nxt;
        nxt = nn;
    };
    for (int base = 0; base < n_kt; base += 64) {
        TileChunk ch = chunk_at(base);
        TileRef cur = next(ch, base);
        if (!(cur.fl & kMore)) continue;
        TileRef nxt = next(ch, base);
        // the last iteration of the chunk before read V slot 0 or 1; all slots are
        // free behind this barrier
        lds_barrier();
        load_k(cur, 0);
        load_ids(cur, 0);
        load_v(cur, 0);
        load_k(nxt, 1);
        load_ids(nxt, 1);
        sync_tiles();
        qk(Ks0, sa);
        rules(sa, cur.t * BN);
        if (cur.t >= 0) {
            mask_max(sa, cur, ids[sp][0] + cur.t % TPD * BN);
        } else {
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                for (int e = 0; e < 16; ++e) sa[blk][e] = kHidden;
        }
        while (cur.fl & kMore) {
            iter(0, cur, nxt, next(ch, base), sa, sb);
            if (!(cur.fl & kMore)) break;
            iter(1, cur, nxt, next(ch, base), sb, sa);
        }
        wait_vmem();  // copies of no tile, still counted
    }
    sync_tiles();  // all waves done with the tiles, no copy in flight

    if constexpr (KS == 2) {
        // ---- the second group's part joins the first's (rescaled to the common maximum) ----
        constexpr int NO = (D / 32) * 16, NF = NO + 2;
        static_assert(4 * NF * 64 * 4 <= C::SMEM_ELEMS * (int)sizeof(T), "a group's part fits its tile buffers");
        float* mg = reinterpret_cast<float*>(smem + C::SMEM_ELEMS);
        auto at = [&](int f) FA_INLINE { return mg + (w * NF + f) * 64 + lane; };
        if (sp > 0) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) *at(16 * i + e) = o[i][e];
            *at(NO) = m_run;
            *at(NO + 1) = l_run;
        }
        lds_barrier();
        if (sp == 0) {
            const float m1 = *at(NO), mm = fmaxf(m_run, m1);
            const float a0 = fast_exp2(m_run - mm), a1 = fast_exp2(m1 - mm);
            l_run = __builtin_fmaf(*at(NO + 1), a1, l_run * a0);
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[i][e] = __builtin_fmaf(*at(16 * i + e), a1, o[i][e] * a0);
            m_run = mm;
        }
    }

    // ---- epilogue: normalise, LSE, O^T through LDS as rows ----
    const ScoredParams& pe = late_args();
    const float l_tot = pair_sum(l_run);
    const float inv = l_tot > 0.f || l_tot != l_tot ? 1.f / l_tot : 0.f;
    if (pe.lse && sp == 0 && hi == 0 && qi < p.Sq) {
        const int64_t at = (int64_t)(b * pe.H + h) * pe.Sq + qi;
        const float lse = l_tot > 0.f ? (m_run + __log2f(l_tot)) * kLn2 : l_tot == 0.f ? -INFINITY : l_tot;
        if (SLOPE && pe.lse_near) pe.lse_near[at] = lse;
        pe.lse[at] = has_slope<CAP, SLOPE>(pe) ? __builtin_fmaf(-pe.slopes[b * pe.slopes_sb + h], rule.far(qi), lse) : lse;
    }
    store_rows<T, D>(smem + w * 32 * C::OW, C::OW, o, inv, (T*)pe.o + b * pe.o_sb + h * pe.o_sh, pe.o_ss,
                     qw0, pe.Sq, pe.cols, lane, sp == 0);
}

// ---------------------------------------------------------------------------
// dQ, and per query the rows LSE * log2 e and delta = rowsum(dO O) that the
// dK/dV pass reads after it.  Cap: both passes hold 4 P (the exponent is 2 larger), as
// the derivative comes divided by 4: dS through it is then what it is, and fp16 rounds
// neither it nor P sooner as a subnormal number.
// SLOPE: P is e^(s - LSE) with the LSE over distances from the nearest key: lse_near,
// or lse less what it holds for them.
// DSLOPE: also -d loss / d slope of each row,
//   sum_j |d| P (dP - delta) = sum |d| dS - sum |d| P sum dS,  dS = P (dP - delta'),
// over P and dS that are divided by sum P: with delta' from the rounded output, what
// is subtracted is small, and delta itself is as good as the sums (the sum over all
// rows is returned in float32, whose digits the rounding would cost).
template <typename T, int D, int CAP, bool SLOPE, bool DSLOPE, int KS>
__global__ __launch_bounds__(256 * KS, (KS == 1 ? DqCfg<T, D>::MIN_BLOCKS : 1)) void scored_dq_kernel(const ScoredParams p) {
    using C = DqCfg<T, D>;
    constexpr int BN = C::BN, KW = C::KW;
    static_assert(BN == 64, "one range of document ids a tile");
    __shared__ __attribute__((aligned(16))) char smem[C::SMEM_BYTES * KS];
    __shared__ __attribute__((aligned(16))) int ids[KS][2][64];  // document ids of the tiles

    const int tid = threadIdx.x;
    const int lane = tid & 63, wg = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, hi = lane >> 5;
    const int w = wg & 3, sp = KS == 1 ? 0 : wg >> 2;  // (& 3: its range decides copies at compile time)
    const BlockOrder ord = block_order<32 * (KS == 1 ? C::MIN_BLOCKS : 1)>(p, p.H);
    const int qt = p.n_tiles - 1 - ord.rank;
    const int h = ord.head, b = ord.b;
    const int hk = h / p.group;
    const int q0 = qt * C::BM, qw0 = q0 + 32 * w, qi = qw0 + l32;
    const SeqRule rule(p, b);

    constexpr int QR = C::F32 ? D / 8 : D / 16;
    uint4 qreg[QR], doreg[QR];
    float del = 0.f;
    {
        const T* qrow = (const T*)p.q + b * p.q_sb + (int64_t)qi * p.q_ss + h * p.q_sh;
        const T* drow = (const T*)p.dout + b * p.do_sb + (int64_t)qi * p.do_ss + h * p.do_sh;
        const T* orow = (const T*)p.o + b * p.o_sb + (int64_t)qi * p.o_ss + h * p.o_sh;
#pragma unroll
        for (int i = 0; i < QR; ++i) {
            const int d0 = C::F32 ? 8 * i + 4 * hi : 16 * i + 8 * hi;
            const bool ok = qi < p.Sq && d0 < p.cols;
            qreg[i] = ok ? *reinterpret_cast<const uint4*>(qrow + d0) : make_uint4(0u, 0u, 0u, 0u);
            doreg[i] = ok ? *reinterpret_cast<const uint4*>(drow + d0) : make_uint4(0u, 0u, 0u, 0u);
            const uint4 ov = ok ? *reinterpret_cast<const uint4*>(orow + d0) : make_uint4(0u, 0u, 0u, 0u);
            float part = 0.f;
            if constexpr (C::F32) {
                const f32x4 x = __builtin_bit_cast(f32x4, ov), y = __builtin_bit_cast(f32x4, doreg[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) part = __builtin_fmaf(x[e], y[e], part);
            } else {
                const s16x8 x = __builtin_bit_cast(s16x8, ov), y = __builtin_bit_cast(s16x8, doreg[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) part = __builtin_fmaf(Elem<T>::unpack1(x[e]), Elem<T>::unpack1(y[e]), part);
            }
            del += part;
        }
        del = pair_sum(del);
    }
    const float* const lse_rows = SLOPE && p.lse_near ? p.lse_near : p.lse;
    float lse_in = qi < p.Sq ? lse_rows[(int64_t)(b * p.H + h) * p.Sq + qi] : -INFINITY;
    const float slope2 = has_slope<CAP, SLOPE>(p) ? p.slopes[b * p.slopes_sb + h] * kLog2e : 0.f;
    // of distances from the nearest key; a row that sees nothing, and rows past the
    // last: P = exp2(s - inf) = 0
    if (has_slope<CAP, SLOPE>(p) && !p.lse_near)
        lse_in = __builtin_fmaf(p.slopes[b * p.slopes_sb + h], rule.far(qi), lse_in);
    const float lse2 = (lse_in == -INFINITY ? INFINITY : lse_in * kLog2e) - (CAP ? 2.f : 0.f);
    if (sp == 0 && hi == 0) {
        const int64_t wi = ((int64_t)b * p.H + h) * p.ws_stride + qi;  // qi < sq_pad
        p.lse2[wi] = lse2;
        p.lse2[wi + p.sq_pad] = qi < p.Sq ? del : 0.f;
    }

    const int lim_hi = rule.lim(min(q0 + C::BM, p.Sq) - 1);
    const int n_kt = (max(lim_hi, 0) + BN - 1) / BN;
    const int wlim_lo = rule.lim(qw0), wlim_hi = qw0 < p.Sq ? rule.lim(min(qw0 + 31, p.Sq - 1)) : 0;
    const int lim_l = rule.lim(qi);
    const bool docs = p.q_docs != nullptr;
    const int* kdoc = p.k_docs + (docs ? (int64_t)b * p.k_docs_pad : 0);
    const int2* krng = p.k_rng + (docs ? (int64_t)b * (p.k_docs_pad / 64) : 0);
    int2 qr = {0, 0}, wr = {0, 0};
    int qd = -2;
    if (docs) {
        const int2* qrng = p.q_rng + (int64_t)b * (p.q_docs_pad / 64) + q0 / 64;
        const int2 a = uniform2(qrng[0]), c = q0 + 64 < p.q_docs_pad ? uniform2(qrng[1]) : a;
        qr = docs_join(a, c);
        wr = w < 2 ? a : c;
        const int id = qi < p.Sq ? p.q_docs[(int64_t)b * p.q_docs_pad + qi] : -1;
        if (id >= 0) qd = id;
    }
    // key tiles [base, base + 64)
    auto chunk_at = [&](int base) FA_INLINE -> TileChunk {
        const int t = base + lane, k0 = t * BN;
        bool v = t < n_kt, a = v && k0 < wlim_hi;
        TileChunk c;
        c.lim = __ballot(k0 + BN <= wlim_lo);
        c.doc = ~0ull;
        c.neg = 0;
        if (docs) {
            const int2 r = v ? krng[t] : make_int2(-1, -1);
            v = v && docs_meet(r, qr);
            a = a && v && docs_meet(r, wr);
            c.doc = __ballot(docs_one(r, wr));
            c.neg = __ballot(r.x < 0);
        }
        c.vis = __ballot(v);
        c.act = __ballot(a);
        return c;
    };
    // the next tile of a chunk.  KS = 2: of this group, with kMore and kNeg of the
    // groups together (they share the barriers)
    auto next = [&](TileChunk& c, int base) FA_INLINE -> TileRef {
        auto one = [&]() FA_INLINE -> TileRef {
            if (c.vis == 0) return TileRef{-1, 0u};
            const int i = (int)__builtin_ctzll(c.vis);
            c.vis &= c.vis - 1;
            return c.ref(base, i);
        };
        TileRef r = one();
        if constexpr (KS == 2) {
            const TileRef r2 = one();
            const unsigned both = (r.fl | r2.fl) & (kMore | kNeg);
            if (sp) r = r2;
            r.fl |= both;
        }
        return r;
    };

    f32x16 dq[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) dq[i] = f32x16{};
    const float c = p.scale_log2;
    Cap<(C::F32 || CAP == kCapWide)> cap(p);
    const int qpos = rule.near(qi);
    // sums of P, dS, |d| P, |d| dS (DSLOPE)
    [[maybe_unused]] float sum_p = 0.f, sum_ds = 0.f, sum_d = 0.f, sum_dds = 0.f;

    const T* kbase = (const T*)p.k + b * p.k_sb + hk * p.k_sh;
    const T* vbase = (const T*)p.v + b * p.v_sb + hk * p.v_sh;
    const bool copy_k = w < C::NW / 2;
    typename C::Rows rows;
    rows.init(copy_k ? p.k_ss : p.v_ss, lane, w % (C::NW / 2), p.cols);
    auto buf = [&](int s) FA_INLINE -> char* { return smem + sp * C::SMEM_BYTES + s * C::BUF_BYTES; };
    auto issue = [&](const TileRef& r, int s) FA_INLINE {
        const int k0 = max(r.t, 0) * BN, nv = r.t < 0 ? 0 : rule.len - k0;
        const T* src = copy_k ? kbase + (int64_t)k0 * p.k_ss : vbase + (int64_t)k0 * p.v_ss;
        // (float32: copies that the compiler tracks; with the others it runs out of
        // scalar registers for their addresses)
        if constexpr (C::F32)
            rows.load(src, copy_k ? p.k_ss : p.v_ss, nv, (T*)(buf(s) + (copy_k ? 0 : C::KALLOC)));
        else
            rows.load_untracked(src, copy_k ? p.k_ss : p.v_ss, nv, (const T*)(buf(s) + (copy_k ? 0 : C::KALLOC)));
        if (docs && w == 0 && r.t >= 0)
            dma_load4_untracked(buffer_words(kdoc + k0, 256), lds_addr(ids[sp][s]), 4 * lane);
    };
    auto sync_tiles = [&]() FA_INLINE {
        wait_vmem();
        lds_barrier();
    };
    // ---- S^T = K Q^T, dP^T = V dO^T of 32 keys ----
    auto sdp = [&](const T* Ks, const T* Vs, f32x16& s, f32x16& dp) FA_INLINE {
        s = f32x16{};
        dp = f32x16{};
        const T* krow = Ks + l32 * KW;
        const T* vrow = Vs + l32 * KW;
#pragma unroll
        for (int i = 0; i < QR; ++i) {
            if constexpr (C::F32) {
                if (i % 4 == 0 && 8 * i >= live_cols<D>(p)) break;
                const f32x4 ak = *reinterpret_cast<const f32x4*>(krow + 8 * i + 4 * hi);
                const f32x4 av = *reinterpret_cast<const f32x4*>(vrow + 8 * i + 4 * hi);
                const f32x4 bq = __builtin_bit_cast(f32x4, qreg[i]), bd = __builtin_bit_cast(f32x4, doreg[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s = mfma_f32(ak[e], bq[e], s);
                    dp = mfma_f32(av[e], bd[e], dp);
                }
            } else {
                const s16x8 ak = *reinterpret_cast<const s16x8*>(krow + 16 * i + 8 * hi);
                const s16x8 av = *reinterpret_cast<const s16x8*>(vrow + 16 * i + 8 * hi);
                s = Elem<T>::mfma(ak, __builtin_bit_cast(s16x8, qreg[i]), s);
                dp = Elem<T>::mfma(av, __builtin_bit_cast(s16x8, doreg[i]), dp);
            }
        }
    };
    // ---- 16 keys (half ks of the 32): dX^T = P^T (dP^T - delta) cap', then
    // dQ^T += K^T dX^T ----
    auto half = [&](int k0, const T* Ks, const int* id, int ks, const f32x16& s, const f32x16& dp, unsigned fl) FA_INLINE {
        const int ka = k0 + 16 * ks + 4 * hi;  // of element 0; element e is key ka + 8 (e / 4) + e % 4
        const float d0 = (float)(qpos - ka);
        float ds[8];
        [[maybe_unused]] float pe[8];  // P
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int r = 8 * ks + e;
            const float ad = __builtin_fabsf(d0 - (float)(8 * (e >> 2) + (e & 3)));
            float pv;
            if constexpr (CAP) {
                float t = cap.value(s[r]) - lse2;
                if (SLOPE) t = __builtin_fmaf(-slope2, ad, t);
                pv = fast_exp2(t);
            } else {
                pv = fast_exp2(__builtin_fmaf(s[r], c, SLOPE ? __builtin_fmaf(-slope2, ad, -lse2) : -lse2));
            }
            pe[e] = pv;
            ds[e] = pv * (dp[r] - del);
            if (CAP) ds[e] *= cap.slope();
        }
        if (!(fl & kLim)) {
            stay_branch();
            const int lim = lim_l - ka;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (8 * (e >> 2) + (e & 3) >= lim) pe[e] = ds[e] = 0.f;
        }
        if (!(fl & kDoc)) {
            stay_branch();
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int4 kd = *reinterpret_cast<const int4*>(id + 16 * ks + 8 * g + 4 * hi);
                if (kd.x != qd) pe[4 * g] = ds[4 * g] = 0.f;
                if (kd.y != qd) pe[4 * g + 1] = ds[4 * g + 1] = 0.f;
                if (kd.z != qd) pe[4 * g + 2] = ds[4 * g + 2] = 0.f;
                if (kd.w != qd) pe[4 * g + 3] = ds[4 * g + 3] = 0.f;
            }
        }
        if constexpr (DSLOPE) {
            float xp[2] = {0.f, 0.f}, x0[2] = {0.f, 0.f}, x1[2] = {0.f, 0.f}, x2[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float ad = __builtin_fabsf(d0 - (float)(8 * (e >> 2) + (e & 3)));
                // dS before the cap's derivative (a masked dP may be anything)
                const float dsn = CAP ? (pe[e] == 0.f ? 0.f : pe[e] * (dp[8 * ks + e] - del)) : ds[e];
                xp[e & 1] += pe[e];
                x0[e & 1] += dsn;
                x1[e & 1] = __builtin_fmaf(pe[e], ad, x1[e & 1]);
                x2[e & 1] = __builtin_fmaf(dsn, ad, x2[e & 1]);
            }
            sum_p += xp[0] + xp[1];
            sum_ds += x0[0] + x0[1];
            sum_d += x1[0] + x1[1];
            sum_dds += x2[0] + x2[1];
            // summed here: moved on, P and dP stay in registers until then, and spill
            // (2 x 4096 x 32 heads of 128: backward with the slopes' gradient 1683 -> 1141 us)
            asm volatile("" : "+v"(sum_p), "+v"(sum_ds), "+v"(sum_d), "+v"(sum_dds));
        }
        if constexpr (C::F32) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                if (32 * i >= live_cols<D>(p)) break;
#pragma unroll
                for (int t = 0; t < 8; ++t)
                    dq[i] = mfma_f32(Ks[(16 * ks + 8 * (t >> 2) + 4 * hi + (t & 3)) * KW + l32 + 32 * i], ds[t], dq[i]);
            }
        } else {
            const int trow = 4 * hi + ((lane & 15) >> 2);
            const int tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            const s16x8 bs8 = pack8<T>(ds);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const T* kp = Ks + (16 * ks + trow) * KW + 32 * i + tcol;
                const s16x8 a = cat4(lds_read_tr16(kp), lds_read_tr16(kp + 8 * KW));
                dq[i] = Elem<T>::mfma(a, bs8, dq[i]);
            }
        }
    };

    // two buffers in turn: tile j is read while tile j + 1 lands in the other,
    // last read before the barrier that opens the iteration
    int bc = 0;
    for (int base = 0; base < n_kt; base += 64) {
        TileChunk ch = chunk_at(base);
        TileRef cur = next(ch, base);
        if (!(cur.fl & kMore)) continue;
        issue(cur, bc);
        while (cur.fl & kMore) {
            sync_tiles();
            const TileRef nxt = next(ch, base);
            issue(nxt, bc ^ 1);
            T* const Ks = (T*)buf(bc);
            const T* const Vs = (const T*)(buf(bc) + C::KALLOC);
            const int* const id = ids[sp][bc];
            if (cur.fl & kNeg) {
                if (cur.t >= 0) clear_rows<T, BN, D, KW, 256>(Ks, id, tid & 255);
                lds_barrier();
            }
            if (cur.fl & kAct) {
                const int k0 = cur.t * BN;
                f32x16 s0, dp0, s1, dp1;
                sdp(Ks, Vs, s0, dp0);
                sdp(Ks + 32 * KW, Vs + 32 * KW, s1, dp1);
                half(k0, Ks, id, 0, s0, dp0, cur.fl);
                half(k0, Ks, id, 1, s0, dp0, cur.fl);
                half(k0 + 32, Ks + 32 * KW, id + 32, 0, s1, dp1, cur.fl);
                half(k0 + 32, Ks + 32 * KW, id + 32, 1, s1, dp1, cur.fl);
            }
            bc ^= 1;
            cur = nxt;
        }
    }
    sync_tiles();
    if constexpr (DSLOPE) {
        sum_p = pair_sum(sum_p);
        sum_ds = pair_sum(sum_ds);
        sum_d = pair_sum(sum_d);
        sum_dds = pair_sum(sum_dds);
    }
    if constexpr (KS == 2) {
        constexpr int NO = (D / 32) * 16, NF = NO + (DSLOPE ? 4 : 0);
        static_assert(4 * NF * 64 * 4 <= C::SMEM_BYTES, "a group's part fits its tile buffers");
        float* mg = reinterpret_cast<float*>(smem + C::SMEM_BYTES);
        auto at = [&](int f) FA_INLINE { return mg + (w * NF + f) * 64 + lane; };
        if (sp > 0) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) *at(16 * i + e) = dq[i][e];
            if (DSLOPE) {
                *at(NO) = sum_p;
                *at(NO + 1) = sum_ds;
                *at(NO + 2) = sum_d;
                *at(NO + 3) = sum_dds;
            }
        }
        lds_barrier();
        if (sp == 0) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) dq[i][e] += *at(16 * i + e);
            if (DSLOPE) {
                sum_p += *at(NO);
                sum_ds += *at(NO + 1);
                sum_d += *at(NO + 2);
                sum_dds += *at(NO + 3);
            }
        }
    }
    const ScoredParams& pe = late_args();
    if constexpr (DSLOPE) {
        // (sums of 4 P and 4 dS under a cap: their quotients are the same)
        const float inv = sum_p == 0.f ? 0.f : 1.f / sum_p;  // a row that sees nothing
        if (sp == 0 && hi == 0 && qi < pe.Sq)
            pe.dslope_rows[((int64_t)b * pe.H + h) * pe.Sq + qi] = __builtin_fmaf(sum_ds * inv, sum_d, -sum_dds) * inv;
    }
    store_rows<T, D>((T*)smem + w * 32 * C::OW, C::OW, dq, pe.scale,
                     (T*)pe.dq + b * pe.dq_sb + h * pe.dq_sh, pe.dq_ss, qw0, pe.Sq, pe.cols, lane, sp == 0);
}

// ---------------------------------------------------------------------------
// dK and dV of 128 keys of one (batch, KV head): the query heads of the group one
// after the other, each over the query tiles that the keys are seen by (or this
// part's of them), the last first (so that the workgroups of a head read the same
// tiles at about the same time).  K and V rows in registers, as in
// dkdv_kernel.
// 16-bit inputs at D = 128: K, V and the sums take 192 of the 256 registers a
// lane has (two workgroups a CU); with 64-query tiles in two slots, the LDS left
// nothing to put beside them, 60 registers spilled, and each reload waited for
// the tile copies in flight.  There the tiles are of 32 queries in three slots,
// copied two ahead, and 5 of 8 row chunks of K stay in LDS (backward of 2 x 4096 x
// 32 heads, cap: 1188 -> 1140 us; packed documents 374 -> 339 us).
template <typename T, int D>
struct ScoredDkdvCfg {
    static constexpr bool F32 = Elem<T>::kF32, SMALL = !F32 && D == 128;
    static constexpr int NW = 4, BK = 32 * NW;
    static constexpr int NSUB = SMALL ? 1 : 2, BQ = 32 * NSUB, NSLOT = SMALL ? 3 : 2;
    static constexpr int RW = DkdvCfg<T, D>::RW;
    using Rows = DmaRowGroups<T, BQ, D, RW, NW / 2>;
    static constexpr int QALLOC = BQ * RW * (int)sizeof(T);
    static constexpr int SLOT_BYTES = 2 * QALLOC + 2 * BQ * 4;  // Q rows, dO rows, LSE * log2 e, delta
    // K chunks in LDS: of each wave's 32 rows, 64 lanes x 16 bytes each
    static constexpr int KST = SMALL ? 5 : 0, KST_BYTES = KST * NW * 1024;
    static constexpr int OW = D + (F32 ? 4 : 8);
    static constexpr int RAW = NSLOT * SLOT_BYTES + KST_BYTES, STAGE = NW * 32 * OW * (int)sizeof(T);
    static constexpr int SMEM_BYTES = RAW > STAGE ? RAW : STAGE;
    // copies that each wave has issued for a tile, at least: rows, LSE and delta
    static constexpr int MIN_COPIES = Rows::NI / (NW / 2) + (SMALL ? 1 : 2);
    static_assert(SLOT_BYTES % 16 == 0, "16-byte aligned slots");
};

// FAR: queries may stand off the keys, whose distances start at the nearest one (one
// clamp a score, which in every call would cost 2 x 4096, 32 on 8 heads of 128, bf16,
// slopes: 1410 -> 1463 us a step).
template <typename T, int D, int CAP, bool SLOPE, bool FAR>
__global__ __launch_bounds__(256, (!(Elem<T>::kF32 && D == 128) ? 2 : 1)) void scored_dkdv_kernel(const ScoredParams p) {
    using C = ScoredDkdvCfg<T, D>;
    constexpr int BQ = C::BQ, RW = C::RW, NSLOT = C::NSLOT;
    constexpr int TPD = 64 / BQ;  // tiles per range of document ids
    __shared__ __attribute__((aligned(16))) char smem[C::SMEM_BYTES];
    __shared__ __attribute__((aligned(16))) int ids[NSLOT][64];  // document ids of the tiles
    // each key's first query and document id: needed by partly seen tiles only,
    // and registers are short
    __shared__ int key_first[C::BK], key_doc[C::BK];

    const int tid = threadIdx.x;
    const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6) & 3, l32 = lane & 31, hi = lane >> 5;
    const BlockOrder ord = block_order<32 * (!(Elem<T>::kF32 && D == 128) ? 2 : 1)>(p, p.Hkv * p.kv_parts);
    const int kt = ord.rank;  // the first keys are seen by the most queries
    const int part = ord.head % p.kv_parts, hk = ord.head / p.kv_parts, b = ord.b;
    // of 64 query tiles, this part's: every kv_parts-th (1, 2, 4 or 8)
    const uint64_t own = (p.kv_parts == 1 ? ~0ull : p.kv_parts == 2 ? 0x5555555555555555ull
                          : p.kv_parts == 4 ? 0x1111111111111111ull : 0x0101010101010101ull) << part;
    const int k0 = kt * C::BK, kw0 = k0 + 32 * w, kj = kw0 + l32;
    const SeqRule rule(p, b);

    constexpr int KR = C::F32 ? D / 8 : D / 16, KREG = KR - C::KST;
    uint4 kreg[KREG], vreg[KR];
    // this lane's K chunks KREG .. KR - 1
    char* const kst = smem + NSLOT * C::SLOT_BYTES + w * C::KST * 1024 + lane * 16;
    {
        const T* krow = (const T*)p.k + b * p.k_sb + (int64_t)kj * p.k_ss + hk * p.k_sh;
        const T* vrow = (const T*)p.v + b * p.v_sb + (int64_t)kj * p.v_ss + hk * p.v_sh;
#pragma unroll
        for (int i = 0; i < KR; ++i) {
            const int d0 = C::F32 ? 8 * i + 4 * hi : 16 * i + 8 * hi;
            const bool ok = kj < rule.len && d0 < p.cols;
            const uint4 x = ok ? *reinterpret_cast<const uint4*>(krow + d0) : make_uint4(0u, 0u, 0u, 0u);
            if (i < KREG)
                kreg[i < KREG ? i : 0] = x;
            else
                *reinterpret_cast<uint4*>(kst + (i - KREG) * 1024) = x;  // read by this lane only
            vreg[i] = ok ? *reinterpret_cast<const uint4*>(vrow + d0) : make_uint4(0u, 0u, 0u, 0u);
        }
        // the dP products start from delta and take -V: they give delta - dP, and
        // the products below sum -dX into dK, whose final scale is negative
#pragma unroll
        for (int i = 0; i < KR; ++i) vreg[i] = C::F32 ? neg32x4(vreg[i]) : neg16x8(vreg[i]);
    }

    // ---- the query tiles that the keys are seen by ----
    const int first0 = rule.first(k0);                 // of the block's keys: none of them sooner
    const int wfirst_lo = rule.first(kw0), wfirst_hi = rule.first(kw0 + 31);
    key_first[32 * w + l32] = rule.first(kj);
    const int n_qt = (p.Sq + BQ - 1) / BQ;
    const int t_lo = first0 == INT_MAX ? n_qt : min(n_qt, first0 / BQ);  // tiles [t_lo, n_qt)
    const bool docs = p.q_docs != nullptr;
    const int* qdoc = p.q_docs + (docs ? (int64_t)b * p.q_docs_pad : 0);
    const int2* qrng = p.q_rng + (docs ? (int64_t)b * (p.q_docs_pad / 64) : 0);
    int2 kr = {0, 0}, wr = {0, 0};
    int kd = -2;  // no query's id
    if (docs) {
        const int2* krng = p.k_rng + (int64_t)b * (p.k_docs_pad / 64) + k0 / 64;
        const int2 a = uniform2(krng[0]), c = k0 + 64 < p.k_docs_pad ? uniform2(krng[1]) : a;
        kr = docs_join(a, c);
        wr = w < 2 ? a : c;
        const int id = kj < p.Sk ? p.k_docs[(int64_t)b * p.k_docs_pad + kj] : -1;
        if (id >= 0) kd = id;
    }
    key_doc[32 * w + l32] = kd;
    // query tiles [base, base + 64)
    auto chunk_at = [&](int base) FA_INLINE -> TileChunk {
        const int t = base + lane, qa = t * BQ, qz = min(qa + BQ, p.Sq) - 1;  // first and last query
        bool v = t >= t_lo && t < n_qt, a = v && qz >= wfirst_lo;
        TileChunk c;
        c.lim = __ballot(qa >= wfirst_hi);
        c.doc = ~0ull;
        c.neg = 0;
        if (docs) {
            const int2 r = v ? qrng[t / TPD] : make_int2(-1, -1);
            v = v && docs_meet(r, kr);
            a = a && v && docs_meet(r, wr);
            c.doc = __ballot(docs_one(r, wr));
            c.neg = __ballot(r.x < 0);
        }
        c.vis = __ballot(v) & own;
        c.act = __ballot(a);
        return c;
    };

    f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        dk[i] = f32x16{};
        dv[i] = f32x16{};
    }
    const float c = p.scale_log2;
    Cap<(C::F32 || CAP == kCapWide)> cap(p);

    const bool copy_q = w < C::NW / 2;
    typename C::Rows rows;
    rows.init(copy_q ? p.q_ss : p.do_ss, lane, w & 1, p.cols);
    auto buf = [&](int s) FA_INLINE -> char* { return smem + s * C::SLOT_BYTES; };
    // a tile of no queries (t < 0) is copied too: nothing is read, but the counts stay exact
    auto issue = [&](const TileRef& r, int hh, int s) FA_INLINE {
        const int qb0 = max(r.t, 0) * BQ, nv = r.t < 0 ? 0 : p.Sq - qb0;
        char* bp = buf(s);
        const T* src = copy_q ? (const T*)p.q + b * p.q_sb + (int64_t)qb0 * p.q_ss + hh * p.q_sh
                              : (const T*)p.dout + b * p.do_sb + (int64_t)qb0 * p.do_ss + hh * p.do_sh;
        if constexpr (C::F32)
            rows.load(src, copy_q ? p.q_ss : p.do_ss, nv, (T*)(bp + (copy_q ? 0 : C::QALLOC)));
        else
            rows.load_untracked(src, copy_q ? p.q_ss : p.do_ss, nv, (const T*)(bp + (copy_q ? 0 : C::QALLOC)));
        const float* wrow = p.lse2 + ((int64_t)b * p.H + hh) * p.ws_stride + qb0;  // qb0 + BQ <= sq_pad
        const u32x4 rs = buffer_words(wrow, r.t < 0 ? 0 : (p.ws_stride - qb0) * 4);
        const uint32_t f = lds_addr(bp + 2 * C::QALLOC);
        if constexpr (BQ == 32) {  // one instruction: 32 of each
            dma_load4_untracked(rs, f, 4 * (hi ? p.sq_pad + l32 : l32));
        } else {
            dma_load4_untracked(rs, f, 4 * lane);
            dma_load4_untracked(rs, f + 4 * BQ, 4 * (p.sq_pad + lane));
        }
        if (docs && w == 0 && r.t >= 0)
            dma_load4_untracked(buffer_words(qdoc + qb0 / 64 * 64, 256), lds_addr(ids[s]), 4 * lane);
    };
    // ---- S = Q K^T, delta - dP (dP = dO V^T) of 32 queries ----
    auto sdp = [&](int s, int st, f32x16& sc, f32x16& dpc) FA_INLINE {
        sc = f32x16{};
        dpc = delta16((const float*)(buf(s) + 2 * C::QALLOC) + BQ + 32 * st, hi);
        const T* qrow = (const T*)buf(s) + (32 * st + l32) * RW;
        const T* drow = (const T*)(buf(s) + C::QALLOC) + (32 * st + l32) * RW;
#pragma unroll
        for (int i = 0; i < KR; ++i) {
            if constexpr (C::F32) {
                if (i % 4 == 0 && 8 * i >= live_cols<D>(p)) break;
                const f32x4 aq = *reinterpret_cast<const f32x4*>(qrow + 8 * i + 4 * hi);
                const f32x4 ad = *reinterpret_cast<const f32x4*>(drow + 8 * i + 4 * hi);
                const f32x4 bk = __builtin_bit_cast(f32x4, kreg[i]), bv = __builtin_bit_cast(f32x4, vreg[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc = mfma_f32(aq[e], bk[e], sc);
                    dpc = mfma_f32(ad[e], bv[e], dpc);
                }
            } else {
                const s16x8 aq = *reinterpret_cast<const s16x8*>(qrow + 16 * i + 8 * hi);
                const s16x8 ad = *reinterpret_cast<const s16x8*>(drow + 16 * i + 8 * hi);
                const s16x8 bk = i < KREG ? __builtin_bit_cast(s16x8, kreg[i < KREG ? i : 0])
                                          : *reinterpret_cast<const s16x8*>(kst + (i - KREG) * 1024);
                sc = Elem<T>::mfma(aq, bk, sc);
                dpc = Elem<T>::mfma(ad, __builtin_bit_cast(s16x8, vreg[i]), dpc);
            }
        }
    };
    // ---- 16 queries (half ks of the 32): P and -dX = P (delta - dP) cap', packed ----
    constexpr int NPK = C::F32 ? 1 : 2;
    auto half = [&](int qb0, int s, int st, int ks, float slope2, f32x16& sc, f32x16& dpc, s16x8 (&bp)[NPK], s16x8 (&bs)[NPK],
                    unsigned fl) FA_INLINE {
        const float* lse2 = (const float*)(buf(s) + 2 * C::QALLOC) + 32 * st + 16 * ks + 4 * hi;
        const int qa = qb0 + 16 * ks + 4 * hi;  // of element 0; element e is query qa + 8 (e / 4) + e % 4
        const float d0 = (float)(qa + rule.off - kj);
        float pd[8], ds[8];
#pragma unroll
        for (int gg = 0; gg < 2; ++gg) {
            const f32x4 l4 = *reinterpret_cast<const f32x4*>(lse2 + 8 * gg);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 8 * ks + 4 * gg + e;
                float d = d0 + (float)(8 * gg + e);
                if constexpr (FAR)  // from the key nearest to the query
                    d = __builtin_amdgcn_fmed3f(d, (float)-kj, (float)(max(rule.len, 1) - 1 - kj));
                const float ad = __builtin_fabsf(d);
                float pv;
                if constexpr (CAP) {
                    float t = cap.value(sc[r]) - l4[e];
                    if (SLOPE) t = __builtin_fmaf(-slope2, ad, t);
                    pv = fast_exp2(t);
                } else {
                    pv = fast_exp2(__builtin_fmaf(sc[r], c, SLOPE ? __builtin_fmaf(-slope2, ad, -l4[e]) : -l4[e]));
                }
                pd[4 * gg + e] = pv;
                ds[4 * gg + e] = CAP ? pv * dpc[r] * cap.slope() : pv * dpc[r];
            }
        }
        if (!(fl & kLim)) {
            stay_branch();
            const int lim = key_first[32 * w + l32] - qa;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (8 * (e >> 2) + (e & 3) < lim) pd[e] = ds[e] = 0.f;
        }
        if (!(fl & kDoc)) {
            stay_branch();
            const int kd = key_doc[32 * w + l32];
#pragma unroll
            for (int gg = 0; gg < 2; ++gg) {
                const int4 id = *reinterpret_cast<const int4*>(ids[s] + (qb0 & 63) + 16 * ks + 8 * gg + 4 * hi);
                if (id.x != kd) pd[4 * gg] = ds[4 * gg] = 0.f;
                if (id.y != kd) pd[4 * gg + 1] = ds[4 * gg + 1] = 0.f;
                if (id.z != kd) pd[4 * gg + 2] = ds[4 * gg + 2] = 0.f;
                if (id.w != kd) pd[4 * gg + 3] = ds[4 * gg + 3] = 0.f;
            }
        }
        if constexpr (C::F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sc[8 * ks + e] = pd[e];
                dpc[8 * ks + e] = ds[e];
            }
        } else {
            bp[ks] = pack8<T>(pd);
            bs[ks] = pack8<T>(ds);
            asm volatile("" : "+v"(bp[ks]), "+v"(bs[ks]));  // packed here: the unpacked values would stay in registers
        }
    };
    // ---- dV^T += dO^T P, dK^T -= Q^T dX ----
    auto acc = [&](int s, int st, const f32x16& pd, const f32x16& ds, const s16x8 (&bp)[NPK], const s16x8 (&bs)[NPK]) FA_INLINE {
        const T* Qs = (const T*)buf(s) + 32 * st * RW;
        const T* Ds = (const T*)(buf(s) + C::QALLOC) + 32 * st * RW;
        if constexpr (C::F32) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                if (32 * i >= live_cols<D>(p)) break;
#pragma unroll
                for (int t = 0; t < 16; ++t) {
                    const int qr = 8 * (t >> 2) + 4 * hi + (t & 3);
                    dv[i] = mfma_f32(Ds[qr * RW + 32 * i + l32], pd[t], dv[i]);
                    dk[i] = mfma_f32(Qs[qr * RW + 32 * i + l32], ds[t], dk[i]);
                }
            }
        } else {
            const int trow = 4 * hi + ((lane & 15) >> 2);
            const int tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const int off = (16 * ks + trow) * RW + 32 * i + tcol;
                    const s16x8 ad = cat4(lds_read_tr16(Ds + off), lds_read_tr16(Ds + off + 8 * RW));
                    const s16x8 aq = cat4(lds_read_tr16(Qs + off), lds_read_tr16(Qs + off + 8 * RW));
                    dv[i] = Elem<T>::mfma(ad, bp[ks], dv[i]);
                    dk[i] = Elem<T>::mfma(aq, bs[ks], dk[i]);
                }
        }
    };

    // chunks of 64 query tiles from the last one, and within a chunk the heads of
    // the part, each over the chunk's tiles from the last one.  A tile is copied
    // NSLOT - 1 ahead, into the slot that was read before the barrier that opens
    // the iteration.
    int bc = 0;  // slot of the current tile
    auto slot_after = [&](int s, int n) FA_INLINE { return s + n >= NSLOT ? s + n - NSLOT : s + n; };
    for (int base = n_qt > 0 ? (n_qt - 1) / 64 * 64 : -1; base >= 0 && base + 64 > t_lo; base -= 64) {
        const TileChunk ch = chunk_at(base);
        if (ch.vis == 0) continue;
        uint64_t left = ch.vis;
        int g = 0;
        auto next = [&]() FA_INLINE -> TileRef {
            if (left == 0) {
                if (g + 1 >= p.group) return TileRef{-1, 0u};
                ++g;
                left = ch.vis;
            }
            const int i = 63 - (int)__builtin_clzll(left);
            left &= ~(1ull << i);
            return ch.ref(base, i);
        };
        TileRef cur = next();
        int cur_h = hk * p.group;
        issue(cur, cur_h, bc);
        [[maybe_unused]] TileRef nxt = {-1, 0u};
        [[maybe_unused]] int nxt_h = cur_h;
        if constexpr (NSLOT == 3) {
            nxt = next();
            nxt_h = hk * p.group + g;
            issue(nxt, nxt_h, slot_after(bc, 1));
        }
        while (cur.fl & kMore) {
            if constexpr (NSLOT == 3) {
                wait_vmem_below<C::MIN_COPIES>();  // the current tile's copies; the next one's may be in flight
                barrier_no_fence();
            } else {
                wait_vmem();
                lds_barrier();
            }
            const TileRef nn = next();
            const int nn_h = hk * p.group + g;
            issue(nn, nn_h, slot_after(bc, NSLOT - 1));
            const int q0 = cur.t * BQ;
            if (cur.fl & kNeg) {
                const int* const id = ids[bc] + (q0 & 63);
                clear_rows<T, BQ, D, RW, 256>((T*)buf(bc), id, tid);
                clear_rows<T, BQ, D, RW, 256>((T*)(buf(bc) + C::QALLOC), id, tid);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                barrier_no_fence();
            }
            if (cur.fl & kAct) {
                const float slope2 = has_slope<CAP, SLOPE>(p) ? p.slopes[b * p.slopes_sb + cur_h] * kLog2e : 0.f;
#pragma unroll
                for (int st = 0; st < C::NSUB; ++st) {
                    f32x16 sc, dpc;
                    s16x8 bp[NPK], bs[NPK];
                    if constexpr (C::SMALL) __builtin_amdgcn_sched_barrier(0);
                    sdp(bc, st, sc, dpc);
                    if constexpr (C::SMALL) __builtin_amdgcn_sched_barrier(0);
                    half(q0 + 32 * st, bc, st, 0, slope2, sc, dpc, bp, bs, cur.fl);
                    half(q0 + 32 * st, bc, st, 1, slope2, sc, dpc, bp, bs, cur.fl);
                    if constexpr (C::SMALL) __builtin_amdgcn_sched_barrier(0);
                    acc(bc, st, sc, dpc, bp, bs);
                }
            }
            bc = slot_after(bc, 1);
            if constexpr (NSLOT == 3) {
                cur = nxt;
                cur_h = nxt_h;
                nxt = nn;
                nxt_h = nn_h;
            } else {
                cur = nn;
                cur_h = nn_h;
            }
        }
        // three slots: the copies of no tile issued last go to slots that the next
        // chunk's first tiles take; they land before those (in issue order)
        if constexpr (NSLOT == 3) {
            wait_vmem();
            barrier_no_fence();
        }
    }
    wait_vmem();
    lds_barrier();
    const ScoredParams& pe = late_args();
    if (pe.kv_parts > 1) {  // float32 parts, for kv_sum_kernel
        if (kj < pe.Sk) {
            float* row = pe.kv_part + ((((int64_t)part * pe.B + b) * pe.Hkv + hk) * 2 * pe.Sk + kj) * D + 4 * hi;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    f32x4 x, y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = dk[i][4 * g + e];
                        y[e] = dv[i][4 * g + e];
                    }
                    *reinterpret_cast<f32x4*>(row + 32 * i + 8 * g) = x;
                    *reinterpret_cast<f32x4*>(row + (int64_t)pe.Sk * D + 32 * i + 8 * g) = y;
                }
        }
        return;
    }
    T* const Os = (T*)smem + w * 32 * C::OW;
    store_rows<T, D>(Os, C::OW, dk, -pe.scale, (T*)pe.dk + b * pe.dk_sb + hk * pe.dk_sh, pe.dk_ss, kw0,
                     pe.Sk, pe.cols, lane, true);
    lds_barrier();
    store_rows<T, D>(Os, C::OW, dv, CAP ? 0.25f : 1.f, (T*)pe.dv + b * pe.dv_sb + hk * pe.dv_sh, pe.dv_ss, kw0, pe.Sk, pe.cols, lane, true);
}

// dK and dV from the float32 parts of a KV head (every n-th query tile each): one
// thread 4 columns of a key, the parts in order
template <typename T, int D>
__global__ __launch_bounds__(256) void kv_sum_kernel(const ScoredParams p, const float k_mul, const float v_mul) {
    const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int col = (int)(gid % (D / 4)) * 4;
    const int64_t r = gid / (D / 4);  // ((b Hkv + hk) 2 + which) Sk + key
    if (r >= (int64_t)p.B * p.Hkv * 2 * p.Sk || col >= p.cols) return;
    const int key = (int)(r % p.Sk), which = (int)(r / p.Sk % 2);
    const int64_t bh = r / (2 * (int64_t)p.Sk);
    const int hk = (int)(bh % p.Hkv), b = (int)(bh / p.Hkv);
    const float* x = p.kv_part + r * D + col;
    const int64_t step = (int64_t)p.B * p.Hkv * 2 * p.Sk * D;
    f32x4 acc = *reinterpret_cast<const f32x4*>(x);
    for (int n = 1; n < p.kv_parts; ++n) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(x + n * step);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += y[e];
    }
    const float mul = which ? v_mul : k_mul;
    T* out = which ? (T*)p.dv + b * p.dv_sb + (int64_t)key * p.dv_ss + hk * p.dv_sh
                   : (T*)p.dk + b * p.dk_sb + (int64_t)key * p.dk_ss + hk * p.dk_sh;
    if constexpr (Elem<T>::kF32) {
        *reinterpret_cast<f32x4*>(out + col) = f32x4{acc[0] * mul, acc[1] * mul, acc[2] * mul, acc[3] * mul};
    } else {
        s16x4 v4;
#pragma unroll
        for (int e = 0; e < 4; ++e) v4[e] = Elem<T>::pack1(acc[e] * mul);
        *reinterpret_cast<s16x4*>(out + col) = v4;
    }
}

// ---------------------------------------------------------------------------
// launchers (instantiated in fa_scored_{fwd,bwd}_*.hip)
// Grids whose blocks get two groups of waves (a workgroup of 512 threads a CU), each
// on every other tile, so that the longest walk takes half: those of fewer
// workgroups than CUs, and causal ones of at most two workgroups a CU on every XCD,
// whose last blocks' walks are the time.  A group has the start and the end of a
// block to do for half of its tiles, so short walks take one; the walks over
// documents are as long as these, which the host does not know: there only long
// sequences count.  Forward / backward us, one group against two (bf16 unless said):
//   1 x 256, 16 heads of 128: 12 / 38, 13 / 40; 1 x 1024: 27 / 84, 24 / 80
//   2 x 1777, 12 heads of 64, slopes: 40 / 113, 34 / 104 (336 workgroups)
//   2 x 1500, 16 heads of 128: 41 / 139, 36 / 135 (384); 4 x 1024: 33 / 112, 37 / 118 (512)
//   1 x 4096, 16 heads of 128: 99 / 322, 87 / 304 (512)
//   1 x 1777, 36 heads of 128: 53 / 192, 69 / 210 (504, of which an XCD has 70)
//   4 x 512, 20 heads of 64 in float32: 59 / 178, 48 / 167 (320)
//   2 x 2304, 16 heads of 64: 43 / 122, 49 / 131 (576)
//   2 x 1536, 11 heads of 64, not causal: 35 / 98, 45 / 109 (264)
//   documents of 5 to 603 tokens, 2 x 2048, 16 heads of 128: 35 / 101, 42 / 108 (512)
//   up to 1596: 3 x 3718, 4 heads of 80: 58 / 151, 50 / 143 (360)
//   up to 1759: 1 x 4096, 16 heads of 128: 61 / 198, 60 / 197; 700 each: 39 / 158, 49 / 159
//   up to 3517: 1 x 8192, 8 heads of 128: 106 / 307, 93 / 290; 700 each: 39 / 150, 49 / 161
//   up to 521: 2 x 1777, 12 heads of 64 in float32: 71 / 228, 78 / 236
template <typename T>
inline bool two_groups(const ScoredParams& p, int64_t nb) {
    if (nb < 256) return p.Sk >= 512;
    const int64_t on_xcd = ((int64_t)p.B * p.H + 7) / 8 * p.n_tiles;
    return p.causal && nb <= 512 && on_xcd <= 64 && p.Sk >= (p.q_docs ? 3500 : Elem<T>::kF32 ? 500 : 1500);
}
template <typename T, int D, int CAP, bool SLOPE>
hipError_t launch_scored_fwd_t(ScoredParams p, hipStream_t s) {
    using C = FwdCfg<T, D>;
    p.n_tiles = (p.Sq + C::BM - 1) / C::BM;
    const int64_t nb = (int64_t)p.n_tiles * p.H * p.B;
    if (nb <= 0) return hipSuccess;
    if (two_groups<T>(p, nb)) {
        hipLaunchKernelGGL((scored_fwd_kernel<T, D, CAP, SLOPE, 2>), dim3((unsigned)nb), dim3(512), 0, s, p);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((scored_fwd_kernel<T, D, CAP, SLOPE, 1>), dim3((unsigned)nb), dim3(256), 0, s, p);
    return hipGetLastError();
}

template <typename T, int D, int CAP, bool SLOPE>
hipError_t launch_scored_bwd_t(ScoredParams p, hipStream_t s) {
    using CQ = DqCfg<T, D>;
    using CK = DkdvCfg<T, D>;
    p.n_tiles = (p.Sq + CQ::BM - 1) / CQ::BM;
    const int64_t nq = (int64_t)p.n_tiles * p.H * p.B;
    constexpr bool kTwo = !(CQ::F32 && D == 128);  // (whose tiles take the whole LDS)
    const int ks = kTwo && two_groups<T>(p, nq) ? 2 : 1;
    auto dq = [&](auto dslope, auto two) {
        hipLaunchKernelGGL((scored_dq_kernel<T, D, CAP, SLOPE, decltype(dslope)::value, decltype(two)::value ? 2 : 1>),
                           dim3((unsigned)nq), dim3(256 * ks), 0, s, p);
    };
    auto dq_ks = [&](auto dslope) {
        if constexpr (kTwo)
            if (ks == 2) return dq(dslope, std::true_type{});
        dq(dslope, std::false_type{});
    };
    if (nq > 0) {
        if constexpr (SLOPE) {
            if (p.dslope_rows)
                dq_ks(std::true_type{});
            else
                dq_ks(std::false_type{});
        } else {
            dq_ks(std::false_type{});
        }
    }
    p.n_tiles = (p.Sk + CK::BK - 1) / CK::BK;
    const int64_t nk = (int64_t)p.n_tiles * p.Hkv * p.B * p.kv_parts;
    // whether a query may stand off its sequence's keys
    const bool far = p.slopes && (p.lens || p.offsets || p.offset0 < 0 || (int64_t)p.offset0 + p.Sq > p.Sk);
    auto dkdv = [&](auto f) {
        hipLaunchKernelGGL((scored_dkdv_kernel<T, D, CAP, SLOPE, decltype(f)::value>), dim3((unsigned)nk), dim3(256), 0, s, p);
    };
    if (nk > 0) {
        if constexpr (SLOPE) {
            if (far)
                dkdv(std::true_type{});
            else
                dkdv(std::false_type{});
        } else {
            dkdv(std::false_type{});
        }
    }
    if (nk > 0 && p.kv_parts > 1) {
        const int64_t nt = (int64_t)p.B * p.Hkv * 2 * p.Sk * (D / 4);
        hipLaunchKernelGGL((kv_sum_kernel<T, D>), dim3((unsigned)((nt + 255) / 256)), dim3(256), 0, s, p,
                           -p.scale, CAP ? 0.25f : 1.f);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t launch_scored_fwd(const ScoredParams& p, int D, hipStream_t s) {
    const bool cap = p.cap > 0.f, slope = p.slopes != nullptr;
    [[maybe_unused]] const bool wide = p.cap > kWideCap;
#define FA_CASE(DD)                                                                                    \
    if (D == DD) {                                                                                     \
        if constexpr (!Elem<T>::kF32)                                                                  \
            if (wide) return launch_scored_fwd_t<T, DD, kCapWide, true>(p, s);                         \
        if (cap)                                                                                       \
            return slope ? launch_scored_fwd_t<T, DD, kCapQuick, true>(p, s)                           \
                         : launch_scored_fwd_t<T, DD, kCapQuick, false>(p, s);                         \
        return slope ? launch_scored_fwd_t<T, DD, kCapNone, true>(p, s)                                \
                     : launch_scored_fwd_t<T, DD, kCapNone, false>(p, s);                              \
    }
    FA_CASE(32)
    FA_CASE(64)
    FA_CASE(128)
#undef FA_CASE
    return hipErrorInvalidValue;
}
template <typename T>
hipError_t launch_scored_bwd(const ScoredParams& p, int D, hipStream_t s) {
    const bool cap = p.cap > 0.f, slope = p.slopes != nullptr;
    [[maybe_unused]] const bool wide = p.cap > kWideCap;
#define FA_CASE(DD)                                                                                    \
    if (D == DD) {                                                                                     \
        if constexpr (!Elem<T>::kF32)                                                                  \
            if (wide) return launch_scored_bwd_t<T, DD, kCapWide, true>(p, s);                         \
        if (cap)                                                                                       \
            return slope ? launch_scored_bwd_t<T, DD, kCapQuick, true>(p, s)                           \
                         : launch_scored_bwd_t<T, DD, kCapQuick, false>(p, s);                         \
        return slope ? launch_scored_bwd_t<T, DD, kCapNone, true>(p, s)                                \
                     : launch_scored_bwd_t<T, DD, kCapNone, false>(p, s);                              \
    }
    FA_CASE(32)
    FA_CASE(64)
    FA_CASE(128)
#undef FA_CASE
    return hipErrorInvalidValue;
}

}  // namespace fa
