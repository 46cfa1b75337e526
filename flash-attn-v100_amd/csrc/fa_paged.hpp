// Attention of the newest tokens of each sequence, one after another or as a tree
// of drafted ones, over a cache whose keys lie in pages; gfx950.
//
// A row is one (sequence, new token, query head); a unit is 32, 128 or 256 rows of one
// sequence and KV head.  The keys of all sequences, in steps, make one list that groups
// of workgroups (one workgroup for each unit of a sequence) share out evenly, so that
// sequences of any lengths keep the device equally busy: a workgroup walks its part of
// the list, unit after unit, and a unit that it holds only a part of leaves its rows'
// maximum, sum and unnormalised output in float32 for paged_join_kernel:
//   O = sum_x 2^(m_x - m) O_x / sum_x 2^(m_x - m) l_x,  m = max_x m_x.
// Scores, their maximum and sum and O are float32; probabilities are rounded to the inputs'
// 16-bit type where they enter a product, half a step of it each.
//
// Units of 32 rows (single tokens, small trees, float32): the four waves of a workgroup walk
// tiles of 32 keys of their own, K and V through LDS that no other wave waits for.  Bound
// by K and V: 32 tokens on 32 and 8 heads of 128 over up to 4096 keys (345 MB) take 75 us
// at 4.6 TB/s, and the same without the products 71; a bare loop that reads the same rows takes 62
// to 70, for the quarter of the addresses that one channel group serves answers later.
// Units of 128 or 256 rows (trees of many rows a KV head, chunks of prompts): the waves, on 32
// rows each, share tiles of 64 keys, which are read once for all of them.  16 trees of 64 on
// 32 and 8 heads of 128 over up to 8192 keys: 120 us back to back (140 on a device idle between
// calls), 630 TFLOP/s of the products of what is seen; the matrix units are busy for 31% of it:
// each product of 32 x 32 x 16 has 9 vector instructions beside it (exponentials at a
// quarter of their rate), and all waves go through both behind one barrier a tile, so that they
// mostly follow one another; one workgroup of two waves a SIMD (O and q take the registers of more).
//
// Keys come in blocks of 16 tokens, which never leave a page: one lookup and one
// buffer descriptor a block, whose range ends with the sequence, so that what lies
// behind it lands as zeros.  A tree's rows hide keys among the newest tokens only: each
// row's ancestors are bits, and a tile of 32 keys takes its 32 of them.
#pragma once

#include "fa_common.hpp"
#include "fa_ops_params.hpp"
#include "fa_scored.hpp"

namespace fa {

constexpr int kTreeNodes = 256;
constexpr int kTreeWords = kTreeNodes / 32;

template <typename T, int D>
struct PagedCfg {
    static constexpr bool F32 = Elem<T>::kF32;
    static constexpr int NW = 4;
    static constexpr int EPC = 16 / (int)sizeof(T);
    static constexpr int CW = D / EPC;        // 16-byte chunks of a row
    static constexpr int ROWB = CW * 16;
    static constexpr int NI16 = CW / 4;       // copies of 64 chunks in a block of 16 rows
    static constexpr int TILE = 32 * D;       // a wave's 32 keys
    static constexpr int REGION = 2 * TILE;
    static constexpr int STEP = NW * 32;      // keys of a step
    static constexpr int SMEM = NW * REGION;
    static_assert((D / 32) * 16 * 64 * 4 <= REGION * (int)sizeof(T), "a wave's O part fits its region");
    static constexpr int PER_CU = F32 && D == 128 ? 1 : 2;
};

// Rows lie in LDS without padding, the chunks of row r at places c ^ row_swizzle(r).  What
// one instruction reads then spreads over all banks: the same chunk of 16 rows (K), and 64
// bytes of each of 4 rows (V^T).
template <int CW>
__device__ FA_INLINE inline int row_swizzle(int r) {
    if constexpr (CW == 4) return (r >> 2) & 3;
    if constexpr (CW == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
    return ((r & 3) << 2) | ((r >> 2) & 3);
}

// The kernel's arguments, to be read by scalar loads where they are used: read first
// and kept, they took more scalar registers than there are (200 reads of lanes of vector
// registers in the loop over tiles).
typedef const __attribute__((address_space(4))) PagedParams PagedArgs;
__device__ FA_INLINE inline PagedArgs& paged_args() {
    uint64_t a = (uint64_t)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return *(PagedArgs*)(uintptr_t)a;
}
// scalar loads of what no kernel of the call writes
typedef const __attribute__((address_space(4))) int const_int;
__device__ FA_INLINE inline int uniform_load(const int* p, int64_t at) {
    return ((const_int*)(uintptr_t)p)[at];
}
// filled tokens of a sequence; of one that is the same for a wave
__device__ FA_INLINE inline int filled_here(PagedArgs& p, int b) {
    return p.lens ? max(0, min(p.Sk, uniform_load(p.lens, __builtin_amdgcn_readfirstlane(b)))) : p.Sk;
}
__device__ FA_INLINE inline int filled_tokens(PagedArgs& p, int b) { return p.lens ? max(0, min(p.Sk, p.lens[b])) : p.Sk; }
__device__ FA_INLINE inline void put_row_lse(PagedArgs& p, int b, int h, int i, float m, float l) {
    p.lse[((int64_t)b * p.H + h) * p.Sq + i] = l > 0.f ? (m + __log2f(l)) * kLn2 : l == 0.f ? -INFINITY : l;
}


// 16 tokens of a sequence: their page, -1 where there is none, and the first one's row
struct Block16 {
    int page, row;
};
// the lookups of one sequence
struct PageTable {
    const int* row;  // null: its tokens are all on page b
    int b, last_col, pages, blocks;
    unsigned magic;
    __device__ FA_INLINE inline PageTable(PagedArgs& p, int b_)
        : row(p.table ? p.table + b_ * p.table_sb : nullptr), b(b_), last_col(p.table_cols - 1), pages(p.pages), blocks(p.page_blocks),
          magic(p.page_magic) {}
    __device__ FA_INLINE inline Block16 block(int blk) const {
        const int col = blocks == 1 ? blk : (int)__umulhi((unsigned)blk, magic);
        int page = b;
        if (row) page = uniform_load(row, min(col, last_col));
        return {(unsigned)page < (unsigned)pages ? page : -1, 16 * (blk - col * blocks)};
    }
    // bits of a tile's keys that have a page, from block blk on
    template <int BLOCKS>
    __device__ FA_INLINE inline uint64_t have(int blk) const {
        uint64_t w = 0;
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i) w |= block(blk + i).page < 0 ? 0ull : 0xFFFFull << (16 * i);
        return w;
    }
    // Whether one of blocks [b0, b1) has no page.  Callers round b1 up to whole tiles: where
    // pages are smaller than those, a column behind the last key's that holds none counts too, and
    // the part takes the loop of hidden keys throughout, with the same results (trees of 64 over up
    // to 8192 keys: 132 us with pages of 64, 190 with pages of 16).
    __device__ FA_INLINE inline bool holes(int b0, int b1, int lane) const {
        if (!row || b0 >= b1) return false;
        bool none = false;
        for (int col = b0 / blocks + lane; col <= min((b1 - 1) / blocks, last_col); col += 64)
            none |= (unsigned)row[col] >= (unsigned)pages;
        return __ballot(none) != 0ull;
    }
};

// copies of 16-row blocks of one KV head's keys or values
template <typename T, int D>
struct PageCopy {
    using C = PagedCfg<T, D>;
    const T* base;  // the pool's, of the KV head
    int64_t sp, ss;
    int cols;
    int off[C::NI16];
    __device__ FA_INLINE inline void init(const T* b, int64_t page_stride, int64_t row_stride, int n_cols, int lane) {
        base = b;
        sp = page_stride;
        ss = row_stride;
        cols = n_cols;
#pragma unroll
        for (int x = 0; x < C::NI16; ++x) {
            const int c = 64 * x + lane, row = c / C::CW, chunk = (c % C::CW) ^ row_swizzle<C::CW>(row);
            off[x] = chunk < cols / C::EPC ? (row * (int)ss + chunk * C::EPC) * (int)sizeof(T) : kOffNowhere;
        }
    }
    // rows from nv on, and all of a block without a page, land as zeros
    __device__ FA_INLINE inline void load(Block16 k, int nv, const T* lds) const {
        const T* at = base + (int64_t)max(k.page, 0) * sp + (int64_t)k.row * ss;
        const u32x4 rs = row_buffer_words<T, D, 16>(at, ss, k.page < 0 ? 0 : nv, cols);
        const uint32_t l0 = lds_addr(lds);
#pragma unroll
        for (int x = 0; x < C::NI16; ++x) dma_load16_untracked(rs, l0 + 1024 * x, off[x]);
    }
};

// ---------------------------------------------------------------------------
// Trees.  bits[i]: the nodes that node i sees (its ancestors and itself), none for what
// is no token.  A node's bits are its parent's and its own: ceil(log2 N) rounds, each
// joining the bits of the node that a node points to and pointing on to where that one
// points (-1: the context, -2: no token).
struct TreeBits {
    unsigned bits[kTreeNodes][kTreeWords];
    int up[kTreeNodes];
};
__device__ FA_INLINE inline void tree_init(PagedArgs& p, TreeBits& t, int b, int tid) {
    const int N = p.Sq, W = (N + 31) >> 5;
    lds_barrier();  // (the last unit's rows have read theirs)
    int up = -2;
    if (tid < N) {
        up = p.parents[b * p.parents_sb + tid];
        if (up < -1 || up >= tid) up = -2;
        for (int w = 0; w < W; ++w) t.bits[tid][w] = w == (tid >> 5) ? 1u << (tid & 31) : 0u;
        t.up[tid] = up;
    }
    for (int n = 1; n < N; n *= 2) {
        lds_barrier();
        unsigned more[kTreeWords];
        int next = up;
        if (up >= 0) {
            for (int w = 0; w < kTreeWords; ++w) more[w] = w < W ? t.bits[up][w] : 0u;
            next = t.up[up];
        }
        lds_barrier();
        if (up >= 0) {
            for (int w = 0; w < kTreeWords; ++w)
                if (w < W) t.bits[tid][w] |= more[w];
            t.up[tid] = up = next;
        }
    }
    if (tid < N && up != -1)
        for (int w = 0; w < W; ++w) t.bits[tid][w] = 0u;
    lds_barrier();
}
// the 32 keys from tree position s on (it may be negative: the context) that node i sees
__device__ FA_INLINE inline unsigned tree_word(const TreeBits& t, int i, int s, int W) {
    const int w = s >> 5;
    auto word = [&](int x) FA_INLINE { return x < 0 ? ~0u : x < W ? t.bits[i][x] : 0u; };
    const uint64_t two = ((uint64_t)word(w + 1) << 32) | word(w);
    return (unsigned)(two >> (s & 31));
}

// ---------------------------------------------------------------------------
// Work.  A sequence's units (of every KV head) have the same keys, in steps: one at least,
// and p.extra more that stand for what a unit costs beside its keys.  The steps of all
// sequences, one after the other, are shared out evenly to W groups of workgroups, one
// workgroup of a group for each unit: they walk the same tokens side by side, whose
// heads lie side by side in memory (and several units of one KV head read its tiles
// through one L2).  Where no sequence is longer than a group's share, or than p.alone
// steps, there is a group for each sequence.
struct PagedWork {
    int T, W;      // steps, groups
    bool whole;    // a group for each sequence
    int st0, inc0; // of sequence `lane`: its steps, and those up to its end
    template <int STEP>
    __device__ FA_INLINE inline static int steps(PagedArgs& p, int b) {
        return b < p.B ? max(1, (filled_tokens(p, b) + STEP - 1) / STEP) + p.extra : 0;
    }
    template <int STEP>
    __device__ FA_INLINE inline static int steps_here(PagedArgs& p, int b) {
        return max(1, (filled_here(p, b) + STEP - 1) / STEP) + p.extra;
    }
    __device__ FA_INLINE inline static int scan(int x, int lane) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(x, d);
            if (lane >= d) x += y;
        }
        return x;
    }
    template <int STEP>
    __device__ FA_INLINE inline void init(PagedArgs& p, int lane) {
        if (!p.part) {  // (nothing may be shared: no lengths are needed to know it)
            whole = true;
            W = p.B;
            return;
        }
        int sum = 0, most = 0;
        if (p.lens) {
            most = st0 = steps<STEP>(p, lane);
            for (int b0 = 64; b0 < p.B; b0 += 64) {
                const int st = steps<STEP>(p, b0 + lane);
                sum += st;
                most = max(most, st);
            }
            inc0 = scan(st0, lane);
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) {
                if (p.B > 64) sum += __shfl_xor(sum, x);
                most = max(most, __shfl_xor(most, x));
            }
            sum += __builtin_amdgcn_readlane(inc0, 63);
        } else {
            most = steps<STEP>(p, 0);
            sum = most * p.B;
        }
        T = __builtin_amdgcn_readfirstlane(sum);
        W = min(p.groups, (T + p.least - 1) / p.least);
        whole = W <= 1 || __builtin_amdgcn_readfirstlane(most) - p.extra <= max(p.alone, (T + W - 1) / W);
        if (whole) W = p.B;
    }
    // the first step of group g (floor(g T / W)), and whose step x is; in 32 bits where they
    // suffice
    __device__ FA_INLINE inline int first(int g) const {
        return (int64_t)T * W < INT_MAX ? (int)((unsigned)(g * T) / (unsigned)W) : (int)((int64_t)g * T / W);
    }
    __device__ FA_INLINE inline int whose(int x) const {
        return (int64_t)T * W < INT_MAX ? (int)((unsigned)((x + 1) * W - 1) / (unsigned)T) : (int)((((int64_t)x + 1) * W - 1) / T);
    }
    // the sequence of step x, its first step and its steps
    template <int STEP>
    __device__ FA_INLINE inline void locate(PagedArgs& p, int x, int lane, int& b, int& start, int& len) const {
        if (!p.lens) {
            len = steps<STEP>(p, 0);
            b = x / len;
            start = b * len;
            return;
        }
        int before = 0;
        for (int b0 = 0;; b0 += 64) {
            const int st = b0 ? steps<STEP>(p, b0 + lane) : st0, inc = b0 ? scan(st, lane) : inc0;
            const uint64_t past = __ballot(before + inc > x);
            if (past || b0 + 64 >= p.B) {
                const int l = past ? (int)__builtin_ctzll(past) : 63;
                b = b0 + l;
                len = __builtin_amdgcn_readlane(st, l);
                start = before + __builtin_amdgcn_readlane(inc, l) - len;
                return;
            }
            before += __builtin_amdgcn_readlane(inc, 63);
        }
    }
    // for the join: the first and the last group of every sequence (the same one where it is whole)
    template <int STEP>
    __device__ FA_INLINE inline void spans(PagedArgs& p, int lane) const {
        int before = 0;
        for (int b0 = 0; b0 < p.B; b0 += 64) {
            const int b = b0 + lane, st = b0 || whole || !p.lens ? steps<STEP>(p, b) : st0;
            const int inc = scan(st, lane), start = before + inc - st;
            if (b < p.B) p.spans[b] = whole ? make_int2(0, 0) : make_int2(whose(start), whose(start + st - p.extra - 1));
            before += __builtin_amdgcn_readlane(inc, 63);
        }
    }
};
// parts: a workgroup (g) leaves at most two, of the sequence that it begins with (2 g) and
// of the one that it ends with, begun by it (2 g + 1).  Those of 32 rows lie together, in
// accumulator order (part_of), so that a store of a wave is 1 KB in a row: as rows, 64
// places of 16 bytes a store, 256 rows took 8 us.
template <int ROWS>
__device__ FA_INLINE inline int64_t part_at(int g, bool begun) { return ((int64_t)2 * g + (begun ? 1 : 0)) * ROWS; }

// four columns of a lane's row, 32 n + 8 q4 + 4 (lane / 32) and on, in the part whose first row is `row`
template <int D>
__device__ FA_INLINE inline f32x4* part_of(float* part, int64_t row, int n, int q4, int lane) {
    return reinterpret_cast<f32x4*>(part + row * D) + (4 * n + q4) * 64 + lane;
}

// one row of a unit: keys [0, lim) at most, of which it sees all below `all`
struct PagedRow {
    int i, h, lim, all;
    bool live, valid;  // exists; and sees keys
    int qpos;
    __device__ FA_INLINE inline PagedRow(PagedArgs& p, int row, int hk) {
        live = row < p.Sq * p.group;
        const int rr = live ? row : 0;
        i = rr / p.group;
        h = hk * p.group + (rr - i * p.group);
    }
    __device__ FA_INLINE inline void rule(const TreeBits* t, int words, int len, int c) {
        valid = live && c + i >= 0;
        qpos = c + i;
        lim = all = c + i + 1;
        if (t) {
            int n = 0;
            for (int w = 0; w < words; ++w) n += __popc(t->bits[i][w]);
            valid = valid && n > 0;
            qpos = c + n - 1;
            lim = len;
            all = max(c, 0);
        }
        if (!valid) lim = 0;
    }
};
// keys that some of the rows below `rows` of a unit may see
__device__ FA_INLINE inline int keys_of(PagedArgs& p, const TreeBits* t, int rows, int len, int c) {
    return t ? len : max(0, min(len, c + min(p.Sq, (rows - 1) / p.group + 1)));
}

// A lane's place in a tile, as an LDS address that the compiler does not see through: the
// places of the columns after it are that ^ a constant (a tile begins at a multiple of
// its row's bytes), one instruction each, which it would otherwise keep in registers
// from tile to tile.
typedef __attribute__((address_space(3))) const char* lds_chars;
__device__ FA_INLINE inline uint32_t lds_place(const void* tile, int bytes) {
    uint32_t a = lds_addr(tile) + bytes;
    asm volatile("" : "+v"(a));
    return a;
}
template <typename V>
__device__ FA_INLINE inline V lds_at(uint32_t a) {
    return *reinterpret_cast<__attribute__((address_space(3))) const V*>((lds_chars)(uintptr_t)a);
}
__device__ FA_INLINE inline s16x4 lds_tr16_at(uint32_t a) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)a);
}

// Order of the instructions of a block: reads of LDS ahead of the matrix instructions that
// take them, `ahead` of them at first and then EACH for one (the compiler's own order
// reads one operand, waits for it and multiplies).
template <int MFMAS, int EACH, int AHEAD>
__device__ FA_INLINE inline void reads_ahead() {
    constexpr int kMfma = 0x008, kRead = 0x100;
    __builtin_amdgcn_sched_group_barrier(kRead, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < MFMAS; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
        if (AHEAD + EACH * i < EACH * MFMAS) __builtin_amdgcn_sched_group_barrier(kRead, EACH, 0);
    }
}

// STEPS times a read of LDS and the products that take it, read AHEAD steps ahead
template <int STEPS, int AHEAD, typename V, typename R, typename M>
__device__ FA_INLINE inline void read_ahead(R&& read, M&& products) {
    V v[STEPS];
#pragma unroll
    for (int i = 0; i < (AHEAD < STEPS ? AHEAD : STEPS); ++i) v[i] = read(i);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        if (i + AHEAD < STEPS) v[i + AHEAD] = read(i + AHEAD);
        __builtin_amdgcn_sched_barrier(0);  // (else they are read where they are used)
        products(i, v[i]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Scores of one block of 32 keys (D / 16 products) beside the exponentials of another, then
// that one's values (D / 16 products, two reads each) beside the maximum of the scores
template <int D>
__device__ FA_INLINE inline void block_order() {
    constexpr int kMfma = 0x008, kRead = 0x100, kVector = 0x002, N = D / 16, AHEAD = N < 4 ? N : 4;
    __builtin_amdgcn_sched_group_barrier(kRead, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kVector, 64 / N, 0);
        if (AHEAD + i < N)
            __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
        else
            __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kVector, 2, 0);
        __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
    }
}

// the products of a wave's 32 rows with 32 keys (K tile), log2 units before
// the rules (float32, whose products bound it: only over columns that exist)
// (ORDERED: its place among other instructions is the caller's to say)
template <typename T, int D, bool ORDERED = false>
__device__ FA_INLINE inline void tile_scores(f32x16& s, const T* Ks, const uint4 (&q)[Elem<T>::kF32 ? D / 8 : D / 16], int cols,
                                            int l32, int hi) {
    using C = PagedCfg<T, D>;
    const uint32_t at = lds_place(Ks, l32 * C::ROWB + ((hi ^ row_swizzle<C::CW>(l32)) << 4));
    s = f32x16{};
    if constexpr (C::F32) {
        auto go = [&](auto steps) FA_INLINE {
            read_ahead<decltype(steps)::value, 2, f32x4>([&](int kk) FA_INLINE { return lds_at<f32x4>(at ^ (kk << 5)); },
                                                         [&](int kk, const f32x4& a) FA_INLINE {
                                                             const f32x4 b = __builtin_bit_cast(f32x4, q[kk]);
#pragma unroll
                                                             for (int e = 0; e < 4; ++e) s = mfma_f32(a[e], b[e], s);
                                                         });
        };
        if (cols > 3 * D / 4)
            go(template_int<D / 8>{});
        else
            go(template_int<3 * D / 32>{});
    } else {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
            s = Elem<T>::mfma(lds_at<s16x8>(at ^ (kk << 5)), __builtin_bit_cast(s16x8, q[kk]), s);
        if constexpr (!ORDERED) reads_ahead<D / 16, 1, D / 16 < 6 ? D / 16 : 6>();
    }
}

// O^T += V^T P^T over 32 keys
template <typename T, int D, bool ORDERED = false>
__device__ FA_INLINE inline void tile_values(const T* Vs, const f32x16& s, f32x16 (&o)[D / 32], int cols, int lane) {
    using C = PagedCfg<T, D>;
    const int l32 = lane & 31, hi = lane >> 5;
    if constexpr (C::F32) {
        // rows 8 (x / 4) + 4 hi + x % 4: their swizzles differ from that of row 4 hi by x alone
        const uint32_t at = lds_place(Vs, 4 * hi * C::ROWB + (((l32 >> 2) ^ row_swizzle<C::CW>(4 * hi)) << 4) + 4 * (l32 & 3));
        auto go = [&](auto blocks) FA_INLINE {
            constexpr int N = decltype(blocks)::value;
            struct Row {
                float v[N];
            };
            read_ahead<16, 2, Row>(
                [&](int x) FA_INLINE {
                    const int r = 8 * (x >> 2) + (x & 3);
                    Row row;
#pragma unroll
                    for (int n = 0; n < N; ++n) row.v[n] = lds_at<float>((at ^ (((8 * n) ^ row_swizzle<C::CW>(r)) << 4)) + r * C::ROWB);
                    return row;
                },
                [&](int x, const Row& row) FA_INLINE {
#pragma unroll
                    for (int n = 0; n < N; ++n) o[n] = mfma_f32(row.v[n], s[x], o[n]);
                });
        };
        if (D <= 64 || cols > 96)
            go(template_int<D / 32>{});
        else
            go(template_int<(D > 32 ? D / 32 - 1 : 1)>{});
    } else {
        const int r0 = 4 * hi + ((lane & 15) >> 2);
        const int chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        const uint32_t at = lds_place(Vs, r0 * C::ROWB + ((chunk ^ row_swizzle<C::CW>(r0)) << 4) + 8 * (lane & 1));
        s16x8 pk[2];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            float tmp[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) tmp[e] = s[8 * ks + e];
            pk[ks] = pack8<T>(tmp);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int n = 0; n < D / 32; ++n) {
                const s16x8 a = cat4(lds_tr16_at((at ^ (n << 6)) + 16 * ks * C::ROWB),
                                     lds_tr16_at((at ^ ((n << 6) ^ (row_swizzle<C::CW>(8) << 4))) + (16 * ks + 8) * C::ROWB));
                o[n] = Elem<T>::mfma(a, pk[ks], o[n]);
            }
        if constexpr (!ORDERED) reads_ahead<D / 16, 2, D / 16 < 4 ? D / 8 : 8>();
    }
}

// Whether a value of the tile is an infinity or NaN: 0 times it, for a key that a row does
// not see, would not be 0
template <typename T, int D>
__device__ FA_INLINE inline bool tile_odd(const T* Vs, int lane) {
    using C = PagedCfg<T, D>;
    // the largest magnitude, as integers: an infinity's or above
    constexpr unsigned short M = std::is_same<T, bf16>::value ? 0x7F80 : 0x7C00;
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    unsigned top = 0u;
    u16x2 top2 = {0, 0};
#pragma unroll 4
    for (int x = 0; x < 32 * C::CW / 64; ++x) {
        const uint4 v = *reinterpret_cast<const uint4*>((const char*)Vs + 16 * (64 * x + lane));
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (C::F32)
                top = max(top, w[e] & 0x7FFFFFFFu);
            else
                top2 = __builtin_elementwise_max(top2, __builtin_bit_cast(u16x2, w[e] & 0x7FFF7FFFu));
        }
    }
    return __ballot(C::F32 ? top >= 0x7F800000u : top2.x >= M || top2.y >= M) != 0ull;
}
// tile_values key by key, each to the rows that see it (bit x of seen: key x)
template <typename T, int D>
__device__ FA_INLINE inline void tile_values_seen(const T* Vs, const f32x16& s, unsigned seen, f32x16 (&o)[D / 32], int lane) {
    using C = PagedCfg<T, D>;
    const int l32 = lane & 31, hi = lane >> 5;
#pragma unroll 1
    for (int x = 0; x < 32; ++x) {
        float mine = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) mine = e == 4 * (x >> 3) + (x & 3) ? s[e] : mine;
        const float p = __shfl(mine, l32 + 8 * (x & 4));
        const bool sees = (seen >> x) & 1;
        const char* row = (const char*)Vs + x * C::ROWB;
        const int sw = row_swizzle<C::CW>(x);
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
            asm volatile("" ::: "memory");  // (the next columns' values are not read ahead: they would need registers)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                float v[4];
                if constexpr (C::F32) {
                    const f32x4 y = *reinterpret_cast<const f32x4*>(row + (((8 * n + 2 * q4 + hi) ^ sw) << 4));
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = y[e];
                } else {
                    const s16x4 y = *reinterpret_cast<const s16x4*>(row + (((4 * n + q4) ^ sw) << 4) + 8 * hi);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = Elem<T>::unpack1(y[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = __builtin_fmaf(p, v[e], o[n][4 * q4 + e]);
                    o[n][4 * q4 + e] = sees ? y : o[n][4 * q4 + e];
                }
            }
        }
    }
}

// what the rules take from the arguments, read once
template <bool EXACT>
struct TileRules {
    Cap<EXACT> cap;
    bool capped, slope;
    float mul, unit, slope2;  // scores times mul, unless unit, their factor in the exponent, is that
    int words;  // of bits of a tree
    __device__ FA_INLINE inline TileRules(PagedArgs& p, int b, int h)
        : cap(p), capped(p.cap > 0.f), slope(p.slopes != nullptr), mul(p.scale_log2), words((p.Sq + 31) >> 5) {
        unit = capped || slope ? 1.f : mul;
        slope2 = slope ? p.slopes[b * p.slopes_sb + h] * kLog2e : 0.f;
    }
};
// What a row sees of the 32 keys from k0 on, with bits for the blocks that have a page
__device__ FA_INLINE inline unsigned row_sees(const TreeBits* t, const PagedRow& r, int words, int k0, int c, unsigned have) {
    unsigned w;
    if (t) {
        w = tree_word(*t, r.i, k0 - c, words);
    } else {
        const int n = r.lim - k0;
        w = n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
    }
    return r.valid ? w & have : 0u;
}

// scores of 32 keys through the rules, hidden ones -infinity.  HIDDEN: some row may not
// see some key
template <bool EXACT, bool HIDDEN>
__device__ FA_INLINE inline void tile_rules(f32x16& s, TileRules<EXACT>& u, const PagedRow& r, const TreeBits* t, int k0, int c,
                                           unsigned& seen, unsigned have, int hi) {
    const bool steps = u.slope && HIDDEN && t;  // distances along the tree
    if (u.capped) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = u.cap.value(s[e]);
    } else if (u.slope) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= u.mul;
    }
    if (u.slope && !steps) {
        const float d0 = (float)(r.qpos - k0 - 4 * hi);
#pragma unroll
        for (int e = 0; e < 16; ++e)
            s[e] = __builtin_fmaf(-u.slope2, __builtin_fabsf(d0 - (float)(8 * (e >> 2) + (e & 3))), s[e]);
    }
    if constexpr (HIDDEN) {
        seen = row_sees(t, r, u.words, k0, c, have);
        const unsigned mine = seen >> (4 * hi);
        if (steps) {
            // the tokens from a key to the row's own are those that it sees behind the key
            const int end = k0 - c + 32;
            int above = max(-end, 0);
            for (int w = max(end, 0) >> 5; w < u.words; ++w) {
                const unsigned x = t->bits[r.i][w];
                above += __popc(w == (end >> 5) ? x & (~0u << (end & 31)) : x);
            }
            const unsigned word = tree_word(*t, r.i, k0 - c, u.words);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int x = 8 * (e >> 2) + (e & 3);
                const int d = above + __popc((word >> (x + 4 * hi)) >> 1);
                s[e] = __builtin_fmaf(-u.slope2, (float)d, s[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (!((mine >> (8 * (e >> 2) + (e & 3))) & 1)) s[e] = -INFINITY;
    }
}

// The running maximum and sum of a row over 32 more scores, which become
// probabilities: e^(s - m) with an m that is at most 8 (of log2) behind the largest, so
// that O is rescaled when a maximum grows by more
template <int D>
__device__ FA_INLINE inline void soft_max(const f32x16& s, float unit, float& m_run, float& l_run, f32x16 (&o)[D / 32]) {
    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 16; ++e) m4[e & 3] = fmaxf(m4[e & 3], s[e]);
    const float m_new = fmaxf(m_run, unit * pair_max(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]))));
    if (__ballot(m_new > m_run + 8.0f) != 0ull) {
        const float alpha = fast_exp2(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int n = 0; n < D / 32; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[n][e] *= alpha;
        m_run = m_new;
    }
}
__device__ FA_INLINE inline void soft_exp(f32x16& s, float unit, float m_run, float& l_run) {
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        s[e] = fast_exp2(__builtin_fmaf(s[e], unit, -m_run));
        ps[e & 3] += s[e];
    }
    l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
}

// A row's q, in the operand order of the products (float32: 4 of each 8 columns a lane)
template <typename T, int D>
__device__ FA_INLINE inline void load_q(PagedArgs& p, const PagedRow& row, int b, int hi, uint4 (&q)[Elem<T>::kF32 ? D / 8 : D / 16]) {
    constexpr int STEP = Elem<T>::kF32 ? 8 : 16;
    const T* at = (const T*)p.q + b * p.q_sb + (int64_t)row.i * p.q_ss + row.h * p.q_sh;
#pragma unroll
    for (int kk = 0; kk < D / STEP; ++kk) {
        const int d0 = STEP * kk + STEP / 2 * hi;
        q[kk] = row.live && d0 < p.cols ? *reinterpret_cast<const uint4*>(at + d0) : make_uint4(0u, 0u, 0u, 0u);
    }
}

// 32 rows of a unit over its steps [s0, s1): each wave walks tiles of its own.  part:
// the rows' place among the parts, below 0 where this is all of the unit.  The first
// tiles are on their way before anything else is waited for.
template <typename T, int D, bool EXACT>
__device__ FA_INLINE inline void paged_unit32(T* smem, float (*stat)[2][32], TreeBits* tree, bool new_tree, int b, int hk, int rt,
                                             int s0, int s1, int64_t part, int tid) {
    using C = PagedCfg<T, D>;
    constexpr int NW = C::NW;
    PagedArgs& p = paged_args();
    const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
    const int l32 = lane & 31, hi = lane >> 5;
    PagedRow row(p, 32 * rt + l32, hk);
    uint4 q[C::F32 ? D / 8 : D / 16];
    load_q<T, D>(p, row, b, hi, q);
    TileRules<EXACT> rules(p, b, row.h);
    const int len = filled_here(p, b), c = len - p.Sq;
    const int n_keys = keys_of(p, tree, 32 * (rt + 1), len, c);
    const int nt = (n_keys + 31) / 32, t1 = min(NW * s1, nt);

    T* Ks = smem + w * C::REGION;
    T* Vs = Ks + C::TILE;
    PageCopy<T, D> kc, vc;
    kc.init((const T*)p.k + hk * p.k_sh, p.k_sp, p.k_ss, p.cols, lane);
    vc.init((const T*)p.v + hk * p.v_sh, p.v_sp, p.v_ss, p.cols, lane);
    // the two blocks of a tile, looked up a tile before the copy that needs them; what is
    // past the end reads nothing, but is issued, so that the vmcnt counts stay exact
    const PageTable table(p, b);
    // (those behind the sequence are of some page, and their copies read nothing)
    auto blocks = [&](int t, Block16& x, Block16& y) FA_INLINE {
        x = table.block(2 * t);
        y = table.block(2 * t + 1);
    };
    auto copy = [&](const PageCopy<T, D>& pc, int t, Block16 x, Block16 y, const T* dst) FA_INLINE {
        const int nv = t < t1 ? n_keys - 32 * t : 0;
        pc.load(x, nv, dst);
        pc.load(y, nv - 16, dst + 16 * D);
    };
    int t = NW * s0 + w;
    Block16 bx, by;
    blocks(t, bx, by);
    copy(kc, t, bx, by, Ks);
    copy(vc, t, bx, by, Vs);
    blocks(t + NW, bx, by);

    if (new_tree) tree_init(p, *tree, b, tid);
    row.rule(tree, rules.words, len, c);
    const bool holes = table.holes(2 * NW * s0, 2 * t1, lane);
    int lim_max = row.lim, lim_min = row.valid ? row.all : INT_MAX;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        lim_max = max(lim_max, __shfl_xor(lim_max, x));
        lim_min = min(lim_min, __shfl_xor(lim_min, x));
    }
    lim_min = __builtin_amdgcn_readfirstlane(lim_min);
    const bool uneven = tree || lim_min != __builtin_amdgcn_readfirstlane(lim_max);  // rows see different keys
    wait_vmem();
    asm volatile("" ::: "memory");

    f32x16 o[D / 32];
#pragma unroll
    for (int n = 0; n < D / 32; ++n) o[n] = f32x16{};
    float m_run = -1e30f, l_run = 0.f;
    // tiles that every row sees, then the others: the loop over the first ones has no registers
    // to give to the rules of the second
    auto tile = [&](auto hidden) FA_INLINE {
        constexpr bool HIDDEN = decltype(hidden)::value;
        wait_vmem_below<2 * C::NI16>();  // K(t); only V(t) may be in flight
        asm volatile("" ::: "memory");
        f32x16 s;
        tile_scores<T, D>(s, Ks, q, kc.cols, l32, hi);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K(t) read before it is overwritten
        copy(kc, t + NW, bx, by, Ks);

        unsigned have = ~0u, seen = ~0u;
        if (HIDDEN && holes) have = (unsigned)table.template have<2>(2 * t);
        tile_rules<EXACT, HIDDEN>(s, rules, row, tree, 32 * t, c, seen, have, hi);
        soft_max<D>(s, rules.unit, m_run, l_run, o);
        soft_exp(s, rules.unit, m_run, l_run);

        wait_vmem_below<2 * C::NI16>();  // V(t); only K(t + 4) may be in flight
        asm volatile("" ::: "memory");
        if (HIDDEN && uneven && tile_odd<T, D>(Vs, lane)) {
            stay_branch();
            tile_values_seen<T, D>(Vs, s, seen, o, lane);
        } else {
            tile_values<T, D>(Vs, s, o, vc.cols, lane);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V(t) read before it is overwritten
        copy(vc, t + NW, bx, by, Vs);
        blocks(t + 2 * NW, bx, by);
    };
    const int tv = holes ? 0 : min(t1, lim_min / 32);
    for (; t < tv; t += NW) tile(std::false_type{});
    for (; t < t1; t += NW) tile(std::true_type{});
    wait_vmem();  // no copy in flight when the region takes the O part
    asm volatile("" ::: "memory");

    // ---- the waves' parts, rescaled to their common maximum ----
    PagedArgs& pe = paged_args();
    const float l_w = pair_sum(l_run);
    float* mine = reinterpret_cast<float*>(Ks);
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) mine[(16 * n + e) * 64 + lane] = o[n][e];
    if (hi == 0) {
        stat[w][0][l32] = m_run;
        stat[w][1][l32] = l_w;
    }
    lds_barrier();
    float mm = stat[0][0][l32];
#pragma unroll
    for (int x = 1; x < NW; ++x) mm = fmaxf(mm, stat[x][0][l32]);
    float a[NW], l_tot = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
        a[x] = fast_exp2(stat[x][0][l32] - mm);
        l_tot = __builtin_fmaf(stat[x][1][l32], a[x], l_tot);
    }
    if (!row.valid) {  // (such a row went along with the others)
        mm = -1e30f;
        l_tot = 0.f;
    }
    const bool whole = part < 0;
    if (!whole && w == 0 && hi == 0 && row.live) pe.stat[part + l32] = make_float2(mm, l_tot);
    if (whole && w == 0 && hi == 0 && row.live && pe.lse) put_row_lse(pe, b, row.h, row.i, mm, l_tot);
    const float inv = l_tot > 0.f || l_tot != l_tot ? 1.f / l_tot : 0.f;
#pragma unroll
    for (int n0 = 0; n0 < D / 32; n0 += NW) {
        const int n = n0 + w;
        if (n >= D / 32) break;
        f32x16 om = f32x16{};
#pragma unroll
        for (int x = 0; x < NW; ++x) {
            const float* px = reinterpret_cast<const float*>(smem + x * C::REGION);
#pragma unroll
            for (int e = 0; e < 16; ++e) om[e] = __builtin_fmaf(px[(16 * n + e) * 64 + lane], a[x], om[e]);
        }
        if (!row.valid) om = f32x16{};
        if (!row.live) continue;
        if (!whole) {
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *part_of<D>(pe.part, part, n, q4, lane) = f32x4{om[4 * q4], om[4 * q4 + 1], om[4 * q4 + 2], om[4 * q4 + 3]};
        } else {
            T* ob = (T*)pe.o + b * pe.o_sb + (int64_t)row.i * pe.o_ss + row.h * pe.o_sh + 32 * n + 4 * hi;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                if (32 * n + 8 * q4 + 4 * hi >= pe.cols) continue;
                if constexpr (C::F32) {
                    f32x4 v4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v4[e] = om[4 * q4 + e] * inv;
                    *reinterpret_cast<f32x4*>(ob + 8 * q4) = v4;
                } else {
                    s16x4 v4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v4[e] = Elem<T>::pack1(om[4 * q4 + e] * inv);
                    *reinterpret_cast<s16x4*>(ob + 8 * q4) = v4;
                }
            }
        }
    }
    lds_barrier();  // the regions and stat are free for the next unit
}

// rows [first, first + n) of a sequence without a token
template <typename T, int D>
__device__ FA_INLINE inline void empty_unit(PagedArgs& p, int b, int hk, int first, int n, int tid, int threads) {
    constexpr int CW = PagedCfg<T, D>::CW, EPC = PagedCfg<T, D>::EPC;
    for (int x = tid; x < n * CW; x += threads) {
        const PagedRow row(p, first + x / CW, hk);
        const int col = x % CW * EPC;
        if (!row.live || col >= p.cols) continue;
        *reinterpret_cast<uint4*>((T*)p.o + b * p.o_sb + (int64_t)row.i * p.o_ss + row.h * p.o_sh + col) = make_uint4(0u, 0u, 0u, 0u);
        if (col == 0 && p.lse) put_row_lse(p, b, row.h, row.i, 0.f, 0.f);
    }
}

// A wave's 32 rows of O from its LDS (chunks at row_swizzle's places) to their places in
// memory, whole rows a store
template <typename T, int D>
__device__ FA_INLINE inline void store_tile(PagedArgs& p, const T* tile, int b, const PagedRow& row, int lane) {
    using C = PagedCfg<T, D>;
    const int64_t mine = row.live ? (int64_t)row.i * p.o_ss + row.h * p.o_sh : -1;
    T* const ob = (T*)p.o + b * p.o_sb;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // written by this wave alone
#pragma unroll
    for (int x = 0; x < 32 * C::CW / 64; ++x) {
        const int r = (64 * x + lane) / C::CW, chunk = lane % C::CW;
        const int64_t at = __shfl(mine, r);
        const uint4 v = *reinterpret_cast<const uint4*>(tile + r * D + ((chunk ^ row_swizzle<C::CW>(r)) * C::EPC));
        if (at >= 0 && chunk * C::EPC < p.cols) *reinterpret_cast<uint4*>(ob + at + chunk * C::EPC) = v;
    }
}

// ---------------------------------------------------------------------------
// Units of 32 NW rows whose NW waves, on 32 rows each, share tiles of 64 keys: K and V
// are read once for all of them.  NW = 8 for 128 columns only: up to 64 leave registers for
// three workgroups of four waves a CU (28 trees of 91 over up to 13755 keys, 4 heads of 64:
// 130 us with two, 113 with three, 118 with four, which spill).  NS tiles in LDS, of which
// NS - 1 are on their way or read; a wave copies one block of 16 keys (NW = 8) or one of K and
// one of V.
template <typename T, int D, int NW>
struct WideCfg {
    using C = PagedCfg<T, D>;
    static constexpr int STEP = 64;
    static constexpr int TILE = STEP * D;
    static constexpr int NS = NW == 8 ? 4 : 2;
    static constexpr int SMEM = NS * 2 * TILE;
    static constexpr int COPIES = 8 / NW * C::NI16;  // of a wave, a tile
    static constexpr int PER_CU = NW == 8 ? 1 : D < 128 ? 3 : 2;
};

template <typename T, int D, bool EXACT, int NW>
__device__ FA_INLINE inline void paged_unit_wide(T* smem, TreeBits* tree, bool new_tree, int b, int hk, int rt, int s0, int s1,
                                                int64_t part, int tid) {
    using C = PagedCfg<T, D>;
    using X = WideCfg<T, D, NW>;
    PagedArgs& p = paged_args();
    const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6) & (NW - 1);
    const int l32 = lane & 31, hi = lane >> 5;
    PagedRow row(p, 32 * (NW * rt + w) + l32, hk);
    uint4 q[D / 16];
    load_q<T, D>(p, row, b, hi, q);
    TileRules<EXACT> rules(p, b, row.h);
    const int len = filled_here(p, b), c = len - p.Sq;
    // (all waves copy for all)
    const int n_keys = keys_of(p, tree, 32 * NW * (rt + 1), len, c), t1 = min(s1, (n_keys + 63) / 64);

    PageCopy<T, D> kc, vc;
    if (NW == 4 || w < 4) kc.init((const T*)p.k + hk * p.k_sh, p.k_sp, p.k_ss, p.cols, lane);
    if (NW == 4) vc.init((const T*)p.v + hk * p.v_sh, p.v_sp, p.v_ss, p.cols, lane);
    if (NW == 8 && w >= 4) kc.init((const T*)p.v + hk * p.v_sh, p.v_sp, p.v_ss, p.cols, lane);
    const PageTable table(p, b);
    auto look = [&](int t) FA_INLINE { return table.block(4 * t + (w & 3)); };
    // tile t, to slot t % NS; what is past the end reads nothing, but is issued, so that the
    // vmcnt counts stay exact
    auto issue = [&](int t, Block16 at) FA_INLINE {
        const int nv = t < t1 ? n_keys - 64 * t - 16 * (w & 3) : 0;
        T* const dst = smem + (t & (X::NS - 1)) * 2 * X::TILE + 16 * (w & 3) * D;
        kc.load(at, nv, NW == 8 ? dst + (w >> 2) * X::TILE : dst);
        if (NW == 4) vc.load(at, nv, dst + X::TILE);
    };
#pragma unroll
    for (int x = 0; x < X::NS - 1; ++x) issue(s0 + x, look(s0 + x));
    Block16 next = look(s0 + X::NS - 1);

    if (new_tree) tree_init(p, *tree, b, tid);
    row.rule(tree, rules.words, len, c);
    const bool holes = table.holes(4 * s0, 4 * t1, lane);
    int lim_min = row.valid ? row.all : INT_MAX;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) lim_min = min(lim_min, __shfl_xor(lim_min, x));
    lim_min = __builtin_amdgcn_readfirstlane(lim_min);
    const bool uneven = lim_min < n_keys;  // a row does not see what others, or other waves' rows, see
    wait_vmem();
    asm volatile("" ::: "memory");

    f32x16 o[D / 32];
#pragma unroll
    for (int n = 0; n < D / 32; ++n) o[n] = f32x16{};
    float m_run = -1e30f, l_run = 0.f;
    auto next_tile = [&](int t) FA_INLINE {
        wait_vmem_below<(X::NS - 2) * X::COPIES>();  // this wave's part of tile t
        barrier_no_fence();                          // everyone's, and tile t - 1 has been read
        issue(t + X::NS - 1, next);
        next = look(t + X::NS);
        return smem + (t & (X::NS - 1)) * 2 * X::TILE;
    };
    // (as in paged_unit32: what every row sees first; the others in blocks of 32 keys)
    const int tv = holes ? s0 : min(t1, lim_min / 64);
    int t = s0;
    for (; t < tv; ++t) {
        const T* const Ks = next_tile(t);
        const T* const Vs = Ks + X::TILE;
        // the second block's scores beside the first one's exponentials, the first one's values
        // beside the second one's maximum
        unsigned seen;
        f32x16 sa, sb;
        tile_scores<T, D>(sa, Ks, q, D, l32, hi);
        tile_rules<EXACT, false>(sa, rules, row, tree, 64 * t, c, seen, ~0u, hi);
        soft_max<D>(sa, rules.unit, m_run, l_run, o);
        tile_scores<T, D, true>(sb, Ks + 32 * D, q, D, l32, hi);
        soft_exp(sa, rules.unit, m_run, l_run);
        tile_values<T, D, true>(Vs, sa, o, D, lane);
        block_order<D>();
        tile_rules<EXACT, false>(sb, rules, row, tree, 64 * t + 32, c, seen, ~0u, hi);
        soft_max<D>(sb, rules.unit, m_run, l_run, o);
        soft_exp(sb, rules.unit, m_run, l_run);
        tile_values<T, D>(Vs + 32 * D, sb, o, D, lane);
    }
    for (; t < t1; ++t) {
        const T* const Ks = next_tile(t);
#pragma unroll 1
        for (int x = 0; x < 2; ++x) {
            const T* const Vs = Ks + X::TILE + x * 32 * D;
            f32x16 s;
            tile_scores<T, D>(s, Ks + x * 32 * D, q, D, l32, hi);
            unsigned have = ~0u, seen;
            if (holes) have = (unsigned)table.template have<2>(4 * t + 2 * x);
            tile_rules<EXACT, true>(s, rules, row, tree, 64 * t + 32 * x, c, seen, have, hi);
            soft_max<D>(s, rules.unit, m_run, l_run, o);
            soft_exp(s, rules.unit, m_run, l_run);
            if (uneven && tile_odd<T, D>(Vs, lane)) {
                stay_branch();
                tile_values_seen<T, D>(Vs, s, seen, o, lane);
            } else {
                tile_values<T, D>(Vs, s, o, D, lane);
            }
        }
    }
    wait_vmem();  // (copies of no tile)

    PagedArgs& pe = paged_args();
    float l_tot = pair_sum(l_run);
    if (!row.valid) {  // (such a row went along with the others)
        m_run = -1e30f;
        l_tot = 0.f;
#pragma unroll
        for (int n = 0; n < D / 32; ++n) o[n] = f32x16{};
    }
    barrier_no_fence();  // the slots have been read: they take the rows of O, or the next unit's tiles
    if (part >= 0) {
        if (row.live && hi == 0) pe.stat[part + 32 * w + l32] = make_float2(m_run, l_tot);
#pragma unroll
        for (int n = 0; n < D / 32; ++n)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                if (row.live) *part_of<D>(pe.part, part + 32 * w, n, q4, lane) =
                    f32x4{o[n][4 * q4], o[n][4 * q4 + 1], o[n][4 * q4 + 2], o[n][4 * q4 + 3]};
    } else {
        if (row.live && hi == 0 && pe.lse) put_row_lse(pe, b, row.h, row.i, m_run, l_tot);
        const float inv = l_tot > 0.f || l_tot != l_tot ? 1.f / l_tot : 0.f;
        T* const mine = smem + w * 32 * D;
#pragma unroll
        for (int n = 0; n < D / 32; ++n)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                s16x4 v4;
#pragma unroll
                for (int e = 0; e < 4; ++e) v4[e] = Elem<T>::pack1(o[n][4 * q4 + e] * inv);
                *reinterpret_cast<s16x4*>(mine + l32 * D + (((4 * n + q4) ^ row_swizzle<C::CW>(l32)) << 3) + 4 * hi) = v4;
            }
        store_tile<T, D>(pe, mine, b, row, lane);
        barrier_no_fence();  // read, before the next unit's copies
    }
}

// ---------------------------------------------------------------------------
// One workgroup's part of the list.  NW: waves that share tiles (units of 32 NW rows);
// 1: units of 32 rows, 4 waves.
template <typename T, int D, int NW>
struct PagedShape {
    using X = WideCfg<T, D, NW>;
    static constexpr int THREADS = 64 * NW, STEP = X::STEP, ROWS = 32 * NW, SMEM = X::SMEM, PER_CU = X::PER_CU;
};
template <typename T, int D>
struct PagedShape<T, D, 1> {
    using C = PagedCfg<T, D>;
    static constexpr int THREADS = 256, STEP = C::STEP, ROWS = 32, SMEM = C::SMEM, PER_CU = C::PER_CU;
};

template <typename T, int D, bool EXACT, bool TREE, int NW>
__global__ __launch_bounds__((PagedShape<T, D, NW>::THREADS), (NW == 8 ? 2 * PagedShape<T, D, NW>::PER_CU : PagedShape<T, D, NW>::PER_CU)) void paged_kernel(const PagedParams) {
    using S = PagedShape<T, D, NW>;
    PagedArgs& p = paged_args();
    __shared__ __attribute__((aligned(1024))) T smem[S::SMEM];
    __shared__ typename std::conditional<TREE, TreeBits, int>::type bits;
    TreeBits* tree = nullptr;
    if constexpr (TREE) tree = &bits;
    const int tid = threadIdx.x, lane = tid & 63;
    PagedWork wk;
    wk.init<S::STEP>(p, lane);
    if (p.part && blockIdx.x == gridDim.x - 1 && tid < 64) wk.spans<S::STEP>(p, lane);
    const int units = p.Hkv * p.unit_tiles, extra = p.extra;
    if ((int64_t)blockIdx.x >= (int64_t)wk.W * units) return;
    const int g = xcd_remap((int)blockIdx.x, wk.W * units), group = g / units, u = g - group * units;
    const int tiles = p.unit_tiles, hk = u / tiles, rt = u - hk * tiles;
    int x = 0, end = 0, b = 0, start = 0, len = 0, last_b = -1;  // len: of a unit, with the extra steps
    if (wk.whole) {
        b = group;
        len = PagedWork::steps_here<S::STEP>(p, b);
        end = len;
    } else {
        x = wk.first(group);
        end = wk.first(group + 1);
    }
    while (x < end) {
        if (!wk.whole) wk.locate<S::STEP>(paged_args(), x, lane, b, start, len);
        const int s0 = x - start, n = len - extra, s1 = min(n, end - start);
        x = min(end, start + len);
        if (s0 >= s1) continue;  // (the extra steps of a unit that ended in another workgroup)
        const int64_t part = s1 - s0 == n ? -1 : part_at<S::ROWS>(g, s0 == 0);
        if (n == 1 && filled_here(paged_args(), b) == 0) {
            empty_unit<T, D>(paged_args(), b, hk, rt * S::ROWS, S::ROWS, tid, S::THREADS);
        } else if constexpr (NW == 1) {
            __shared__ float stat[PagedCfg<T, D>::NW][2][32];
            paged_unit32<T, D, EXACT>(smem, stat, tree, TREE && b != last_b, b, hk, rt, s0, s1, part, tid);
        } else {
            paged_unit_wide<T, D, EXACT, NW>(smem, tree, TREE && b != last_b, b, hk, rt, s0, s1, part, tid);
        }
        last_b = b;
    }
}

// The parts of 32 rows (blockIdx.x: KV head, unit, its rows) of a unit that several
// workgroups shared: for 32 columns G waves, each of which takes every G-th part, two at
// a time, and whose sums meet in LDS.  Units of 32 rows are few, in as many parts as there are
// workgroups for each: 64 with 8 KV heads, up to 512 with one.  Four waves, 16 where a
// sequence may be in more than 40 parts (us with 4 and 16: one token of 8 heads over 8192 keys, 32
// parts, 15.7 and 16.4; 15 tokens of 2 heads in 54 parts 16.9 and 16.4; one of 8 heads over 65536 in 64 parts
// 39.6 and 38.5; one of one head over 131072 in 512 31.7 and 24.6), 32 columns a workgroup (one token over
// 65536 keys: 39 us a call, 45 with two and all columns); wide units are in two or three, and
// what a workgroup finds out about its unit serves all columns (16 trees of 64 over up to 8192:
// 13 us, 18 with 32 columns).
template <int D, int NW, bool MANY>
struct JoinShape {
    static constexpr int G = NW > 1 ? 2 : MANY ? 16 : 4, BLOCKS = NW == 1 ? 1 : D / 32;  // of 32 columns
};
template <typename T, int D, int NW, bool MANY>
__global__ __launch_bounds__((64 * JoinShape<D, NW, MANY>::G * JoinShape<D, NW, MANY>::BLOCKS)) void paged_join_kernel(const PagedParams) {
    using S = PagedShape<T, D, NW>;
    using J = JoinShape<D, NW, MANY>;
    constexpr int G = J::G, OUT = G < 4 ? G : 4;  // waves that write the sums
    PagedArgs& p = paged_args();
    __shared__ float sums[J::BLOCKS][G][16][64], stat[G][2][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, hi = lane >> 5, b = blockIdx.z;
    const int w = wave % G, block = wave / G, n = blockIdx.y * J::BLOCKS + block;
    // (found again from the lengths, it took 1.3 us of the 6.2 of a join of 32 tokens' parts)
    const int2 span = p.spans[b];
    const int g0 = __builtin_amdgcn_readfirstlane(span.x), g1 = __builtin_amdgcn_readfirstlane(span.y);
    if (g0 == g1) return;
    const int units = p.Hkv * p.unit_tiles, u = blockIdx.x / NW, r0 = 32 * (blockIdx.x % NW);
    const PagedRow row(p, S::ROWS * (u % p.unit_tiles) + r0 + l32, u / p.unit_tiles);
    float m = -1e30f, l = 0.f;
    f32x4 acc[4];
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) acc[q4] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int g = g0 + w; g <= g1; g += 2 * G) {
        float2 st[2];
        f32x4 v[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const bool in = g + G * x <= g1;
            const int gx = in ? g + G * x : g;
            const int64_t part = part_at<S::ROWS>(gx * units + u, gx == g0) + r0;  // g0 begins the sequence
            if (in && row.live) {
                st[x] = p.stat[part + l32];
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) v[x][q4] = *part_of<D>(p.part, part, n, q4, lane);
            } else {
                st[x] = make_float2(-1e30f, 0.f);
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) v[x][q4] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
        const float m0 = fmaxf(m, fmaxf(st[0].x, st[1].x)), a0 = fast_exp2(m - m0);
        const float a[2] = {fast_exp2(st[0].x - m0), fast_exp2(st[1].x - m0)};
        l = __builtin_fmaf(st[1].y, a[1], __builtin_fmaf(st[0].y, a[0], l * a0));
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                acc[q4][e] = __builtin_fmaf(v[1][q4][e], a[1], __builtin_fmaf(v[0][q4][e], a[0], acc[q4][e] * a0));
        m = m0;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) sums[block][w][e][lane] = acc[e >> 2][e & 3];
    if (block == 0 && hi == 0) {
        stat[w][0][l32] = m;
        stat[w][1][l32] = l;
    }
    __syncthreads();
    if (!row.live || w >= OUT) return;
    float mm = stat[0][0][l32], l_tot = 0.f, a[G];
#pragma unroll
    for (int x = 1; x < G; ++x) mm = fmaxf(mm, stat[x][0][l32]);
#pragma unroll
    for (int x = 0; x < G; ++x) {
        a[x] = fast_exp2(stat[x][0][l32] - mm);
        l_tot = __builtin_fmaf(stat[x][1][l32], a[x], l_tot);
    }
    const float inv = l_tot > 0.f || l_tot != l_tot ? 1.f / l_tot : 0.f;
    if (n == 0 && w == 0 && hi == 0 && p.lse) put_row_lse(p, b, row.h, row.i, mm, l_tot);
    T* ob = (T*)p.o + b * p.o_sb + (int64_t)row.i * p.o_ss + row.h * p.o_sh + 32 * n + 4 * hi;
#pragma unroll
    for (int q = 0; q < 4 / OUT; ++q) {
        const int q4 = w * (4 / OUT) + q;
        if (32 * n + 8 * q4 + 4 * hi >= p.cols) continue;
        float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < G; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(sums[block][x][4 * q4 + e][lane], a[x], o[e]);
        if constexpr (Elem<T>::kF32) {
            *reinterpret_cast<f32x4*>(ob + 8 * q4) = f32x4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        } else {
            s16x4 v4;
#pragma unroll
            for (int e = 0; e < 4; ++e) v4[e] = Elem<T>::pack1(o[e] * inv);
            *reinterpret_cast<s16x4*>(ob + 8 * q4) = v4;
        }
    }
}

template <typename T, int D, int NW>
hipError_t launch_paged_t(const PagedParams& p, hipStream_t s) {
    using S = PagedShape<T, D, NW>;
    const dim3 grid((unsigned)p.o_wgs), block(S::THREADS);
    constexpr bool F32 = Elem<T>::kF32;
    if (p.parents) {
        if (F32 || p.cap > kWideCap)
            hipLaunchKernelGGL((paged_kernel<T, D, true, true, NW>), grid, block, 0, s, p);
        else
            hipLaunchKernelGGL((paged_kernel<T, D, F32, true, NW>), grid, block, 0, s, p);
    } else {
        if (F32 || p.cap > kWideCap)
            hipLaunchKernelGGL((paged_kernel<T, D, true, false, NW>), grid, block, 0, s, p);
        else
            hipLaunchKernelGGL((paged_kernel<T, D, F32, false, NW>), grid, block, 0, s, p);
    }
    if (p.part) {
        auto join = [&](auto many) {
            using J = JoinShape<D, NW, decltype(many)::value>;
            const dim3 tiles((unsigned)(p.Hkv * p.unit_tiles * NW), D / 32 / J::BLOCKS, (unsigned)p.B);
            hipLaunchKernelGGL((paged_join_kernel<T, D, NW, decltype(many)::value>), tiles, dim3(64 * J::G * J::BLOCKS), 0, s, p);
        };
        if (NW == 1 && p.many)
            join(std::integral_constant<bool, NW == 1>{});
        else
            join(std::false_type{});
    }
    return hipGetLastError();
}
template <typename T, int D>
hipError_t launch_paged_d(const PagedParams& p, hipStream_t s) {
    if constexpr (!Elem<T>::kF32) {
        if constexpr (D == 128) {
            if (p.wide == 8) return launch_paged_t<T, D, 8>(p, s);
        }
        if (p.wide == 4) return launch_paged_t<T, D, 4>(p, s);
    }
    return launch_paged_t<T, D, 1>(p, s);
}

template <typename T>
hipError_t launch_paged(const PagedParams& p, int D, hipStream_t s) {
    switch (D) {
        case 32: return launch_paged_d<T, 32>(p, s);
        case 64: return launch_paged_d<T, 64>(p, s);
        case 128: return launch_paged_d<T, 128>(p, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace fa
