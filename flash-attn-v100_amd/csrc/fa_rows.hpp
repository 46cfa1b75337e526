// Attention of a few new tokens a sequence over its cache, and over a prefix
// that all sequences of the batch share; gfx950.
//
// A row is one (sequence, new token, query head).  The keys of every unit of rows
// are split over workgroups:
//   * a sequence's own keys: units of 32 rows (of one sequence and KV head), whose
//     keys a workgroup's 4 waves walk in turn, 32 at a time, each copying its own
//     tiles (direct to LDS, both of a tile's copies in flight) with no barrier;
//   * the prefix: the rows of all sequences together, units of 128 whose waves
//     share 64-key tiles, so that K and V are read once for 128 rows, not once a
//     sequence; units of 32 where there are no more than 64 rows.
// A split leaves its rows' maximum, sum and unnormalised output in float32, and
// rows_join_kernel puts the parts of a row together:
//   O = sum_x 2^(m_x - m) O_x / sum_x 2^(m_x - m) l_x,  m = max_x m_x.
// Query i of a sequence with n keys of its own stands at own position
// n - Sq + i and sees its keys up to there; in distances the prefix lies before
// them.  Bound by the K and V bytes, and over the prefix by the products of its
// rows: 16 tokens over caches of up to 8192 keys, 32 on 8 heads of 128: 78 us, 4.6
// TB/s; 64 tokens after 8192 shared ones and up to 512 of their own: 37 us (51 us
// when units of 32 rows read the prefix); 8 x 5 tokens after 20001, 16 on 2 heads:
// 25 us (43).  Small calls are bound by the launch: 9 us for 8 heads over 512
// keys, with 4 waves a workgroup as with 8.  float32, whose tiles are copied and waited
// for one by one: 16 tokens over 8192 keys, 32 on 8 heads of 128: 270 us with the join, 4.0
// TB/s; 64 tokens after 8192 and 512: 229 us, of which the products are 61 on the float32
// matrix instruction.
#pragma once

#include "fa_common.hpp"
#include "fa_fwd_decode.hpp"
#include "fa_ops_params.hpp"
#include "fa_scored.hpp"

namespace fa {

template <typename T, int D>
struct RowsCfg {
    static constexpr bool F32 = Elem<T>::kF32;
    static constexpr int NW = 4;
    // a wave's own tiles (rows of one 32-row unit): 32 keys, rows of an even
    // number of 16-byte chunks, so that a tile is whole copy instructions
    static constexpr int BN = 32;
    static constexpr int KW = D + (F32 ? 4 : 16);
    static constexpr int VW = F32 ? D + 8 : D + (D == 128 ? 32 : 16);
    static constexpr int KTILE = BN * KW, VTILE = BN * VW;
    static constexpr int REGION = KTILE + VTILE;
    static_assert((D / 32) * 16 * 64 * 4 <= REGION * (int)sizeof(T), "a wave's O part fits its region");
    // tiles shared by the waves of a 128-row unit
    using S = FwdCfg<T, D>;
    static constexpr int SMEM = NW * REGION > S::SMEM_ELEMS ? NW * REGION : S::SMEM_ELEMS;
    // two workgroups a CU where registers and LDS allow it
    static constexpr int PER_CU = F32 && D == 128 ? 1 : 2;
};

// filled keys of a sequence's own, and the position among them of query 0
__device__ FA_INLINE inline int own_len(const RowsParams& p, int b) {
    return p.lens ? max(0, min(p.Sk, p.lens[b])) : p.Sk;
}
__device__ FA_INLINE inline int own_pos(const RowsParams& p, int b, int len) {
    return p.tail ? len - p.Sq : max(-kMaxOffset, min(kMaxOffset, p.offsets ? p.offsets[b] : p.offset0));
}
// the key nearest to a position: distances are taken from there, as SeqRule::near
__device__ FA_INLINE inline int near_key(int pos, int len) { return max(0, min(len - 1, pos)); }
// the LSE of a row from its maximum and sum, with what the distance to there adds (a
// query after a prefix stands on one of the own keys, or sees nothing)
__device__ FA_INLINE inline void put_lse(const RowsParams& p, int b, int h, int i, float m, float l) {
    const int64_t at = ((int64_t)b * p.H + h) * p.Sq + i;
    float lse = l > 0.f ? (m + __log2f(l)) * kLn2 : l == 0.f ? -INFINITY : l;
    if (p.lse_near) p.lse_near[at] = lse;
    if (p.slopes && !p.tail) {
        const int len = own_len(p, b), own = own_pos(p, b, len) + i;
        lse = __builtin_fmaf(-p.slopes[b * p.slopes_sb + h], (float)abs(own - near_key(own, len)), lse);
    }
    p.lse[at] = lse;
}

// one row of a unit: its query and the keys [0, lim) it sees
struct UnitRow {
    int b, i, h, lim;
    bool live;
    int qpos;  // of the nearest key (the prefix before the own ones)
    __device__ FA_INLINE inline UnitRow(const RowsParams& p, bool pre, int row, int hk, int bs) {
        const int per_seq = p.Sq * p.group, n_rows = pre ? p.B * per_seq : per_seq;
        live = row < n_rows;
        const int rr = live ? row : 0;
        b = pre ? rr / per_seq : bs;
        const int ig = pre ? rr % per_seq : rr;
        i = ig / p.group;
        h = hk * p.group + ig % p.group;
        const int len = own_len(p, b);
        const int own = own_pos(p, b, len) + i;  // the query's position among the sequence's own keys
        lim = pre ? p.P : p.causal ? min(len, own + 1) : len;
        if (!live || (p.masked_neg && own < 0)) lim = 0;
        qpos = pre ? p.P + own : near_key(own, len);
    }
};

// scores of 16 keys of a 32-key block in log2 units
template <bool EXACT>
__device__ FA_INLINE inline void row_rules(f32x16& s, const RowsParams& p, Cap<EXACT>& cap, bool slope, float slope2, float d0) {
    if (p.cap > 0.f) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = cap.value(s[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= p.scale_log2;
    }
    if (slope) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            s[e] = __builtin_fmaf(-slope2, __builtin_fabsf(d0 - (float)(8 * (e >> 2) + (e & 3))), s[e]);
    }
}

// 32 rows over split `split` of the keys [0, n_keys) (a sequence's own ones, or a
// prefix that few rows read; p.joined: the prefix, then the own ones): each wave
// walks tiles of its own
template <typename T, int D, bool EXACT>
__device__ FA_INLINE inline void unit32(const RowsParams& p, bool pre, T* smem, float (*stat)[2][32], int id, int lane, int w) {
    using C = RowsCfg<T, D>;
    constexpr int BN = C::BN, KW = C::KW, VW = C::VW, NW = C::NW;
    const int l32 = lane & 31, hi = lane >> 5;
    const int splits = pre ? p.p_splits : p.o_splits, rts = pre ? p.p_rt : p.o_rt;
    const int split = id % splits, unit = id / splits, rt = unit % rts, bk = unit / rts;
    const int hk = bk % p.Hkv, bs = bk / p.Hkv;  // bs: the sequence (own keys)
    const UnitRow row(p, pre, 32 * rt + l32, hk, bs);
    // keys that some row of the tile sees, and that all do
    int lim_max = row.lim, lim_min = row.live ? row.lim : INT_MAX;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        lim_max = max(lim_max, __shfl_xor(lim_max, x));
        lim_min = min(lim_min, __shfl_xor(lim_min, x));
    }
    lim_max = __builtin_amdgcn_readfirstlane(lim_max);
    lim_min = __builtin_amdgcn_readfirstlane(lim_min);
    const int n_keys = max(lim_max, 0);
    // tiles of the prefix before the own ones (a row that sees any key sees the
    // prefix and a key of its own)
    const int pt = p.joined && n_keys > 0 ? (p.P + BN - 1) / BN : 0;
    const int nt = pt + (n_keys + BN - 1) / BN;
    const int t0 = (int)((int64_t)nt * split / splits), t1 = (int)((int64_t)nt * (split + 1) / splits);

    const int64_t k_ss = pre ? p.kp_ss : p.k_ss, v_ss = pre ? p.vp_ss : p.v_ss;
    const T* __restrict__ kbase = pre ? (const T*)p.kp + hk * p.kp_sh : (const T*)p.k + bs * p.k_sb + hk * p.k_sh;
    const T* __restrict__ vbase = pre ? (const T*)p.vp + hk * p.vp_sh : (const T*)p.v + bs * p.v_sb + hk * p.v_sh;
    T* Ks = smem + w * C::REGION;
    T* Vs = Ks + C::KTILE;
    DmaTile<T, BN, D, KW, 1> kd;
    kd.init(k_ss, lane, 0, p.cols);
    DmaTile<T, BN, D, VW, 1> vd;
    vd.init(v_ss, lane, 0, p.cols);
    constexpr int NKI = decltype(kd)::NI, NVI = decltype(vd)::NI;
    // tiles past the split's end read nothing but are issued, so that the vmcnt
    // counts stay exact (float32 tiles are copied and waited for one by one)
    DmaTile<T, BN, D, KW, 1> kpd;  // rows of the prefix, before own ones
    kpd.init(p.kp_ss, lane, 0, p.cols);
    DmaTile<T, BN, D, VW, 1> vpd;
    vpd.init(p.vp_ss, lane, 0, p.cols);
    auto copy = [&](auto& tile, const T* base, int64_t ss, int k0, int nv, T* dst) FA_INLINE {
        if constexpr (C::F32)
            tile.load(base + (int64_t)k0 * ss, ss, nv, dst, lane);
        else
            tile.load_untracked(base + (int64_t)k0 * ss, ss, nv, dst, lane);
    };
    auto copy_k = [&](int t) FA_INLINE {
        const int k0 = (t < pt ? t : t - pt) * BN;
        if (t < pt)
            copy(kpd, (const T*)p.kp + hk * p.kp_sh, p.kp_ss, k0, t < t1 ? p.P - k0 : 0, Ks);
        else
            copy(kd, kbase, k_ss, k0, t < t1 ? n_keys - k0 : 0, Ks);
    };
    auto copy_v = [&](int t) FA_INLINE {
        const int k0 = (t < pt ? t : t - pt) * BN;
        if (t < pt)
            copy(vpd, (const T*)p.vp + hk * p.vp_sh, p.vp_ss, k0, t < t1 ? p.P - k0 : 0, Vs);
        else
            copy(vd, vbase, v_ss, k0, t < t1 ? n_keys - k0 : 0, Vs);
    };

    constexpr int QR = C::F32 ? D / 8 : D / 16;
    uint4 qreg[QR];
    {
        const T* qrow = (const T*)p.q + row.b * p.q_sb + (int64_t)row.i * p.q_ss + row.h * p.q_sh;
#pragma unroll
        for (int kk = 0; kk < QR; ++kk) {
            const int d0 = C::F32 ? hi * (D / 2) + 4 * kk : 16 * kk + 8 * hi;
            qreg[kk] = row.live && d0 < p.cols ? *reinterpret_cast<const uint4*>(qrow + d0) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    const bool slope = p.slopes != nullptr;
    const float slope2 = slope ? p.slopes[row.b * p.slopes_sb + row.h] * kLog2e : 0.f;
    wait_vmem();
    asm volatile("" ::: "memory");

    f32x16 o[D / 32];
#pragma unroll
    for (int n = 0; n < D / 32; ++n) o[n] = f32x16{};
    float m_run = -1e30f, l_run = 0.f;
    Cap<EXACT> cap(p);

    int t = t0 + w;
    copy_k(t);
    copy_v(t);
    for (; t < t1; t += NW) {
        const bool first = t < pt;
        const int k0 = (first ? t : t - pt) * BN;
        // ---- S^T = K Q^T ----
        if constexpr (C::F32)
            wait_vmem();
        else
            wait_vmem_below<NVI>();  // K(t); only V(t) may be in flight
        asm volatile("" ::: "memory");
        f32x16 s = f32x16{};
        const T* krow = Ks + l32 * KW;
#pragma unroll
        for (int kk = 0; kk < QR; ++kk) {
            if constexpr (C::F32) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(krow + hi * (D / 2) + 4 * kk);
                const f32x4 bq = __builtin_bit_cast(f32x4, qreg[kk]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s = mfma_f32(a[e], bq[e], s);
            } else {
                const s16x8 a = *reinterpret_cast<const s16x8*>(krow + 16 * kk + 8 * hi);
                s = Elem<T>::mfma(a, __builtin_bit_cast(s16x8, qreg[kk]), s);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K(t) read before it is overwritten
        if constexpr (!C::F32) copy_k(t + NW);

        row_rules(s, p, cap, slope, slope2, (float)(row.qpos - k0 + (first ? p.P : 0) - 4 * hi));
        if (k0 + BN > (first && lim_min > 0 ? p.P : lim_min)) {
            stay_branch();
            const int lm = (first && row.lim > 0 ? p.P : row.lim) - k0 - 4 * hi;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (8 * (e >> 2) + (e & 3) >= lm) s[e] = -INFINITY;
        }
        // ---- softmax ----
        float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 16; ++e) m2[e & 1] = fmaxf(m2[e & 1], s[e]);
        const float m_new = fmaxf(m_run, pair_max(fmaxf(m2[0], m2[1])));
        if (__ballot(m_new > m_run + 8.0f) != 0ull) {
            const float alpha = fast_exp2(m_run - m_new);
            l_run *= alpha;
#pragma unroll
            for (int n = 0; n < D / 32; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[n][e] *= alpha;
            m_run = m_new;
        }
        float ps[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = fast_exp2(s[e] - m_run);
            ps[e & 1] += s[e];
        }
        l_run += ps[0] + ps[1];

        // ---- O^T += V^T P^T ----
        if constexpr (C::F32) {
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const T* vrow = Vs + (8 * (x >> 2) + 4 * hi + (x & 3)) * VW + l32;
#pragma unroll
                for (int n = 0; n < D / 32; ++n) o[n] = mfma_f32(vrow[32 * n], s[x], o[n]);
            }
        } else {
            wait_vmem_below<NKI>();  // V(t); only K(t + 4) may be in flight
            asm volatile("" ::: "memory");
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks) {
                float tmp[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) tmp[e] = s[8 * ks + e];
                const s16x8 pk = pack8<T>(tmp);
#pragma unroll
                for (int n = 0; n < D / 32; ++n) {
                    const T* vp = Vs + (16 * ks + 4 * hi + ((lane & 15) >> 2)) * VW + 32 * n + 16 * ((lane >> 4) & 1) +
                                  4 * (lane & 3);
                    const s16x8 a = cat4(lds_read_tr16(vp), lds_read_tr16(vp + 8 * VW));
                    o[n] = Elem<T>::mfma(a, pk, o[n]);
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V(t) read before it is overwritten
        if constexpr (C::F32) copy_k(t + NW);
        copy_v(t + NW);
    }
    wait_vmem();  // no copy in flight when the region takes the O part
    asm volatile("" ::: "memory");

    // ---- the waves' parts, rescaled to their common maximum ----
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
    const bool only = p.p_splits + p.o_splits == 1;  // no other part of these rows
    const int64_t prow = (pre ? 0 : p.p_rows) + (int64_t)id * 32 + l32;
    if (!only && w == 0 && hi == 0) p.stat[prow] = make_float2(mm, l_tot);
    if (only && w == 0 && hi == 0 && row.live && p.lse) put_lse(late_args<RowsParams>(), row.b, row.h, row.i, mm, l_tot);
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
        if (!only) {
            float* op = p.part + prow * D + 32 * n + 4 * hi;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<f32x4*>(op + 8 * q4) = f32x4{om[4 * q4], om[4 * q4 + 1], om[4 * q4 + 2], om[4 * q4 + 3]};
        } else if (row.live) {
            T* ob = (T*)p.o + row.b * p.o_sb + (int64_t)row.i * p.o_ss + row.h * p.o_sh + 32 * n + 4 * hi;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                if (32 * n + 8 * q4 + 4 * hi >= p.cols) continue;
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
}

// 128 rows of all sequences over split `split` of the prefix: the waves share its
// tiles (64 keys, double-buffered), each on 32 rows
template <typename T, int D, bool EXACT>
__device__ FA_INLINE inline void unit128(const RowsParams& p, T* smem, int id, int lane, int w) {
    using C = FwdCfg<T, D>;
    constexpr int BN = C::BN, NB = C::NB, KW = C::KW, VW = C::VW;
    const int l32 = lane & 31, hi = lane >> 5;
    const int split = id % p.p_splits, unit = id / p.p_splits, rt = unit % p.p_rt, hk = unit / p.p_rt;
    const UnitRow row(p, true, 128 * rt + 32 * w + l32, hk, 0);
    const int nt = (p.P + BN - 1) / BN;
    const int t0 = (int)((int64_t)nt * split / p.p_splits), t1 = (int)((int64_t)nt * (split + 1) / p.p_splits);
    const T* __restrict__ kbase = (const T*)p.kp + hk * p.kp_sh;
    const T* __restrict__ vbase = (const T*)p.vp + hk * p.vp_sh;
    T* const Ks0 = smem;
    T* const Vs0 = smem + 2 * C::KTILE;
    DmaTile<T, BN, D, KW, C::NW> kd;
    kd.init(p.kp_ss, lane, w, p.cols);
    DmaTile<T, BN, D, VW, C::NW> vd;
    vd.init(p.vp_ss, lane, w, p.cols);
    auto copy = [&](int t, int slot) FA_INLINE {
        const int nv = t < t1 ? p.P - t * BN : 0;
        if constexpr (C::F32) {
            kd.load(kbase + (int64_t)(t * BN) * p.kp_ss, p.kp_ss, nv, Ks0 + slot * C::KTILE, lane);
            vd.load(vbase + (int64_t)(t * BN) * p.vp_ss, p.vp_ss, nv, Vs0 + slot * C::VTILE, lane);
        } else {
            kd.load_untracked(kbase + (int64_t)(t * BN) * p.kp_ss, p.kp_ss, nv, Ks0 + slot * C::KTILE, lane);
            vd.load_untracked(vbase + (int64_t)(t * BN) * p.vp_ss, p.vp_ss, nv, Vs0 + slot * C::VTILE, lane);
        }
    };
    constexpr int QR = C::F32 ? D / 8 : D / 16;
    uint4 qreg[QR];
    {
        const T* qrow = (const T*)p.q + row.b * p.q_sb + (int64_t)row.i * p.q_ss + row.h * p.q_sh;
#pragma unroll
        for (int kk = 0; kk < QR; ++kk) {
            const int d0 = C::F32 ? hi * (D / 2) + 4 * kk : 16 * kk + 8 * hi;
            qreg[kk] = row.live && d0 < p.cols ? *reinterpret_cast<const uint4*>(qrow + d0) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    const bool slope = p.slopes != nullptr;
    const float slope2 = slope ? p.slopes[row.b * p.slopes_sb + row.h] * kLog2e : 0.f;
    const int lim_w = __builtin_amdgcn_readfirstlane(__ballot(row.live && row.lim == 0) != 0ull ? 0 : p.P);  // seen by all
    f32x16 o[D / 32];
#pragma unroll
    for (int n = 0; n < D / 32; ++n) o[n] = f32x16{};
    float m_run = -1e30f, l_run = 0.f;
    Cap<EXACT> cap(p);

    int slot = 0;
    copy(t0, 0);
    for (int t = t0; t < t1; ++t) {
        wait_vmem();
        lds_barrier();
        copy(t + 1, slot ^ 1);
        const int k0 = t * BN;
        f32x16 s[NB];
#pragma unroll
        for (int blk = 0; blk < NB; ++blk) {
            s[blk] = f32x16{};
            const T* krow = Ks0 + slot * C::KTILE + (32 * blk + l32) * KW;
#pragma unroll
            for (int kk = 0; kk < QR; ++kk) {
                if constexpr (C::F32) {
                    const f32x4 a = *reinterpret_cast<const f32x4*>(krow + hi * (D / 2) + 4 * kk);
                    const f32x4 bq = __builtin_bit_cast(f32x4, qreg[kk]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[blk] = mfma_f32(a[e], bq[e], s[blk]);
                } else {
                    const s16x8 a = *reinterpret_cast<const s16x8*>(krow + 16 * kk + 8 * hi);
                    s[blk] = Elem<T>::mfma(a, __builtin_bit_cast(s16x8, qreg[kk]), s[blk]);
                }
            }
        }
#pragma unroll
        for (int blk = 0; blk < NB; ++blk)
            row_rules(s[blk], p, cap, slope, slope2, (float)(row.qpos - k0 - 32 * blk - 4 * hi));
        if (k0 + BN > lim_w) {
            stay_branch();
            const int lm = row.lim - k0 - 4 * hi;
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (32 * blk + 8 * (e >> 2) + (e & 3) >= lm) s[blk][e] = -INFINITY;
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int blk = 0; blk < NB; ++blk)
#pragma unroll
            for (int e = 0; e < 16; ++e) m4[e & 3] = fmaxf(m4[e & 3], s[blk][e]);
        const float m_new = fmaxf(m_run, pair_max(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]))));
        if (__ballot(m_new > m_run + 8.0f) != 0ull) {
            const float alpha = fast_exp2(m_run - m_new);
            l_run *= alpha;
#pragma unroll
            for (int n = 0; n < D / 32; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[n][e] *= alpha;
            m_run = m_new;
        }
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int blk = 0; blk < NB; ++blk)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[blk][e] = fast_exp2(s[blk][e] - m_run);
                ps[e & 3] += s[blk][e];
            }
        l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        const T* const Vs = Vs0 + slot * C::VTILE;
        if constexpr (C::F32) {
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const T* vrow = Vs + (32 * blk + 8 * (x >> 2) + 4 * hi + (x & 3)) * VW + l32;
#pragma unroll
                    for (int n = 0; n < D / 32; ++n) o[n] = mfma_f32(vrow[32 * n], s[blk][x], o[n]);
                }
        } else {
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks) {
                float tmp[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) tmp[e] = s[ks >> 1][8 * (ks & 1) + e];
                const s16x8 pk = pack8<T>(tmp);
#pragma unroll
                for (int n = 0; n < D / 32; ++n) {
                    const T* vp = Vs + (16 * ks + 4 * hi + ((lane & 15) >> 2)) * VW + 32 * n + 16 * ((lane >> 4) & 1) +
                                  4 * (lane & 3);
                    const s16x8 a = cat4(lds_read_tr16(vp), lds_read_tr16(vp + 8 * VW));
                    o[n] = Elem<T>::mfma(a, pk, o[n]);
                }
            }
        }
        slot ^= 1;
    }
    wait_vmem();  // (copies of no tile)
    const float l_w = pair_sum(l_run);
    const int64_t prow = (int64_t)id * 128 + 32 * w + l32;
    if (hi == 0) p.stat[prow] = make_float2(m_run, l_w);
    float* op = p.part + prow * D + 4 * hi;
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<f32x4*>(op + 32 * n + 8 * q4) = f32x4{o[n][4 * q4], o[n][4 * q4 + 1], o[n][4 * q4 + 2], o[n][4 * q4 + 3]};
}

// The units of the prefix, then those of the sequences' own keys, in one launch
// (the products of the ones beside the bytes of the others).  EXACT: the cap by its
// series (a branch on it in this kernel costs single tokens 0.2 of 9.0 us).
template <typename T, int D, bool EXACT>
__global__ __launch_bounds__(256, (RowsCfg<T, D>::PER_CU)) void rows_kernel(const RowsParams p) {
    using C = RowsCfg<T, D>;
    __shared__ __attribute__((aligned(16))) T smem[C::SMEM];
    __shared__ float stat[C::NW][2][32];
    const int tid = threadIdx.x;
    const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
    const bool pre = (int64_t)blockIdx.x < p.p_wgs;
    // splits of a unit are consecutive ids, on one XCD's share of the grid
    const int id = xcd_remap(pre ? (int)blockIdx.x : (int)(blockIdx.x - p.p_wgs), (int)(pre ? p.p_wgs : p.o_wgs));
    if (pre && p.p_unit == 128)
        unit128<T, D, EXACT>(p, smem, id, lane, w);
    else
        unit32<T, D, EXACT>(p, pre, smem, stat, id, lane, w);
}

// The parts of every row, rescaled to their common maximum: D / 4 threads a row (4
// columns each), times G groups that share its parts and meet in LDS.  Bound by the
// latency of two rounds of loads: 5 us for 64 x 32 rows of 12 parts, 6 us for 640
// rows of 57 (17 us with one group a row).
template <typename T, int D>
__global__ __launch_bounds__(256) void rows_join_kernel(const RowsParams p, const int64_t n_rows, const int G) {
    constexpr int TPR = D / 4, SLOTS = 256 / TPR;  // row-groups of a workgroup
    __shared__ float sm[SLOTS][2], sacc[SLOTS][D];
    const int slot = (int)threadIdx.x / TPR, col = (int)(threadIdx.x % TPR) * 4;
    const int g = slot % G;
    const int64_t r = (int64_t)blockIdx.x * (SLOTS / G) + slot / G;
    const bool live = r < n_rows;
    const int64_t rr = live ? r : 0;
    // r = (b H + h) Sq + i
    const int i = (int)(rr % p.Sq), h = (int)((rr / p.Sq) % p.H), b = (int)(rr / ((int64_t)p.Sq * p.H));
    const int hk = h / p.group, ig = i * p.group + h % p.group, per_seq = p.Sq * p.group;
    const int U = p.p_unit;
    const int64_t gp = (int64_t)b * per_seq + ig;  // row of the prefix units
    const int64_t pbase = ((int64_t)hk * p.p_rt + gp / U) * p.p_splits * U + gp % U;
    const int64_t obase = p.p_rows + (((int64_t)b * p.Hkv + hk) * p.o_rt + (ig >> 5)) * p.o_splits * 32 + (ig & 31);
    const int n = p.p_splits + p.o_splits;
    auto part_row = [&](int x) FA_INLINE { return x < p.p_splits ? pbase + (int64_t)U * x : obase + 32 * (int64_t)(x - p.p_splits); };
    float mm = -1e30f, l_tot = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    // four parts at a time, whose loads wait for nothing
    for (int x0 = g; x0 < n; x0 += 4 * G) {
        float2 st[4];
        f32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = x0 + j * G < n;
            const int64_t pr = part_row(in ? x0 + j * G : x0);
            st[j] = p.stat[pr];
            v[j] = *reinterpret_cast<const f32x4*>(p.part + pr * D + col);
            if (!in) {
                st[j] = make_float2(-1e30f, 0.f);
                v[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
        const float m0 = fmaxf(mm, fmaxf(fmaxf(st[0].x, st[1].x), fmaxf(st[2].x, st[3].x)));
        const float a0 = fast_exp2(mm - m0);
        l_tot *= a0;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] *= a0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = fast_exp2(st[j].x - m0);
            l_tot = __builtin_fmaf(st[j].y, a, l_tot);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(v[j][e], a, acc[e]);
        }
        mm = m0;
    }
    if (G > 1) {
        if (col == 0) {
            sm[slot][0] = mm;
            sm[slot][1] = l_tot;
        }
        *reinterpret_cast<f32x4*>(&sacc[slot][col]) = acc;
        __syncthreads();
        if (g != 0) return;
        float m2 = mm;
        for (int x = 1; x < G; ++x) m2 = fmaxf(m2, sm[slot + x][0]);
        const float a0 = fast_exp2(mm - m2);
        l_tot *= a0;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] *= a0;
        for (int x = 1; x < G; ++x) {
            const float a = fast_exp2(sm[slot + x][0] - m2);
            l_tot = __builtin_fmaf(sm[slot + x][1], a, l_tot);
            const f32x4 v = *reinterpret_cast<const f32x4*>(&sacc[slot + x][col]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(v[e], a, acc[e]);
        }
        mm = m2;
    }
    if (!live) return;
    const float inv = l_tot > 0.f || l_tot != l_tot ? 1.f / l_tot : 0.f;
    if (col == 0 && p.lse) put_lse(p, b, h, i, mm, l_tot);
    if (col >= p.cols) return;
    T* ob = (T*)p.o + b * p.o_sb + (int64_t)i * p.o_ss + h * p.o_sh + col;
    if constexpr (Elem<T>::kF32) {
        *reinterpret_cast<f32x4*>(ob) = f32x4{acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    } else {
        s16x4 v4;
#pragma unroll
        for (int e = 0; e < 4; ++e) v4[e] = Elem<T>::pack1(acc[e] * inv);
        *reinterpret_cast<s16x4*>(ob) = v4;
    }
}

template <typename T, int D>
hipError_t launch_rows_t(const RowsParams& p, hipStream_t s) {
    const dim3 grid((unsigned)(p.p_wgs + p.o_wgs));
    if (Elem<T>::kF32 || p.cap > kWideCap)
        hipLaunchKernelGGL((rows_kernel<T, D, true>), grid, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((rows_kernel<T, D, Elem<T>::kF32>), grid, dim3(256), 0, s, p);
    const int n = p.p_splits + p.o_splits;
    if (n > 1) {
        const int64_t n_rows = (int64_t)p.B * p.H * p.Sq;
        constexpr int SLOTS = 256 / (D / 4);
        const int G = n > 16 ? 8 : n > 4 ? 4 : 1;  // up to 8 row-groups a workgroup at D = 128
        const int64_t per = SLOTS / G;
        hipLaunchKernelGGL((rows_join_kernel<T, D>), dim3((unsigned)((n_rows + per - 1) / per)), dim3(256), 0, s, p, n_rows, G);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t launch_rows(const RowsParams& p, int D, hipStream_t s) {
    switch (D) {
        case 32: return launch_rows_t<T, 32>(p, s);
        case 64: return launch_rows_t<T, 64>(p, s);
        case 128: return launch_rows_t<T, 128>(p, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace fa
