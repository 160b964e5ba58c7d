// Windowed attention with first tokens that stay visible: the backward. With p_ij = 2^(c q_i . k_j - lse_i) from
// recomputed scores, delta_i = dO_i . o_i (a launch of its own) and ds_ij = p_ij (dO_i . v_j - delta_i):
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij dO_i
// Two passes, each over the scores of every visible block, so that no sum is shared between workgroups (no atomics:
// the same bits in every run): one by queries (dq), one by keys (dk, dv, over all the query heads of a group). Seven
// products of 2 D a pair where five would do with dq summed by atomics. p and ds are rounded to the tensors' type for the products
// that take them, as the matrix units read 16 bits: against 64 bits the gradients are off by 2.4e-3 of their norm in bf16 and
// 3.0e-4 in f16, where their own rounding alone gives 1.7e-3 and 2.1e-4.
//
// Measured on MI355X (whole calls): 2 x 24 heads of 64 x 1088, window 128 both ways, 64 first tokens, bf16 41 us; 3 x 16 heads of
// 128 on 2, up to 2049 tokens, causal window of 512, 4 first tokens, f16 131 us (350 TFLOP/s of five products). Bound by the work
// of a block on its SIMD, as the forward: the matrix units are busy for 37% of the time with heads of 128 and 22% with heads of
// 64; the sums fill a lane's registers, so that two waves a SIMD is all there is. Not kept: pairs of waves that share a tile,
// one for dk and one for dv (dK/dV pass 116 us against 78), three waves a SIMD with heads of 64 (47 us against 40).
//
// By queries: S^T = K Q^T and dP^T = V dO^T leave a lane with one query, dq^T += K^T dS^T reads K transposed.
// By keys: S = Q K^T and dP = dO V^T leave it with one key, dv^T += dO^T P and dk^T += Q^T dS read dO and Q transposed.
#include <algorithm>
#include <type_traits>

#include "wattn.h"

namespace {
using namespace sa3k;
using namespace sa3k::wattn;

struct BwdArgs {
    AttnShape s;
    const void *q, *k, *v, *o, *dO;
    const float* lse;
    float* delta;   // [B][H][Sq]
    void *dq, *dk, *dv;
    KeySplit split;
    float* part;    // per (sample, key/value head, share) dk [128][D] and dv [128][D], of tiles with more than one share
};

template <class T>
__device__ __forceinline__ float dot8(typename Vec<T>::x8 a, typename Vec<T>::x8 b) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf((float)a[e], (float)b[e], s);
    return s;
}

// four values a lane at dims 32 i + 8 vg + 4 hl of its row
template <class T, int D>
__device__ __forceinline__ void store_row(T* p, const f32x16 (&x)[D / 32], float f, int hl) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int vg = 0; vg < 4; ++vg) {
            typename Vec<T>::x4 y = {(T)(x[i][4 * vg] * f), (T)(x[i][4 * vg + 1] * f), (T)(x[i][4 * vg + 2] * f),
                                     (T)(x[i][4 * vg + 3] * f)};
            *reinterpret_cast<typename Vec<T>::x4*>(p + 32 * i + 8 * vg + 4 * hl) = y;
        }
}

// delta = dO . o of every row: D / 8 lanes a row, 8 dims each. One pass over dO and o (3 x 16 x 2049 rows of 128 f16: 9.2 us with
// the launch).
template <class T, int D>
__global__ __launch_bounds__(kThreads) void wattn_delta_kernel(BwdArgs a) {
    constexpr int L = D / 8;
    const AttnShape& s = a.s;
    const int64_t i = (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L;   // row [b][q][h]: heads lie together
    const int h = (int)(i % s.H);
    const int64_t bq = i / s.H;
    const int b = (int)(bq / s.Sq), q = (int)(bq - (int64_t)b * s.Sq);
    const bool ok = b < s.B && q < clamp_len(s.q_len, min(b, s.B - 1), s.Sq);
    const int64_t off = b * s.os[0] + (int64_t)q * s.os[1] + h * s.os[2] + (threadIdx.x % L) * 8;
    float d = dot8<T>(ld_global(static_cast<const T*>(a.dO) + off, ok), ld_global(static_cast<const T*>(a.o) + off, ok));
#pragma unroll
    for (int o = 1; o < L; o <<= 1) d += __shfl_xor(d, o, 64);
    if (ok && threadIdx.x % L == 0) a.delta[((int64_t)b * s.H + h) * s.Sq + q] = d;
}

// 128 queries of one head a workgroup (`index` of them), 32 a wave; key tiles as in the forward.
template <class T, int D>
__device__ __forceinline__ void dq_body(const BwdArgs& a, int index, char* lds) {
    typedef typename Vec<T>::x8 x8;
    constexpr int TILE = BLK * D * 2, STAGES = 2, LOADS = 2 * (D / 64) * (BLK * 8 / kThreads);
    const AttnShape& s = a.s;
    const Place pl = place(s, (s.Sq + 127) / 128, index);
    const int nq = clamp_len(s.q_len, pl.b, s.Sq), nk = clamp_len(s.k_len, pl.b, s.Sk), off = nk - nq;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hl = lane >> 5;
    const int c32 = lane & 31;
    const int q0 = pl.blk * 128;
    if (q0 >= nq) return;   // (workgroup-uniform)
    const int q0w = q0 + wave * 32, q = q0w + c32;
    const float c = s.scale * kLog2e;
    const int64_t qoff = pl.b * s.qs[0] + (int64_t)q * s.qs[1] + pl.h * s.qs[2];
    const int64_t ooff = pl.b * s.os[0] + (int64_t)q * s.os[1] + pl.h * s.os[2];
    const T* kp = static_cast<const T*>(a.k) + pl.b * s.ks[0] + pl.kh * s.ks[2];
    const T* vp = static_cast<const T*>(a.v) + pl.b * s.vs[0] + pl.kh * s.vs[2];
    const int64_t row = ((int64_t)pl.b * s.H + pl.h) * s.Sq + q;
    x8 qf[D / 16], dof[D / 16];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        qf[ks] = ld_global(static_cast<const T*>(a.q) + qoff + ks * 16 + hl * 8, q < nq);
        dof[ks] = ld_global(static_cast<const T*>(a.dO) + ooff + ks * 16 + hl * 8, q < nq);
    }
    const float lse = q < nq ? a.lse[row] : 0.f, delta = q < nq ? a.delta[row] : 0.f;

    Seen see = seen_by(q + off, nk, s.left, s.right, s.sinks, s.causal);
    if (q >= nq) see = Seen{0, 0, 0};
    const int ql = min(q0w + 32, nq) - 1;
    const Seen sa = seen_by(q0w + off, nk, s.left, s.right, s.sinks, s.causal);
    const Seen sb = seen_by(ql + off, nk, s.left, s.right, s.sinks, s.causal);
    const KeyBlocks kb = key_blocks(q0 + off, min(q0 + 128, nq) - 1 + off, nk, s.left, s.right, s.sinks, s.causal, BLK);
    f32x16 dq[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) dq[i][v] = 0.f;

    LaneOff at;
    at.init(lane);
    const uint32_t base = lds_addr(lds);
    auto issue = [&](int st, int i) {
        const int row0 = key_block(kb, i) * BLK;
        tile_dma<D, BLK, kThreads>(kp, s.ks[1], nk, row0, base + st * 2 * TILE, tid, wave);
        tile_dma<D, BLK, kThreads>(vp, s.vs[1], nk, row0, base + st * 2 * TILE + TILE, tid, wave);
    };
    for (int it = 0; it < STAGES - 1 && it < kb.count; ++it) issue(it, it);
    for (int it = 0, st = 0; it < kb.count; ++it, st = st + 1 < STAGES ? st + 1 : 0) {
        wait_tile<STAGES - 2, LOADS>(kb.count - 1 - it);
        if (it + STAGES - 1 < kb.count) issue(st > 0 ? st - 1 : STAGES - 1, it + STAGES - 1);
        const int k0 = key_block(kb, it) * BLK, k1 = k0 + BLK - 1;
        const bool near = (k1 >= sa.lo && k0 < sb.lo + sb.n) || k0 < sb.first;
        if (q0w >= nq || !near) continue;   // this wave sees nothing of this block
        const bool all = q0w + 32 <= nq && ((k0 >= sb.lo && k1 < sa.lo + sa.n) || k1 < sa.first);
        Bits bits;
        bits.set(k0, see.lo, see.n, see.first, lane);
        const uint32_t kt = base + st * 2 * TILE, vt = kt + TILE;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // K and V fragments first, then their products in turn, then the transposed K while the weights are worked out
            x8 kf[D / 16], vf[D / 16];
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                kf[ks] = rd_row<T, BLK>(kt, at, h, ks);
                vf[ks] = rd_row<T, BLK>(vt, at, h, ks);
            }
            f32x16 sc, dp;
#pragma unroll
            for (int v = 0; v < 16; ++v) sc[v] = dp[v] = 0.f;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                sc = Vec<T>::mfma(kf[ks], qf[ks], sc);
                dp = Vec<T>::mfma(vf[ks], dof[ks], dp);
            }
            x8 tf[2][D / 32];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) tf[j][i] = rd_tr<T, BLK>(kt, at, 2 * h + j, i);
            __builtin_amdgcn_sched_barrier(0);
            x8 ds[2];
            if (all) {
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    ds[v >> 3][v & 7] = (T)(ex2(__builtin_fmaf(sc[v], c, -lse)) * (dp[v] - delta));
            } else {
#pragma unroll
                for (int v = 0; v < 16; ++v)   // (a row that sees nothing has lse = -inf)
                    ds[v >> 3][v & 7] = (T)keep(ex2(__builtin_fmaf(sc[v], c, -lse)) * (dp[v] - delta), bits.spread(h, v));
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) dq[i] = Vec<T>::mfma(tf[j][i], ds[j], dq[i]);
        }
    }
    settle(dq);
    if (q < nq) store_row<T, D>(static_cast<T*>(a.dq) + qoff, dq, s.scale, hl);
}

// 128 keys of one key/value head a workgroup, 32 a wave; tiles of 64 queries' q and dO with their lse and delta.
template <class T, int D>
__device__ __forceinline__ void dkdv_body(const BwdArgs& a, int index, char* lds, float (&vec)[2][2][BLK]) {
    typedef typename Vec<T>::x8 x8;
    constexpr int TILE = BLK * D * 2, STAGES = 2, LOADS = 2 * (D / 64) * (BLK * 8 / kThreads) + 1;
    const AttnShape& s = a.s;
    const int BK = s.B * s.K, bk = index % BK, item = index / BK;
    const int b = bk / s.K, kh = bk - b * s.K;
    const KeyItem ki = key_item(a.split, item);
    const int nq = clamp_len(s.q_len, b, s.Sq), nk = clamp_len(s.k_len, b, s.Sk), off = nk - nq;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hl = lane >> 5;
    const int c32 = lane & 31;
    const int k0 = ki.tile * kKeyTile;
    if (k0 >= nk) return;   // (workgroup-uniform)
    const int k0w = k0 + wave * 32, key = k0w + c32;
    const float c = s.scale * kLog2e;
    const int64_t koff = b * s.ks[0] + (int64_t)key * s.ks[1] + kh * s.ks[2];
    const int64_t voff = b * s.vs[0] + (int64_t)key * s.vs[1] + kh * s.vs[2];
    x8 kf[D / 16], vf[D / 16];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        kf[ks] = ld_global(static_cast<const T*>(a.k) + koff + ks * 16 + hl * 8, key < nk);
        vf[ks] = ld_global(static_cast<const T*>(a.v) + voff + ks * 16 + hl * 8, key < nk);
    }
    // the queries that see this lane's key, the wave's, the workgroup's
    Span mine = seen_from(key, key, nq, off, s.left, s.right, s.sinks, s.causal);
    if (key >= nk) mine = Span{0, -1};
    const unsigned mine_n = (unsigned)max(0, mine.hi - mine.lo + 1);
    const int klw = min(k0w + 31, nk - 1);
    const Span reach = seen_from(k0w, klw, nq, off, s.left, s.right, s.sinks, s.causal);
    const Span wg = seen_from(k0, min(k0 + kKeyTile, nk) - 1, nq, off, s.left, s.right, s.sinks, s.causal);
    // queries that see every one of the wave's keys: of those past the first tokens the lowest reaches least far up
    const int kfw = klw >= s.sinks ? max(k0w, s.sinks) : k0w;
    const Span fa = seen_from(kfw, kfw, nq, off, s.left, s.right, s.sinks, s.causal);
    const Span fb = seen_from(klw, klw, nq, off, s.left, s.right, s.sinks, s.causal);
    const int full_lo = max(fa.lo, fb.lo), full_hi = k0w + 32 <= nk ? min(fa.hi, fb.hi) : -1;
    const int qb_lo = wg.lo / BLK, nqb = wg.hi >= wg.lo ? wg.hi / BLK + 1 - qb_lo : 0, total = nqb * s.G;
    const int per = (total + ki.splits - 1) / ki.splits;
    const int lo = min(total, ki.split * per), hi = min(total, lo + per);

    f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) dk[i][v] = dv[i][v] = 0.f;
    LaneOff at;
    at.init(lane);
    const uint32_t base = lds_addr(lds);
    auto issue = [&](int st, int it) {
        const int g = it / nqb, row0 = (qb_lo + it - g * nqb) * BLK, h = kh * s.G + g;
        const T* qp = static_cast<const T*>(a.q) + b * s.qs[0] + h * s.qs[2];
        const T* op = static_cast<const T*>(a.dO) + b * s.os[0] + h * s.os[2];
        tile_dma<D, BLK, kThreads>(qp, s.qs[1], nq, row0, base + st * 2 * TILE, tid, wave);
        tile_dma<D, BLK, kThreads>(op, s.os[1], nq, row0, base + st * 2 * TILE + TILE, tid, wave);
        const int64_t r = ((int64_t)b * s.H + h) * s.Sq;
        // (two waves load each, the same values, so that every wave has the same number of loads under way)
        vec_dma((wave & 1 ? a.delta : a.lse) + r, nq, row0, vec[st][wave & 1], lane);
    };
    for (int it = 0; it < STAGES - 1 && lo + it < hi; ++it) issue(it, lo + it);
    for (int it = lo, st = 0; it < hi; ++it, st = st + 1 < STAGES ? st + 1 : 0) {
        wait_tile<STAGES - 2, LOADS>(hi - 1 - it);
        if (it + STAGES - 1 < hi) issue(st > 0 ? st - 1 : STAGES - 1, it + STAGES - 1);
        const int q0 = (qb_lo + it % nqb) * BLK, q1 = q0 + BLK - 1;
        if (k0w >= nk || q0 > reach.hi || q1 < reach.lo) continue;   // nothing of this block sees the wave's keys
        const bool all = q0 >= full_lo && q1 <= full_hi;
        Bits bits;
        bits.set(q0, mine.lo, (int)mine_n, 0, lane);
        const uint32_t qt = base + st * 2 * TILE, ot = qt + TILE;
#pragma unroll 1   // (unrolled, more sums are alive than a lane's 256 registers hold)
        for (int h = 0; h < 2; ++h) {
            // fragments in batches, each read while the batch before is multiplied
            constexpr int FB = D == 64 ? 4 : 1, NB = D / 16 / FB;   // FB fragments of q and of dO a batch
            f32x16 sc, dp;
#pragma unroll
            for (int v = 0; v < 16; ++v) sc[v] = dp[v] = 0.f;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                x8 qf[FB], of[FB];
#pragma unroll
                for (int k4 = 0; k4 < FB; ++k4) {
                    qf[k4] = rd_row<T, BLK>(qt, at, h, FB * nb + k4);
                    of[k4] = rd_row<T, BLK>(ot, at, h, FB * nb + k4);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k4 = 0; k4 < FB; ++k4) {
                    sc = Vec<T>::mfma(qf[k4], kf[FB * nb + k4], sc);
                    dp = Vec<T>::mfma(of[k4], vf[FB * nb + k4], dp);
                }
            }
            x8 p[2], ds[2];
            const uint32_t word = h ? bits.w[1] : bits.w[0];
            // MASK 0: every pair visible, 1: by the bits, 2: by the bits if not all are. For heads of 64 the code is written out
            // for both; for heads of 128 that spills sums, and a branch an element costs less.
            auto weights = [&](auto mask) {
                constexpr int MASK = decltype(mask)::value;
#pragma unroll
                for (int vg = 0; vg < 4; ++vg) {
                    const float4 l4 = *reinterpret_cast<const float4*>(&vec[st][0][32 * h + 8 * vg + 4 * hl]);
                    const float4 d4 = *reinterpret_cast<const float4*>(&vec[st][1][32 * h + 8 * vg + 4 * hl]);
                    const float ls[4] = {l4.x, l4.y, l4.z, l4.w}, dl[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int v = 4 * vg + u;
                        float w = ex2(__builtin_fmaf(sc[v], c, -ls[u]));
                        float x = w * (dp[v] - dl[u]);
                        if (MASK == 1 || (MASK == 2 && !all)) {
                            const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)word, 8 * vg + u, 1);
                            w = keep(w, m);
                            x = keep(x, m);
                        }
                        p[v >> 3][v & 7] = (T)w;
                        ds[v >> 3][v & 7] = (T)x;
                    }
                }
            };
            if constexpr (D == 128) {
                weights(std::integral_constant<int, 2>{});
            } else {
                if (all) weights(std::integral_constant<int, 0>{});
                else weights(std::integral_constant<int, 1>{});
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                x8 tf[D / 32];
#pragma unroll
                for (int i = 0; i < D / 32; ++i) tf[i] = rd_tr<T, BLK>(ot, at, 2 * h + j, i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) dv[i] = Vec<T>::mfma(tf[i], p[j], dv[i]);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) tf[i] = rd_tr<T, BLK>(qt, at, 2 * h + j, i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) dk[i] = Vec<T>::mfma(tf[i], ds[j], dk[i]);
            }
        }
    }
    settle(dk);
    settle(dv);
    if (key >= nk) return;
    if (ki.splits == 1) {
        store_row<T, D>(static_cast<T*>(a.dk) + koff, dk, s.scale, hl);
        store_row<T, D>(static_cast<T*>(a.dv) + voff, dv, 1.f, hl);
        return;
    }
    float* pk = a.part + ((int64_t)bk * a.split.shares() + item) * (2 * kKeyTile * D) + (wave * 32 + c32) * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int vg = 0; vg < 4; ++vg) {
            float* p = pk + 32 * i + 8 * vg + 4 * hl;
            *reinterpret_cast<float4*>(p) =
                make_float4(dk[i][4 * vg] * s.scale, dk[i][4 * vg + 1] * s.scale, dk[i][4 * vg + 2] * s.scale,
                            dk[i][4 * vg + 3] * s.scale);
            *reinterpret_cast<float4*>(p + kKeyTile * D) =
                make_float4(dv[i][4 * vg], dv[i][4 * vg + 1], dv[i][4 * vg + 2], dv[i][4 * vg + 3]);
        }
}

// Both passes in one launch: the workgroups by keys, which run longer, first, then those by queries, so that neither
// pass's last turn leaves the chip partly empty.
template <class T, int D>
__global__ __launch_bounds__(kThreads, 2) void wattn_bwd_kernel(BwdArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[2 * 2 * BLK * D * 2];
    __shared__ __attribute__((aligned(16))) float vec[2][2][BLK];   // lse, delta
    const int by_key = a.s.Sk > 0 ? a.s.B * a.s.K * a.split.items() : 0, i = blockIdx.x;
    if (i < by_key) dkdv_body<T, D>(a, i, lds, vec);
    else dq_body<T, D>(a, i - by_key, lds);
}

// dk and dv of the tiles with more than one share: the shares' sums in their order, 8 dims a thread. (3 x 2 x 2049 keys of 128:
// 9.0 us.)
template <class T, int D>
__global__ __launch_bounds__(kThreads) void wattn_dkdv_sum_kernel(BwdArgs a, int tiles) {
    typedef typename Vec<T>::x8 x8;
    constexpr int CPR = D / 8, ROWS = kThreads / CPR, GROUPS = kKeyTile / ROWS;
    const AttnShape& s = a.s;
    const int BK = s.B * s.K, bk = blockIdx.x % BK, rest = blockIdx.x / BK;
    const int b = bk / s.K, kh = bk - b * s.K, tile = rest / GROUPS;
    const int r = (rest - tile * GROUPS) * ROWS + threadIdx.x / CPR, d0 = (threadIdx.x % CPR) * 8;
    const int key = tile * kKeyTile + r;
    if (key >= clamp_len(s.k_len, b, s.Sk)) return;
    const bool first = tile < a.split.first_tiles;
    const int n = first ? a.split.first : a.split.rest;
    const int item = first ? tile * n : a.split.first_tiles * a.split.first + (tile - a.split.first_tiles) * n;
    const float* p = a.part + ((int64_t)bk * a.split.shares() + item) * (2 * kKeyTile * D) + (int64_t)r * D + d0;
    float x[2][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[0][e] = x[1][e] = 0.f;
    for (int z = 0; z < n; ++z, p += 2 * kKeyTile * D)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 y = *reinterpret_cast<const float4*>(p + u * kKeyTile * D + e);
                x[u][e] += y.x;
                x[u][e + 1] += y.y;
                x[u][e + 2] += y.z;
                x[u][e + 3] += y.w;
            }
    x8 yk, yv;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        yk[e] = (T)x[0][e];
        yv[e] = (T)x[1][e];
    }
    *reinterpret_cast<x8*>(static_cast<T*>(a.dk) + b * s.ks[0] + (int64_t)key * s.ks[1] + kh * s.ks[2] + d0) = yk;
    *reinterpret_cast<x8*>(static_cast<T*>(a.dv) + b * s.vs[0] + (int64_t)key * s.vs[1] + kh * s.vs[2] + d0) = yv;
}

template <class T, int D>
void bwd_run(sa3k_ctx* ctx, BwdArgs& a) {
    const AttnShape& s = a.s;
    a.split = key_split(s);
    // tiles whose shares a second launch adds up: those with first tokens only, or all
    const int summed = a.split.rest > 1 ? a.split.tiles : a.split.first > 1 ? a.split.first_tiles : 0;
    const size_t nd = ((size_t)s.B * s.H * s.Sq + 63) / 64 * 64;
    const size_t np = (size_t)s.B * s.K * a.split.shares() * 2 * kKeyTile * D;
    a.delta = layer_workspace(ctx, (nd + np) * sizeof(float));
    a.part = a.delta + nd;
    if (s.Sq > 0) {
        KernelScope ks(ctx, "window_attn_delta");
        launch_k(ctx, false, wattn_delta_kernel<T, D>, dim3((unsigned)ceil_div((int64_t)s.B * s.H * s.Sq, kThreads / (D / 8))),
                 dim3(kThreads), 0, a);
        SA3K_LAUNCHED();
    }
    {
        const int64_t by_key = s.Sk > 0 ? (int64_t)s.B * s.K * a.split.items() : 0, by_query = ceil_div(s.Sq, 128) * s.B * s.H;
        if (by_key + by_query == 0) return;
        KernelScope ks(ctx, "window_attn_bwd");
        launch_k(ctx, summed == 0, wattn_bwd_kernel<T, D>, dim3((unsigned)(by_key + by_query)), dim3(kThreads), 0, a);
        SA3K_LAUNCHED();
    }
    if (summed) {
        KernelScope ks(ctx, "window_attn_dkdv_sum");
        launch_k(ctx, true, wattn_dkdv_sum_kernel<T, D>, dim3((unsigned)(s.B * s.K) * summed * (kKeyTile * D / 8 / kThreads)),
                 dim3(kThreads), 0, a, summed);
        SA3K_LAUNCHED();
    }
}

}  // namespace

extern "C" {

SA3K_API int sa3k_window_attn_bwd(sa3k_ctx* ctx, const sa3k_window_attn* d, const void* q, const void* k, const void* v,
                                  const void* o, const float* lse, const void* dO, const int32_t* q_len,
                                  const int32_t* k_len, void* dq, void* dk, void* dv) {
    return sa3k_guard(ctx, "sa3k_window_attn_bwd", [&] {
        AttnPtrs p;
        p.q = q; p.k = k; p.v = v; p.o = o; p.lse = lse; p.dO = dO; p.q_len = q_len; p.k_len = k_len;
        p.dq = dq; p.dk = dk; p.dv = dv;
        int code;
        const char* msg = attn_check(d, p, true, &code);
        require_ok(msg, code);
        if (d->batch == 0) return;
        DeviceScope dev(ctx);
        BwdArgs a{};
        a.s = attn_shape(*d, q_len, k_len);
        a.q = q; a.k = k; a.v = v; a.o = o; a.lse = lse; a.dO = dO;
        a.dq = dq; a.dk = dk; a.dv = dv;
        const bool b16 = d->type == SA3K_TYPE_BF16;
        if (d->head_dim == 64) b16 ? bwd_run<bf16, 64>(ctx, a) : bwd_run<f16, 64>(ctx, a);
        else b16 ? bwd_run<bf16, 128>(ctx, a) : bwd_run<f16, 128>(ctx, a);
    });
}

}  // extern "C"
