// Windowed attention with first tokens that stay visible: the forward.
//   o_i = sum_j p_ij v_j / l_i, p_ij = 2^(c q_i . k_j - m_i), l_i = sum_j p_ij, lse_i = m_i + log2 l_i, c = scale log2 e
// in one pass over the key blocks that any of a workgroup's queries sees, with a running m and l. m moves only
// when a block's maximum exceeds it by more than kLazy, so o is rescaled a few times a row instead of every block;
// weights stay below 2^kLazy and o / l and lse are the same quantities.
//
// Every product is computed transposed so that a lane owns one query: S^T = K Q^T (A: 32 keys from LDS, B: the wave's
// 32 queries in registers) leaves lane l with query l % 32 and keys 8 (v / 4) + 4 (l / 32) + v % 4, v = 0 .. 15, of a
// 32-key half; O^T += V^T P^T (A: V read transposed from LDS, B: P^T as the lane holds it) leaves it with its own query's
// dims, so neither maximum, sum nor rescale needs another lane than l ^ 32.
//
// Weights are rounded to the tensors' type for the product with V, whose operands the matrix units take in 16 bits; their sum l is
// of the weights before that, in f32. That adds half a step a weight to o: against 64 bits o is off by 2.3e-3 of its norm in
// bf16 and 2.8e-4 in f16, where rounding o alone gives 1.7e-3 and 2.1e-4. (Both halves of a weight, high and low, would be exact at
// twice the products with V.)
//
// Measured on MI355X: 2 x 24 heads of 64 x 1088, window 128 both ways, 64 first tokens, bf16 14.7 us (270 TFLOP/s of visible
// pairs); 32 heads of 128 on 8 x 8192, causal window of 1024, 166 to 172 us (750 to 778 TFLOP/s); one query of each of 8 samples, 32 heads on 8,
// a window of 4096 keys, 32.0 us (4.2 TB/s of keys and values).
#include <algorithm>

#include "wattn.h"

namespace {
using namespace sa3k;
using namespace sa3k::wattn;

constexpr int QW = 32;          // queries a wave
constexpr float kLazy = 8.f;    // weights stay below 2^8

struct FwdArgs {
    AttnShape s;
    const void *q, *k, *v;
    void* o;
    float* lse;
    // keys split over workgroups: per (sample, key/value head, chunk of 32 rows, split) o [32][D], m [32] and l [32]
    float* part;
    int splits, chunks;
};

// One query's running softmax over blocks of 64 keys: the state a lane holds.
template <class T, int D>
struct Running {
    typedef typename Vec<T>::x8 x8;
    f32x16 o[D / 32];
    float m = -INFINITY, l = 0.f;

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[i][v] = 0.f;
    }
    // R keys kbase .. of the tiles kt, vt (this query's row sees of them what `see` says; all: every key)
    template <int R>
    __device__ __forceinline__ void block(uint32_t kt, uint32_t vt, const LaneOff& off, const x8 (&qf)[D / 16], int kbase,
                                          const Seen& see, bool all, float c, int lane) {
        constexpr int HALVES = R / 32;
        // Every fragment of K first, then the products, the two halves in turn: left to itself the compiler reads each
        // fragment right before its product and waits for it there.
        f32x16 s[HALVES];
        x8 kf[HALVES][D / 16];
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
            for (int h = 0; h < HALVES; ++h) kf[h][ks] = rd_row<T, R>(kt, off, h, ks);
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int v = 0; v < 16; ++v) s[h][v] = 0.f;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
            for (int h = 0; h < HALVES; ++h) s[h] = Vec<T>::mfma(kf[h][ks], qf[ks], s[h]);
        // the fragments of V arrive while the weights are worked out
        x8 vf[HALVES * 2][D / 32];
#pragma unroll
        for (int j = 0; j < HALVES * 2; ++j)
#pragma unroll
            for (int i = 0; i < D / 32; ++i) vf[j][i] = rd_tr<T, R>(vt, off, j, i);
        __builtin_amdgcn_sched_barrier(0);
        if (!all) {   // (wave-uniform)
            Bits bits;
            bits.set(kbase, see.lo, see.n, see.first, lane);
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int v = 0; v < 16; ++v) s[h][v] = keep_or_none(s[h][v], bits.spread(h, v));
        }
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int v = 0; v < 16; ++v) mx = fmaxf(mx, s[h][v]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c;
        // a maximum moved far (the difference is exact where it matters; m + kLazy may round to m + 16 past 2^27)
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(mx - m > kLazy) != 0, 0)) {
            const float mn = fmaxf(m, mx);
            const float al = ex2(m - (mn == -INFINITY ? 0.f : mn));   // 0 when m was -inf
            m = mn;
            l *= al;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[i][v] *= al;
        }
        const float base = m == -INFINITY ? 0.f : m;   // -inf only while no key was visible: every weight is 0
        x8 p[HALVES][2];
        float ps[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float e = ex2(__builtin_fmaf(s[h][v], c, -base));
                ps[v & 1] += e;
                p[h][v >> 3][v & 7] = (T)e;
            }
        l += ps[0] + ps[1];
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) o[i] = Vec<T>::mfma(vf[2 * h + j][i], p[h][j], o[i]);
    }
};

// 128 queries of one head a workgroup, 32 a wave; tiles of 64 keys, whose loads run STAGES - 1 tiles ahead (three or four
// stages gained nothing). Bound by the work of a block on its SIMD: of a block's time the matrix units are busy for 42% with heads
// of 128 and 18% with heads of 64, the rest are the exponentials, the conversions and the reads of K and V, which the two waves
// of a SIMD hide in each other only partly. A grid that passes over the chip little more than once, as 2 x 24 x 1088 does, lasts
// as long as its eight blocks one after the other, 1.3 us each. Two heads of a group a workgroup, which halves the loads of
// keys and values, was slower (198 us against 178 at 8192 tokens: one workgroup a CU).
template <class T, int D>
__global__ __launch_bounds__(kThreads, 2) void wattn_fwd_kernel(FwdArgs a) {
    constexpr int TILE = BLK * D * 2, STAGES = 2, LOADS = 2 * (D / 64) * (BLK * 8 / kThreads);
    __shared__ __attribute__((aligned(1024))) char lds[STAGES * 2 * TILE];
    const AttnShape& s = a.s;
    const Place pl = place(s, (s.Sq + 127) / 128, blockIdx.x);
    const int nq = clamp_len(s.q_len, pl.b, s.Sq), nk = clamp_len(s.k_len, pl.b, s.Sk), off = nk - nq;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hl = lane >> 5;
    const int q0 = pl.blk * 128;
    if (q0 >= nq) return;   // (workgroup-uniform) nothing but rows past the sample
    const int q0w = q0 + wave * QW, q = q0w + (lane & 31);
    const float c = s.scale * kLog2e;

    const T* qp = static_cast<const T*>(a.q) + pl.b * s.qs[0] + (int64_t)q * s.qs[1] + pl.h * s.qs[2];
    const T* kp = static_cast<const T*>(a.k) + pl.b * s.ks[0] + pl.kh * s.ks[2];
    const T* vp = static_cast<const T*>(a.v) + pl.b * s.vs[0] + pl.kh * s.vs[2];
    typename Vec<T>::x8 qf[D / 16];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = ld_global(qp + ks * 16 + hl * 8, q < nq);

    Seen see = seen_by(q + off, nk, s.left, s.right, s.sinks, s.causal);
    if (q >= nq) see = Seen{0, 0, 0};
    // the wave's reach: its first query sees the lowest keys, its last one the highest and the most first tokens
    const int ql = min(q0w + QW, nq) - 1;
    const Seen sa = seen_by(q0w + off, nk, s.left, s.right, s.sinks, s.causal);
    const Seen sb = seen_by(ql + off, nk, s.left, s.right, s.sinks, s.causal);
    const KeyBlocks kb = key_blocks(q0 + off, min(q0 + 128, nq) - 1 + off, nk, s.left, s.right, s.sinks, s.causal, BLK);

    Running<T, D> run;
    run.clear();
    LaneOff at;
    at.init(lane);
    const uint32_t base = lds_addr(lds);
    auto issue = [&](int st, int i) {
        const int row0 = key_block(kb, i) * BLK;
        tile_dma<D, BLK, kThreads>(kp, s.ks[1], nk, row0, base + st * 2 * TILE, tid, wave);
        tile_dma<D, BLK, kThreads>(vp, s.vs[1], nk, row0, base + st * 2 * TILE + TILE, tid, wave);
    };
    for (int i = 0; i < STAGES - 1 && i < kb.count; ++i) issue(i, i);
    for (int i = 0, st = 0; i < kb.count; ++i, st = st + 1 < STAGES ? st + 1 : 0) {
        wait_tile<STAGES - 2, LOADS>(kb.count - 1 - i);
        if (i + STAGES - 1 < kb.count) issue(st > 0 ? st - 1 : STAGES - 1, i + STAGES - 1);
        const int k0 = key_block(kb, i) * BLK, k1 = k0 + BLK - 1;
        const bool near = q0w < nq && ((k1 >= sa.lo && k0 < sb.lo + sb.n) || k0 < sb.first);
        const bool all = q0w + QW <= nq && ((k0 >= sb.lo && k1 < sa.lo + sa.n) || k1 < sa.first);
        if (near) run.template block<BLK>(base + st * 2 * TILE, base + st * 2 * TILE + TILE, at, qf, k0, see, all, c, lane);
    }
    settle(run.o);
    if (q >= nq) return;
    const float l = run.l + __shfl_xor(run.l, 32, 64);
    if (a.lse && hl == 0) a.lse[((int64_t)pl.b * s.H + pl.h) * s.Sq + q] = run.m + log2f(l);
    const float il = l == 0.f ? 0.f : 1.f / l;   // no visible key: o = 0
    T* op = static_cast<T*>(a.o) + pl.b * s.os[0] + (int64_t)q * s.os[1] + pl.h * s.os[2];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int vg = 0; vg < 4; ++vg) {
            const f32x16& x = run.o[i];
            typename Vec<T>::x4 y = {(T)(x[4 * vg] * il), (T)(x[4 * vg + 1] * il), (T)(x[4 * vg + 2] * il),
                                     (T)(x[4 * vg + 3] * il)};
            *reinterpret_cast<typename Vec<T>::x4*>(op + 32 * i + 8 * vg + 4 * hl) = y;
        }
}

// Few queries over many keys: 32 rows = (query, member of the group) of one key/value head a workgroup, so that the
// group's heads read the keys once, and the keys split over workgroups and over their four waves, each with tiles of
// its own of 32 keys in two stages (no barrier before the end). The waves' results are joined in LDS, the
// workgroups' by a second launch. Bound by HBM: 8 x one query over windows of 4096 keys, 8 key/value heads of 128 (134 MB), 24.9 us,
// 5.4 TB/s, and the join 4.7.
template <class T, int D>
__global__ __launch_bounds__(kThreads) void wattn_split_kernel(FwdArgs a) {
    constexpr int R = 32, TILE = R * D * 2, LOADS = 2 * (D / 64) * (R * 8 / 64);
    __shared__ __attribute__((aligned(1024))) char lds[4 * 2 * 2 * TILE];   // 4 waves x 2 stages x {K, V}
    __shared__ float wm[4][R], wl[4][R];
    const AttnShape& s = a.s;
    const int BK = s.B * s.K, bk = blockIdx.x % BK, rest = blockIdx.x / BK;
    const int b = bk / s.K, kh = bk - b * s.K, chunk = rest % a.chunks, split = rest / a.chunks;
    const int nq = clamp_len(s.q_len, b, s.Sq), nk = clamp_len(s.k_len, b, s.Sk), off = nk - nq;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hl = lane >> 5;
    const int rows = nq * s.G, r0 = chunk * R, r = r0 + (lane & 31);
    if (r0 >= rows) return;   // (workgroup-uniform)
    const int q = r / s.G, h = kh * s.G + (r - q * s.G);
    const float c = s.scale * kLog2e;

    const T* qp = static_cast<const T*>(a.q) + b * s.qs[0] + (int64_t)q * s.qs[1] + h * s.qs[2];
    const T* kp = static_cast<const T*>(a.k) + b * s.ks[0] + kh * s.ks[2];
    const T* vp = static_cast<const T*>(a.v) + b * s.vs[0] + kh * s.vs[2];
    typename Vec<T>::x8 qf[D / 16];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = ld_global(qp + ks * 16 + hl * 8, r < rows);
    Seen see = seen_by(q + off, nk, s.left, s.right, s.sinks, s.causal);
    if (r >= rows) see = Seen{0, 0, 0};
    const int pa = r0 / s.G + off, pb = (min(r0 + R, rows) - 1) / s.G + off;
    const Seen sa = seen_by(pa, nk, s.left, s.right, s.sinks, s.causal);
    const Seen sb = seen_by(pb, nk, s.left, s.right, s.sinks, s.causal);
    const KeyBlocks kb = key_blocks(pa, pb, nk, s.left, s.right, s.sinks, s.causal, R);
    const int per = (kb.count + a.splits - 1) / a.splits;
    const int lo = min(kb.count, split * per) + wave, hi = min(kb.count, (split + 1) * per);

    Running<T, D> run;
    run.clear();
    LaneOff at;
    at.init(lane);
    const uint32_t mine = lds_addr(lds) + wave * 4 * TILE;
    auto issue = [&](int st, int i) {
        const int row0 = key_block(kb, i) * R;
        tile_dma<D, R, 64>(kp, s.ks[1], nk, row0, mine + st * 2 * TILE, lane, 0);
        tile_dma<D, R, 64>(vp, s.vs[1], nk, row0, mine + st * 2 * TILE + TILE, lane, 0);
    };
    wait_own_loads<0>();   // the queries: from here on only tiles are in flight
    if (lo < hi) issue(0, lo);
    int st = 0;
    for (int i = lo; i < hi; i += 4, st ^= 1) {
        if (i + 4 < hi) {
            wait_own_loads<63>();   // the other stage's reads have returned
            issue(st ^ 1, i + 4);
            wait_own_loads<LOADS>();
        } else {
            wait_own_loads<0>();
        }
        const int k0 = key_block(kb, i) * R, k1 = k0 + R - 1;
        const bool all = r0 + R <= rows && ((k0 >= sb.lo && k1 < sa.lo + sa.n) || k1 < sa.first);
        run.template block<R>(mine + st * 2 * TILE, mine + st * 2 * TILE + TILE, at, qf, k0, see, all, c, lane);
    }
    settle(run.o);
    // join the waves: common maximum, then the sums of the rescaled o and l in wave order
    const float l = run.l + __shfl_xor(run.l, 32, 64);
    if (hl == 0) {
        wm[wave][lane] = run.m;
        wl[wave][lane] = l;
    }
    __syncthreads();   // every wave is done with its tiles
    constexpr int OS = D + 4;   // floats a staged row
    static_assert(2 * R * OS * 4 <= (int)sizeof(lds), "two waves' rows fit the tiles' memory");
    const int c32 = lane & 31;
    const float M = fmaxf(fmaxf(wm[0][c32], wm[1][c32]), fmaxf(wm[2][c32], wm[3][c32]));
    const float f = ex2(run.m - (M == -INFINITY ? 0.f : M));
    float* stage = reinterpret_cast<float*>(lds);
    // two rounds of two waves each, so that the staging fits the tiles' memory
    const int row = tid >> 3, part8 = tid & 7;
    constexpr int PER = D / 8;   // floats of its row that a thread sums
    float acc[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll
    for (int round = 0; round < 2; ++round) {
        if (wave >> 1 == round) {
            float* p = stage + ((wave & 1) * R + c32) * OS + 4 * hl;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int vg = 0; vg < 4; ++vg)
                    *reinterpret_cast<float4*>(p + 32 * i + 8 * vg) =
                        make_float4(run.o[i][4 * vg] * f, run.o[i][4 * vg + 1] * f, run.o[i][4 * vg + 2] * f,
                                    run.o[i][4 * vg + 3] * f);
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int e = 0; e < PER; e += 4) {
                const float4 x = *reinterpret_cast<const float4*>(stage + (w * R + row) * OS + part8 * PER + e);
                acc[e] += x.x;
                acc[e + 1] += x.y;
                acc[e + 2] += x.z;
                acc[e + 3] += x.w;
            }
        __syncthreads();
    }
    const float Mr = fmaxf(fmaxf(wm[0][row], wm[1][row]), fmaxf(wm[2][row], wm[3][row]));
    const float base = Mr == -INFINITY ? 0.f : Mr;
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) L += wl[w][row] * ex2(wm[w][row] - base);
    if (r0 + row >= rows) return;
    if (a.splits > 1) {
        float* p = a.part + (((int64_t)bk * a.chunks + chunk) * a.splits + split) * (R * (D + 2));
#pragma unroll
        for (int e = 0; e < PER; e += 4)
            *reinterpret_cast<float4*>(p + row * D + part8 * PER + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
        if (part8 == 0) {
            p[R * D + row] = Mr;
            p[R * D + R + row] = L;
        }
        return;
    }
    const int qr = (r0 + row) / s.G, hr = kh * s.G + (r0 + row - qr * s.G);
    const float il = L == 0.f ? 0.f : 1.f / L;
    T* op = static_cast<T*>(a.o) + b * s.os[0] + (int64_t)qr * s.os[1] + hr * s.os[2] + part8 * PER;
#pragma unroll
    for (int e = 0; e < PER; e += 8) {
        typename Vec<T>::x8 y;
#pragma unroll
        for (int u = 0; u < 8; ++u) y[u] = (T)(acc[e + u] * il);
        *reinterpret_cast<typename Vec<T>::x8*>(op + e) = y;
    }
    if (a.lse && part8 == 0) a.lse[((int64_t)b * s.H + hr) * s.Sq + qr] = Mr + log2f(L);
}

// The splits' results of eight rows a workgroup, 32 threads a row: o = sum_z o_z 2^(m_z - M) / sum_z l_z 2^(m_z - M), in
// the order of the splits.
template <class T, int D>
__global__ __launch_bounds__(kThreads) void wattn_join_kernel(FwdArgs a) {
    constexpr int R = 32, PER = D / 32;
    const AttnShape& s = a.s;
    const int BK = s.B * s.K, bk = blockIdx.x % BK, rest = blockIdx.x / BK;
    const int b = bk / s.K, kh = bk - b * s.K, chunk = rest >> 2;
    const int row = (rest & 3) * 8 + (threadIdx.x >> 5), d0 = (threadIdx.x & 31) * PER;
    const int r = chunk * R + row;
    if (r >= clamp_len(s.q_len, b, s.Sq) * s.G) return;
    const int64_t step = R * (D + 2);
    const float* p = a.part + ((int64_t)bk * a.chunks + chunk) * a.splits * step;
    const float *pm = p + R * D + row, *plw = pm + R, *po = p + row * D + d0;
    // a lane a split for the maximum and the factors, the row's 32 lanes in step; then the sums, eight splits in flight
    const int z0 = threadIdx.x & 31;
    float M = -INFINITY;
    for (int z = z0; z < a.splits; z += 32) M = fmaxf(M, pm[z * step]);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float base = M == -INFINITY ? 0.f : M;
    float acc[PER], L = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = 0.f;
    for (int zb = 0; zb < a.splits; zb += 32) {
        const int z = zb + z0;
        const float mine = z < a.splits ? ex2(pm[z * step] - base) : 0.f;
        L += z < a.splits ? plw[z * step] * mine : 0.f;
        for (int k = 0; k < 32 && zb + k < a.splits; k += 8) {
            float v[8][PER];
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < PER; ++e) v[u][e] = po[min(zb + k + u, a.splits - 1) * step + e];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float f = __shfl(mine, (threadIdx.x & 32) + k + u, 64);   // 0 past the last split
#pragma unroll
                for (int e = 0; e < PER; ++e) acc[e] = __builtin_fmaf(v[u][e], f, acc[e]);
            }
        }
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) L += __shfl_xor(L, o, 64);
    const int q = r / s.G, h = kh * s.G + (r - q * s.G);
    const float il = L == 0.f ? 0.f : 1.f / L;
    T* op = static_cast<T*>(a.o) + b * s.os[0] + (int64_t)q * s.os[1] + h * s.os[2] + d0;
#pragma unroll
    for (int e = 0; e < PER; ++e) op[e] = (T)(acc[e] * il);
    if (a.lse && d0 == 0) a.lse[((int64_t)b * s.H + h) * s.Sq + q] = M + log2f(L);
}

template <class T, int D>
void fwd_run(sa3k_ctx* ctx, FwdArgs& a) {
    const AttnShape& s = a.s;
    if (attn_split_keys(s)) {
        a.chunks = (int)ceil_div((int64_t)s.Sq * s.G, 32);
        a.splits = attn_splits(s, a.chunks);
        if (a.splits > 1)
            a.part = layer_workspace(ctx, (size_t)s.B * s.K * a.chunks * a.splits * 32 * (D + 2) * sizeof(float));
        {
            KernelScope ks(ctx, "window_attn_split");
            launch_k(ctx, a.splits == 1, wattn_split_kernel<T, D>, dim3((unsigned)(s.B * s.K) * a.chunks * a.splits),
                     dim3(kThreads), 0, a);
            SA3K_LAUNCHED();
        }
        if (a.splits > 1) {
            KernelScope ks(ctx, "window_attn_join");
            launch_k(ctx, true, wattn_join_kernel<T, D>, dim3((unsigned)(s.B * s.K) * a.chunks * 4), dim3(kThreads), 0, a);
            SA3K_LAUNCHED();
        }
        return;
    }
    KernelScope ks(ctx, "window_attn_fwd");
    const unsigned grid = (unsigned)(ceil_div(s.Sq, 128) * s.B * s.H);
    launch_k(ctx, true, wattn_fwd_kernel<T, D>, dim3(grid), dim3(kThreads), 0, a);
    SA3K_LAUNCHED();
}

}  // namespace

extern "C" {

SA3K_API int sa3k_window_attn_fwd(sa3k_ctx* ctx, const sa3k_window_attn* d, const void* q, const void* k, const void* v,
                                  const int32_t* q_len, const int32_t* k_len, void* o, float* lse) {
    return sa3k_guard(ctx, "sa3k_window_attn_fwd", [&] {
        AttnPtrs p;
        p.q = q; p.k = k; p.v = v; p.o = o; p.lse = lse; p.q_len = q_len; p.k_len = k_len;
        int code;
        const char* msg = attn_check(d, p, false, &code);
        require_ok(msg, code);
        if (d->batch == 0 || d->q_tokens == 0) return;
        DeviceScope dev(ctx);
        FwdArgs a{};
        a.s = attn_shape(*d, q_len, k_len);
        a.q = q; a.k = k; a.v = v; a.o = o; a.lse = lse;
        const bool b16 = d->type == SA3K_TYPE_BF16;
        if (d->head_dim == 64) b16 ? fwd_run<bf16, 64>(ctx, a) : fwd_run<f16, 64>(ctx, a);
        else b16 ? fwd_run<bf16, 128>(ctx, a) : fwd_run<f16, 128>(ctx, a);
    });
}

}  // extern "C"
