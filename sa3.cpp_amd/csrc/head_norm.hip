// RMS norm of the heads of q and k with the position rotation in the same pass, forward and backward; a new token's k and v
// into their row of a cache in the same launch.
//   forward    r = 1 / sqrt(mean x^2 + eps), n = x r gain, y = R n, R turning each pair (a, b) of the first rope_dims
//              elements by its angle: (a cos - b sin, b cos + a sin)
//   backward   w = R^T dy, dgain = sum over tokens and heads w x r, h = w gain, dx = r (h - x r mean(h x r))
// The statistics are worked out again in the backward, from the x it reads anyway. All arithmetic in f32, each output rounded once.
//
// Eight elements of a head a lane, 4 to 32 lanes a head, several heads a wave. A wave takes up to three such groups of heads of one row
// (token) and one tensor, so that nothing but the lane's own head is chosen inside it; the row's sines and cosines, which the heads share,
// are worked out a pair a lane while the loads are under way. Angles are taken modulo a turn in whole numbers (head_turns), so a position a
// million tokens out is as good as the first.
//
// Forward bound by HBM, or by a launch. Measured on MI355X: 8192 x (32 + 8) heads of 128 f16 33.0 us with its inputs in the memory-side
// cache (5.1 TB/s), 38 a call without, f32 70 a call (4.8 TB/s); 2 x 1088 x (24 + 24) heads of 64 bf16 8.4 (3.2 TB/s, one round of loads); 8
// new tokens 5.2. Backward 3 x 2049 x (16 + 2) heads of 128 f32 27.5 (5.1 TB/s) and 4.9 for the second launch; 2 x 1088 x (24 + 24) bf16
// 12.8 and 3.9, bound by latency: two waves a SIMD, two rows each one after the other, that wait for 56% of their time; vector instructions
// take a third of the SIMDs' cycles. (A wave over all of a row's heads, choosing the tensor for each group: 12.7 and 28.8 us in place of 8.4
// and 12.6.)
#include <algorithm>

#include "head_norm.h"
#include "headprep.h"
#include "layer_ops_dev.h"

namespace {
using namespace sa3k;

constexpr int kFwdWaves = 4, kBwdWaves = 4;   // of a workgroup

struct HeadTensor {   // q, k or v
    const void *x, *dy;
    void* y;
    const float* gain;
    int64_t xs[3], ys[3], dys[3];   // strides of samples, tokens, heads
    int heads, first;               // first: of the workgroups' parts
};
struct HeadArgs {
    HeadTensor t[3];
    const int32_t *pos, *slot, *len;
    int batch, tokens, dim, rope, near, cache;
    int kinds, parts;                                   // tensors there are, one after the other in t; parts of a row
    int kind[3];                                        // which each is: 0 q, 1 k, 2 v
    float eps;
    uint64_t turn[kHeadMaxDim / 2];
};

// sin and cos of t / 2^32 turns, by the Taylor series on the eighth of a turn to either side of a quarter (the first terms left out
// are (pi / 4)^11 / 11! = 1.8e-9 and (pi / 4)^12 / 12! = 1.2e-10)
__device__ __forceinline__ float2 cos_sin(uint32_t t) {
    const uint32_t quarter = (t + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(t - (quarter << 30)) * 1.46291807926715968e-9f;   // 2 pi / 2^32
    const float z = x * x;
    float s = __builtin_fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
    s = __builtin_fmaf(z, s, 8.33333333e-3f);
    s = __builtin_fmaf(z, s, -1.66666667e-1f);
    s = __builtin_fmaf(z * x, s, x);
    float c = __builtin_fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
    c = __builtin_fmaf(z, c, -1.38888889e-3f);
    c = __builtin_fmaf(z, c, 4.16666667e-2f);
    c = __builtin_fmaf(z, c, -0.5f);
    c = __builtin_fmaf(z, c, 1.f);
    float2 r = quarter & 1 ? make_float2(-s, c) : make_float2(c, s);
    if (quarter & 2) r = make_float2(-r.x, -r.y);
    return r;
}

template <class T>
__device__ __forceinline__ float inverse_root(float v) {
    if constexpr (sizeof(T) == 4) {
        return 1.f / sqrtf(v);
    } else {   // off by 2^-23, against the 2^-9 or 2^-12 of the output's rounding; the instruction takes what is below 2^-126 as 0
        const bool small = v < 0x1p-126f;
        const float r = __builtin_amdgcn_rsqf(small ? v * 0x1p64f : v);
        return small ? r * 0x1p32f : r;
    }
}

// The row (a token of a sample) of a wave
struct Row {
    int64_t row;
    int b, t;
    bool on;   // the token is in its sequence
};
__device__ __forceinline__ Row row_of(const HeadArgs& a, int64_t row) {
    Row r;
    r.row = row;
    r.b = __builtin_amdgcn_readfirstlane((int)((uint32_t)row / (uint32_t)a.tokens));   // (batch x tokens stays below 2^31)
    r.t = (int)((uint32_t)row - (uint32_t)r.b * (uint32_t)a.tokens);
    r.on = !(a.len && r.t >= a.len[r.b]);
    return r;
}
// cos and sin of the row's angles for this lane's eight elements (with neighbours four pairs, else eight): each pair's by one lane of
// the wave, exchanged through `tab`, this wave's place in LDS (kTab long: lanes whose elements are not turned read on)
constexpr int kTab = kHeadMaxDim / 2 + 8;
// The sines come with the sign of the lane's share: w[e] turns (y, partner's y) to y w.x + partner's w.y. back: the other way round.
__device__ __forceinline__ void row_turns(const HeadArgs& a, const Row& r, int c, int lane, bool back, float2* tab, float2 (&w)[8]) {
    if (a.rope == 0) return;   // (uniform)
    const int pairs = a.rope >> 1;
    const int64_t pos = a.pos ? a.pos[r.row] : (int64_t)r.t;
    for (int p = lane; p < pairs; p += 64) tab[p] = cos_sin((uint32_t)(((uint64_t)pos * a.turn[p] + 0x80000000u) >> 32));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int h = a.rope >> 4;   // lanes of half the turned elements
    const int at = 8 * c >= a.rope ? 0 : a.near ? 4 * c : 8 * (c < h ? c : c - h);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        w[e] = tab[at + e];
        w[e].y = back != (!a.near && c < h) ? -w[e].y : w[e].y;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();   // (the next row's angles come after these reads)
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// which tensor a workgroup's part is of
__device__ __forceinline__ int tensor_of(const HeadArgs& a, int part) {
    int i = 0;
    if (a.kinds > 1 && part >= a.t[1].first) i = 1;
    if (a.kinds > 2 && part >= a.t[2].first) i = 2;
    return i;
}
// eight elements of a head, from element `at` on
template <class T>
struct Eight {
    u32x4a r[sizeof(T) / 2];
    __device__ __forceinline__ void load(const void* p, int64_t at) {
        const SA3K_GLOBAL T* q = (const SA3K_GLOBAL T*)p + at;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r[i] = load16(q + i * (16 / sizeof(T)));
    }
    __device__ __forceinline__ void store(void* p, int64_t at) const {
        SA3K_GLOBAL T* q = (SA3K_GLOBAL T*)p + at;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) store16(q + i * (16 / sizeof(T)), r[i]);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const Pack<T, 8> q = __builtin_bit_cast(Pack<T, 8>, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)q.v[e];
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        Pack<T, 8> q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q.v[e] = (T)v[e];
        *this = __builtin_bit_cast(Eight, q);
    }
};

// over the lanes of a head, the same bits in each
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
    v = dpp_add<0xB1>(v);                                    // lane ^ 1
    v = dpp_add<0x4E>(v);                                    // lane ^ 2
    if constexpr (LPH > 4) v = dpp_add<0x141>(v);            // the mirrored lane of eight
    if constexpr (LPH > 8) v = dpp_add<0x140>(v);            // of sixteen
    if constexpr (LPH > 16) v += __shfl_xor(v, 16, 64);
    return v;
}

// y's pairs turned by w. Elements 8c .. 8c + 7 of the head; rope and its half are multiples of eight, so a lane's elements are all
// turned or none, and the partners of (i, i + rope / 2) are one lane's.
__device__ __forceinline__ void rotate(const HeadArgs& a, const float2 (&w)[8], int c, int lane, float (&y)[8]) {
    if (a.rope == 0) return;   // (uniform)
    const bool turned = 8 * c < a.rope;
    if (a.near) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float p = y[e], q = y[e + 1], s = w[e / 2].y;
            y[e] = turned ? __builtin_fmaf(p, w[e / 2].x, -q * s) : p;
            y[e + 1] = turned ? __builtin_fmaf(q, w[e / 2].x, p * s) : q;
        }
        return;
    }
    const int h = a.rope >> 4;
    const bool first = c < h;
    const int from = !turned ? lane : first ? lane + h : lane - h;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float o = __shfl(y[e], from, 64);
        y[e] = turned ? __builtin_fmaf(y[e], w[e].x, o * w[e].y) : y[e];
    }
}

__device__ __forceinline__ void load_gain(const HeadArgs& a, const float* p, int c, float (&g)[8]) {
    if (p && 8 * c < a.dim) {
        const SA3K_GLOBAL float* q = (const SA3K_GLOBAL float*)p + 8 * c;
        const u32x4a lo = load16(q), hi = load16(q + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            g[e] = __uint_as_float(lo[e]);
            g[4 + e] = __uint_as_float(hi[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = 1.f;
    }
}

__device__ __forceinline__ void clear(float (&v)[8], bool keep) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = keep ? v[e] : 0.f;
}

// A wave takes kGroups groups of heads of one row and tensor at the most, whose loads are all under way at once. A lane past the last
// head, or past a head's elements, reads the last ones and stores nothing.
template <class T, int LPH>
__global__ __launch_bounds__(64 * kFwdWaves) void head_norm_fwd_kernel(HeadArgs a) {
    __shared__ float2 tabs[kFwdWaves][kTab];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane % LPH;
    const int part = (int)(blockIdx.x % (uint32_t)a.parts);
    const int64_t row = (int64_t)(blockIdx.x / (uint32_t)a.parts) * kFwdWaves + wave;
    if (row >= (int64_t)a.batch * a.tokens) return;
    const int ti = tensor_of(a, part), kind = a.kind[ti];
    const HeadTensor& tn = a.t[ti];
    const Row r = row_of(a, row);
    if (!r.on) return;
    const int h0 = (part - tn.first) * kGroups * (64 / LPH) + lane / LPH, e0 = min(8 * c, a.dim - 8), heads = tn.heads;
    const int64_t from = r.b * tn.xs[0] + r.t * tn.xs[1] + e0, xh = tn.xs[2];
    Eight<T> x[kGroups];
#pragma unroll
    for (int u = 0; u < kGroups; ++u) x[u].load(tn.x, from + min(h0 + u * (64 / LPH), heads - 1) * xh);
    const int slot = a.slot && kind ? a.slot[row] : r.t;
    const bool kept = !(a.slot && kind) || (slot >= 0 && slot < a.cache);
    float2 w[8];
    float gain[8];
    if (kind < 2) {   // (uniform)
        load_gain(a, tn.gain, c, gain);
        row_turns(a, r, c, lane, false, tabs[wave], w);   // (while the loads are under way)
    }
    if (!kept) return;   // (uniform)
    const float inv = 1.f / (float)a.dim;
    const bool tail = a.dim < 8 * LPH;   // (uniform) lanes past a head's elements, which hold a copy of its last
    const int64_t to = r.b * tn.ys[0] + slot * tn.ys[1] + e0, yh = tn.ys[2];
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
        const int h = h0 + u * (64 / LPH);
        if (u && h - lane / LPH >= heads) break;   // (uniform)
        if (kind < 2) {   // (uniform)
            float y[8], s = 0.f;
            x[u].get(y);
            if (tail) clear(y, 8 * c < a.dim);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = __builtin_fmaf(y[e], y[e], s);
            const float rt = inverse_root<T>(__builtin_fmaf(head_sum<LPH>(s), inv, a.eps));
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] *= rt * gain[e];
            rotate(a, w, c, lane, y);
            x[u].set(y);
        }
        if (h < heads && 8 * c < a.dim) x[u].store(tn.y, to + h * yh);
    }
}

// part [parts][workgroups of a part][dim]: each workgroup's sums of its gain's gradient (null: none)
template <class T, int LPH>
__global__ __launch_bounds__(64 * kBwdWaves, 4) void head_norm_bwd_kernel(HeadArgs a, float* part) {
    __shared__ union {
        float2 tabs[kBwdWaves][kTab];
        float sums[kBwdWaves][LPH * 8];
    } lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane % LPH;
    const int64_t rows = (int64_t)a.batch * a.tokens;
    const int mine = (int)(blockIdx.x % (uint32_t)a.parts), block = (int)(blockIdx.x / (uint32_t)a.parts);
    const int blocks = (int)(gridDim.x / (uint32_t)a.parts);
    const HeadTensor& tn = a.t[tensor_of(a, mine)];
    const int h0 = (mine - tn.first) * kGroups * (64 / LPH) + lane / LPH, e0 = min(8 * c, a.dim - 8), heads = tn.heads;
    const float inv = 1.f / (float)a.dim;
    const bool tail = a.dim < 8 * LPH;   // (uniform) lanes past a head's elements, which hold a copy of its last
    float gain[8], dg[8];
    load_gain(a, tn.gain, c, gain);
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[e] = 0.f;
    for (int64_t row = (int64_t)block * kBwdWaves + wave; row < rows; row += (int64_t)blocks * kBwdWaves) {
        const Row r = row_of(a, row);
        if (!r.on) continue;   // (uniform)
        const int64_t xat = r.b * tn.xs[0] + r.t * tn.xs[1] + e0, dat = r.b * tn.dys[0] + r.t * tn.dys[1] + e0;
        const int64_t yat = r.b * tn.ys[0] + r.t * tn.ys[1] + e0;
        Eight<T> x[kGroups], dy[kGroups];
#pragma unroll
        for (int u = 0; u < kGroups; ++u) {
            const int h = min(h0 + u * (64 / LPH), heads - 1);
            x[u].load(tn.x, xat + h * tn.xs[2]);
            dy[u].load(tn.dy, dat + h * tn.dys[2]);
        }
        float2 w[8];
        row_turns(a, r, c, lane, true, lds.tabs[wave], w);   // (while the loads are under way)
#pragma unroll
        for (int u = 0; u < kGroups; ++u) {
            const int hd = h0 + u * (64 / LPH);
            if (u && hd - lane / LPH >= heads) break;   // (uniform)
            const bool on = hd < heads && 8 * c < a.dim;
            float d[8], xf[8], h[8], s = 0.f, t = 0.f;
            dy[u].get(d);
            x[u].get(xf);
            if (tail) {
                clear(d, 8 * c < a.dim);
                clear(xf, 8 * c < a.dim);
            }
            rotate(a, w, c, lane, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[e] = d[e] * gain[e];
                s = __builtin_fmaf(xf[e], xf[e], s);
                t = __builtin_fmaf(h[e], xf[e], t);
            }
            const float rt = inverse_root<T>(__builtin_fmaf(head_sum<LPH>(s), inv, a.eps));
            const float mean = head_sum<LPH>(t) * rt * inv;
            // (uniform) the group's last heads are a copy, of no gradient to the gain
            if (hd - lane / LPH + 64 / LPH > heads) clear(d, on);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float xh = xf[e] * rt;
                dg[e] = __builtin_fmaf(d[e], xh, dg[e]);
                h[e] = rt * (h[e] - xh * mean);
            }
            x[u].set(h);
            if (on) x[u].store(tn.y, yat + hd * tn.ys[2]);
        }
    }
    if (!part) return;
    // over the wave's heads, then the waves in their order
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v = dg[e];
#pragma unroll
        for (int o = LPH; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
        if (lane < LPH) lds.sums[wave][8 * c + e] = v;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += 64 * kBwdWaves) {
        float v = 0.f;
#pragma unroll
        for (int n = 0; n < kBwdWaves; ++n) v += lds.sums[n][i];
        part[((int64_t)mine * blocks + block) * a.dim + i] = v;
    }
}

// the gains' gradients from the workgroups' sums: of q (blockIdx.y 0) the first nq rows, of k the nk after them
__global__ __launch_bounds__(kColumnSumThreads) void head_norm_sum_kernel(const float* __restrict__ part, int nq, int nk, int dim,
                                                                          float* dq, float* dk, int accumulate) {
    float* d = blockIdx.y ? dk : dq;
    if (!d) return;
    column_sums(blockIdx.y ? part + (int64_t)nq * dim : part, blockIdx.y ? nk : nq, dim,
                [&](int64_t i, float t) { d[i] = accumulate ? d[i] + t : t; });
}

// Workgroups of the backward with gains' gradients, at the most: each writes 4 dim bytes that the second launch reads again.
constexpr int kHeadBwdGroups = 1024;

HeadArgs head_args(const sa3k_head_norm& d, const HeadPtrs& p, bool bwd) {
    HeadArgs a{};
    const void *x[3] = {p.q, p.k, p.v}, *dy[3] = {p.dqo, p.dko, nullptr}, *gain[3] = {p.q_gain, p.k_gain, nullptr};
    void* y[3] = {p.qo, p.ko, p.vo};
    const int64_t *xs[3] = {d.q_stride, d.k_stride, d.v_stride}, *os[3] = {d.q_out_stride, d.k_out_stride, d.v_out_stride};
    int parts = 0;
    for (int i = 0; i < 3; ++i) {
        if (!x[i]) continue;
        HeadTensor& t = a.t[a.kinds];
        a.kind[a.kinds++] = i;
        t.x = x[i];
        t.dy = dy[i];
        t.y = y[i];
        t.gain = static_cast<const float*>(gain[i]);
        for (int n = 0; n < 3; ++n) {
            t.xs[n] = xs[i][n];
            t.ys[n] = (bwd ? xs : os)[i][n];
            t.dys[n] = os[i][n];
        }
        t.heads = i == 0 ? d.heads : d.kv_heads;
        t.first = parts;
        parts += head_parts(t.heads, d.head_dim);
    }
    a.parts = parts;
    a.pos = static_cast<const int32_t*>(p.pos);
    a.slot = static_cast<const int32_t*>(p.slot);
    a.len = static_cast<const int32_t*>(p.len);
    a.batch = d.batch; a.tokens = d.tokens;
    a.dim = d.head_dim; a.rope = d.rope_dims; a.near = d.neighbours; a.cache = d.cache_tokens; a.eps = d.eps;
    head_turns(d.rope_dims, d.rope_base, a.turn);
    return a;
}

void head_sums(sa3k_ctx* ctx, const HeadPtrs& p, const float* part, int nq, int nk, int dim) {
    KernelScope ks(ctx, "head_norm_bwd_sum");
    launch_k(ctx, true, head_norm_sum_kernel, dim3((unsigned)ceil_div(dim, 64), 2), dim3(kColumnSumThreads), 0, part, nq, nk, dim,
             static_cast<float*>(p.dq_gain), static_cast<float*>(p.dk_gain), p.accumulate);
    SA3K_LAUNCHED();
}

template <class T, int LPH>
void head_launch(sa3k_ctx* ctx, const HeadArgs& a, const HeadPtrs& p, bool bwd) {
    const int64_t rows = (int64_t)a.batch * a.tokens;
    int of[3] = {0, 0, 0};   // parts of each
    for (int i = 0; i < a.kinds; ++i) of[a.kind[i]] = head_parts(a.t[i].heads, a.dim);
    if (!bwd) {
        KernelScope ks(ctx, "head_norm_fwd");
        launch_k(ctx, true, head_norm_fwd_kernel<T, LPH>, dim3((unsigned)(ceil_div(rows, kFwdWaves) * a.parts)),
                 dim3(64 * kFwdWaves), 0, a);
        SA3K_LAUNCHED();
        return;
    }
    const bool sums = p.dq_gain || p.dk_gain;
    const int64_t blocks = ceil_div(rows, kBwdWaves), most = sums ? std::max<int64_t>(1, kHeadBwdGroups / a.parts) : 1 << 20;
    const int grid = (int)ceil_div(blocks, ceil_div(blocks, most));   // workgroups of the same number of rounds each
    float* part = sums ? layer_workspace(ctx, (size_t)grid * a.parts * (size_t)a.dim * sizeof(float)) : nullptr;
    {
        KernelScope ks(ctx, "head_norm_bwd");
        launch_k(ctx, !sums, head_norm_bwd_kernel<T, LPH>, dim3((unsigned)(grid * a.parts)), dim3(64 * kBwdWaves), 0, a, part);
        SA3K_LAUNCHED();
    }
    if (sums) head_sums(ctx, p, part, of[0] * grid, of[1] * grid, a.dim);
}
template <class T>
void head_run(sa3k_ctx* ctx, const HeadArgs& a, const HeadPtrs& p, bool bwd) {
    switch (head_lanes(a.dim)) {
    case 4: return head_launch<T, 4>(ctx, a, p, bwd);
    case 8: return head_launch<T, 8>(ctx, a, p, bwd);
    case 16: return head_launch<T, 16>(ctx, a, p, bwd);
    default: return head_launch<T, 32>(ctx, a, p, bwd);
    }
}
void head_dispatch(sa3k_ctx* ctx, const sa3k_head_norm& d, const HeadPtrs& p, bool bwd) {
    DeviceScope dev(ctx);
    if (d.batch == 0 || d.tokens == 0) {
        if (bwd && !p.accumulate && (p.dq_gain || p.dk_gain)) head_sums(ctx, p, nullptr, 0, 0, d.head_dim);   // over nothing
        return;
    }
    const HeadArgs a = head_args(d, p, bwd);
    if (d.type == SA3K_TYPE_F32) head_run<float>(ctx, a, p, bwd);
    else if (d.type == SA3K_TYPE_F16) head_run<f16>(ctx, a, p, bwd);
    else head_run<bf16>(ctx, a, p, bwd);
}

}  // namespace

extern "C" {

SA3K_API int sa3k_head_norm_fwd(sa3k_ctx* ctx, const sa3k_head_norm* d, const void* q, const void* k, const void* v,
                                const float* q_gain, const float* k_gain, const int32_t* pos, const int32_t* slot,
                                const int32_t* len, void* q_out, void* k_out, void* v_out) {
    return sa3k_guard(ctx, "sa3k_head_norm_fwd", [&] {
        HeadPtrs p;
        p.q = q; p.k = k; p.v = v; p.q_gain = q_gain; p.k_gain = k_gain; p.pos = pos; p.slot = slot; p.len = len;
        p.qo = q_out; p.ko = k_out; p.vo = v_out;
        int code;
        const char* msg = head_norm_check(d, p, false, &code);
        require_ok(msg ? msg : head_norm_apart(*d, p, false), code);
        head_dispatch(ctx, *d, p, false);
    });
}

SA3K_API int sa3k_head_norm_bwd(sa3k_ctx* ctx, const sa3k_head_norm* d, const void* q, const void* k, const void* dq_out,
                                const void* dk_out, const float* q_gain, const float* k_gain, const int32_t* pos,
                                const int32_t* len, void* dq, void* dk, float* dq_gain, float* dk_gain, int accumulate) {
    return sa3k_guard(ctx, "sa3k_head_norm_bwd", [&] {
        HeadPtrs p;
        p.q = q; p.k = k; p.dqo = dq_out; p.dko = dk_out; p.q_gain = q_gain; p.k_gain = k_gain; p.pos = pos; p.len = len;
        p.qo = dq; p.ko = dk; p.dq_gain = dq_gain; p.dk_gain = dk_gain; p.accumulate = accumulate;
        int code;
        const char* msg = head_norm_check(d, p, true, &code);
        require_ok(msg ? msg : head_norm_apart(*d, p, true), code);
        head_dispatch(ctx, *d, p, true);
    });
}

}  // extern "C"
