// RMS norm of the heads of q and k with the position rotation in the same pass, forward and backward; a new token's k and v
// into their row of a cache in the same launch.
//   forward    r = 1 / sqrt(mean x^2 + eps), n = x r gain, y = R n, R turning each pair (a, b) of the first rope_dims
//              elements by its angle: (a cos - b sin, b cos + a sin)
//   backward   w = R^T dy, dgain = sum over tokens and heads w x r, h = w gain, dx = r (h - x r mean(h x r))
// The statistics are worked out again in the backward, from the x it reads anyway. All arithmetic in f32, each output rounded once.
//
// Eight elements of a head a lane, 4 to 32 lanes a head, several heads a wave; a wave's heads are all q, all k or all v, so that
// pointers, strides and gains are the wave's own. A workgroup takes whole rows (tokens): their sines and cosines, shared by all heads,
// go through LDS once. Angles are exact modulo a turn (head_turns), so a position a million tokens out is as good as the first.
#include <algorithm>

#include "head_norm.h"
#include "layer_ops_dev.h"

namespace {
using namespace sa3k;

constexpr int kThreads = 256, kWaves = kThreads / 64;

struct HeadArgs {
    const void *x[3], *dy[2];
    void* y[3];
    int64_t xs[3][3], ys[3][3], dys[2][3];   // strides of samples, tokens, heads
    const float* gain[2];
    const int32_t *pos, *slot, *len;
    int batch, tokens, heads[3], groups[3];   // of q, k, v; groups: of as many heads as a wave takes
    int dim, rope, near, cache, rows;         // rows: a workgroup takes at once
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
    if constexpr (sizeof(T) == 4) return 1.f / sqrtf(v);
    else return __builtin_amdgcn_rsqf(v);   // off by 2^-23, against the 2^-9 or 2^-12 of the output's rounding
}

// the angles' cos and sin of `n` rows from row0 on into tab [n][rope / 2]
__device__ __forceinline__ void fill_turns(const HeadArgs& a, int64_t row0, int n, float2* tab) {
    const int pairs = a.rope >> 1;
    for (int i = threadIdx.x; i < n * pairs; i += kThreads) {
        const int r = i / pairs, p = i - r * pairs;
        const uint32_t row = (uint32_t)row0 + (uint32_t)r;
        const int64_t pos = a.pos ? a.pos[row] : (int64_t)(row % (uint32_t)a.tokens);
        tab[i] = cos_sin((uint32_t)(((uint64_t)pos * a.turn[p]) >> 32));
    }
}

// One wave's share of a row's group of heads: which tensor, and where this lane's eight elements lie
struct Item {
    int kind, b, t, slot;   // 0 q, 1 k, 2 v
    int row;                // of the workgroup's
    int64_t head;
    bool on;                // the lane has elements of a head, and the token is in its sequence
    bool store;             // and they have a place to go to
};
template <int LPH>
__device__ __forceinline__ Item item_of(const HeadArgs& a, int64_t row0, int n, int i, int lane) {
    constexpr int HPW = 64 / LPH;
    const int groups = a.groups[0] + a.groups[1] + a.groups[2];
    Item m;
    m.row = __builtin_amdgcn_readfirstlane(i / groups);
    int g = __builtin_amdgcn_readfirstlane(i - m.row * groups);
    m.kind = g < a.groups[0] ? 0 : g < a.groups[0] + a.groups[1] ? 1 : 2;
    g -= m.kind > 0 ? a.groups[0] : 0;
    g -= m.kind > 1 ? a.groups[1] : 0;
    const bool in = m.row < n;
    const uint32_t row = (uint32_t)row0 + (uint32_t)(in ? m.row : 0);   // (batch x tokens stays below 2^31)
    m.b = (int)(row / (uint32_t)a.tokens);
    m.t = (int)(row - (uint32_t)m.b * (uint32_t)a.tokens);
    m.head = g * HPW + lane / LPH;
    m.on = in && m.head < a.heads[m.kind] && (lane % LPH) * 8 < a.dim && !(a.len && m.t >= a.len[m.b]);
    m.slot = a.slot && m.kind > 0 && in ? a.slot[row] : m.t;
    m.store = m.on && !(a.slot && m.kind > 0 && (m.slot < 0 || m.slot >= a.cache));
    return m;
}
__device__ __forceinline__ int64_t place(const int64_t* s, int b, int t, int64_t head, int lane_off) {
    return b * s[0] + t * s[1] + head * s[2] + lane_off;
}

template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
    for (int o = 1; o < LPH; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// y's pairs turned by the angles in tab (sign -1: back). Elements 8c .. 8c + 7 of the head; rope and its half are
// multiples of eight, so a lane's elements are all turned or none, and the partners of (i, i + rope / 2) are one lane's.
template <int LPH>
__device__ __forceinline__ void rotate(const HeadArgs& a, const float2* tab, int c, int lane, float sign, float (&y)[8]) {
    if (a.rope == 0) return;   // (uniform)
    const bool turned = 8 * c < a.rope;
    if (a.near) {
        if (!turned) return;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float2 w = tab[4 * c + e / 2];
            const float p = y[e], q = y[e + 1], s = sign * w.y;
            y[e] = __builtin_fmaf(p, w.x, -q * s);
            y[e + 1] = __builtin_fmaf(q, w.x, p * s);
        }
        return;
    }
    const int h = a.rope >> 4;   // lanes of half the turned elements
    const bool first = c < h;
    const int from = !turned ? lane : first ? lane + h : lane - h;
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = __shfl(y[e], from, 64);
    if (!turned) return;
    const float sg = first ? -sign : sign;
    const float2* w = tab + 8 * (first ? c : c - h);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf(y[e], w[e].x, o[e] * (sg * w[e].y));
}

template <int LPH>
__device__ __forceinline__ void load_gain(const HeadArgs& a, int c, float (&g)[2][8]) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) g[k][e] = a.gain[k] && 8 * c < a.dim ? a.gain[k][8 * c + e] : 1.f;
}

template <class T, int LPH>
__global__ __launch_bounds__(kThreads) void head_norm_fwd_kernel(HeadArgs a) {
    constexpr int U = 4;   // groups of heads whose loads a wave has under way
    __shared__ float2 tab[kThreads];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane % LPH;
    const int64_t rows = (int64_t)a.batch * a.tokens;
    float gain[2][8];
    load_gain<LPH>(a, c, gain);
    const float inv = 1.f / (float)a.dim;
    for (int64_t row0 = (int64_t)blockIdx.x * a.rows; row0 < rows; row0 += (int64_t)gridDim.x * a.rows) {
        const int n = (int)min((int64_t)a.rows, rows - row0), items = n * (a.groups[0] + a.groups[1] + a.groups[2]);
        if (row0 != (int64_t)blockIdx.x * a.rows) __syncthreads();   // (the rows before are done with the table)
        fill_turns(a, row0, n, tab);
        __syncthreads();
        for (int i0 = wave; i0 < items; i0 += kWaves * U) {
            Pack<T, 8> x[U];
            Item m[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                m[u] = item_of<LPH>(a, row0, n, i0 + u * kWaves, lane);
                if (m[u].on) {
                    x[u] = *reinterpret_cast<const Pack<T, 8>*>(static_cast<const T*>(a.x[m[u].kind]) +
                                                               place(a.xs[m[u].kind], m[u].b, m[u].t, m[u].head, 8 * c));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[u].v[e] = (T)0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i0 + u * kWaves >= items) break;   // (uniform)
                T* out = static_cast<T*>(a.y[m[u].kind]) + place(a.ys[m[u].kind], m[u].b, m[u].slot, m[u].head, 8 * c);
                if (m[u].kind == 2) {   // (uniform)
                    if (m[u].store) *reinterpret_cast<Pack<T, 8>*>(out) = x[u];
                    continue;
                }
                float y[8], s = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    y[e] = (float)x[u].v[e];
                    s = __builtin_fmaf(y[e], y[e], s);
                }
                const float r = inverse_root<T>(__builtin_fmaf(head_sum<LPH>(s), inv, a.eps));
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] *= r * (m[u].kind ? gain[1][e] : gain[0][e]);
                rotate<LPH>(a, tab + m[u].row * (a.rope >> 1), c, lane, 1.f, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[u].v[e] = (T)y[e];
                if (m[u].store) *reinterpret_cast<Pack<T, 8>*>(out) = x[u];
            }
        }
    }
}

// part [gridDim.x][2][dim]: this workgroup's sums of the gains' gradients (null: none)
template <class T, int LPH>
__global__ __launch_bounds__(kThreads) void head_norm_bwd_kernel(HeadArgs a, float* part) {
    constexpr int U = 2;
    __shared__ float2 tab[kThreads];
    __shared__ float sums[kWaves][2][LPH * 8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane % LPH;
    const int64_t rows = (int64_t)a.batch * a.tokens;
    float gain[2][8], dg[2][8];
    load_gain<LPH>(a, c, gain);
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[0][e] = dg[1][e] = 0.f;
    const float inv = 1.f / (float)a.dim;
    for (int64_t row0 = (int64_t)blockIdx.x * a.rows; row0 < rows; row0 += (int64_t)gridDim.x * a.rows) {
        const int n = (int)min((int64_t)a.rows, rows - row0), items = n * (a.groups[0] + a.groups[1]);
        __syncthreads();   // (the rows before are done with the table)
        fill_turns(a, row0, n, tab);
        __syncthreads();
        for (int i0 = wave; i0 < items; i0 += kWaves * U) {
            Pack<T, 8> x[U], dy[U];
            Item m[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                m[u] = item_of<LPH>(a, row0, n, i0 + u * kWaves, lane);
                const int k = m[u].kind;
                if (m[u].on) {
                    x[u] = *reinterpret_cast<const Pack<T, 8>*>(static_cast<const T*>(a.x[k]) +
                                                               place(a.xs[k], m[u].b, m[u].t, m[u].head, 8 * c));
                    dy[u] = *reinterpret_cast<const Pack<T, 8>*>(static_cast<const T*>(a.dy[k]) +
                                                                place(a.dys[k], m[u].b, m[u].t, m[u].head, 8 * c));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[u].v[e] = dy[u].v[e] = (T)0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i0 + u * kWaves >= items) break;   // (uniform)
                const int k = m[u].kind;
                float w[8], xf[8], s = 0.f, t = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = (float)dy[u].v[e];
                    xf[e] = (float)x[u].v[e];
                }
                rotate<LPH>(a, tab + m[u].row * (a.rope >> 1), c, lane, -1.f, w);
                float h[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[e] = w[e] * (k ? gain[1][e] : gain[0][e]);
                    s = __builtin_fmaf(xf[e], xf[e], s);
                    t = __builtin_fmaf(h[e], xf[e], t);
                }
                const float r = inverse_root<T>(__builtin_fmaf(head_sum<LPH>(s), inv, a.eps));
                const float mean = head_sum<LPH>(t) * r * inv;
                if (m[u].on) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float xh = xf[e] * r;
                        if (k) dg[1][e] = __builtin_fmaf(w[e], xh, dg[1][e]);
                        else dg[0][e] = __builtin_fmaf(w[e], xh, dg[0][e]);
                        x[u].v[e] = (T)(r * (h[e] - xh * mean));
                    }
                    *reinterpret_cast<Pack<T, 8>*>(static_cast<T*>(a.y[k]) + place(a.ys[k], m[u].b, m[u].t, m[u].head, 8 * c)) = x[u];
                }
            }
        }
    }
    if (!part) return;
    // over the wave's heads, then the waves in their order
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = dg[k][e];
#pragma unroll
            for (int o = LPH; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
            if (lane < LPH) sums[wave][k][8 * c + e] = v;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.dim; i += kThreads) {
        const int k = i >= a.dim, d = k ? i - a.dim : i;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v += sums[w][k][d];
        part[(int64_t)blockIdx.x * 2 * a.dim + i] = v;
    }
}

// the gains' gradients from the workgroups' sums
__global__ __launch_bounds__(kColumnSumThreads) void head_norm_sum_kernel(const float* __restrict__ part, int parts, int dim,
                                                                          float* dq, float* dk, int accumulate) {
    column_sums(part, parts, 2 * (int64_t)dim, [&](int64_t i, float t) {
        float* d = i < dim ? dq : dk;
        const int64_t e = i < dim ? i : i - dim;
        if (d) d[e] = accumulate ? d[e] + t : t;
    });
}

// Workgroups of the backward with gains' gradients, at the most: each writes 8 dim bytes that the second launch reads again.
constexpr int kHeadBwdGroups = 1024;

void copy3(int64_t (&to)[3], const int64_t* from) {
    for (int i = 0; i < 3; ++i) to[i] = from[i];
}

HeadArgs head_args(const sa3k_head_norm& d, const HeadPtrs& p, bool bwd) {
    HeadArgs a{};
    a.x[0] = p.q; a.x[1] = p.k; a.x[2] = p.v;
    a.y[0] = p.qo; a.y[1] = p.ko; a.y[2] = p.vo;
    a.dy[0] = p.dqo; a.dy[1] = p.dko;
    copy3(a.xs[0], d.q_stride); copy3(a.xs[1], d.k_stride); copy3(a.xs[2], d.v_stride);
    copy3(a.ys[0], bwd ? d.q_stride : d.q_out_stride); copy3(a.ys[1], bwd ? d.k_stride : d.k_out_stride);
    copy3(a.ys[2], d.v_out_stride);
    copy3(a.dys[0], d.q_out_stride); copy3(a.dys[1], d.k_out_stride);
    a.gain[0] = static_cast<const float*>(p.q_gain);
    a.gain[1] = static_cast<const float*>(p.k_gain);
    a.pos = static_cast<const int32_t*>(p.pos);
    a.slot = static_cast<const int32_t*>(p.slot);
    a.len = static_cast<const int32_t*>(p.len);
    a.batch = d.batch; a.tokens = d.tokens;
    const int per_wave = 64 / head_lanes(d.head_dim);
    for (int i = 0; i < 3; ++i) {
        a.heads[i] = !a.x[i] ? 0 : i == 0 ? d.heads : d.kv_heads;
        a.groups[i] = (int)ceil_div(a.heads[i], per_wave);
    }
    a.dim = d.head_dim; a.rope = d.rope_dims; a.near = d.neighbours; a.cache = d.cache_tokens; a.eps = d.eps;
    a.rows = head_rows((int64_t)d.batch * d.tokens, d.rope_dims / 2);
    head_turns(d.rope_dims, d.rope_base, a.turn);
    return a;
}

template <class T, int LPH>
void head_launch(sa3k_ctx* ctx, const HeadArgs& a, const HeadPtrs& p, bool bwd) {
    const int64_t blocks = ceil_div((int64_t)a.batch * a.tokens, a.rows);
    if (!bwd) {
        KernelScope ks(ctx, "head_norm_fwd");
        launch_k(ctx, true, head_norm_fwd_kernel<T, LPH>, dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(kThreads), 0, a);
        SA3K_LAUNCHED();
        return;
    }
    const bool sums = p.dq_gain || p.dk_gain;
    const int64_t rounds = ceil_div(blocks, sums ? kHeadBwdGroups : 1 << 20);
    const int grid = (int)ceil_div(blocks, rounds);   // workgroups of the same number of rounds each
    float* part = sums ? layer_workspace(ctx, (size_t)grid * 2 * (size_t)a.dim * sizeof(float)) : nullptr;
    {
        KernelScope ks(ctx, "head_norm_bwd");
        launch_k(ctx, !sums, head_norm_bwd_kernel<T, LPH>, dim3((unsigned)grid), dim3(kThreads), 0, a, part);
        SA3K_LAUNCHED();
    }
    if (sums) {
        KernelScope ks(ctx, "head_norm_bwd_sum");
        launch_k(ctx, true, head_norm_sum_kernel, dim3((unsigned)ceil_div(2 * a.dim, 64)), dim3(kColumnSumThreads), 0, part, grid,
                 a.dim, static_cast<float*>(p.dq_gain), static_cast<float*>(p.dk_gain), p.accumulate);
        SA3K_LAUNCHED();
    }
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
        if (bwd && !p.accumulate && (p.dq_gain || p.dk_gain)) {   // sums over nothing
            head_norm_sum_kernel<<<(unsigned)ceil_div(2 * d.head_dim, 64), kColumnSumThreads, 0, ctx->stream>>>(
                nullptr, 0, d.head_dim, static_cast<float*>(p.dq_gain), static_cast<float*>(p.dk_gain), 0);
            SA3K_LAUNCHED();
        }
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
        require_ok(msg, code);
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
        require_ok(msg, code);
        head_dispatch(ctx, *d, p, true);
    });
}

}  // extern "C"
