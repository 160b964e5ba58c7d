// Layer norm, forward and backward, with the residual sum in front of it and the gradients of gain and
// offset.
//   forward    s = x [+ r, rounded to the tensors' type], mu = mean s, rstd = 1 / sqrt(mean (s - mu)^2 + eps),
//              y = (s - mu) rstd gamma + beta
//   backward   xh = (x - mu) rstd, h = dy gamma, dx = rstd (h - mean h - xh mean(h xh)) [+ dsum],
//              dgamma = sum over rows dy xh, dbeta = sum over rows dy
// All sums in f32 over a row that stays in registers, the variance from the differences to the mean.
// Both passes are bound by HBM: every element is read once and written once. Measured on MI355X, where a large copy reaches
// 5.0 TB/s: forward 8704 x 1536 bf16 with a residual and its sum stored 20.8 us (5.1 TB/s; a call 25.8), 16384 x 1024 bf16
// 13.6 us (4.9 TB/s); backward with gain and offset 4099 x 1025 f32 18.1 us and 4.2 for the second launch; one row 6 us, the
// launch itself.
//
// A group of TG threads takes a row: a wave where that leaves at most 32 elements a lane (up to 2048
// columns; four rows a workgroup, no barrier), 256 threads up to 8192 columns, 512 above. (The backward of 4099 x 1025 f32 by 256
// threads a row: 22.1 us.) Lane l's chunk j is columns (j TG + l) V .. + V - 1, V elements of 16 bytes, read at whatever
// address they lie. The backward's lanes own the same columns in every row, so dgamma and dbeta add up in registers
// over the workgroup's rows; the workgroup's sums go to a workspace row, and a second launch adds those
// in a fixed order (no atomics: the same bits in every run).
#include <algorithm>

#include "layer_ops_dev.h"

namespace {
using namespace sa3k;

template <class T>
constexpr int kVec = 16 / (int)sizeof(T);

// chunk j of this lane; columns past the end are left as they are (zeros)
template <class T, int TG, int CH>
__device__ __forceinline__ void load_row(const T* p, int cols, int lane, float (&v)[CH * kVec<T>]) {
    constexpr int V = kVec<T>;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = (j * TG + lane) * V;
        if (c + V <= cols) {
            const Pack<T, V> q = *reinterpret_cast<const Pack<T, V>*>(p + c);
#pragma unroll
            for (int e = 0; e < V; ++e) v[j * V + e] = (float)q.v[e];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[j * V + e] = c + e < cols ? (float)p[c + e] : 0.f;
        }
    }
}
template <class T, int TG, int CH>
__device__ __forceinline__ void store_row(T* p, int cols, int lane, const float (&v)[CH * kVec<T>]) {
    constexpr int V = kVec<T>;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = (j * TG + lane) * V;
        if (c + V <= cols) {
            Pack<T, V> q;
#pragma unroll
            for (int e = 0; e < V; ++e) q.v[e] = (T)v[j * V + e];
            *reinterpret_cast<Pack<T, V>*>(p + c) = q;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c + e < cols) p[c + e] = (T)v[j * V + e];
        }
    }
}
// this lane's share of a vector of `cols` floats (null: fill)
template <class T, int TG, int CH>
__device__ __forceinline__ void load_vec(const float* p, float fill, int cols, int lane, float (&v)[CH * kVec<T>]) {
    constexpr int V = kVec<T>;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = (j * TG + lane) * V;
        if (p && c + V <= cols) {
            const Pack<float, V> q = *reinterpret_cast<const Pack<float, V>*>(p + c);
#pragma unroll
            for (int e = 0; e < V; ++e) v[j * V + e] = q.v[e];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[j * V + e] = p && c + e < cols ? p[c + e] : fill;
        }
    }
}

// Sums of N values over the row's group of TG threads, the same bits in every lane. red: LDS of
// 2 x N x TG / 64 floats, whose halves alternate (phase), so that one barrier a sum is enough.
template <int TG, int N>
__device__ __forceinline__ void group_sum(float (&s)[N], float* red, int& phase) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) s[i] += __shfl_xor(s[i], o, 64);
    if constexpr (TG > 64) {
        constexpr int W = TG / 64;
        float* r = red + (phase & 1) * N * W;
        ++phase;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) r[i * W + (threadIdx.x >> 6)] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) t += r[i * W + w];
            s[i] = t;
        }
    }
}

template <int TG>
constexpr int kNormThreads = TG < 256 ? 256 : TG;

template <class T, int TG, int CH>
__global__ __launch_bounds__(kNormThreads<TG>) void norm_fwd_kernel(NormArgs a) {
    constexpr int V = kVec<T>, E = CH * V, RPB = kNormThreads<TG> / TG;
    __shared__ float red[TG > 64 ? 2 * (TG / 64) : 1];
    const int lane = threadIdx.x % TG, cols = (int)a.cols;
    int phase = 0;
    float gm[E], bt[E];
    load_vec<T, TG, CH>(a.gamma, 1.f, cols, lane, gm);
    load_vec<T, TG, CH>(a.beta, 0.f, cols, lane, bt);
    const float inv = 1.f / (float)cols;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TG; row < a.rows; row += (int64_t)gridDim.x * RPB) {
        float x[E];
        load_row<T, TG, CH>(static_cast<const T*>(a.x) + row * a.ldx, cols, lane, x);
        if (a.r) {
            float r[E];
            load_row<T, TG, CH>(static_cast<const T*>(a.r) + row * a.ldr, cols, lane, r);
            // the norm is of the sum as it is stored: the backward reads that sum again
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = (float)(T)(x[e] + r[e]);
            if (a.sum) store_row<T, TG, CH>(static_cast<T*>(a.sum) + row * a.ldsum, cols, lane, x);
        }
        float s[1] = {0.f};
#pragma unroll
        for (int e = 0; e < E; ++e) s[0] += x[e];
        group_sum<TG>(s, red, phase);
        const float mu = s[0] * inv;
        float q[1] = {0.f};
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = (j * TG + lane) * V + e < cols ? x[j * V + e] - mu : 0.f;
                x[j * V + e] = d;
                q[0] = __builtin_fmaf(d, d, q[0]);
            }
        group_sum<TG>(q, red, phase);
        const float rs = 1.f / sqrtf(q[0] * inv + a.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = __builtin_fmaf(x[e] * rs, gm[e], bt[e]);
        store_row<T, TG, CH>(static_cast<T*>(a.y) + row * a.ldy, cols, lane, x);
        if (lane == 0) {
            if (a.mean) a.mean[row] = mu;
            if (a.rstd) a.rstd[row] = rs;
        }
    }
}

// part: [gridDim.x][2][cols] sums of this workgroup's rows (null: no gradient of gain and offset)
template <class T, int TG, int CH>
__global__ __launch_bounds__(kNormThreads<TG>) void norm_bwd_kernel(NormArgs a, float* part) {
    constexpr int V = kVec<T>, E = CH * V, RPB = kNormThreads<TG> / TG;
    __shared__ float red[TG > 64 ? 4 * (TG / 64) : 1];
    __shared__ float acc[TG == 64 ? 2 * TG * E : 1];
    const int lane = threadIdx.x % TG, cols = (int)a.cols;
    int phase = 0;
    float gm[E], dg[E], db[E];
    load_vec<T, TG, CH>(a.gamma, 1.f, cols, lane, gm);
#pragma unroll
    for (int e = 0; e < E; ++e) dg[e] = db[e] = 0.f;
    const float inv = 1.f / (float)cols;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TG; row < a.rows; row += (int64_t)gridDim.x * RPB) {
        const float mu = a.mean[row], rs = a.rstd[row];
        float x[E], dy[E];
        load_row<T, TG, CH>(static_cast<const T*>(a.x) + row * a.ldx, cols, lane, x);
        load_row<T, TG, CH>(static_cast<const T*>(a.dy) + row * a.lddy, cols, lane, dy);
        float r[E];
        if (a.r) {
            load_row<T, TG, CH>(static_cast<const T*>(a.r) + row * a.ldr, cols, lane, r);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) r[e] = 0.f;
        }
        float s[2] = {0.f, 0.f};
        // columns past the end hold dy = 0: they add nothing to any sum
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = (x[e] - mu) * rs;
            db[e] += dy[e];
            dg[e] = __builtin_fmaf(dy[e], x[e], dg[e]);
            dy[e] *= gm[e];
            s[0] += dy[e];
            s[1] = __builtin_fmaf(dy[e], x[e], s[1]);
        }
        group_sum<TG>(s, red, phase);
        const float m0 = s[0] * inv, m1 = s[1] * inv;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = __builtin_fmaf(dy[e] - m0 - x[e] * m1, rs, r[e]);
        store_row<T, TG, CH>(static_cast<T*>(a.y) + row * a.ldy, cols, lane, x);
    }
    if (!part) return;
    if constexpr (TG == 64) {   // the four waves' sums, added in wave order
        for (int w = 0; w < RPB; ++w) {
            if ((int)(threadIdx.x >> 6) == w) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float* p = acc + (e * TG + lane);
                    dg[e] += w ? p[0] : 0.f;
                    db[e] += w ? p[TG * E] : 0.f;
                    p[0] = dg[e];
                    p[TG * E] = db[e];
                }
            }
            __syncthreads();
        }
        if ((int)(threadIdx.x >> 6) != RPB - 1) return;
    }
    float* o = part + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int c = (j * TG + lane) * V + e;
            if (c < cols) {
                o[c] = dg[j * V + e];
                o[cols + c] = db[j * V + e];
            }
        }
}

// dgamma and dbeta from the workgroups' sums
__global__ __launch_bounds__(kColumnSumThreads) void norm_bwd_sum_kernel(const float* __restrict__ part, int parts, int cols,
                                                                         float* dgamma, float* dbeta, int accumulate) {
    column_sums(part, parts, 2 * (int64_t)cols, [&](int64_t i, float t) {
        float* d = i < cols ? dgamma : dbeta;
        const int64_t c = i < cols ? i : i - cols;
        if (d) d[c] = accumulate ? d[c] + t : t;
    });
}

// Workgroups of the backward with gradients of gain and offset, at the most. Each writes 8 cols bytes that the second launch
// reads again, and fewer of them have fewer loads in flight. Measured on MI355X, us at 128 / 256 / 512 / 1024 workgroups:
//   a wave a row            8704 x 1536 bf16  - / 34.0 / 26.9 / 33.8      4099 x 1025 f32    - / 20.3 / 19.2 / 23.0
//   a workgroup a row       4096 x 8192 bf16  126 / 74.7 / 87.5 / 114     512 x 4096 bf16    15.5 / 16.4 / 24.2 / 24.2
template <int TG>
constexpr int kNormBwdGroups = TG == 64 ? 512 : 256;

template <class T, int TG, int CH>
void norm_launch(sa3k_ctx* ctx, const NormArgs& a, bool bwd) {
    constexpr int RPB = kNormThreads<TG> / TG;
    const int64_t blocks = ceil_div(a.rows, RPB);
    const dim3 thr(kNormThreads<TG>);
    if (!bwd) {
        KernelScope ks(ctx, "layer_norm_fwd");
        launch_k(ctx, true, norm_fwd_kernel<T, TG, CH>, dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), thr, 0, a);
        SA3K_LAUNCHED();
        return;
    }
    const bool sums = a.dgamma || a.dbeta;
    // workgroups of the same number of rounds each
    const int64_t rounds = ceil_div(blocks, sums ? kNormBwdGroups<TG> : 1 << 20);
    const int grid = (int)ceil_div(blocks, rounds);
    float* part = sums ? layer_workspace(ctx, (size_t)grid * 2 * (size_t)a.cols * sizeof(float)) : nullptr;
    {
        KernelScope ks(ctx, "layer_norm_bwd");
        launch_k(ctx, !sums, norm_bwd_kernel<T, TG, CH>, dim3((unsigned)grid), thr, 0, a, part);
        SA3K_LAUNCHED();
    }
    if (sums) {
        KernelScope ks(ctx, "layer_norm_bwd_sum");
        launch_k(ctx, true, norm_bwd_sum_kernel, dim3((unsigned)ceil_div(2 * a.cols, 64)), dim3(kColumnSumThreads), 0, part, grid,
                 (int)a.cols, a.dgamma, a.dbeta, a.accumulate);
        SA3K_LAUNCHED();
    }
}

// the group that takes a row, and how many chunks a lane holds
template <class T>
void norm_run(sa3k_ctx* ctx, const NormArgs& a, bool bwd) {
    constexpr int V = kVec<T>, M = 32 / V;   // at most 32 elements a lane
    const int64_t ch = ceil_div(a.cols, V);
    if (ch <= 64) norm_launch<T, 64, 1>(ctx, a, bwd);
    else if (ch <= 128) norm_launch<T, 64, 2>(ctx, a, bwd);
    else if (ch <= 192) norm_launch<T, 64, 3>(ctx, a, bwd);
    else if (ch <= 256) norm_launch<T, 64, 4>(ctx, a, bwd);
    else if (M > 4 && ch <= 64 * 6) norm_launch<T, 64, (M > 4 ? 6 : 4)>(ctx, a, bwd);
    else if (M > 4 && ch <= 64 * 8) norm_launch<T, 64, M>(ctx, a, bwd);
    else if (M == 4 && ch <= 256 * 2) norm_launch<T, 256, (M == 4 ? 2 : 4)>(ctx, a, bwd);   // (f32: a wave takes these)
    else if (ch <= 256 * 4) norm_launch<T, 256, 4>(ctx, a, bwd);
    else if (M > 4 && ch <= 256 * 8) norm_launch<T, 256, M>(ctx, a, bwd);
    else norm_launch<T, 512, M>(ctx, a, bwd);
}

void norm_dispatch(sa3k_ctx* ctx, const NormArgs& a, bool bwd) {
    DeviceScope dev(ctx);
    if (a.rows == 0) {
        if (bwd && !a.accumulate)
            for (float* d : {a.dgamma, a.dbeta})
                if (d) {
                    norm_bwd_sum_kernel<<<(unsigned)ceil_div(2 * a.cols, 64), kColumnSumThreads, 0, ctx->stream>>>(
                        nullptr, 0, (int)a.cols, d == a.dgamma ? d : nullptr, d == a.dgamma ? nullptr : d, 0);
                    SA3K_LAUNCHED();
                }
        return;
    }
    if (a.type == SA3K_TYPE_F32) norm_run<float>(ctx, a, bwd);
    else if (a.type == SA3K_TYPE_F16) norm_run<f16>(ctx, a, bwd);
    else norm_run<bf16>(ctx, a, bwd);
}

}  // namespace

extern "C" {

SA3K_API int sa3k_layer_norm_fwd(sa3k_ctx* ctx, int type, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                 int64_t rows, int64_t cols, const float* gamma, const float* beta, float eps, void* sum,
                                 int64_t ldsum, void* y, int64_t ldy, float* mean, float* rstd) {
    return sa3k_guard(ctx, "sa3k_layer_norm_fwd", [&] {
        NormArgs a;
        a.type = type; a.rows = rows; a.cols = cols;
        a.x = x; a.ldx = ldx; a.r = residual; a.ldr = ldr;
        a.y = y; a.ldy = ldy; a.sum = sum; a.ldsum = ldsum;
        a.gamma = gamma; a.beta = beta; a.eps = eps; a.mean = mean; a.rstd = rstd;
        int code;
        const char* msg = norm_check(a, false, &code);
        require_ok(msg, code);
        norm_dispatch(ctx, a, false);
    });
}

SA3K_API int sa3k_layer_norm_bwd(sa3k_ctx* ctx, int type, const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                 const void* dsum, int64_t lddsum, int64_t rows, int64_t cols, const float* gamma,
                                 const float* mean, const float* rstd, void* dx, int64_t lddx, float* dgamma,
                                 float* dbeta, int accumulate) {
    return sa3k_guard(ctx, "sa3k_layer_norm_bwd", [&] {
        NormArgs a;
        a.type = type; a.rows = rows; a.cols = cols;
        a.x = x; a.ldx = ldx; a.r = dsum; a.ldr = lddsum; a.dy = dy; a.lddy = lddy;
        a.y = dx; a.ldy = lddx; a.gamma = gamma;
        a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
        a.dgamma = dgamma; a.dbeta = dbeta; a.accumulate = accumulate;
        int code;
        const char* msg = norm_check(a, true, &code);
        require_ok(msg, code);
        norm_dispatch(ctx, a, true);
    });
}

}  // extern "C"
