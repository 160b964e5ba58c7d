// Gated products and their backward:
//   g = X Wg^T + bg, u = X Wu^T + bu, Y = act(g) u
//   dg = dY u act'(g), du = dY act(g);  dX = dg Wg + du Wu, dWg = dg^T X, dWu = du^T X, db = column sums
// on the tile kernels of prod_dev.h. Forward: a tile holds the same columns of both weights, so that g and u meet in one
// workgroup's epilogue and X is read once for both. Backward: one pass over dY, g and u writes dg and du side by side, rounded to the
// tensors' type as the matrix units read 16 bits (db is of both before that); dX is one product over both (K = gate's
// columns, then up's), and so are the weights' gradients (rows of gate's, then of up's).
#include "gated.h"
#include "prod_dev.h"

namespace {

// act(z) and its slope
__device__ __forceinline__ float2 act_and_slope(float z, int act) {
    float v[1] = {z};
    act_values(v, act);
    return make_float2(v[0], act_slope(z, act));
}

// Few rows (at most 16): 16 columns of the output a workgroup, whose eight waves split K in steps of 32 and read both weights
// straight from memory into the MFMA's registers (each element once); the waves' sums are joined in LDS. Bound by HBM and the
// latency of a launch.
template <class T>
__global__ __launch_bounds__(512) void gated_few_kernel(GemmArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int W = 8, U = 6;
    __shared__ float red[2][W][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15;
    const int64_t n0 = (int64_t)blockIdx.x * 16, wn = n0 + r;
    const int64_t steps = (a.K + 31) / 32;
    const T* gp = static_cast<const T*>(a.B) + min(wn, a.N - 1) * a.ldb;
    const T* up = static_cast<const T*>(a.B2) + min(wn, a.N - 1) * a.ldb;
    const T* xp = static_cast<const T*>(a.A) + min((int64_t)r, a.M - 1) * a.lda;
    f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    // eight of K at k, zeros past its end (rows and columns past theirs repeat the last one: never stored)
    auto ld = [&](const T* p, int64_t k) {
        x8 v;
        if (k + 8 <= a.K) {
            const Pack<T, 8> q = *reinterpret_cast<const Pack<T, 8>*>(p + k);
            v = __builtin_bit_cast(x8, q);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = k + e < a.K ? p[k + e] : (T)0.f;
        }
        return v;
    };
    for (int64_t s0 = wave; s0 < steps; s0 += W * U) {
        x8 g[U], u[U], x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t k = (s0 + i * W) * 32 + 8 * (lane >> 4);
            g[i] = ld(gp, k);
            u[i] = ld(up, k);
            x[i] = ld(xp, k);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if constexpr (__is_same(T, bf16)) {
                acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(g[i], x[i], acc[0], 0, 0, 0);
                acc[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u[i], x[i], acc[1], 0, 0, 0);
            } else {
                acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(g[i], x[i], acc[0], 0, 0, 0);
                acc[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(u[i], x[i], acc[1], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) red[i][wave][r][4 * (lane >> 4) + v] = acc[i][v];
    __syncthreads();
    if (tid >= 256) return;
    const int64_t m = tid >> 4, n = n0 + (tid & 15);
    if (m >= a.M || n >= a.N) return;
    float g[1] = {0.f}, u = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        g[0] += red[0][w][m][tid & 15];
        u += red[1][w][m][tid & 15];
    }
    if (a.bias) g[0] += a.bias[n];
    if (a.bias2) u += a.bias2[n];
    if (a.Z) static_cast<T*>(a.Z)[m * a.ldz + n] = (T)g[0];
    if (a.Z2) static_cast<T*>(a.Z2)[m * a.ldz + n] = (T)u;
    act_values(g, a.act);
    static_cast<T*>(a.C)[m * a.ldc + n] = (T)(g[0] * u);
}

struct DzArgs {
    const void *dY, *G, *U;
    int64_t lddy, ldz, M, N, half;
    int act;
    void* dz;            // [M][2 half]: dg, then du, zeros behind each (null: not stored)
    float* part;         // [gridDim.y][2][N] column sums of this workgroup's rows (null: none, or a single row of workgroups)
    float *dbg, *dbu;    // a single row of workgroups writes these itself (each may be null)
    int accumulate;
};
// A workgroup takes 256 columns, 8 a thread, eight rows at a time. Bound by HBM.
template <class T>
__global__ __launch_bounds__(256) void gated_dz_kernel(DzArgs a) {
    __shared__ float red[2][8][256 + 8];
    const int c = (threadIdx.x & 31) * 8, rl = threadIdx.x >> 5;
    const int64_t n = (int64_t)blockIdx.x * 256 + c;
    float sg[8], su[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sg[e] = su[e] = 0.f;
    // (lanes past the last column go along, as zeros: a run of such instructions with few lanes enabled takes longer)
    for (int64_t m = (int64_t)blockIdx.y * 8 + rl; m < a.M; m += (int64_t)gridDim.y * 8) {
        float d[8], g[8], u[8];
        load8(static_cast<const T*>(a.dY) + m * a.lddy, n, a.N, d);
        load8(static_cast<const T*>(a.G) + m * a.ldz, n, a.N, g);
        load8(static_cast<const T*>(a.U) + m * a.ldz, n, a.N, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float2 f = act_and_slope(g[e], a.act);
            g[e] = d[e] * u[e] * f.y;
            u[e] = d[e] * f.x;
        }
        if (a.dz) {
            T* p = static_cast<T*>(a.dz) + m * 2 * a.half;
            store8(p, n, a.half, g);
            store8(p + a.half, n, a.half, u);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sg[e] += g[e];
            su[e] += u[e];
        }
    }
    if (!a.part && !a.dbg && !a.dbu) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        red[0][rl][c + e] = sg[e];
        red[1][rl][c + e] = su[e];
    }
    __syncthreads();
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= a.N) return;
    float t[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        t[0] += red[0][w][threadIdx.x];
        t[1] += red[1][w][threadIdx.x];
    }
    if (a.part) {
        float* p = a.part + (int64_t)blockIdx.y * 2 * a.N + j;
        p[0] = t[0];
        p[a.N] = t[1];
    } else {
        if (a.dbg) a.dbg[j] = a.accumulate ? a.dbg[j] + t[0] : t[0];
        if (a.dbu) a.dbu[j] = a.accumulate ? a.dbu[j] + t[1] : t[1];
    }
}

// the biases' gradients from the workgroups' sums
__global__ __launch_bounds__(kColumnSumThreads) void gated_db_kernel(const float* __restrict__ part, int parts, int64_t N, float* dbg,
                                                                     float* dbu, int accumulate) {
    column_sums(part, parts, 2 * N, [&](int64_t i, float t) {
        float* d = i < N ? dbg : dbu;
        const int64_t c = i < N ? i : i - N;
        if (d) d[c] = accumulate ? d[c] + t : t;
    });
}

template <class T>
void fwd_run(sa3k_ctx* ctx, const GatedArgs& p) {
    GemmArgs a{};
    a.A = p.X; a.lda = p.ldx; a.B = p.Wg; a.B2 = p.Wu; a.ldb = p.ldw;
    a.M = p.M; a.N = p.N; a.K = p.K;
    a.C = p.Y; a.ldc = p.ldy; a.act = p.act; a.bias = p.bg; a.bias2 = p.bu; a.Z = p.Go; a.Z2 = p.Uo; a.ldz = p.ldz;
    if (p.M <= kFewRows) {
        KernelScope ks(ctx, "gated_linear_few", 4.0 * (double)a.M * (double)a.N * (double)a.K);
        launch_k(ctx, true, gated_few_kernel<T>, dim3((unsigned)ceil_div(a.N, 16)), dim3(512), 0, a);
        SA3K_LAUNCHED();
        return;
    }
    const bool padded = !loads16(p.X, p.ldx, p.K) || !loads16(p.Wg, p.ldw, p.K) || !loads16(p.Wu, p.ldw, p.K);
    const int64_t Kp = padded ? up8(p.K) : p.K;
    const ProdPlan plan = prod_plan(p.M, 2 * p.N, Kp);
    Scratch s;
    // (they share K: if one is padded, all are)
    const size_t ox = s.take(padded ? (size_t)p.M * Kp * 2 : 0), og = s.take(padded ? (size_t)p.N * Kp * 2 : 0);
    const size_t ou = s.take(padded ? (size_t)p.N * Kp * 2 : 0), os = s.take(split_bytes(plan, p.M, 2 * up8(p.N)));
    char* ws = s.need ? reinterpret_cast<char*>(layer_workspace(ctx, s.need)) : nullptr;
    if (padded) {
        pad<T>(ctx, PadArgs{{p.X, p.Wg}, {p.ldx, p.ldw}, {p.M, p.N}, p.K, {ws + ox, ws + og}}, "gated_linear_pad");
        pad<T>(ctx, PadArgs{{p.Wu, nullptr}, {p.ldw, 0}, {p.N, 0}, p.K, {ws + ou, nullptr}}, "gated_linear_pad");
        a.A = ws + ox;
        a.B = ws + og;
        a.B2 = ws + ou;
        a.lda = a.ldb = a.K = Kp;
    }
    tile_run<T, kGatedForward>(ctx, a, plan, reinterpret_cast<float*>(ws + os), "gated_linear_fwd", "gated_linear_sum");
}

// Row shares of the pass over dY, g and u: one for up to 64 rows (which saves the launch that adds up shares), else about 128,
// each of the same number of rounds of eight rows.
int dz_parts(int64_t M) {
    if (M <= 64) return 1;
    const int64_t groups = std::max<int64_t>(1, ceil_div(M, 8)), rounds = ceil_div(groups, 128);
    return (int)ceil_div(groups, rounds);
}

template <class T>
void bwd_run(sa3k_ctx* ctx, const GatedArgs& p) {
    const int64_t M = p.M, N = p.N, K = p.K, half = gated_half(N), Kp = up8(K);
    const bool do_x = p.dX && M > 0, do_w = p.dWg != nullptr, products = do_x || do_w, sums = p.dbg || p.dbu;
    const bool px = do_w && M > 0 && !loads16(p.X, p.ldx, K);
    const bool pw = do_x && (!loads16(p.Wg, p.ldw, K) || !loads16(p.Wu, p.ldw, K));
    ProdPair plan{false, prod_plan(M > 0 ? M : 1, K, 2 * half), prod_plan(2 * half, K, M > 0 ? M : 1)};
    if (do_x && do_w) plan = prod_pair({M, K, 2 * half}, {2 * half, K, M});
    const int parts = dz_parts(M);
    Scratch s;
    const size_t oz = s.take(products ? (size_t)M * 2 * half * 2 : 0), ox = s.take(px ? (size_t)M * Kp * 2 : 0);
    const size_t og = s.take(pw ? (size_t)N * Kp * 2 : 0), ou = s.take(pw ? (size_t)N * Kp * 2 : 0);
    const size_t ob = s.take(sums && parts > 1 ? (size_t)parts * 2 * N * 4 : 0);
    const size_t sx = do_x ? split_bytes(plan.a, M, Kp) : 0, sw = do_w ? split_bytes(plan.b, 2 * half, Kp) : 0;
    const size_t osx = s.take(plan.together ? sx : std::max(sx, sw)), osw = plan.together ? s.take(sw) : osx;
    char* ws = s.need ? reinterpret_cast<char*>(layer_workspace(ctx, s.need)) : nullptr;
    float* part = sums && parts > 1 ? reinterpret_cast<float*>(ws + ob) : nullptr;
    if (products || sums) {
        DzArgs z{p.dY, p.G, p.U, p.lddy, p.ldz, M, N, half, p.act, products && M > 0 ? ws + oz : nullptr, part,
                 part ? nullptr : p.dbg, part ? nullptr : p.dbu, p.accumulate};
        KernelScope ks(ctx, "gated_linear_dz");
        launch_k(ctx, !products && !part, gated_dz_kernel<T>, dim3((unsigned)ceil_div(half, 256), (unsigned)parts), dim3(256), 0, z);
        SA3K_LAUNCHED();
    }
    if (part) {
        KernelScope ks(ctx, "gated_linear_db");
        launch_k(ctx, !products, gated_db_kernel, dim3((unsigned)ceil_div(2 * N, 64)), dim3(kColumnSumThreads), 0, part, parts, N,
                 p.dbg, p.dbu, p.accumulate);
        SA3K_LAUNCHED();
    }
    pad<T>(ctx, PadArgs{{p.Wg, p.Wu}, {p.ldw, p.ldw}, {pw ? N : 0, pw ? N : 0}, K, {ws + og, ws + ou}}, "gated_linear_pad");
    pad<T>(ctx, PadArgs{{p.X, nullptr}, {p.ldx, 0}, {px ? M : 0, 0}, K, {ws + ox, nullptr}}, "gated_linear_pad");
    GemmArgs x{}, w{};
    x.half = w.half = half;
    x.each = w.each = N;
    if (do_x) {   // [M][K] = (dg | du) [M][2 half] . (Wg, Wu) [N][K] each
        x.A = ws + oz; x.lda = 2 * half;
        x.B = pw ? ws + og : p.Wg;
        x.B2 = pw ? ws + ou : p.Wu;
        x.ldb = pw ? Kp : p.ldw;
        x.M = M; x.N = K; x.K = 2 * half;
        x.C = p.dX; x.ldc = p.lddx;
    }
    if (do_w) {   // [2 half][K] = (dg | du)^T [2 half][M] . X [M][K]
        w.A = ws + oz; w.lda = 2 * half;
        w.B = px ? ws + ox : p.X;
        w.ldb = px ? Kp : p.ldx;
        w.M = 2 * half; w.N = K; w.K = M;
        w.C = p.dWg; w.C2 = p.dWu; w.ldc = p.lddw;
        w.c_f32 = p.dw_type == SA3K_TYPE_F32;
        w.accumulate = p.accumulate;
    }
    float *part_x = reinterpret_cast<float*>(ws + osx), *part_w = reinterpret_cast<float*>(ws + osw);
    if (plan.together) {
        const int64_t nx = plan_into<kGatedInput>(x, plan.a, part_x), nw = plan_into<kGatedWeight>(w, plan.b, part_w);
        {
            KernelScope ks(ctx, "gated_linear_dx_dw", 8.0 * (double)M * (double)N * (double)K);
            launch_k(ctx, x.splits == 1 && w.splits == 1, prod_pair_kernel<T, kGatedInput, kGatedWeight>, dim3((unsigned)(nx + nw)),
                     dim3(256), 0, x, w, (int)nx);
            SA3K_LAUNCHED();
        }
        sum_splits<T, kGatedInput>(ctx, x, "gated_linear_sum");
        sum_splits<T, kGatedWeight>(ctx, w, "gated_linear_sum");
        return;
    }
    if (do_x) tile_run<T, kGatedInput>(ctx, x, plan.a, part_x, "gated_linear_dx", "gated_linear_sum");
    if (do_w) tile_run<T, kGatedWeight>(ctx, w, plan.b, part_w, "gated_linear_dw", "gated_linear_sum");
}

}  // namespace

extern "C" {

SA3K_API int sa3k_gated_linear_fwd(sa3k_ctx* ctx, int type, int act, const void* X, int64_t ldx, const void* Wg, const void* Wu,
                                   int64_t ldw, const float* bg, const float* bu, int64_t M, int64_t N, int64_t K, void* Y,
                                   int64_t ldy, void* G, void* U, int64_t ldz) {
    return sa3k_guard(ctx, "sa3k_gated_linear_fwd", [&] {
        GatedArgs p;
        p.type = type; p.act = act; p.M = M; p.N = N; p.K = K;
        p.X = X; p.ldx = ldx; p.Wg = Wg; p.Wu = Wu; p.ldw = ldw; p.bg = bg; p.bu = bu;
        p.Y = Y; p.ldy = ldy; p.Go = G; p.Uo = U; p.ldz = ldz;
        int code;
        const char* msg = gated_check(p, false, &code);
        require_ok(msg, code);
        if (M == 0) return;
        DeviceScope dev(ctx);
        if (type == SA3K_TYPE_BF16) fwd_run<bf16>(ctx, p);
        else fwd_run<f16>(ctx, p);
    });
}

SA3K_API int sa3k_gated_linear_bwd(sa3k_ctx* ctx, int type, int act, const void* dY, int64_t lddy, const void* G, const void* U,
                                   int64_t ldz, const void* X, int64_t ldx, const void* Wg, const void* Wu, int64_t ldw, int64_t M,
                                   int64_t N, int64_t K, void* dX, int64_t lddx, void* dWg, void* dWu, int dw_type, int64_t lddw,
                                   float* dbg, float* dbu, int accumulate) {
    return sa3k_guard(ctx, "sa3k_gated_linear_bwd", [&] {
        GatedArgs p;
        p.type = type; p.act = act; p.M = M; p.N = N; p.K = K;
        p.dY = dY; p.lddy = lddy; p.G = G; p.U = U; p.ldz = ldz; p.X = X; p.ldx = ldx; p.Wg = Wg; p.Wu = Wu; p.ldw = ldw;
        p.dX = dX; p.lddx = lddx; p.dWg = dWg; p.dWu = dWu; p.dw_type = dw_type; p.lddw = lddw; p.dbg = dbg; p.dbu = dbu;
        p.accumulate = accumulate;
        int code;
        const char* msg = gated_check(p, true, &code);
        require_ok(msg, code);
        DeviceScope dev(ctx);
        if (type == SA3K_TYPE_BF16) bwd_run<bf16>(ctx, p);
        else bwd_run<f16>(ctx, p);
    });
}

}  // extern "C"
