// Products with bias, activation and residual in the epilogue, and their backward:
//   z = X W^T + b, Y = act(z) + R;   dz = dY act'(z), dX = dz W, dW = dz^T X, db = sum over rows dz
// on the tile kernels of prod_dev.h.
#include "prod_dev.h"

namespace {

// Few rows (at most 16): 16 columns of the output a workgroup, whose eight waves split K in steps of 32 and read W
// straight from memory into the MFMA's registers (each element once); the waves' sums are joined in LDS. Bound by the latency
// of a launch and a few rounds of loads: 1 x 1536 x 6144 bf16 7.2 us, 19 MB of W.
template <class T>
__global__ __launch_bounds__(512) void prod_few_kernel(GemmArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int W = 8, U = 8;
    __shared__ float red[W][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15;
    const int64_t n0 = (int64_t)blockIdx.x * 16, wn = n0 + r;
    const int64_t steps = (a.K + 31) / 32;
    const T* wp = static_cast<const T*>(a.B) + min(wn, a.N - 1) * a.ldb;
    const T* xp = static_cast<const T*>(a.A) + min((int64_t)r, a.M - 1) * a.lda;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
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
        x8 w[U], x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = (s0 + u * W) * 32 + 8 * (lane >> 4);
            w[u] = ld(wp, k);
            x[u] = ld(xp, k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (__is_same(T, bf16)) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[u], x[u], acc, 0, 0, 0);
            else acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[u], x[u], acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) red[wave][r][4 * (lane >> 4) + v] = acc[v];
    __syncthreads();
    if (tid < 256) {
        const int64_t m = tid >> 4, n = n0 + (tid & 15);
        if (m >= a.M || n >= a.N) return;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += red[w][m][tid & 15];
        if (a.bias) v += a.bias[n];
        if (a.Z) static_cast<T*>(a.Z)[m * a.ldz + n] = (T)v;
        float y[1] = {v};
        act_values(y, a.act);
        v = y[0];
        if (a.R) v += (float)static_cast<const T*>(a.R)[m * a.ldr + n];
        static_cast<T*>(a.C)[m * a.ldc + n] = (T)v;
    }
}

// dz = dY act'(z) [M][pitch] (null: not stored) and its column sums over this workgroup's rows, part [gridDim.y][N] (null:
// none; a single row of workgroups writes db itself). A workgroup takes 256 columns, 8 a thread, eight rows at a time.
// dz is rounded to the tensors' type, as the matrix units read 16 bits; db is of dz before that. Against 64 bits dX and dW are off by
// 2.3e-3 of their norm in bf16, where their own rounding alone gives 1.7e-3.
// Bound by HBM: 2176 x 6144 bf16 gelu 17.2 us, 80 MB, 4.7 TB/s.
template <class T>
__global__ __launch_bounds__(256) void prod_dz_kernel(const T* dY, int64_t lddy, const T* Z, int64_t ldz, int64_t M, int64_t N,
                                                      int act, T* dz, int64_t pitch, float* part, int accumulate) {
    __shared__ float red[8][256 + 8];
    const int c = (threadIdx.x & 31) * 8, rl = threadIdx.x >> 5;
    const int64_t n = (int64_t)blockIdx.x * 256 + c;
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = 0.f;
    // (lanes past the last column go along, as zeros: see finish8)
    for (int64_t m = (int64_t)blockIdx.y * 8 + rl; m < M; m += (int64_t)gridDim.y * 8) {
        float d[8];
        load8(dY + m * lddy, n, N, d);
        if (act) {   // (uniform)
            float z[8];
            load8(Z + m * ldz, n, N, z);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] *= act_slope(z[e], act);
        }
        if (dz) store8(dz + m * pitch, n, pitch, d);   // (columns past N: 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += d[e];
    }
    if (!part) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) red[rl][c + e] = s[e];
    __syncthreads();
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= N) return;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += red[w][threadIdx.x];
    if (gridDim.y == 1 && accumulate) t += part[j];
    part[(int64_t)blockIdx.y * N + j] = t;
}

// db (+)= the workgroups' sums
__global__ __launch_bounds__(kColumnSumThreads) void prod_db_kernel(const float* __restrict__ part, int parts, int64_t N,
                                                                    float* db, int accumulate) {
    column_sums(part, parts, N, [&](int64_t i, float t) { db[i] = accumulate ? db[i] + t : t; });
}

template <class T>
void fwd_run(sa3k_ctx* ctx, const ProdArgs& p) {
    GemmArgs a{};
    a.A = p.X; a.lda = p.ldx; a.B = p.W; a.ldb = p.ldw;
    a.M = p.M; a.N = p.N; a.K = p.K;
    a.C = p.Y; a.ldc = p.ldy; a.act = p.act; a.bias = p.bias; a.R = p.R; a.ldr = p.ldr; a.Z = p.Zo; a.ldz = p.ldz;
    if (p.M <= kFewRows) {
        KernelScope ks(ctx, "linear_act_few", 2.0 * (double)a.M * (double)a.N * (double)a.K);
        launch_k(ctx, true, prod_few_kernel<T>, dim3((unsigned)ceil_div(a.N, 16)), dim3(512), 0, a);
        SA3K_LAUNCHED();
        return;
    }
    const bool px = !loads16(p.X, p.ldx, p.K), pw = !loads16(p.W, p.ldw, p.K);
    const int64_t Kp = px || pw ? up8(p.K) : p.K;
    const ProdPlan plan = prod_plan(p.M, p.N, Kp);
    Scratch s;
    // (if one operand is padded, both are: they share K)
    const size_t ox = s.take(px || pw ? (size_t)p.M * Kp * 2 : 0), ow = s.take(px || pw ? (size_t)p.N * Kp * 2 : 0);
    const size_t os = s.take(split_bytes(plan, p.M, up8(p.N)));
    char* ws = s.need ? reinterpret_cast<char*>(layer_workspace(ctx, s.need)) : nullptr;
    if (px || pw) {
        pad<T>(ctx, PadArgs{{p.X, p.W, nullptr}, {p.ldx, p.ldw, 0}, {p.M, p.N, 0}, p.K, {ws + ox, ws + ow, nullptr}}, "linear_act_pad");
        a.A = ws + ox;
        a.B = ws + ow;
        a.lda = a.ldb = a.K = Kp;
    }
    tile_run<T, kForward>(ctx, a, plan, reinterpret_cast<float*>(ws + os), "linear_act_fwd", "linear_act_sum");
}

// Row shares of the pass over dY and z: one for up to 64 rows (which saves the launch that adds up shares), else about 128, each
// of the same number of rounds of eight rows.
int dz_parts(int64_t M) {
    if (M <= 64) return 1;
    const int64_t groups = std::max<int64_t>(1, ceil_div(M, 8)), rounds = ceil_div(groups, 128);
    return (int)ceil_div(groups, rounds);
}

template <class T>
void bwd_run(sa3k_ctx* ctx, const ProdArgs& p) {
    const int64_t M = p.M, N = p.N, K = p.K, Np = up8(N), Kp = up8(K);
    const bool products = p.dX || p.dW;
    // dz as the products read it: dY itself, or its own rows
    const bool own_dz = products && M > 0 && (p.act != SA3K_ACT_NONE || !loads16(p.dY, p.lddy, N));
    const bool px = p.dW && M > 0 && !loads16(p.X, p.ldx, K), pw = p.dX && M > 0 && !loads16(p.W, p.ldw, K);
    const bool do_x = p.dX && M > 0, do_w = p.dW != nullptr;
    ProdPair plan{false, prod_plan(M > 0 ? M : 1, K, N), prod_plan(N, K, M > 0 ? M : 1)};
    if (do_x && do_w) plan = prod_pair({M, K, N}, {N, K, M});
    const int parts = dz_parts(M);
    Scratch s;
    const size_t oz = s.take(own_dz ? (size_t)M * Np * 2 : 0), ox = s.take(px ? (size_t)M * Kp * 2 : 0);
    const size_t ow = s.take(pw ? (size_t)N * Kp * 2 : 0), ob = s.take(p.db && parts > 1 ? (size_t)parts * N * 4 : 0);
    const size_t sx = do_x ? split_bytes(plan.a, M, Kp) : 0, sw = do_w ? split_bytes(plan.b, N, Kp) : 0;
    const size_t osx = s.take(plan.together ? sx : std::max(sx, sw)), osw = plan.together ? s.take(sw) : osx;
    char* ws = s.need ? reinterpret_cast<char*>(layer_workspace(ctx, s.need)) : nullptr;
    T* dz = own_dz ? reinterpret_cast<T*>(ws + oz) : nullptr;
    float* part = !p.db ? nullptr : parts > 1 ? reinterpret_cast<float*>(ws + ob) : p.db;
    if (own_dz || p.db) {
        KernelScope ks(ctx, "linear_act_dz");
        launch_k(ctx, !products && parts == 1, prod_dz_kernel<T>, dim3((unsigned)ceil_div(N, 256), (unsigned)parts), dim3(256), 0,
                 static_cast<const T*>(p.dY), p.lddy, static_cast<const T*>(p.Z), p.ldz, M, N, p.act, dz, Np, part, p.accumulate);
        SA3K_LAUNCHED();
    }
    if (p.db && parts > 1) {
        KernelScope ks(ctx, "linear_act_db");
        launch_k(ctx, !products, prod_db_kernel, dim3((unsigned)ceil_div(N, 64)), dim3(kColumnSumThreads), 0, part, parts, N, p.db,
                 p.accumulate);
        SA3K_LAUNCHED();
    }
    const void* g = own_dz ? dz : p.dY;
    const int64_t ldg = own_dz ? Np : p.lddy;
    GemmArgs x{}, w{};
    pad<T>(ctx, PadArgs{{p.W, p.X, nullptr}, {p.ldw, p.ldx, 0}, {pw ? N : 0, px ? M : 0, 0}, K, {ws + ow, ws + ox, nullptr}}, "linear_act_pad");
    if (do_x) {   // [M][K] = dz [M][N] . W [N][K]
        x.A = g; x.lda = ldg;
        x.B = pw ? ws + ow : p.W;
        x.ldb = pw ? Kp : p.ldw;
        x.M = M; x.N = K; x.K = N;
        x.C = p.dX; x.ldc = p.lddx;
    }
    if (do_w) {   // [N][K] = dz^T [N][M] . X [M][K]
        w.A = g; w.lda = ldg;
        w.B = px ? ws + ox : p.X;
        w.ldb = px ? Kp : p.ldx;
        w.M = N; w.N = K; w.K = M;
        w.C = p.dW; w.ldc = p.lddw;
        w.c_f32 = p.dw_type == SA3K_TYPE_F32;
        w.accumulate = p.accumulate;
    }
    float *part_x = reinterpret_cast<float*>(ws + osx), *part_w = reinterpret_cast<float*>(ws + osw);
    if (plan.together) {
        const int64_t nx = plan_into<kInput>(x, plan.a, part_x), nw = plan_into<kWeight>(w, plan.b, part_w);
        {
            KernelScope ks(ctx, "linear_act_dx_dw", 4.0 * (double)M * (double)N * (double)K);
            launch_k(ctx, x.splits == 1 && w.splits == 1, prod_pair_kernel<T, kInput, kWeight>, dim3((unsigned)(nx + nw)), dim3(256), 0, x, w,
                     (int)nx);
            SA3K_LAUNCHED();
        }
        sum_splits<T, kInput>(ctx, x, "linear_act_sum");
        sum_splits<T, kWeight>(ctx, w, "linear_act_sum");
        return;
    }
    if (do_x) tile_run<T, kInput>(ctx, x, plan.a, part_x, "linear_act_dx", "linear_act_sum");
    if (do_w) tile_run<T, kWeight>(ctx, w, plan.b, part_w, "linear_act_dw", "linear_act_sum");
}

}  // namespace

extern "C" {

SA3K_API int sa3k_linear_act_fwd(sa3k_ctx* ctx, int type, int act, const void* X, int64_t ldx, const void* W, int64_t ldw,
                                 const float* bias, const void* residual, int64_t ldr, int64_t M, int64_t N, int64_t K,
                                 void* Y, int64_t ldy, void* Z, int64_t ldz) {
    return sa3k_guard(ctx, "sa3k_linear_act_fwd", [&] {
        ProdArgs p;
        p.type = type; p.act = act; p.M = M; p.N = N; p.K = K;
        p.X = X; p.ldx = ldx; p.W = W; p.ldw = ldw; p.bias = bias; p.R = residual; p.ldr = ldr;
        p.Y = Y; p.ldy = ldy; p.Zo = Z; p.ldz = ldz;
        int code;
        const char* msg = prod_check(p, false, &code);
        require_ok(msg, code);
        if (M == 0) return;
        DeviceScope dev(ctx);
        if (type == SA3K_TYPE_BF16) fwd_run<bf16>(ctx, p);
        else fwd_run<f16>(ctx, p);
    });
}

SA3K_API int sa3k_linear_act_bwd(sa3k_ctx* ctx, int type, int act, const void* dY, int64_t lddy, const void* Z, int64_t ldz,
                                 const void* X, int64_t ldx, const void* W, int64_t ldw, int64_t M, int64_t N, int64_t K,
                                 void* dX, int64_t lddx, void* dW, int dw_type, int64_t lddw, float* db, int accumulate) {
    return sa3k_guard(ctx, "sa3k_linear_act_bwd", [&] {
        ProdArgs p;
        p.type = type; p.act = act; p.M = M; p.N = N; p.K = K;
        p.dY = dY; p.lddy = lddy; p.Z = Z; p.ldz = ldz; p.X = X; p.ldx = ldx; p.W = W; p.ldw = ldw;
        p.dX = dX; p.lddx = lddx; p.dW = dW; p.dw_type = dw_type; p.lddw = lddw; p.db = db; p.accumulate = accumulate;
        int code;
        const char* msg = prod_check(p, true, &code);
        require_ok(msg, code);
        DeviceScope dev(ctx);
        if (type == SA3K_TYPE_BF16) bwd_run<bf16>(ctx, p);
        else bwd_run<f16>(ctx, p);
    });
}

}  // extern "C"
