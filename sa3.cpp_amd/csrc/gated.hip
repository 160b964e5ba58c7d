// Gated products and their backward:
//   g = X Wg^T + bg, u = X Wu^T + bu, Y = act(g) u
//   dg = dY u act'(g), du = dY act(g);  dX = dg Wg + du Wu, dWg = dg^T X, dWu = du^T X, db = column sums
// on the tile kernels of prod_dev.h. Forward: a tile holds the same columns of both weights, so that g and u meet in one
// workgroup's epilogue and X is read once for both. Backward: one pass over dY, g and u writes dg and du side by side, rounded to the
// tensors' type as the matrix units read 16 bits (db is of both before that; beside the rounding of 16-bit results this makes their
// error 1.4 times as large: 0.00235 of dX in bf16 against 0.00166, 0.00029 in f16 against 0.00021, and no more); dX is one product over
// both (K = gate's columns, then up's), and so are the weights' gradients (rows of gate's, then of up's).
//
// Bound by MFMA with the loads beside it (prod_dev.h), few rows by HBM. Measured on MI355X, us a call, over several cards: 2176 x 1536 ->
// 6144 bf16 silu with g and u stored 102 to 106 (800 TFLOP/s; its 432 tiles fill 256 CUs to 84%), without 92 to 96, 8191 x 4096 -> 8192 f16
// gelu_tanh 948 to 978 (1125 to 1160 TFLOP/s), backward 2176 x 1536 -> 6144 199 to 202 (kernels by themselves: 27 the pass over dY, g and u,
// 170 to 181 both products, 12 the split sums), 1031 x 1001 -> 2731 f16 59 to 60. Plans: gated_plan, gated_pair.
#include "gated.h"
#include "prod_dev.h"

namespace {

// Sixteen bytes of 16-bit elements wherever they begin, from whole dwords. A load off the dwords takes the memory pipe several times
// as long: 1 x 1535 -> 6144 21.8 us with such loads, 1 x 1534 9.3. (The dwords read each hold one of the eight elements.)
template <class T>
__device__ __forceinline__ u32x4a load16_any(const T* p) {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    const uint32_t odd = (uint32_t)at & 2u;
    const SA3K_GLOBAL uint32_t* q = (const SA3K_GLOBAL uint32_t*)(at & ~(uint64_t)3);
    const u32x4at4 w = *(const SA3K_GLOBAL u32x4at4*)q;
    const uint32_t last = q[3 + (odd >> 1)], shift = odd * 8;
    return u32x4a{__builtin_amdgcn_alignbit(w[1], w[0], shift), __builtin_amdgcn_alignbit(w[2], w[1], shift),
                  __builtin_amdgcn_alignbit(w[3], w[2], shift), __builtin_amdgcn_alignbit(last, w[3], shift)};
}
inline bool off_dwords(const void* p, int64_t ld) { return p && (reinterpret_cast<uintptr_t>(p) % 4 != 0 || ld % 2 != 0); }

// Few rows, RB blocks of 16: 16 columns of the output a workgroup, whose eight waves split K in steps of 32 and read both weights
// straight from memory into the MFMA's registers (each element once); the waves' sums are joined in LDS. Bound by HBM and the
// latency of a launch: 1 x 1536 -> 6144 bf16 9.0 us, 38 MB (4.2 TB/s), 1 x 1535 12.5, 16 x 4095 -> 6144 31 (its loads as they lie: 76).
template <class T, int RB, bool ODD>   // ODD: rows may begin off a dword
__global__ __launch_bounds__(512) void gated_few_kernel(GemmArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int W = 8, U = RB == 1 ? 6 : 4;
    __shared__ float red[2][W][16 * RB][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15;
    const int64_t n0 = (int64_t)blockIdx.x * 16, wn = n0 + r;
    const int64_t steps = (a.K + 31) / 32;
    const T* gp = static_cast<const T*>(a.B) + min(wn, a.N - 1) * a.ldb;
    const T* up = static_cast<const T*>(a.B2) + min(wn, a.N - 1) * a.ldb;
    const T* xp[RB];
    f32x4 acc[2][RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        xp[b] = static_cast<const T*>(a.A) + min((int64_t)(16 * b + r), a.M - 1) * a.lda;
        acc[0][b] = acc[1][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // eight of K at k, zeros past its end (rows and columns past theirs repeat the last one: never stored)
    auto ld = [&](const T* p, int64_t k) {
        x8 v;
        if (k + 8 <= a.K) {
            if constexpr (ODD) {
                v = __builtin_bit_cast(x8, load16_any(p + k));
            } else {
                const Pack<T, 8> q = *reinterpret_cast<const Pack<T, 8>*>(p + k);
                v = __builtin_bit_cast(x8, q);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = k + e < a.K ? p[k + e] : (T)0.f;
        }
        return v;
    };
    for (int64_t s0 = wave; s0 < steps; s0 += W * U) {
        x8 g[U], u[U], x[U][RB];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t k = (s0 + i * W) * 32 + 8 * (lane >> 4);
            g[i] = ld(gp, k);
            u[i] = ld(up, k);
#pragma unroll
            for (int b = 0; b < RB; ++b) x[i][b] = ld(xp[b], k);
        }
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                if constexpr (__is_same(T, bf16)) {
                    acc[0][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(g[i], x[i][b], acc[0][b], 0, 0, 0);
                    acc[1][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u[i], x[i][b], acc[1][b], 0, 0, 0);
                } else {
                    acc[0][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(g[i], x[i][b], acc[0][b], 0, 0, 0);
                    acc[1][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(u[i], x[i][b], acc[1][b], 0, 0, 0);
                }
            }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int v = 0; v < 4; ++v) red[i][wave][16 * b + r][4 * (lane >> 4) + v] = acc[i][b][v];
    __syncthreads();
    if (tid >= 256 * RB) return;
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
    int act, cols, rows;   // cols: workgroups that share the columns; rows: that share the rows
    void* dz;              // [M][2 half]: dg, then du, zeros behind each (null: not stored)
    float* part;           // [rows][2][N] column sums of this workgroup's rows (null: none, or a single row of workgroups)
    float *dbg, *dbu;      // a single row of workgroups writes these itself (each may be null)
    int accumulate;
};
// dg and du of COLS columns a workgroup, 8 a thread, 2048 / COLS rows at a time. Bound by HBM: 2176 x 6144 bf16 silu, 134 MB, 26 us.
// The workgroups behind those pad the products' operands, which need nothing of this pass: a launch less.
template <class T, int COLS>
__global__ __launch_bounds__(256) void gated_dz_kernel(DzArgs a, PadArgs pads) {
    constexpr int TPR = COLS / 8, ROWS = 256 / TPR;   // threads a row, rows at a time
    if ((int)blockIdx.x >= a.cols * a.rows) {
        pad_body<T>(pads, (int)blockIdx.x - a.cols * a.rows, (int)gridDim.x - a.cols * a.rows);
        return;
    }
    __shared__ float red[2][ROWS][COLS + 8];
    const int by = (int)blockIdx.x / a.cols, bx = (int)blockIdx.x - by * a.cols;
    const int c = ((int)threadIdx.x % TPR) * 8, rl = (int)threadIdx.x / TPR;
    const int64_t n = (int64_t)bx * COLS + c;
    float sg[8], su[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sg[e] = su[e] = 0.f;
    // (lanes past the last column go along, as zeros: a run of such instructions with few lanes enabled takes longer)
    for (int64_t m = (int64_t)by * ROWS + rl; m < a.M; m += (int64_t)a.rows * ROWS) {
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
    for (int i = (int)threadIdx.x; i < 2 * COLS; i += 256) {
        const int w = i / COLS, k = i % COLS;
        const int64_t j = (int64_t)bx * COLS + k;
        if (j >= a.N) continue;
        float t = 0.f;
#pragma unroll 8
        for (int r = 0; r < ROWS; ++r) t += red[w][r][k];
        if (a.part) {
            a.part[((int64_t)by * 2 + w) * a.N + j] = t;
        } else {
            float* d = w ? a.dbu : a.dbg;
            if (d) d[j] = a.accumulate ? d[j] + t : t;
        }
    }
}

// The biases' gradients from the workgroups' sums: 16 columns a workgroup, a sixteenth of the rows a thread, eight in flight; added in
// row order within a thread, then thread by thread
struct DbArgs {
    const float* part;
    int parts, accumulate;
    int64_t N;
    float *dbg, *dbu;
};
__device__ __forceinline__ void db_body(const DbArgs& a, int64_t block) {
    __shared__ float s[16][17];
    const int k = threadIdx.x & 15, w = threadIdx.x >> 4, per = (a.parts + 15) / 16;
    const int lo = min(a.parts, w * per), hi = min(a.parts, lo + per);
    const int64_t i = block * 16 + k;
    float t = 0.f;
    if (i < 2 * a.N)
        for (int r = lo; r < hi; r += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = a.part[(int64_t)min(r + u, hi - 1) * 2 * a.N + i];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (r + u < hi) t += v[u];
        }
    s[w][k] = t;
    __syncthreads();
    if (w || i >= 2 * a.N) return;
    t = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) t += s[r][k];
    float* d = i < a.N ? a.dbg : a.dbu;
    const int64_t c = i < a.N ? i : i - a.N;
    if (d) d[c] = a.accumulate ? d[c] + t : t;
}
// what is left to add up after a backward's products, in one launch: dX's splits (x_wgs workgroups), dW's (w_wgs), the biases' gradients
template <class T>
__global__ __launch_bounds__(256) void gated_sums_kernel(GemmArgs x, GemmArgs w, DbArgs db, int64_t x_wgs, int64_t w_wgs) {
    const int64_t b = blockIdx.x;
    if (b < x_wgs) sum_body<T, kGatedInput>(x, b);
    else if (b < x_wgs + w_wgs) sum_body<T, kGatedWeight>(w, b - x_wgs);
    else db_body(db, b - x_wgs - w_wgs);
}

template <class T>
void fwd_run(sa3k_ctx* ctx, const GatedArgs& p) {
    GemmArgs a{};
    a.A = p.X; a.lda = p.ldx; a.B = p.Wg; a.B2 = p.Wu; a.ldb = p.ldw;
    a.M = p.M; a.N = p.N; a.K = p.K;
    a.C = p.Y; a.ldc = p.ldy; a.act = p.act; a.bias = p.bg; a.bias2 = p.bu; a.Z = p.Go; a.Z2 = p.Uo; a.ldz = p.ldz;
    const bool padded = !loads16(p.X, p.ldx, p.K) || !loads16(p.Wg, p.ldw, p.K) || !loads16(p.Wu, p.ldw, p.K);
    if (const int blocks = few_blocks(p.M, p.N, p.K, padded)) {
        KernelScope ks(ctx, "gated_linear_few", 4.0 * (double)a.M * (double)a.N * (double)a.K);
        const bool odd = off_dwords(p.X, p.ldx) || off_dwords(p.Wg, p.ldw) || off_dwords(p.Wu, p.ldw);
        launch_k(ctx, true, blocks == 1 ? (odd ? gated_few_kernel<T, 1, true> : gated_few_kernel<T, 1, false>)
                                        : (odd ? gated_few_kernel<T, 2, true> : gated_few_kernel<T, 2, false>),
                 dim3((unsigned)ceil_div(a.N, 16)), dim3(512), 0, a);
        SA3K_LAUNCHED();
        return;
    }
    const int64_t Kp = padded ? up8(p.K) : p.K;
    const ProdPlan plan = gated_plan(p.M, p.N, Kp);
    Scratch s;
    // (they share K: if one is padded, all are)
    const size_t ox = s.take(padded ? (size_t)p.M * Kp * 2 : 0), og = s.take(padded ? (size_t)p.N * Kp * 2 : 0);
    const size_t ou = s.take(padded ? (size_t)p.N * Kp * 2 : 0), os = s.take(split_bytes(plan, p.M, 2 * up8(p.N)));
    char* ws = s.need ? reinterpret_cast<char*>(layer_workspace(ctx, s.need)) : nullptr;
    if (padded) {
        pad<T>(ctx, PadArgs{{p.X, p.Wg, p.Wu}, {p.ldx, p.ldw, p.ldw}, {p.M, p.N, p.N}, p.K, {ws + ox, ws + og, ws + ou}},
               "gated_linear_pad");
        a.A = ws + ox;
        a.B = ws + og;
        a.B2 = ws + ou;
        a.lda = a.ldb = a.K = Kp;
    }
    tile_run<T, kGatedForward>(ctx, a, plan, reinterpret_cast<float*>(ws + os), "gated_linear_fwd", "gated_linear_sum");
}

// The pass over dY, g and u: 256 columns a workgroup; 64, and four times the rows at a time, for up to 64 rows, whose column sums one
// row of workgroups then adds up itself without a launch for the shares. Row shares: all there are rounds for where no column sums are
// asked for, else about 128, each of the same number of rounds.
struct DzPlan {
    int cols, rows;   // columns a workgroup, row shares
};
DzPlan dz_plan(int64_t M, int64_t half, bool sums) {
    if (M <= 64) return DzPlan{64, sums ? 1 : (int)std::max<int64_t>(1, ceil_div(M, 32))};
    const int64_t groups = ceil_div(M, 8), most = sums ? 128 : std::min<int64_t>(4096, (1 << 22) / ceil_div(half, 256));
    const int64_t rounds = ceil_div(groups, most);
    return DzPlan{256, (int)ceil_div(groups, rounds)};
}

template <class T>
void bwd_run(sa3k_ctx* ctx, const GatedArgs& p) {
    const int64_t M = p.M, N = p.N, K = p.K, half = gated_half(N), Kp = up8(K);
    const bool do_x = p.dX && M > 0, do_w = p.dWg != nullptr, products = do_x || do_w, sums = p.dbg || p.dbu;
    const bool px = do_w && M > 0 && !loads16(p.X, p.ldx, K);
    const bool pw = do_x && (!loads16(p.Wg, p.ldw, K) || !loads16(p.Wu, p.ldw, K));
    ProdPair plan{false, prod_plan(M > 0 ? M : 1, K, 2 * half), prod_plan(2 * half, K, M > 0 ? M : 1)};
    if (do_x && do_w) plan = gated_pair(M, N, K, plan.a, plan.b);
    const DzPlan dz = dz_plan(M, half, sums);
    Scratch s;
    const size_t oz = s.take(products ? (size_t)M * 2 * half * 2 : 0), ox = s.take(px ? (size_t)M * Kp * 2 : 0);
    const size_t og = s.take(pw ? (size_t)N * Kp * 2 : 0), ou = s.take(pw ? (size_t)N * Kp * 2 : 0);
    const size_t ob = s.take(sums && dz.rows > 1 ? (size_t)dz.rows * 2 * N * 4 : 0);
    const size_t sx = do_x ? split_bytes(plan.a, M, Kp) : 0, sw = do_w ? split_bytes(plan.b, 2 * half, Kp) : 0;
    const size_t osx = s.take(sx), osw = s.take(sw);
    char* ws = s.need ? reinterpret_cast<char*>(layer_workspace(ctx, s.need)) : nullptr;
    float* part = sums && dz.rows > 1 ? reinterpret_cast<float*>(ws + ob) : nullptr;
    if (products || sums) {
        const DzArgs z{p.dY, p.G, p.U, p.lddy, p.ldz, M, N, half, p.act, (int)ceil_div(half, dz.cols), dz.rows,
                       products && M > 0 ? ws + oz : nullptr, part, part ? nullptr : p.dbg, part ? nullptr : p.dbu, p.accumulate};
        const PadArgs pads{{p.Wg, p.Wu, p.X}, {p.ldw, p.ldw, p.ldx}, {pw ? N : 0, pw ? N : 0, px ? M : 0}, K, {ws + og, ws + ou, ws + ox}};
        const int64_t grid = (int64_t)z.cols * z.rows + pad_blocks(pads);
        KernelScope ks(ctx, "gated_linear_dz");
        launch_k(ctx, !products && !part, dz.cols == 64 ? gated_dz_kernel<T, 64> : gated_dz_kernel<T, 256>, dim3((unsigned)grid), dim3(256),
                 0, z, pads);
        SA3K_LAUNCHED();
    }
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
    const bool pair = plan.together && products;
    if (pair) {
        const int64_t nx = plan_into<kGatedInput>(x, plan.a, part_x), nw = plan_into<kGatedWeight>(w, plan.b, part_w);
        KernelScope ks(ctx, "gated_linear_dx_dw", 8.0 * (double)M * (double)N * (double)K);
        const bool big = plan.a.edge == 256, last = x.splits == 1 && w.splits == 1 && !part;
        launch_k(ctx, last, big ? prod_pair_big_kernel<T, kGatedInput, kGatedWeight> : prod_pair_kernel<T, kGatedInput, kGatedWeight>,
                 dim3((unsigned)(nx + nw)), dim3(big ? 512 : 256), 0, x, w, (int)nx);
        SA3K_LAUNCHED();
    } else {
        if (do_x) tile_launch<T, kGatedInput>(ctx, x, plan.a, part_x, "gated_linear_dx");
        if (do_w) tile_launch<T, kGatedWeight>(ctx, w, plan.b, part_w, "gated_linear_dw");
    }
    const int64_t x_wgs = do_x && x.splits > 1 ? ceil_div(M * (x.pitch / 8), 256) : 0;
    const int64_t w_wgs = do_w && w.splits > 1 ? ceil_div(2 * half * (w.pitch / 8), 256) : 0, db_wgs = part ? ceil_div(2 * N, 16) : 0;
    if (x_wgs + w_wgs + db_wgs == 0) return;
    const DbArgs db{part, dz.rows, p.accumulate, N, p.dbg, p.dbu};
    KernelScope ks(ctx, "gated_linear_sum");
    launch_k(ctx, true, gated_sums_kernel<T>, dim3((unsigned)(x_wgs + w_wgs + db_wgs)), dim3(256), 0, x, w, db, x_wgs, w_wgs);
    SA3K_LAUNCHED();
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
        require_ok(msg ? msg : gated_apart(p, false), code);
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
        require_ok(msg ? msg : gated_apart(p, true), code);
        DeviceScope dev(ctx);
        if (type == SA3K_TYPE_BF16) bwd_run<bf16>(ctx, p);
        else bwd_run<f16>(ctx, p);
    });
}

}  // extern "C"
