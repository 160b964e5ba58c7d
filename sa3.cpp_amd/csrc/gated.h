// Host-side arithmetic of the gated products: their backward's plan and the checks of their arguments. No HIP in here: compiled
// with g++ in the CPU tests too.
#pragma once

#include "layer_ops.h"

namespace sa3k {

struct GatedArgs {
    int type = 0, act = 0;
    int64_t M = 0, N = 0, K = 0;
    const void *X = nullptr, *Wg = nullptr, *Wu = nullptr, *dY = nullptr, *G = nullptr, *U = nullptr;
    void *Y = nullptr, *Go = nullptr, *Uo = nullptr, *dX = nullptr, *dWg = nullptr, *dWu = nullptr;   // Go, Uo: the forward's g and u
    int64_t ldx = 0, ldw = 0, lddy = 0, ldz = 0, ldy = 0, lddx = 0, lddw = 0;
    const float *bg = nullptr, *bu = nullptr;
    float *dbg = nullptr, *dbu = nullptr;
    int dw_type = 0, accumulate = 0;
};

// gate's and up's gradients lie side by side, each padded to whole tiles of 64
inline int64_t gated_half(int64_t N) { return (N + 63) / 64 * 64; }

// The backward products' plan: the other products', or one launch of 256 x 256 tiles for both, dX's workgroups first. Its time is
// the last workgroup's end when 256 CUs take nx workgroups of tx microseconds and then nw of tw: after the last full round of dX's,
// nx % 256 CUs start dW's a tx later than the rest. A tile of 64 along K counts 1.5 microseconds, a workgroup's start and stores 4,
// the launch 5, and it is taken where that is 6% below the other plan's estimate: fitted to 79 shapes from 32 to 8192 rows, on which
// the choice is 0.8% above the better of both on average and never more than 3% above the plan without it. dW's contraction, M, stays
// whole: in two splits it lost on every shape tried. Measured on MI355X (M x K -> N, bf16, whole backward calls, us: the plan without
// this launch / 256 x 256 tiles in dX's best split; * what this chooses): 2176 x 1536 -> 6144 212 / 194*, 4096 x 2048 -> 2048 155 /
// 137*, 8192 x 1536 -> 6144 769 / 626*, 2048 x 2048 -> 8192 312 / 307*, 6000 x 4096 -> 6000 1189 / 1069*, 512 x 4096 -> 11008 280 /
// 240*, 1600 x 4832 -> 712 66 / 58*, 4294 x 1384 -> 4632 310* / 284, 3000 x 1000 -> 3500 133* / 120, 1088 x 1536 -> 6144 113* / 116,
// 815 x 1392 -> 2568 53* / 54, 700 x 1536 -> 6144 81* / 90, 1435 x 3320 -> 1192 74* / 84, 160 x 1920 -> 592 18* / 26.
inline double gated_span(int64_t nx, double tx, int64_t nw, double tw) {
    const int64_t late = nx % 256;
    const double early_from = (double)(nx / 256) * tx, late_from = early_from + tx;
    // no end is before the work shared evenly, nor before the last of dX's
    const double shared = ((double)nx * tx + (double)nw * tw) / 256.0, least = late && late_from > shared ? late_from : shared;
    double best = 1e300;
    for (int side = 0; side < 2; ++side) {   // the last end lies whole workgroups of dW after one of both starts
        const double from = side ? early_from : late_from;
        for (int64_t k = least > from ? (int64_t)((least - from) / tw) : 0;; ++k) {
            const double end = from + (double)k * tw;
            if (late && end < late_from) continue;
            const int64_t by_late = late ? (int64_t)((end - late_from) / tw + 1e-9) * late : 0;
            if (by_late + (int64_t)((end - early_from) / tw + 1e-9) * (256 - late) < nw) continue;
            if (end < best) best = end;
            break;
        }
    }
    return best;
}
inline ProdPair gated_pair(int64_t M, int64_t N, int64_t K) {
    const int64_t cols = 2 * gated_half(N), kx = cols / 64, kw = (M + 63) / 64;
    ProdPair best = prod_pair({M, K, cols}, {cols, K, M});
    double least = 0.94 * (best.together ? best.a.us : best.a.us + best.b.us + 4.0);
    const int64_t nk = (K + 255) / 256, nx = (M + 255) / 256 * nk, nw = (cols + 255) / 256 * nk;
    const double tw = 1.5 * (double)kw + 4.0;
    for (int64_t n = 1; n <= 8; ++n) {
        if (!split_fits(n, kx, M, K)) continue;
        const int64_t per = (kx + n - 1) / n;
        const double t = gated_span(nx * n, 1.5 * (double)per + 4.0, nw, tw) + split_sum_us(n, M, K) + 5.0;
        if (t >= least) continue;
        least = t;
        best = ProdPair{true, ProdPlan{256, (int)n, (int)per, t}, ProdPlan{256, 1, (int)kw, t}};
    }
    return best;
}

// whether an element of x and one of y lie in the same place: rows of both `ld` apart
inline bool rows_meet(const void* x, const void* y, int64_t ld, int64_t rows, int64_t cols, int bytes) {
    if (!x || !y || rows <= 0) return false;
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
    const int64_t d = (int64_t)((a > b ? a - b : b - a) / (uintptr_t)bytes), q = d / ld, r = d % ld;
    return (q < rows && r < cols) || (q + 1 < rows && ld - r < cols);
}

inline const char* gated_check(const GatedArgs& a, bool bwd, int* code) {
    *code = SA3K_ERR_INVALID;
    if (a.type != SA3K_TYPE_BF16 && a.type != SA3K_TYPE_F16) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "type must be bf16 or f16";
    }
    if (a.act < SA3K_ACT_NONE || a.act > SA3K_ACT_GELU_TANH) return "unknown activation";
    if (a.M < 0 || a.M >= kMaxExtent) return "M out of range";
    if (a.N <= 0 || a.K <= 0 || 2 * gated_half(a.N) >= kProdMaxPitch || a.K >= kProdMaxPitch) return "N or K out of range";
    if (bwd && a.accumulate != 0 && a.accumulate != 1) return "accumulate must be 0 or 1";
    if (bwd && !a.dWg != !a.dWu) return "the gradients of both weights, or of neither";
    if (bwd && a.dWg && a.dw_type != a.type && a.dw_type != SA3K_TYPE_F32) return "dw_type must be f32 or type";
    if (bwd && a.dWg && a.accumulate && a.dw_type != SA3K_TYPE_F32) return "only an f32 dW can be added to";
    const void* p[12] = {a.X, a.Wg, a.Wu, a.dY, a.G, a.U, a.Y, a.Go, a.Uo, a.dX, a.dWg, a.dWu};
    const int64_t ld[12] = {a.ldx, a.ldw, a.ldw, a.lddy, a.ldz, a.ldz, a.ldy, a.ldz, a.ldz, a.lddx, a.lddw, a.lddw};
    const int64_t w[12] = {a.K, a.K, a.K, a.N, a.N, a.N, a.N, a.N, a.N, a.K, a.K, a.K};
    for (int i = 0; i < 12; ++i) {
        if (!p[i]) continue;
        if (ld[i] < w[i] || ld[i] >= kProdMaxPitch) return "a row pitch is smaller than its rows or out of range";
        if (!elem_aligned(p[i], i >= 10 ? elem_bytes(a.dw_type) : 2)) return "a tensor is not aligned to its elements";
    }
    const void* f[4] = {a.bg, a.bu, a.dbg, a.dbu};
    for (const void* x : f)
        if (!elem_aligned(x, 4)) return "an f32 vector is not 4-byte aligned";
    // a launch has fewer than 2^24 workgroups: tiles of 64 x 64 at the least, and the split sums' 2048 values
    const int64_t cols = 2 * gated_half(a.N);
    if (((a.M + 63) / 64) * ((cols > a.K ? cols : a.K) / 64 + 1) >= ((int64_t)1 << 23)) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "M x N is too large for one launch";
    }
    if (rows_meet(a.Go, a.Uo, a.ldz, a.M, a.N, 2) || rows_meet(a.dWg, a.dWu, a.lddw, a.N, a.K, elem_bytes(a.dw_type)) ||
        rows_meet(a.dbg, a.dbu, a.N, 1, a.N, 4))
        return "gate's output meets up's";
    if (!bwd) {
        if (!a.Wg || !a.Wu) return "the weights must not be null";
        if (a.M > 0 && (!a.X || !a.Y)) return "X and Y must not be null";
    } else {
        if (a.M > 0 && (!a.dY || !a.G || !a.U)) return "dY, G and U must not be null";
        if (a.M > 0 && a.dWg && !a.X) return "dW needs X";
        if (a.dX && (!a.Wg || !a.Wu)) return "dX needs the weights";
    }
    return nullptr;
}

}  // namespace sa3k
