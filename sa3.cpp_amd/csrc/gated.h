// Host-side arithmetic of the gated products: the checks of their arguments. No HIP in here: compiled with g++ in the CPU
// tests too.
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
