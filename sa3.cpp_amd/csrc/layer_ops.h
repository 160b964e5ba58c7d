// Host-side arithmetic of the layer operators (layer norm, windowed attention, fused products): the
// checks of their arguments and the rules that pick a variant. No HIP in here: compiled with g++ in the
// CPU tests too. A check returns null, or the message of the first thing that is wrong, and sets `code`
// to the status an entry point returns with it.
#pragma once

#include <cstdint>

#include "sa3k.h"

namespace sa3k {

constexpr int64_t kMaxExtent = (int64_t)1 << 31;   // rows, columns and pitches stay below this

inline int elem_bytes(int type) { return type == SA3K_TYPE_F32 ? 4 : 2; }
// null, or a pointer that elements of `bytes` bytes can be read from
inline bool elem_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes) == 0; }

// ------------------------------------------------------------------------------------ layer norm
constexpr int64_t kNormMaxCols = 16384;

struct NormArgs {
    int type = 0;
    int64_t rows = 0, cols = 0;
    const void *x = nullptr, *r = nullptr, *dy = nullptr;   // r: the residual, or the sum's gradient (dsum)
    void *y = nullptr, *sum = nullptr;                      // y: the output, or dx
    int64_t ldx = 0, ldr = 0, lddy = 0, ldy = 0, ldsum = 0;
    const float *gamma = nullptr, *beta = nullptr;
    float eps = 0.f;
    float *mean = nullptr, *rstd = nullptr, *dgamma = nullptr, *dbeta = nullptr;
    int accumulate = 0;
};

inline const char* norm_check(const NormArgs& a, bool bwd, int* code) {
    *code = SA3K_ERR_INVALID;
    if (a.type != SA3K_TYPE_F32 && a.type != SA3K_TYPE_F16 && a.type != SA3K_TYPE_BF16) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "type must be f32, f16 or bf16";
    }
    if (a.rows < 0 || a.rows >= kMaxExtent) return "rows out of range";
    if (a.cols <= 0) return "cols must be positive";
    if (a.cols > kNormMaxCols) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "cols must be at most 16384";
    }
    // ranges are written so that a NaN fails them
    if (!bwd && !(a.eps >= 0.f && a.eps <= 3.0e38f)) return "eps must be finite and not negative";
    if (bwd && a.accumulate != 0 && a.accumulate != 1) return "accumulate must be 0 or 1";
    const int64_t ld[5] = {a.ldx, a.ldr, a.lddy, a.ldy, a.ldsum};
    const void* p[5] = {a.x, a.r, a.dy, a.y, a.sum};
    const int eb = elem_bytes(a.type);
    for (int i = 0; i < 5; ++i) {
        if (!p[i]) continue;
        if (ld[i] < a.cols || ld[i] >= kMaxExtent) return "a row pitch is smaller than cols or out of range";
        if (!elem_aligned(p[i], eb)) return "a tensor is not aligned to its elements";
    }
    const void* f[6] = {a.gamma, a.beta, a.mean, a.rstd, a.dgamma, a.dbeta};
    for (const void* q : f)
        if (!elem_aligned(q, 4)) return "an f32 vector is not 4-byte aligned";
    if (a.rows == 0) return nullptr;   // nothing is read or written but the gradients of gain and offset
    if (!bwd) {
        if (!a.x || !a.y) return "x and y must not be null";
        if (a.sum && !a.r) return "a sum needs a residual";
    } else {
        if (!a.x || !a.dy || !a.y || !a.mean || !a.rstd) return "dy, x, mean, rstd and dx must not be null";
    }
    return nullptr;
}

}  // namespace sa3k
