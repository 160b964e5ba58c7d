// The layer operators' argument checks and variant rules (csrc/layer_ops.h) for the CPU tests.
#include "layer_ops.h"

using namespace sa3k;

static const void* at(int64_t v) { return reinterpret_cast<const void*>((uintptr_t)v); }

extern "C" {

// p: x, r, dy, y, sum, gamma, beta, mean, rstd, dgamma, dbeta as addresses; ld: x, r, dy, y, sum
int norm(int type, int64_t rows, int64_t cols, float eps, int accumulate, int bwd, const int64_t* p, const int64_t* ld) {
    NormArgs a;
    a.type = type; a.rows = rows; a.cols = cols; a.eps = eps; a.accumulate = accumulate;
    a.x = at(p[0]); a.r = at(p[1]); a.dy = at(p[2]);
    a.y = const_cast<void*>(at(p[3])); a.sum = const_cast<void*>(at(p[4]));
    a.gamma = (const float*)at(p[5]); a.beta = (const float*)at(p[6]);
    a.mean = (float*)at(p[7]); a.rstd = (float*)at(p[8]); a.dgamma = (float*)at(p[9]); a.dbeta = (float*)at(p[10]);
    a.ldx = ld[0]; a.ldr = ld[1]; a.lddy = ld[2]; a.ldy = ld[3]; a.ldsum = ld[4];
    int code = -1;
    return norm_check(a, bwd != 0, &code) ? code : 0;
}

}  // extern "C"
