// The gated products' checks of pairs of tensors (csrc/gated.h) for the CPU tests.
#include "gated.h"

using namespace sa3k;

static void* at(int64_t v) { return reinterpret_cast<void*>((uintptr_t)v); }

extern "C" {

// p: X, Wg, Wu, dY, G, U, Y, g output, u output, dX, dWg, dWu, bg, bu, dbg, dbu as addresses; ld: x, w, dy, z, y, dx, dw. 0: nothing
// meets, 1: refused here, 2: the arguments are refused before
int apart(int type, const int64_t* mnk, const int64_t* p, const int64_t* ld, int dw_type, int bwd) {
    GatedArgs a;
    a.type = type; a.act = SA3K_ACT_SILU; a.M = mnk[0]; a.N = mnk[1]; a.K = mnk[2];
    a.X = at(p[0]); a.Wg = at(p[1]); a.Wu = at(p[2]); a.dY = at(p[3]); a.G = at(p[4]); a.U = at(p[5]); a.Y = at(p[6]);
    a.Go = at(p[7]); a.Uo = at(p[8]); a.dX = at(p[9]); a.dWg = at(p[10]); a.dWu = at(p[11]);
    a.bg = (const float*)at(p[12]); a.bu = (const float*)at(p[13]); a.dbg = (float*)at(p[14]); a.dbu = (float*)at(p[15]);
    a.ldx = ld[0]; a.ldw = ld[1]; a.lddy = ld[2]; a.ldz = ld[3]; a.ldy = ld[4]; a.lddx = ld[5]; a.lddw = ld[6];
    a.dw_type = dw_type;
    int code = -1;
    if (gated_check(a, bwd != 0, &code)) return 2;
    return gated_apart(a, bwd != 0) ? 1 : 0;
}
// x, y: address, pitch, rows and width in bytes
int meet(const int64_t* x, const int64_t* y) {
    return rows_meet(Rows{(uintptr_t)x[0], x[1], x[2], x[3]}, Rows{(uintptr_t)y[0], y[1], y[2], y[3]});
}

}  // extern "C"
