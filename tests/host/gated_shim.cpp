// The gated products' argument checks and plans (csrc/gated.h) for the CPU tests.
#include "gated.h"

using namespace sa3k;

static void* at(int64_t v) { return reinterpret_cast<void*>((uintptr_t)v); }

extern "C" {

// p: X, Wg, Wu, dY, G, U, Y, g output, u output, dX, dWg, dWu, bg, bu, dbg, dbu as addresses; ld: x, w, dy, z, y, dx, dw
int gated(int type, int act, const int64_t* mnk, const int64_t* p, const int64_t* ld, int dw_type, int accumulate, int bwd) {
    GatedArgs a;
    a.type = type; a.act = act; a.M = mnk[0]; a.N = mnk[1]; a.K = mnk[2];
    a.X = at(p[0]); a.Wg = at(p[1]); a.Wu = at(p[2]); a.dY = at(p[3]); a.G = at(p[4]); a.U = at(p[5]); a.Y = at(p[6]);
    a.Go = at(p[7]); a.Uo = at(p[8]); a.dX = at(p[9]); a.dWg = at(p[10]); a.dWu = at(p[11]);
    a.bg = (const float*)at(p[12]); a.bu = (const float*)at(p[13]); a.dbg = (float*)at(p[14]); a.dbu = (float*)at(p[15]);
    a.ldx = ld[0]; a.ldw = ld[1]; a.lddy = ld[2]; a.ldz = ld[3]; a.ldy = ld[4]; a.lddx = ld[5]; a.lddw = ld[6];
    a.dw_type = dw_type; a.accumulate = accumulate;
    int code = -1;
    return gated_check(a, bwd != 0, &code) ? code : 0;
}
// forward: edge (of few rows: their blocks), splits; both of the backward's products: together, edge and splits of dX, of dW; dX alone: edge, splits; dW alone
void plans(int64_t M, int64_t N, int64_t K, int* out) {
    const int64_t h = 2 * gated_half(N), Kp = (K + 7) / 8 * 8;
    const ProdPlan f = gated_plan(M, N, Kp), x = prod_plan(M, K, h), w = prod_plan(h, K, M);
    const ProdPair p = gated_pair(M, N, K, x, w);
    const int few = few_blocks(M, N, K, K % 8 != 0);   // (tensors without gaps)
    out[0] = few ? few : f.edge; out[1] = few ? 1 : f.splits;
    out[2] = p.together; out[3] = p.a.edge; out[4] = p.a.splits; out[5] = p.b.edge; out[6] = p.b.splits;
    out[7] = x.edge; out[8] = x.splits; out[9] = w.edge; out[10] = w.splits;
}
double span(int64_t nx, double tx, int64_t nw, double tw, int64_t slots) { return pair_span(nx, tx, nw, tw, slots); }

}  // extern "C"
