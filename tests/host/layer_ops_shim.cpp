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

// i: type, batch, heads, kv_heads, head_dim, q_tokens, k_tokens, left, right, sinks, causal; st: the 12 strides;
// p: q, k, v, o, dO, lse, q_len, k_len, dq, dk, dv as addresses
static sa3k_window_attn shape(const int* i, float scale, const int64_t* st) {
    sa3k_window_attn d;
    d.type = i[0]; d.batch = i[1]; d.heads = i[2]; d.kv_heads = i[3]; d.head_dim = i[4]; d.q_tokens = i[5];
    d.k_tokens = i[6]; d.left = i[7]; d.right = i[8]; d.sinks = i[9]; d.causal = i[10];
    d.scale = scale;
    for (int k = 0; k < 3; ++k) {
        d.q_stride[k] = st[k]; d.k_stride[k] = st[3 + k]; d.v_stride[k] = st[6 + k]; d.o_stride[k] = st[9 + k];
    }
    return d;
}
int attn(const int* i, float scale, const int64_t* st, const int64_t* p, int bwd) {
    const sa3k_window_attn d = shape(i, scale, st);
    AttnPtrs a;
    const void** f[11] = {&a.q, &a.k, &a.v, &a.o, &a.dO, &a.lse, &a.q_len, &a.k_len, &a.dq, &a.dk, &a.dv};
    for (int k = 0; k < 11; ++k) *f[k] = at(p[k]);
    int code = -1;
    return attn_check(&d, a, bwd != 0, &code) ? code : 0;
}
int attn_null() {
    int code = -1;
    return attn_check(nullptr, AttnPtrs(), false, &code) ? code : 0;
}
// out: lo, n, first
void seen(int p, int nk, const int* w, int* out) {
    const Seen s = seen_by(p, nk, w[0], w[1], w[2], w[3]);
    out[0] = s.lo; out[1] = s.n; out[2] = s.first;
}
// the key blocks of positions pa .. pb, at most `most` of them
int blocks(int pa, int pb, int nk, const int* w, int blk, int* out, int most) {
    const KeyBlocks k = key_blocks(pa, pb, nk, w[0], w[1], w[2], w[3], blk);
    for (int i = 0; i < k.count && i < most; ++i) out[i] = key_block(k, i);
    return k.count;
}
void from(int k0, int k1, int nq, int off, const int* w, int* out) {
    const Span s = seen_from(k0, k1, nq, off, w[0], w[1], w[2], w[3]);
    out[0] = s.lo; out[1] = s.hi;
}
// tile, split and splits of every item of the dK/dV pass; splits of the keys of a few queries
int items(const int* i, const int64_t* st, int* out, int most, int* few) {
    const AttnShape a = attn_shape(shape(i, 1.f, st), nullptr, nullptr);
    const KeySplit k = key_split(a);
    for (int n = 0; n < k.items() && n < most; ++n) {
        const KeyItem t = key_item(k, n);
        out[3 * n] = t.tile; out[3 * n + 1] = t.split; out[3 * n + 2] = t.splits;
    }
    *few = attn_splits(a, (a.Sq * a.G + 31) / 32);
    return k.items();
}

// p: X, W, R, dY, Z, Y, z output, dX, dW, bias, db as addresses; ld: x, w, r, dy, z, y, dx, dw
int prod(int type, int act, const int64_t* mnk, const int64_t* p, const int64_t* ld, int dw_type, int accumulate, int bwd) {
    ProdArgs a;
    a.type = type; a.act = act; a.M = mnk[0]; a.N = mnk[1]; a.K = mnk[2];
    a.X = at(p[0]); a.W = at(p[1]); a.R = at(p[2]); a.dY = at(p[3]); a.Z = at(p[4]);
    a.Y = const_cast<void*>(at(p[5])); a.Zo = const_cast<void*>(at(p[6]));
    a.dX = const_cast<void*>(at(p[7])); a.dW = const_cast<void*>(at(p[8]));
    a.bias = (const float*)at(p[9]); a.db = (float*)at(p[10]);
    a.ldx = ld[0]; a.ldw = ld[1]; a.ldr = ld[2]; a.lddy = ld[3]; a.ldz = ld[4]; a.ldy = ld[5]; a.lddx = ld[6]; a.lddw = ld[7];
    a.dw_type = dw_type; a.accumulate = accumulate;
    int code = -1;
    return prod_check(a, bwd != 0, &code) ? code : 0;
}
void plan(int64_t M, int64_t N, int64_t K, int* out) {
    const ProdPlan p = prod_plan(M, N, K);
    out[0] = p.edge; out[1] = p.splits; out[2] = p.per;
}

int split_keys(const int* i, const int64_t* st) { return attn_split_keys(attn_shape(shape(i, 1.f, st), nullptr, nullptr)); }

// together, then edge, splits and per of each
void pair(const int64_t* x, const int64_t* y, int* out) {
    const int64_t a[3] = {x[0], x[1], x[2]}, b[3] = {y[0], y[1], y[2]};
    const ProdPair p = prod_pair(a, b);
    out[0] = p.together;
    out[1] = p.a.edge; out[2] = p.a.splits; out[3] = p.a.per;
    out[4] = p.b.edge; out[5] = p.b.splits; out[6] = p.b.per;
}

}  // extern "C"
