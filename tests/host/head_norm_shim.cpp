// The head norms' argument checks and angles (csrc/head_norm.h) for the CPU tests.
#include "head_norm.h"

using namespace sa3k;

static void* at(int64_t v) { return reinterpret_cast<void*>((uintptr_t)v); }

extern "C" {

// i: type, batch, tokens, heads, kv_heads, head_dim, rope_dims, neighbours, cache_tokens; st: the 18 strides; p: q, k, v, dqo, dko,
// q_gain, k_gain, pos, slot, len, qo, ko, vo, dq_gain, dk_gain as addresses
int head_norm(const int* i, float eps, float base, const int64_t* st, const int64_t* p, int accumulate, int bwd) {
    sa3k_head_norm d;
    d.type = i[0]; d.batch = i[1]; d.tokens = i[2]; d.heads = i[3]; d.kv_heads = i[4]; d.head_dim = i[5]; d.rope_dims = i[6];
    d.neighbours = i[7]; d.cache_tokens = i[8]; d.eps = eps; d.rope_base = base;
    int64_t* s[6] = {d.q_stride, d.k_stride, d.v_stride, d.q_out_stride, d.k_out_stride, d.v_out_stride};
    for (int n = 0; n < 18; ++n) s[n / 3][n % 3] = st[n];
    HeadPtrs h;
    h.q = at(p[0]); h.k = at(p[1]); h.v = at(p[2]); h.dqo = at(p[3]); h.dko = at(p[4]); h.q_gain = at(p[5]); h.k_gain = at(p[6]);
    h.pos = at(p[7]); h.slot = at(p[8]); h.len = at(p[9]); h.qo = at(p[10]); h.ko = at(p[11]); h.vo = at(p[12]);
    h.dq_gain = at(p[13]); h.dk_gain = at(p[14]); h.accumulate = accumulate;
    int code = -1;
    return head_norm_check(&d, h, bwd != 0, &code) ? code : 0;
}
int head_norm_null() {
    int code = -1;
    return head_norm_check(nullptr, HeadPtrs(), false, &code) ? code : 0;
}
void turns(int dims, float base, uint64_t* out) { head_turns(dims, base, out); }
int parts(int heads, int dim) { return head_parts(heads, dim); }
int lanes(int dim) { return head_lanes(dim); }

}  // extern "C"
