// The head norms' check of pairs of tensors (csrc/head_norm.h) for the CPU tests.
#include "head_norm.h"

using namespace sa3k;

static void* at(int64_t v) { return reinterpret_cast<void*>((uintptr_t)v); }

extern "C" {

// p: q, k, v, dqo, dko, q_gain, k_gain, pos, slot, len, qo, ko, vo, dq_gain, dk_gain as addresses. 0: each output has a place of its
// own, 1: refused here, 2: refused before
int apart(int tokens, int cache, const int64_t* p, int bwd) {
    sa3k_head_norm d{};
    d.type = SA3K_TYPE_BF16; d.batch = 2; d.tokens = tokens; d.heads = d.kv_heads = 2; d.head_dim = 64; d.rope_dims = 32;
    d.cache_tokens = cache; d.eps = 1e-6f; d.rope_base = 1e4f;
    int64_t* s[6] = {d.q_stride, d.k_stride, d.v_stride, d.q_out_stride, d.k_out_stride, d.v_out_stride};
    for (int64_t* t : s) {
        t[0] = 4096;
        t[1] = 128;
        t[2] = 64;
    }
    HeadPtrs h;
    h.q = at(p[0]); h.k = at(p[1]); h.v = at(p[2]); h.dqo = at(p[3]); h.dko = at(p[4]); h.q_gain = at(p[5]); h.k_gain = at(p[6]);
    h.pos = at(p[7]); h.slot = at(p[8]); h.len = at(p[9]); h.qo = at(p[10]); h.ko = at(p[11]); h.vo = at(p[12]);
    h.dq_gain = at(p[13]); h.dk_gain = at(p[14]);
    int code = -1;
    if (head_norm_check(&d, h, bwd != 0, &code)) return 2;
    return head_norm_apart(d, h, bwd != 0) ? 1 : 0;
}

}  // extern "C"
