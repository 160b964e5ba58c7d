// The sizes of the layer operators' launches and scratch (csrc/layer_ops.h) for the CPU tests.
#include "layer_ops.h"

using namespace sa3k;

extern "C" {

// i: type, batch, heads, kv_heads, head_dim, q_tokens, k_tokens, left, right, sinks, causal;
// out: tiles, tiles with first tokens, shares of those, shares of the others, workgroups, workgroups with a place in the scratch
void key_shares(const int* i, int* out) {
    sa3k_window_attn d{};
    d.type = i[0]; d.batch = i[1]; d.heads = i[2]; d.kv_heads = i[3]; d.head_dim = i[4]; d.q_tokens = i[5];
    d.k_tokens = i[6]; d.left = i[7]; d.right = i[8]; d.sinks = i[9]; d.causal = i[10];
    const KeySplit k = key_split(attn_shape(d, nullptr, nullptr));
    out[0] = k.tiles; out[1] = k.first_tiles; out[2] = k.first; out[3] = k.rest;
    out[4] = k.items(); out[5] = k.shares();
}

}  // extern "C"
