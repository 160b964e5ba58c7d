// Host-side arithmetic of the head norms with rotation: the checks of their arguments, the frequencies and the shape of
// the launches. No HIP in here: compiled with g++ in the CPU tests too.
#pragma once

#include <cmath>

#include "layer_ops.h"

namespace sa3k {

constexpr int kHeadMaxDim = 256;
constexpr int kHeadMaxTokens = 1 << 28;

struct HeadPtrs {
    const void *q = nullptr, *k = nullptr, *v = nullptr;      // the projections
    const void *dqo = nullptr, *dko = nullptr;                // backward: the outputs' gradients
    const void *q_gain = nullptr, *k_gain = nullptr, *pos = nullptr, *slot = nullptr, *len = nullptr;
    void *qo = nullptr, *ko = nullptr, *vo = nullptr;         // forward: the outputs; backward: dq and dk in qo and ko
    void *dq_gain = nullptr, *dk_gain = nullptr;
    int accumulate = 0;
};

// one tensor's strides over (samples, tokens, heads) and its address; out: it is written
inline const char* head_tensor_check(const void* p, const int64_t* st, const int64_t* n, int dim, int bytes, bool out) {
    if (!elem_aligned(p, bytes)) return "a tensor is not aligned to its elements";
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && (st[i] < 0 || st[i] >= kMaxStride)) return "a stride is negative or out of range";
    if (out && !rows_apart(st, n, dim)) return "the rows of an output overlap";
    return nullptr;
}
// x and y may be the same tensor, not two views of one address
inline bool same_place(const void* x, const void* y, const int64_t* sx, const int64_t* sy, const int64_t* n) {
    if (!x || x != y) return true;
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && sx[i] != sy[i]) return false;
    return true;
}

// lanes that share a head, eight of its elements each
inline int head_lanes(int dim) { return dim <= 32 ? 4 : dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }
// a wave takes this many groups of 64 / lanes heads at the most, and a tensor's heads are that many waves' to a row
constexpr int kGroups = 3;
inline int head_parts(int heads, int dim) {
    const int per = kGroups * (64 / head_lanes(dim));
    return (heads + per - 1) / per;
}

inline const char* head_norm_check(const sa3k_head_norm* d, const HeadPtrs& p, bool bwd, int* code) {
    *code = SA3K_ERR_INVALID;
    if (!d) return "null shape";
    if (d->type != SA3K_TYPE_F32 && d->type != SA3K_TYPE_F16 && d->type != SA3K_TYPE_BF16) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "type must be f32, f16 or bf16";
    }
    if (d->head_dim <= 0 || d->head_dim > kHeadMaxDim || d->head_dim % 8 != 0) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "head_dim must be a multiple of 8, at most 256";
    }
    if (d->rope_dims < 0 || d->rope_dims > d->head_dim) return "rope_dims must lie within head_dim";
    if (d->rope_dims % 16 != 0) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "rope_dims must be a multiple of 16";
    }
    if (d->neighbours != 0 && d->neighbours != 1) return "neighbours must be 0 or 1";
    if (d->batch < 0 || d->batch > 65535 || d->tokens < 0 || d->tokens >= kHeadMaxTokens) return "batch or tokens out of range";
    if ((int64_t)d->batch * d->tokens >= kMaxExtent) return "batch x tokens out of range";
    if (d->heads <= 0 || d->heads > 65535 || d->kv_heads <= 0 || d->kv_heads > 65535) return "heads or kv_heads out of range";
    // ranges are written so that a NaN fails them
    if (!(d->eps >= 0.f && d->eps <= 3.0e38f)) return "eps must be finite and not negative";
    if (!(d->rope_base >= 1.f && d->rope_base <= 3.0e38f)) return "rope_base must be finite and at least 1";
    if (d->cache_tokens < 0 || d->cache_tokens >= kHeadMaxTokens) return "cache_tokens out of range";
    if (p.slot && d->cache_tokens == 0) return "slots need cache_tokens";
    if (bwd && p.accumulate != 0 && p.accumulate != 1) return "accumulate must be 0 or 1";
    const void* f[7] = {p.q_gain, p.k_gain, p.pos, p.slot, p.len, p.dq_gain, p.dk_gain};
    for (const void* x : f)
        if (!elem_aligned(x, 4)) return "gains, positions, slots and lengths must be 4-byte aligned";
    if (p.dq_gain && p.dk_gain) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(p.dq_gain), b = reinterpret_cast<uintptr_t>(p.dk_gain);
        if ((a > b ? a - b : b - a) < 4 * (uintptr_t)d->head_dim) return "the gains' gradients overlap";
    }
    if (d->batch == 0 || d->tokens == 0) return nullptr;   // nothing is read or written but the gains' gradients
    const int eb = elem_bytes(d->type), D = d->head_dim;
    const int64_t nq[3] = {d->batch, d->tokens, d->heads}, nk[3] = {d->batch, d->tokens, d->kv_heads};
    const int64_t nc[3] = {d->batch, p.slot ? d->cache_tokens : d->tokens, d->kv_heads};
    if (!p.q && !p.k && !p.v) return "q, k and v are all null";
    if (!p.q != !p.qo || !p.k != !p.ko || !p.v != !p.vo) return "q, k and v need an output each, and an output its input";
    if (bwd && ((p.q && !p.dqo) || (p.k && !p.dko))) return "q and k need their outputs' gradients";
    if (bwd && ((p.dq_gain && !p.q) || (p.dk_gain && !p.k))) return "a gain's gradient needs its heads";
    // four rows a workgroup, a launch of fewer than 2^24 workgroups
    const int64_t parts = head_parts(d->heads, D) + 2 * (int64_t)head_parts(d->kv_heads, D);
    if (((int64_t)d->batch * d->tokens / 4 + 1) * parts >= ((int64_t)1 << 24)) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "batch x tokens x heads is too large for one launch";
    }
    const char* m = nullptr;
    // backward: dqo and dko lie as the outputs do, dq and dk as q and k do
    const struct { const void* p; const int64_t *st, *n; bool out; } t[8] = {
        {p.q, d->q_stride, nq, false}, {p.k, d->k_stride, nk, false}, {p.v, d->v_stride, nk, false},
        {p.qo, bwd ? d->q_stride : d->q_out_stride, nq, true}, {p.ko, bwd ? d->k_stride : d->k_out_stride, bwd ? nk : nc, true},
        {p.vo, d->v_out_stride, nc, true}, {p.dqo, d->q_out_stride, nq, false}, {p.dko, d->k_out_stride, nk, false}};
    for (const auto& x : t)
        if (x.p && (m = head_tensor_check(x.p, x.st, x.n, D, eb, x.out))) return m;
    if ((p.qo && (p.qo == p.ko || p.qo == p.vo)) || (p.ko && p.ko == p.vo)) return "two outputs are the same tensor";
    if (!bwd && p.slot && ((p.ko && p.ko == p.k) || (p.vo && p.vo == p.v))) return "k and v cannot move within themselves";
    if (!same_place(bwd ? p.dqo : p.q, p.qo, bwd ? d->q_out_stride : d->q_stride, bwd ? d->q_stride : d->q_out_stride, nq) ||
        !same_place(bwd ? p.dko : p.k, p.ko, bwd ? d->k_out_stride : d->k_stride, bwd ? d->k_stride : d->k_out_stride, nk) ||
        !same_place(p.v, p.vo, d->v_stride, d->v_out_stride, nk))
        return "a tensor written in place keeps its strides";
    return nullptr;
}

// What head_norm_check found in order: whether an output begins where another tensor does that it may not be (its own input, forward, and
// its own head's gradient or input, backward, it may). Such calls would read what other workgroups write. (The gains' gradients are written
// when all is read. Tensors that share elements, but not their first, are the caller's to keep apart.)
inline const char* head_norm_apart(const sa3k_head_norm& d, const HeadPtrs& p, bool bwd) {
    if (d.batch == 0 || d.tokens == 0) return nullptr;
    const void* const out[5] = {p.qo, p.ko, p.vo, p.dq_gain, p.dk_gain};
    const void* const in[10] = {p.q, p.k, p.v, p.dqo, p.dko, p.q_gain, p.k_gain, p.pos, p.slot, p.len};
    for (int i = 0; i < 5; ++i) {
        if (!out[i]) continue;
        for (int j = 0; j < i; ++j)
            if (out[i] == out[j]) return "two outputs are the same tensor";
        for (int j = 0; i < 3 && j < 10; ++j)
            if (out[i] == in[j] && j != i && !(bwd && j == i + 3)) return "an output is another head's tensor, or a vector's";
    }
    return nullptr;
}

// Pair i turns by pos base^(-2i / dims) radians. A position is a whole number, so only the fraction of a turn that one
// position makes matters: as 64 bits behind the point, pos times it is exact modulo a turn, and off by |pos| times the fraction's own
// error, wherever pos is. Pair i's is pair (i - n)'s times base^(-2n / dims), n the highest power of two in i: seven products at the
// most, in whole numbers. In units of 2^-64 turns: a power is off by 1 (exp2l) and 1 (its cut), of which a product with a fraction
// below 0.16 turns leaves 0.32, and is rounded to an eighth (fractions are held in quarters), so seven leave 3.1; the exponents' own
// roundings 0.25, the last rounding 0.5: below 4, which is 2^-31 turns at the furthest position. (Repeated products by one power in 80
// bits were off by 7.5 at a base of 1.5; this takes the host 0.28 us for 64 pairs, those took 0.35.)
inline void head_turns(int dims, float base, uint64_t* turn) {
    constexpr long double kOne = 18446744073709551616.0L;   // 2^64
    const long double step = dims > 0 ? -2.0L * log2l((long double)base) / (long double)dims : 0.0L;
    uint64_t f[kHeadMaxDim / 2];   // in quarters of 2^-64 turns
    f[0] = (uint64_t)(4.0L * kOne / 6.283185307179586476925286766559L + 0.5L);
    for (int n = 1; n < dims / 2; n *= 2) {
        const long double p = exp2l(step * (long double)n) * kOne;
        const uint64_t power = p < kOne ? (uint64_t)p : ~(uint64_t)0;
        for (int i = n; i < 2 * n && i < dims / 2; ++i) {
            const unsigned __int128 t = (unsigned __int128)f[i - n] * power + ((uint64_t)1 << 63);
            f[i] = (uint64_t)(t >> 64);
        }
    }
    for (int i = 0; i < dims / 2; ++i) turn[i] = (f[i] + 2) >> 2;
}

}  // namespace sa3k
