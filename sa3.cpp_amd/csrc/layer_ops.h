// Host-side arithmetic of the layer operators (layer norm, windowed attention, fused products): the
// checks of their arguments and the rules that pick a variant. No HIP in here: compiled with g++ in the
// CPU tests too. A check returns null, or the message of the first thing that is wrong, and sets `code`
// to the status an entry point returns with it.
#pragma once

#include <cstdint>

#include "sa3k.h"

#ifdef __HIPCC__
#define SA3K_HD __host__ __device__ inline
#else
#define SA3K_HD inline
#endif

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

// ------------------------------------------------------------------------------------- attention
constexpr int kFar = 1 << 29;           // no bound: further than any two positions (k_tokens, q_tokens < 2^28)
constexpr int kMaxTokens = 1 << 28;
constexpr int64_t kMaxTokenStride = (int64_t)1 << 24;   // 64 rows of it in bytes stay below 2^31
constexpr int64_t kMaxStride = (int64_t)1 << 40;

// an output's rows must not overlap: by growing stride, each step passes everything below it
inline bool rows_apart(const int64_t* st, const int64_t* n, int64_t row) {
    if (n[0] == 0 || n[1] == 0 || n[2] == 0) return true;
    int order[3] = {0, 1, 2};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (st[order[j]] < st[order[i]]) { const int t = order[i]; order[i] = order[j]; order[j] = t; }
    int64_t reach = row;
    for (int i = 0; i < 3; ++i) {
        const int d = order[i];
        if (n[d] <= 1) continue;
        if (st[d] < reach) return false;
        reach += st[d] * (n[d] - 1);
    }
    return true;
}

struct AttnPtrs {
    const void *q = nullptr, *k = nullptr, *v = nullptr, *o = nullptr, *dO = nullptr;
    const void *lse = nullptr, *q_len = nullptr, *k_len = nullptr, *dq = nullptr, *dk = nullptr, *dv = nullptr;
};

inline const char* attn_check(const sa3k_window_attn* d, const AttnPtrs& p, bool bwd, int* code) {
    *code = SA3K_ERR_INVALID;
    if (!d) return "null shape";
    if (d->type != SA3K_TYPE_BF16 && d->type != SA3K_TYPE_F16) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "type must be bf16 or f16";
    }
    if (d->head_dim != 64 && d->head_dim != 128) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "head_dim must be 64 or 128";
    }
    if (d->batch < 0 || d->batch > 65535 || d->heads <= 0 || d->heads > 65535) return "batch or heads out of range";
    if (d->kv_heads <= 0 || d->heads % d->kv_heads != 0) return "heads must be a multiple of kv_heads";
    if (d->q_tokens < 0 || d->q_tokens >= kMaxTokens || d->k_tokens < 0 || d->k_tokens >= kMaxTokens)
        return "q_tokens or k_tokens out of range";
    if (d->sinks < 0) return "sinks must not be negative";
    if (d->causal != 0 && d->causal != 1) return "causal must be 0 or 1";
    if (!(d->scale > 0.f && d->scale <= 1.0e30f)) return "scale must be positive and finite";
    const int64_t nq[3] = {d->batch, d->q_tokens, d->heads}, nk[3] = {d->batch, d->k_tokens, d->kv_heads};
    const int64_t* st[4] = {d->q_stride, d->k_stride, d->v_stride, d->o_stride};
    for (int t = 0; t < 4; ++t)
        for (int i = 0; i < 3; ++i) {
            const int64_t v = st[t][i];
            const int64_t n = (t == 1 || t == 2 ? nk : nq)[i];
            if (n <= 1) continue;   // never used
            if (v < 0 || v >= kMaxStride || v % 8 != 0) return "strides must be multiples of 8, not negative";
            if (i == 1 && (v < d->head_dim || v >= kMaxTokenStride))
                return "tokens must be at least head_dim and less than 2^24 elements apart";
        }
    if (!rows_apart(d->o_stride, nq, d->head_dim)) return "the rows of o overlap";
    if (bwd && (!rows_apart(d->q_stride, nq, d->head_dim) || !rows_apart(d->k_stride, nk, d->head_dim) ||
                !rows_apart(d->v_stride, nk, d->head_dim)))
        return "the rows of q, k or v overlap, and their gradients have the same layout";
    // one grid dimension, of fewer than 2^32 threads: at the most 16 a row
    const int64_t most = (d->q_tokens > d->k_tokens ? d->q_tokens : d->k_tokens) / 64 + 1;
    if (most * d->batch * d->heads >= ((int64_t)1 << 21)) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "batch x heads x tokens is too large for one launch";
    }
    if (!elem_aligned(p.q_len, 4) || !elem_aligned(p.k_len, 4) || !elem_aligned(p.lse, 4))
        return "lengths and lse must be 4-byte aligned";
    const void* t[8] = {p.q, p.k, p.v, p.o, p.dO, p.dq, p.dk, p.dv};
    for (const void* x : t)
        if (!elem_aligned(x, 16)) return "tensors must be 16-byte aligned";
    if (d->batch == 0) return nullptr;
    if (d->q_tokens > 0) {
        if (!p.q || !p.o) return "q and o must not be null";
        if (bwd && (!p.dO || !p.lse || !p.dq)) return "lse, dO and dq must not be null";
    }
    if (d->k_tokens > 0) {
        if (!p.k || !p.v) return "k and v must not be null";
        if (bwd && (!p.dk || !p.dv)) return "dk and dv must not be null";
    }
    return nullptr;
}

// The kernels' view of the shape: bounds resolved, lengths in range, strides of single tokens made valid.
struct AttnShape {
    int B, H, K, G, D, Sq, Sk, left, right, sinks, causal;
    float scale;
    int64_t qs[3], ks[3], vs[3], os[3];
    const int32_t *q_len, *k_len;
};

inline AttnShape attn_shape(const sa3k_window_attn& d, const void* q_len, const void* k_len) {
    AttnShape a;
    a.B = d.batch; a.H = d.heads; a.K = d.kv_heads; a.G = d.heads / d.kv_heads; a.D = d.head_dim;
    a.Sq = d.q_tokens; a.Sk = d.k_tokens;
    a.left = d.left < 0 || d.left > kFar ? kFar : d.left;
    a.right = d.causal ? 0 : d.right < 0 || d.right > kFar ? kFar : d.right;
    a.sinks = d.sinks < d.k_tokens ? d.sinks : d.k_tokens;
    a.causal = d.causal;
    a.scale = d.scale;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = d.q_stride[i];
        a.ks[i] = d.k_stride[i];
        a.vs[i] = d.v_stride[i];
        a.os[i] = d.o_stride[i];
    }
    if (a.Sq <= 1) a.qs[1] = a.os[1] = a.D;
    if (a.Sk <= 1) a.ks[1] = a.vs[1] = a.D;
    a.q_len = static_cast<const int32_t*>(q_len);
    a.k_len = static_cast<const int32_t*>(k_len);
    return a;
}

// The keys a query at position p of a sample with nk keys sees: lo .. lo + n - 1, and 0 .. first - 1.
struct Seen {
    int lo, n, first;
};
SA3K_HD Seen seen_by(int p, int nk, int left, int right, int sinks, int causal) {
    const int last = causal && p < nk - 1 ? p : nk - 1;
    const int lo = p - left > 0 ? p - left : 0;
    const int top = p + right < last ? p + right : last;
    Seen s;
    s.lo = lo;
    s.n = top >= lo ? top - lo + 1 : 0;
    s.first = sinks < last + 1 ? sinks : last + 1;
    if (s.first < 0) s.first = 0;
    return s;
}
// The blocks of `blk` keys that the queries of positions pa .. pb see, in order: `head` blocks from 0, then
// those from `from` on, `count` in all.
struct KeyBlocks {
    int head, from, count;
};
SA3K_HD KeyBlocks key_blocks(int pa, int pb, int nk, int left, int right, int sinks, int causal, int blk) {
    const Seen a = seen_by(pa, nk, left, right, sinks, causal), b = seen_by(pb, nk, left, right, sinks, causal);
    const int ns = (b.first + blk - 1) / blk;          // a later query sees no fewer first tokens
    const int top = b.lo + b.n - 1;                    // nor a lower last key
    KeyBlocks r;
    if (b.n == 0 || top < a.lo) {
        r.head = ns;
        r.from = ns;
        r.count = ns;
        return r;
    }
    const int wl = a.lo / blk, wh = top / blk + 1;
    r.head = ns < wl ? ns : wl;
    r.from = wl;
    r.count = r.head + (wh > ns ? wh : ns) - wl;
    return r;
}
SA3K_HD int key_block(const KeyBlocks& r, int i) { return i < r.head ? i : r.from + (i - r.head); }


// The most keys that a sample's queries see.
inline int64_t keys_seen(const AttnShape& s) {
    const int64_t reach = (int64_t)s.left + s.right + s.Sq + 32;
    return (reach < s.Sk ? reach : s.Sk) + s.sinks;
}
// Whether the keys are split over workgroups and waves, 32 rows (query, member of the group) at a time, instead of running by
// tiles of 128 queries a head. Measured on MI355X (tiles / split, us; bf16, all keys visible but where a window is named):
//   one query, 32 heads of 128 on 8:   1 x 16384 keys 337 / 20.0, 8 x 4096 keys 87 / 30, 8 x 512 keys 14.7 / 11.6
//   32 queries of such heads:          1 x 16384 keys 289 / 35.6, 8 x 2048 keys 41 / 35, 8 x 512 keys 13.3 / 21.7
//   self-attention, by its tiles:      24 tiles 9.6 / 7.3, 64 tiles 19.1 / 11.2, 120 tiles 13.9 / 11.5, 128 tiles 46.5 / 35.8 and
//                                      (window 256) 9.5 / 8.8, 160 tiles 29.1 / 32.5, 192 tiles 18.2 / 20.7, 432 tiles 28.5 / 43
// The split serves where there are rows for one chunk only, or too few tiles for the chip.
inline bool attn_split_keys(const AttnShape& s) {
    const int64_t tiles = (int64_t)s.B * s.H * ((s.Sq + 127) / 128);
    return (int64_t)s.Sq * s.G <= 32 || tiles <= 128 || (s.Sq <= 32 && keys_seen(s) > 1024);
}
// The split count for `chunks` chunks of 32 rows a key/value head: a workgroup a CU in all (8 x one query over windows of 4096
// keys: 128 / 256 / 512 / 1024 workgroups 34.0 / 29.5 / 33.1 / 41.5 us), at least two blocks of 32 keys a wave.
inline int attn_splits(const AttnShape& s, int chunks) {
    const int64_t base = (int64_t)s.B * s.K * chunks, most = keys_seen(s) / (32 * 4 * 2);
    int64_t n = 256 / (base > 0 ? base : 1);
    if (n > most) n = most;
    return n < 1 ? 1 : (int)n;
}

// The dK/dV pass: a workgroup takes a tile of 128 keys and a share of the (query head, block of 64 queries) pairs that
// see it. Tiles with first tokens, which every later query sees, get `first` shares, the others `rest`.
constexpr int kKeyTile = 128;
struct KeySplit {
    int tiles, first_tiles, first, rest;   // first_tiles of the tiles hold first tokens
    SA3K_HD int items() const { return first_tiles * first + (tiles - first_tiles) * rest; }   // workgroups a k/v head
    // those whose sums a second launch adds up, and which have a place in the scratch: they come first among the items
    SA3K_HD int shares() const { return rest > 1 ? items() : first > 1 ? first_tiles * first : 0; }
};
inline KeySplit key_split(const AttnShape& s, int* priced = nullptr) {   // priced: the plans that were
    KeySplit r;
    r.tiles = (s.Sk + kKeyTile - 1) / kKeyTile;
    r.first_tiles = (s.sinks + kKeyTile - 1) / kKeyTile;
    const int64_t all = s.Sq > 0 ? (s.Sq + 63) / 64 : 1, band = ((int64_t)kKeyTile + s.left + s.right + 62) / 64 + 1;
    const int64_t most = s.G * all, usual = s.G * (band < all ? band : all);
    const int64_t pairs = (int64_t)s.B * s.K, later = r.tiles - r.first_tiles;
    // By estimated time in microseconds, measured on MI355X: two workgroups that share a CU take 0.9 (heads of 64) or 1.95 (of
    // 128) each for a block, one alone 1.35 times that, and a workgroup starts within the time of two blocks; the pass by queries
    // in the same launch takes 0.85 of that a block. The launch lasts as long as its work or its longest workgroup; the one that
    // adds up shares 4, its sums 4 MB a microsecond. (What it chooses is within 5% of the best of 1 to 8 shares on eight shapes:
    // 2 x 24 x 1088, window 128 both ways, 64 first tokens: whole 44.6 us, the first tile in two shares 46.6.)
    const double block = s.D == 64 ? 0.9 : 1.95, share = 2.0 * kKeyTile * s.D * 4 * 2 / 4e6;
    const int64_t q_wgs = (int64_t)s.B * s.H * ((s.Sq + 127) / 128), k_all = (s.Sk + 63) / 64;
    const int64_t k_band = ((int64_t)128 + s.left + s.right + 62) / 64 + 1 + (s.sinks + 63) / 64;
    const double by_query = 0.85 * (double)q_wgs * (double)((k_band < k_all ? k_band : k_all) + 2);
    // The work and the sums grow with either count: a plan that is dearer by these alone ends the search in that direction, and so
    // does one whose first tiles' shares are no longer than the others'. (Priced one by one, the plans of 32 on 1 heads of 64 x 1024
    // took 47 us of host time in every call, of 16 on 2 x 8192 with a window of 4096 105 us; now 0.4 and 0.1.)
    double least = 1e300;
    int count = 0;
    r.first = r.rest = 1;
    for (int64_t n = 1; n <= 64 && (n == 1 || usual / n >= 4); ++n) {   // at least four blocks a workgroup
        const int64_t len = (usual + n - 1) / n, f0 = r.first_tiles > 0 ? n : 1;
        bool dearer = false;   // at f0: so is every larger n
        for (int64_t f = f0; f <= 256 && (f == n || f == 1 || most / f >= 4); ++f) {
            const int64_t wgs = pairs * (r.first_tiles * f + later * n);
            const double work = (double)pairs * (double)(r.first_tiles * most + later * usual) + 2.0 * (double)wgs + by_query;
            const double all_of_it = work * block / 256.0;
            const double sums = n > 1 ? 4.0 + (double)wgs * share
                                : r.first_tiles > 0 && f > 1 ? 4.0 + (double)(pairs * r.first_tiles * f) * share : 0.0;
            ++count;
            if (all_of_it + sums >= least) {
                dearer = f == f0;
                break;
            }
            const int64_t flen = (most + f - 1) / f, longest = r.first_tiles > 0 && flen > len ? flen : later > 0 ? len : flen;
            const double last = (double)(longest + 2) * block * (wgs + q_wgs <= 256 ? 1.35 : 2.0);
            const double t = (all_of_it > last ? all_of_it : last) + sums;
            if (t < least) {
                least = t;
                r.rest = (int)n;
                r.first = (int)f;
            }
            if (r.first_tiles == 0 || (later > 0 && flen <= len)) break;
        }
        if (dearer || later == 0) break;   // (with no other tiles n says nothing)
    }
    if (priced) *priced = count;
    return r;
}
struct KeyItem {
    int tile, split, splits;
};
SA3K_HD KeyItem key_item(const KeySplit& r, int i) {
    KeyItem t;
    const int head = r.first_tiles * r.first;
    if (i < head) {
        t.tile = i / r.first;
        t.split = i - t.tile * r.first;
        t.splits = r.first;
    } else {
        const int j = i - head, q = j / r.rest;
        t.tile = r.first_tiles + q;
        t.split = j - q * r.rest;
        t.splits = r.rest;
    }
    return t;
}
// The queries (of nq, at positions i + off) that see some key of k0 .. k1: lo .. hi (hi < lo: none).
struct Span {
    int lo, hi;
};
SA3K_HD Span seen_from(int k0, int k1, int nq, int off, int left, int right, int sinks, int causal) {
    const bool first = k0 < sinks;
    const int plo = causal ? k0 : first ? -kFar : k0 - right, phi = first ? kFar : k1 + left;
    Span r;
    r.lo = plo - off > 0 ? plo - off : 0;
    r.hi = phi - off < nq - 1 ? phi - off : nq - 1;
    return r;
}

// --------------------------------------------------------------------------------------- product
struct ProdArgs {
    int type = 0, act = 0;
    int64_t M = 0, N = 0, K = 0;
    const void *X = nullptr, *W = nullptr, *R = nullptr, *dY = nullptr, *Z = nullptr;
    void *Y = nullptr, *Zo = nullptr, *dX = nullptr, *dW = nullptr;   // Zo: the forward's z
    int64_t ldx = 0, ldw = 0, ldr = 0, lddy = 0, ldz = 0, ldy = 0, lddx = 0, lddw = 0;
    const float* bias = nullptr;
    float* db = nullptr;
    int dw_type = 0, accumulate = 0;
};

constexpr int64_t kProdMaxPitch = (int64_t)1 << 22;   // 256 rows of it in bytes stay below 2^31

inline const char* prod_check(const ProdArgs& a, bool bwd, int* code) {
    *code = SA3K_ERR_INVALID;
    if (a.type != SA3K_TYPE_BF16 && a.type != SA3K_TYPE_F16) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "type must be bf16 or f16";
    }
    if (a.act < SA3K_ACT_NONE || a.act > SA3K_ACT_GELU_TANH) return "unknown activation";
    if (a.M < 0 || a.M >= kMaxExtent) return "M out of range";
    if (a.N <= 0 || a.K <= 0 || a.N >= kProdMaxPitch || a.K >= kProdMaxPitch) return "N or K out of range";
    if (bwd && a.accumulate != 0 && a.accumulate != 1) return "accumulate must be 0 or 1";
    if (bwd && a.dW && a.dw_type != a.type && a.dw_type != SA3K_TYPE_F32) return "dw_type must be f32 or type";
    if (bwd && a.dW && a.accumulate && a.dw_type != SA3K_TYPE_F32) return "only an f32 dW can be added to";
    const void* p[9] = {a.X, a.W, a.R, a.dY, a.Z, a.Y, a.Zo, a.dX, a.dW};
    const int64_t ld[9] = {a.ldx, a.ldw, a.ldr, a.lddy, a.ldz, a.ldy, a.ldz, a.lddx, a.lddw};
    const int64_t w[9] = {a.K, a.K, a.N, a.N, a.N, a.N, a.N, a.K, a.K};
    for (int i = 0; i < 9; ++i) {
        if (!p[i]) continue;
        if (ld[i] < w[i] || ld[i] >= kProdMaxPitch) return "a row pitch is smaller than its rows or out of range";
        if (!elem_aligned(p[i], i == 8 ? elem_bytes(a.dw_type) : 2)) return "a tensor is not aligned to its elements";
    }
    if (!elem_aligned(a.bias, 4) || !elem_aligned(a.db, 4)) return "an f32 vector is not 4-byte aligned";
    // a launch has fewer than 2^24 workgroups: tiles of 64 x 64 at the least, and the split sums' 2048 values
    if (((a.M + 63) / 64) * ((a.N > a.K ? a.N : a.K) / 64 + 1) >= ((int64_t)1 << 23)) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "M x N is too large for one launch";
    }
    if (!bwd) {
        if (!a.W) return "W must not be null";
        if (a.M > 0 && (!a.X || !a.Y)) return "X and Y must not be null";
    } else {
        if (a.M > 0 && !a.dY) return "dY must not be null";
        if (a.M > 0 && a.act != SA3K_ACT_NONE && !a.Z) return "an activation needs Z";
        if (a.M > 0 && a.dW && !a.X) return "dW needs X";
        if (a.dX && !a.W) return "dX needs W";
    }
    return nullptr;
}

// The tiles (square, `edge` wide) of an M x N x K product and the split of its contraction, by estimated time in
// microseconds. Measured on MI355X: a round of 256 x 256 tiles (one workgroup a CU) takes 1.75 a tile of 64 along K, one of
// 128 x 128 tiles 1.0 with two workgroups a CU and 0.57 with one; a workgroup's start and its stores about 4; the
// launch that adds up splits 4 and its traffic at 4 MB a microsecond. What it chooses is within 3% of the best of both tiles
// and 1 to 6 splits on twelve shapes from 128 to 6144 rows (2176 x 6144 x 1536: 128 x 128 whole 58 us, in two splits 63,
// 256 x 256 in four splits 61, whole 125; 4096 x 1024 x 4096: 256 x 256 43, 128 x 128 51).
struct ProdPlan {
    int edge, splits, per;   // per: tiles of 64 along K that a split takes
    double us;
};
inline double split_sum_us(int64_t n, int64_t M, int64_t N) {
    return n > 1 ? 4.0 + 8.0 * (double)n * (double)M * (double)N / 4e6 : 0.0;
}
inline bool split_fits(int64_t n, int64_t kt, int64_t M, int64_t N) {   // no empty split, at most 256 MB of split sums
    return n == 1 || (n <= kt && (n - 1) * ((kt + n - 1) / n) < kt && (double)n * (double)M * (double)(N + 8) <= 67108864.0);
}
inline ProdPlan prod_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t kt = (K + 63) / 64;
    ProdPlan best{128, 1, (int)kt, 1e300};
    for (int edge = 256; edge >= 128; edge /= 2) {
        const int64_t tiles = ((M + edge - 1) / edge) * ((N + edge - 1) / edge);
        for (int64_t n = 1; n <= 16; ++n) {
            if (!split_fits(n, kt, M, N)) continue;
            const int64_t per = (kt + n - 1) / n, wgs = tiles * n, slots = edge == 256 ? 256 : 512;
            const double step = edge == 256 ? 1.75 : wgs <= 256 ? 0.57 : 1.0;
            const double t = (double)((wgs + slots - 1) / slots) * ((double)per * step + 4.0) + split_sum_us(n, M, N);
            if (t < best.us) best = ProdPlan{edge, (int)n, (int)per, t};
        }
    }
    return best;
}
// Two products of a backward pass, in one launch of 128 x 128 tiles or one after the other. Together they last as long as their
// work, half a microsecond a tile of 64 along K with two workgroups a CU, or their longest workgroup; a launch saved is 4. Measured
// on MI355X (M x K -> N, bf16; together / one after the other, us; * what this chooses): 64 x 1536 -> 1536 15.9* / 21.2, 1024 x
// 1024 -> 4096 38.4* / 45.2, 2176 x 1536 -> 6144 103* / 113, 2176 x 6144 -> 1536 104* / 100, 4352 x 1536 -> 6144 183* / 196,
// 4096 x 2048 -> 2048 89* / 83, 8704 x 1536 -> 1536 126* / 107, 8704 x 6144 -> 1536 422* / 387, 4096 x 4096 -> 4096 277 / 236*. The
// half microsecond measures 0.51 (4096 x 4096 -> 4096) to 0.64 (4096 x 2048 -> 2048): above about 4096 rows it favours the one launch too far.
struct ProdPair {
    bool together;
    ProdPlan a, b;
};
inline ProdPair prod_pair(const int64_t (&x)[3], const int64_t (&y)[3]) {   // {M, N, K} of each
    ProdPair best{false, prod_plan(x[0], x[1], x[2]), prod_plan(y[0], y[1], y[2])};
    double least = best.a.us + best.b.us + 4.0;
    const int64_t ka = (x[2] + 63) / 64, kb = (y[2] + 63) / 64;
    const int64_t ta = ((x[0] + 127) / 128) * ((x[1] + 127) / 128), tb = ((y[0] + 127) / 128) * ((y[1] + 127) / 128);
    for (int64_t n = 1; n <= 8; ++n)
        for (int64_t m = 1; m <= 8; ++m) {
            if (!split_fits(n, ka, x[0], x[1]) || !split_fits(m, kb, y[0], y[1])) continue;
            const int64_t pa = (ka + n - 1) / n, pb = (kb + m - 1) / m, wgs = ta * n + tb * m;
            const double work = 0.5 * ((double)(ta * ka) + (double)(tb * kb) + 4.0 * (double)wgs) / 256.0;
            const double last = (double)(pa > pb ? pa : pb) * (wgs <= 256 ? 0.65 : 1.0) + 4.0;
            const double t = (work > last ? work : last) + split_sum_us(n, x[0], x[1]) + split_sum_us(m, y[0], y[1]);
            if (t < least) {
                least = t;
                best = ProdPair{true, ProdPlan{128, (int)n, (int)pa, t}, ProdPlan{128, (int)m, (int)pb, t}};
            }
        }
    return best;
}
// Few rows run on a kernel whose waves split K, without tiles in LDS. Measured on MI355X (few / tiles, us): 1 x 1536 x 6144
// 7.0 / 12.8, 8 rows 7.9 / 13.6, 16 rows 8.9 / 12.1; with a second block of 16 rows, 32 rows 14.3 / 12.8.
constexpr int64_t kFewRows = 16;

}  // namespace sa3k
