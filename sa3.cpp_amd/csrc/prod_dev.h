// The tile kernels of the products and what their callers share (linact.hip: products with bias, activation and residual; gated.hip:
// gated products). In an unnamed namespace: each of these files has the instantiations it uses.
//
// One tile kernel does the products C[m][n] = sum_k A(m, k) B(n, k), on v_mfma_f32_32x32x16 with f32 sums. An operand
// lies K-contiguous ([rows][K]: X, W and dz of dX) or K-major ([K][rows]: W of dX, both of dW); a K-major tile is staged as
// it lies, as sub-tiles of [64 k][64 rows], and read transposed (ds_read_b64_tr_b16), so no operand is ever transposed
// in memory. Tiles of 64 along K go straight into LDS (buffer_load ... lds) through a descriptor that ends where the
// operand does: rows and K past the end are zeros. Two stages; the loads of tile t + 1 run while t is computed.
//
// These loads take 16 bytes: operands whose rows are not 16-byte aligned, or not a multiple of 8 long, are copied once into
// padded rows first (a copy of M K + N K elements against M N K multiply-adds).
#pragma once

#include <algorithm>

#include "wattn.h"

namespace {
using namespace sa3k;
using wattn::buffer_rsrc;
using wattn::dma16;
using wattn::ex2;
using wattn::f32x16;
using wattn::lds_ptr_t;
using wattn::swz;
using wattn::u32x4;
using wattn::Vec;
using wattn::kLog2e;

typedef float f32x4 __attribute__((__vector_size__(4 * sizeof(float))));

// The products: a forward with its epilogue, and the two of a backward. Gated: of two weights, gate and up, side by side.
//   kGatedForward  a tile's B holds as many rows of each weight, in turns of NT / 8 rows; a wave's sums are of the same columns
//                  of both, and the epilogue multiplies them
//   kGatedInput    K is gate's, then up's, each padded to whole tiles of 64 (`half` long in A)
//   kGatedWeight   rows of the output are gate's, then up's, `half` apart in A
enum Product { kForward, kInput, kWeight, kGatedForward, kGatedInput, kGatedWeight };
template <int P>
struct Is {
    static constexpr bool fwd = P == kForward || P == kGatedForward;
    static constexpr bool gated_fwd = P == kGatedForward, gated_dx = P == kGatedInput, gated_dw = P == kGatedWeight;
    static constexpr bool ak = P == kWeight || P == kGatedWeight, bk = !fwd;   // K-major operands
};

struct GemmArgs {
    const void *A, *B;
    int64_t lda, ldb, M, N, K;
    void* C;             // T, or f32
    int64_t ldc;
    int c_f32, accumulate;
    // the forward's epilogue
    int act;
    const float* bias;
    const void* R;
    int64_t ldr;
    void* Z;
    int64_t ldz;
    float* part;         // [splits][M][pitch] sums of the K splits, or null
    int64_t pitch;
    int splits, per;
    // gated: up's weight, bias, z and gradient (gate's are those above), and where it begins (see Product); `each`: columns of one
    const void* B2;
    const float* bias2;
    void *Z2, *C2;
    int64_t half, each;
};

// The activations on the hardware's exp2 and reciprocal. For gelu_tanh, (1 + tanh u) / 2 = 1 / (1 + e^-2u), which is 0 or 1 where
// a large z^3 overflows to an infinity. NaN and infinities go through the formulas as they stand.
//
// For gelu, (1 + erf(z / sqrt 2)) / 2, the part of a normal distribution below z. The part beyond |z| is e^(-z^2 / 2) Q, whose
// exponential is also the slope's, with Q = t (a0 + .. + a6 t^6), t = 1 / (1 + 0.375 |z| / sqrt 2): fitted here to
// e^(x^2) erfc(x) / 2 over x = |z| / sqrt 2 up to 9.6 for the least relative error (a linear program over 4000 points), 6.3e-7; with
// f32 arithmetic 1.2e-6. The exponential's argument adds 1.5 z^2 2^-24. So gelu of a negative z, down to 2^-126, is as
// exact as a positive one's (Abramowitz and Stegun's 7.1.26, bounded by 1.5e-7 of 1 instead, was off by 0.4% of y at z = -6 and
// 1% at -8: bf16 half steps). The library's erff made the pass over dY and z bound by its arithmetic.
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + ex2(-kLog2e * x)); }
// (1 + erf(z / sqrt 2)) / 2, and e^(-z^2 / 2)
__device__ __forceinline__ float normal_below(float z, float& bell) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.265165043f, fabsf(z), 1.f));
    float p = __builtin_fmaf(-0.0675529372f, t, 0.193985501f);
    p = __builtin_fmaf(p, t, -0.0648207571f);
    p = __builtin_fmaf(p, t, 0.141545937f);
    p = __builtin_fmaf(p, t, 0.0833266515f);
    p = __builtin_fmaf(p, t, 0.107845643f);
    p = __builtin_fmaf(p, t, 0.105669648f);
    bell = ex2(-0.5f * kLog2e * z * z);
    const float tail = p * t * bell;   // the part beyond |z|
    return z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float gelu(float z) {
    float bell;
    return z * normal_below(z, bell);
}
// (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) / 2
__device__ __forceinline__ float tanh_gate(float z) { return sigmoid(1.5957691216057308f * (z + 0.044715f * z * z * z)); }
__device__ __forceinline__ float gelu_tanh(float z) { return z * tanh_gate(z); }
// act of N values (one branch for all: their chains of dependent instructions run side by side)
template <int N>
__device__ __forceinline__ void act_values(float (&v)[N], int act) {
    if (act == SA3K_ACT_RELU) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = v[e] <= 0.f ? 0.f : v[e];
    } else if (act == SA3K_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = v[e] * sigmoid(v[e]);
    } else if (act == SA3K_ACT_GELU) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = gelu(v[e]);
    } else if (act == SA3K_ACT_GELU_TANH) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = gelu_tanh(v[e]);
    }
}
__device__ __forceinline__ float act_slope(float z, int act) {
    if (act == SA3K_ACT_RELU) return z <= 0.f ? 0.f : z > 0.f ? 1.f : z;   // (NaN stays NaN)
    if (act == SA3K_ACT_SILU) {
        const float g = sigmoid(z);
        return g * (1.f + z * (1.f - g));
    }
    if (act == SA3K_ACT_GELU) {
        float bell;
        const float below = normal_below(z, bell);
        return below + z * bell * 0.39894228040143268f;
    }
    if (act == SA3K_ACT_GELU_TANH) {
        // Past +-10 g (1 - g) is below 2^-125, and its factors need not grow on: z^2 of a finite z must not overflow. z times 0
        // leaves a NaN or an infinite z a NaN, as the formula does.
        const float g = tanh_gate(z), y = fminf(fmaxf(z, -10.f), 10.f);
        return __builtin_fmaf(y * g * (1.f - g) * 1.5957691216057308f, 1.f + 0.134145f * y * y, g) + 0.f * z;
    }
    return 1.f;
}

// act(z) and its slope, as act_values and act_slope give them, from one exponential
__device__ __forceinline__ float2 act_and_slope(float z, int act) {
    if (act == SA3K_ACT_SILU) {
        const float g = sigmoid(z);
        return make_float2(z * g, g * (1.f + z * (1.f - g)));
    }
    if (act == SA3K_ACT_GELU) {
        float bell;
        const float below = normal_below(z, bell);
        return make_float2(z * below, below + z * bell * 0.39894228040143268f);
    }
    if (act == SA3K_ACT_GELU_TANH) {
        const float g = tanh_gate(z), y = fminf(fmaxf(z, -10.f), 10.f);
        return make_float2(z * g, __builtin_fmaf(y * g * (1.f - g) * 1.5957691216057308f, 1.f + 0.134145f * y * y, g) + 0.f * z);
    }
    return make_float2(act == SA3K_ACT_RELU && z <= 0.f ? 0.f : z, act_slope(z, act));
}

// n .. n + 7 of a row of `cols` elements, zeros past its end
template <class S>
__device__ __forceinline__ void load8(const S* p, int64_t n, int64_t cols, float (&v)[8]) {
    if (n + 8 <= cols) {
        const Pack<S, 8> q = *reinterpret_cast<const Pack<S, 8>*>(p + n);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)q.v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = n + e < cols ? (float)p[n + e] : 0.f;
    }
}
template <class S>
__device__ __forceinline__ void store8(S* p, int64_t n, int64_t cols, const float (&v)[8]) {
    if (n + 8 <= cols) {
        Pack<S, 8> q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q.v[e] = (S)v[e];
        *reinterpret_cast<Pack<S, 8>*>(p + n) = q;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (n + e < cols) p[n + e] = (S)v[e];
    }
}

// What the forward's epilogue reads for columns n .. n + 7: of the bias, and of row m of the residual
__device__ __forceinline__ void bias8(const GemmArgs& a, const float* bias, int64_t n, float (&b)[8]) {
    if (bias) {
        load8(bias, n, a.N, b);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = 0.f;
    }
}
template <class T>
__device__ __forceinline__ void residual8(const GemmArgs& a, int64_t m, int64_t n, Pack<T, 8>& r) {
    const T* p = static_cast<const T*>(a.R) + m * a.ldr;
    if (n + 8 <= a.N) {
        r = *reinterpret_cast<const Pack<T, 8>*>(p + n);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.v[e] = n + e < a.N ? p[n + e] : (T)0.f;
    }
}
// Eight finished sums of row m, columns n .. n + 7. FWD: bias, activation, residual. in: they are in range; lanes whose are not
// work the activation out all the same (with few of a wave's lanes left the same instructions took up to three times as
// long: 712 x 64 x 264, whose last tile has 8 columns, gelu 15.2 us against 9.5).
template <class T, int P>
__device__ __forceinline__ void finish8(const GemmArgs& a, int64_t m, int64_t n, float (&v)[8], const float (&b)[8],
                                        const Pack<T, 8>& r, bool in) {
    if constexpr (Is<P>::fwd) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += b[e];
        if (a.Z && in) store8(static_cast<T*>(a.Z) + m * a.ldz, n, a.N, v);
        act_values(v, a.act);
        if (a.R) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += (float)r.v[e];
        }
        if (in) store8(static_cast<T*>(a.C) + m * a.ldc, n, a.N, v);
    } else if (in) {
        void* C = a.C;
        if constexpr (Is<P>::gated_dw) {   // rows of gate's, then, `half` on, of up's; none between and behind them
            if (m >= a.half) {
                m -= a.half;
                C = a.C2;
            }
            if (m >= a.each) return;
        }
        if (a.c_f32) {
            float* c = static_cast<float*>(C) + m * a.ldc;
            if (a.accumulate) {
                float o[8];
                load8(c, n, a.N, o);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += o[e];
            }
            store8(c, n, a.N, v);
        } else {
            store8(static_cast<T*>(C) + m * a.ldc, n, a.N, v);
        }
    }
}
// The same of a gated forward: gate's and up's finished sums
template <class T>
__device__ __forceinline__ void finish_gated8(const GemmArgs& a, int64_t m, int64_t n, float (&g)[8], float (&u)[8],
                                              const float (&bg)[8], const float (&bu)[8], bool in) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        g[e] += bg[e];
        u[e] += bu[e];
    }
    if (a.Z && in) store8(static_cast<T*>(a.Z) + m * a.ldz, n, a.N, g);
    if (a.Z2 && in) store8(static_cast<T*>(a.Z2) + m * a.ldz, n, a.N, u);
    act_values(g, a.act);
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] *= u[e];
    if (in) store8(static_cast<T*>(a.C) + m * a.ldc, n, a.N, g);
}

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

// One operand's tile: ROWS rows x 64 of K. KMAJOR: stored [K][rows], staged as sub-tiles of [64 k][64 rows]. PAIR: 0 one tensor;
// 1 two, whose rows take turns of NT / 8; 2 two, one after the other along K.
template <class T, int ROWS, int NT, bool KMAJOR, int PAIR = 0>
struct Operand {
    typedef typename Vec<T>::x8 x8;
    static constexpr int PER = ROWS * 8 / NT;   // loads a thread makes for a tile
    struct Desc {
        u32x4 r[PAIR == 1 ? 2 : 1];
    };
    const char *base, *base2;                   // of the tile's first row at K = 0
    int64_t step;                               // bytes from one tile of K to the next
    uint32_t row_bytes, off[PER];
    int rows, kc;                               // rows in range; this thread's chunk of K (K-contiguous)
    int64_t half, each;                         // PAIR 2: where the second begins along K, and how long each is

    __device__ __forceinline__ void init(const void* p, const void* p2, int64_t ld, int64_t row0, int64_t n, int64_t half_,
                                         int64_t each_, int tid) {
        static_assert(PAIR != 1 || !KMAJOR, "rows in turns lie K-contiguous");
        constexpr int RPR = NT / 8;             // rows a round of loads
        row_bytes = (uint32_t)(ld * 2);
        rows = (int)min((int64_t)(PAIR == 1 ? ROWS / 2 : ROWS), n - row0);
        base = static_cast<const char*>(p) + (KMAJOR ? row0 * 2 : row0 * ld * 2);
        if constexpr (PAIR > 0) base2 = static_cast<const char*>(p2) + (KMAJOR ? row0 * 2 : row0 * ld * 2);
        if constexpr (PAIR == 2) {
            half = half_;
            each = each_;
        }
        step = KMAJOR ? 64 * ld * 2 : 128;
        // slot s = q NT + tid of an LDS row of eight 16-byte chunks holds chunk (s % 8) ^ swz(row); NT / 8 is a multiple of 16,
        // so a thread's chunk is the same in every round
        kc = (tid & 7) ^ swz(tid >> 3);
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int s = q * NT + tid;
            if constexpr (KMAJOR)
                off[q] = (uint32_t)((s & 511) >> 3) * row_bytes + (uint32_t)((s >> 9) * 128 + kc * 16);
            else if constexpr (PAIR == 1)
                off[q] = (uint32_t)((q >> 1) * RPR + (tid >> 3)) * row_bytes + (uint32_t)(kc * 16);
            else
                off[q] = (uint32_t)(s >> 3) * row_bytes + (uint32_t)(kc * 16);
        }
    }
    // the descriptor of tile t of K, `left` of K in range from its start on (none: every load gives zeros)
    __device__ __forceinline__ Desc tile(int64_t t, int64_t left) const {
        const char* p = base;
        if constexpr (PAIR == 2) {
            const bool second = t * 64 >= half;
            const int64_t k0 = second ? half : 0;
            left = left <= 0 ? 0 : each - (t * 64 - k0);
            p = second ? base2 : base;
            t -= k0 >> 6;
        }
        const int k = (int)max((int64_t)0, min((int64_t)64, left));
        // The last row in range ends the descriptor: rows past it are zeros. Rows are whole chunks of 8 elements, or padded to
        // that with zeros (a descriptor that ended inside a chunk would drop the dword that crosses its end).
        const uint32_t bytes = k == 0 ? 0u
                               : KMAJOR ? (uint32_t)(k - 1) * row_bytes + (uint32_t)((rows + 7) & ~7) * 2
                                        : (uint32_t)(rows - 1) * row_bytes + (uint32_t)((k + 7) & ~7) * 2;
        Desc d;
        d.r[0] = buffer_rsrc(p + t * step, bytes);
        if constexpr (PAIR == 1) d.r[1] = buffer_rsrc(base2 + t * step, bytes);
        return d;
    }
    // load q of tile t into the LDS piece at lds_addr
    __device__ __forceinline__ void load(const Desc& d, int q, int64_t left, uint32_t lds_addr, int wave) const {
        const bool none = !KMAJOR && kc * 8 >= left;   // a chunk past K lies in the next row: kept out
        dma16(d.r[PAIR == 1 ? q & 1 : 0], none ? 0xFFFFFFF0u : off[q],
              __builtin_amdgcn_readfirstlane(lds_addr + (uint32_t)((q * NT + wave * 64) * 16)));
    }
    __device__ __forceinline__ void issue(int64_t t, int64_t left, uint32_t lds_addr, int wave) const {
        const Desc d = tile(t, left);
#pragma unroll
        for (int q = 0; q < PER; ++q) load(d, q, left, lds_addr, wave);
    }
    // the operand of K step ks (16 of K) for rows r0 .. r0 + 31 of the tile
    static __device__ __forceinline__ x8 frag(const char* t, int r0, int ks, int lane) {
        const int hl = lane >> 5;
        if constexpr (KMAJOR) {
            const char* sub = t + (r0 >> 6) * 8192;
            const int n = (r0 & 63) + 16 * ((lane >> 4) & 1), k = 16 * ks + 8 * hl;
            const typename Vec<T>::x4 a = wattn::ld_tr<T>(sub, k, n, lane), b = wattn::ld_tr<T>(sub, k + 4, n, lane);
            return x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        } else {
            return wattn::ld_row<T, ROWS>(t, r0 + (lane & 31), 2 * ks + hl);
        }
    }
};
template <class T, int P, int EDGE, int NT>
using OperandA = Operand<T, EDGE, NT, Is<P>::ak>;
template <class T, int P, int EDGE, int NT>
using OperandB = Operand<T, EDGE, NT, Is<P>::bk, Is<P>::gated_fwd ? 1 : Is<P>::gated_dx ? 2 : 0>;

// Which tile a workgroup takes, in tiles of EDGE: workgroups go out to the 8 XCDs in turn; XCD c takes the run
// [c n / 8, (c + 1) n / 8) of the items in (split, raster) order, in groups of eight rows of tiles, so that tiles that share
// operands run on one XCD and share its L2.
struct TilePlace {
    int z;
    int64_t m0, n0;
    bool none;
};
template <int EDGE, int COLS>   // COLS: of the output, of one of the weights where there are two
__device__ __forceinline__ TilePlace tile_place(const GemmArgs& a, int L) {   // L: the workgroup's number among this product's
    const int tiles_m = (int)((a.M + EDGE - 1) / EDGE), tiles_n = (int)((a.N + COLS - 1) / COLS);
    const int nwg = (tiles_m * tiles_n + 7) & ~7;   // a split's workgroups
    const int item = (L & 7) * ((nwg * a.splits) >> 3) + (L >> 3);
    TilePlace p;
    p.z = __builtin_amdgcn_readfirstlane(item / nwg);
    const int bid = __builtin_amdgcn_readfirstlane(item - p.z * nwg);
    p.none = bid >= tiles_m * tiles_n;
    const int group = bid / (8 * tiles_n), gsz = min(tiles_m - group * 8, 8), in_g = bid - group * 8 * tiles_n;
    p.m0 = p.none ? 0 : (int64_t)(group * 8 + in_g % gsz) * EDGE;
    p.n0 = p.none ? 0 : (int64_t)(in_g / gsz) * COLS;
    return p;
}

// The end of a tile: 64 rows of its sums at a time, staged in LDS as f32; a thread finishes 8 columns, the same in every
// round, of four of the rows. The bias is read once, a round's residual before its sums are staged, so that the rounds do
// not wait for memory one after the other (with both read in place and the activation branched on for each value, 8191 x 4096 x
// 8192 f16 gelu_tanh with z took 546 us against 513, 2176 x 1536 x 6144 gelu with z 62.5 against 56.2, in turn on one card).
template <class T, int P, int EDGE, int NT, int EROW>
struct Finish {
    static constexpr bool FWD = Is<P>::fwd;
    static constexpr int CPR = EDGE / 8, STEP = NT / CPR, ROUNDS = 64 / STEP;   // threads a row; rows a round
    int64_t m0, n;
    int r0, cq;
    float b[8];
    Pack<T, 8> res[ROUNDS];

    __device__ __forceinline__ void init(const GemmArgs& a, const TilePlace& tp, int tid, bool) {
        cq = (tid % CPR) * 8;
        r0 = tid / CPR;
        m0 = tp.m0;
        n = tp.n0 + cq;
        if (FWD && !a.part) bias8(a, a.bias, n, b);
    }
    __device__ __forceinline__ void fetch(const GemmArgs& a, int rb) {
        if (!FWD || a.part || !a.R) return;   // (uniform)
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
            const int64_t m = m0 + rb + r0 + i * STEP;
            if (m < a.M && n < a.N) residual8<T>(a, m, n, res[i]);
        }
    }
    __device__ __forceinline__ void rows(const GemmArgs& a, int z, const float* st, int rb) {
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
            const int r = r0 + i * STEP;
            const int64_t m = m0 + rb + r;
            const bool in = m < a.M && n < a.N;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 x = *reinterpret_cast<const float4*>(st + r * EROW + cq + e);
                v[e] = x.x;
                v[e + 1] = x.y;
                v[e + 2] = x.z;
                v[e + 3] = x.w;
            }
            if (!a.part) finish8<T, P>(a, m, n, v, b, res[i], in);
            else if (in) store8(a.part + ((int64_t)z * a.M + m) * a.pitch, n, a.pitch, v);
        }
    }
};

// The end of a gated forward's tile. A staged row holds, for each half of the waves, WC columns of gate and then the same of up; a thread
// finishes 8 of them.
template <class T, int EDGE, int NT, int EROW>
struct FinishGated {
    static constexpr int COLS = EDGE / 2, WC = COLS / 2, CPR = COLS / 8, STEP = NT / CPR, ROUNDS = 64 / STEP;
    int64_t m0, n;
    int r0, cq;
    float bg[8], bu[8];

    // added: the sums hold the biases
    __device__ __forceinline__ void init(const GemmArgs& a, const TilePlace& tp, int tid, bool added) {
        const int c = (tid % CPR) * 8;
        cq = (c / WC) * 2 * WC + c % WC;
        r0 = tid / CPR;
        m0 = tp.m0;
        n = tp.n0 + c;
        if (a.part) return;
        bias8(a, added ? nullptr : a.bias, n, bg);
        bias8(a, added ? nullptr : a.bias2, n, bu);
    }
    __device__ __forceinline__ void fetch(const GemmArgs&, int) {}
    __device__ __forceinline__ void rows(const GemmArgs& a, int z, const float* st, int rb) {
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
            const int r = r0 + i * STEP;
            const int64_t m = m0 + rb + r;
            const bool in = m < a.M && n < a.N;
            float g[8], u[8];
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 x = *reinterpret_cast<const float4*>(st + r * EROW + cq + e);
                const float4 y = *reinterpret_cast<const float4*>(st + r * EROW + cq + WC + e);
                g[e] = x.x; g[e + 1] = x.y; g[e + 2] = x.z; g[e + 3] = x.w;
                u[e] = y.x; u[e + 1] = y.y; u[e + 2] = y.z; u[e + 3] = y.w;
            }
            if (!a.part) {
                finish_gated8<T>(a, m, n, g, u, bg, bu, in);
            } else if (in) {   // a row of the splits' sums: gate's, then up's
                float* p = a.part + ((int64_t)z * a.M + m) * a.pitch;
                store8(p, n, a.pitch / 2, g);
                store8(p + a.pitch / 2, n, a.pitch / 2, u);
            }
        }
    }
};
// The end of a wave of a gated forward's 256 x 256 tile, 64 rows x 64 columns of both products, without LDS and without waiting for other
// waves: the products were made with the weights' fragments first, so a lane holds 16 sums of one row of a block of 32 x 32 (column
// 8 (v / 4) + 4 (lane / 32) + v % 4), gate's and up's of the same element. Lanes 32 apart swap their fours for eights (16 bits), lanes 16
// apart halves of their rows, so that a store takes 64 bytes of 16 rows. Measured on MI355X, us a call, in turn on one card (staged
// through LDS as the other products' / so): 2176 x 1536 -> 6144 bf16 106 / 96, with biases, g and u stored 112 / 106, 8192 x 1536 -> 6144 with
// them 340 / 320, 8191 x 4096 -> 8192 f16 1004 / 963. Rows that begin off 16 bytes stay staged: with g and u stored 1952 x 320 -> 2239 27 /
// 35, 2176 x 1536 -> 6145 115 / 132, 4096 x 2048 -> 4100 189 / 194 (of Y alone 21.3 / 19.4, 103 / 99 and 180 / 163: not told apart). The backward's products gained nothing (2176 x 1536 -> 6144 both 197).
template <int A, int B>
__device__ __forceinline__ void swap_lanes(uint32_t (&w)[16], int n, int by) {
#pragma unroll
    for (int e = 0; e < n; ++e) {
        const auto r = by == 32 ? __builtin_amdgcn_permlane32_swap(w[A + e], w[B + e], false, false)
                                : __builtin_amdgcn_permlane16_swap(w[A + e], w[B + e], false, false);
        w[A + e] = r[0];
        w[B + e] = r[1];
    }
}
// a block of 32 x 32 at (m, n) of C [rows][cols]: rounded to T
template <class T>
__device__ __forceinline__ void store_block(void* C, int64_t ld, int64_t m, int64_t n, int64_t rows, int64_t cols, int lane,
                                            const float (&v)[16]) {
    uint32_t w[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const Pack<T, 2> q{{(T)v[2 * e], (T)v[2 * e + 1]}};
        w[e] = __builtin_bit_cast(uint32_t, q);
    }
    swap_lanes<0, 2>(w, 2, 32);   // 0 .. 3: eight columns, the lower lanes' from 0 on, the upper's from 8 on
    swap_lanes<4, 6>(w, 2, 32);   // 4 .. 7: the same from 16 on
    swap_lanes<0, 4>(w, 4, 16);   // 0 .. 3: of rows 0 .. 15; 4 .. 7: of rows 16 .. 31
    n += 16 * ((lane >> 4) & 1) + 8 * (lane >> 5);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t row = m + 16 * h + (lane & 15);
        if (row >= rows) continue;
        const Pack<T, 8> q = __builtin_bit_cast(Pack<T, 8>, u32x4{w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]});
        T* c = static_cast<T*>(C) + row * ld;
        if (n + 8 <= cols) {
            *reinterpret_cast<Pack<T, 8>*>(c + n) = q;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < cols) c[n + e] = q.v[e];
        }
    }
}
// the same in f32, whole fours of columns
__device__ __forceinline__ void store_block_f32(float* C, int64_t ld, int64_t m, int64_t n, int64_t rows, int64_t cols, int lane,
                                                const float (&v)[16]) {
    uint32_t w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(v[e]);
    swap_lanes<0, 4>(w, 4, 16);    // 0 .. 3: sixteen columns of rows 0 .. 15; 4 .. 7: of rows 16 .. 31
    swap_lanes<8, 12>(w, 4, 16);   // 8 ..: the same from 16 on
    n += 8 * ((lane >> 4) & 1) + 4 * (lane >> 5);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int64_t row = m + 16 * (q & 1) + (lane & 15), at = n + 16 * (q >> 1);
        if (row < rows && at < cols)
            *reinterpret_cast<uint4*>(C + row * ld + at) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    }
}
__device__ __forceinline__ void block_of(const f32x16& acc, float (&v)[16]) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = acc[e];
}
// whether the outputs' rows begin on 16 bytes: those of others lie across lines, whose stores of 64 bytes are then two each
template <class T>
__device__ __forceinline__ bool rows_whole(const GemmArgs& a) {
    const uint64_t at = reinterpret_cast<uint64_t>(a.C) | reinterpret_cast<uint64_t>(a.Z) | reinterpret_cast<uint64_t>(a.Z2);
    return ((at | (uint64_t)(a.ldc * (int64_t)sizeof(T)) | (a.Z || a.Z2 ? (uint64_t)(a.ldz * (int64_t)sizeof(T)) : 0)) & 15) == 0;
}
// The sums begin with the biases, whose loads are then under way beside the first tile's (read at the end, 2176 x 1536 -> 6144 took
// 2 us more)
__device__ __forceinline__ void gated_biases(const GemmArgs& a, int64_t n0, int lane, f32x16 (&acc)[2][4]) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const float* bias = w ? a.bias2 : a.bias;
        if (!bias) continue;   // (uniform)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int64_t c = n0 + 32 * j + 8 * q + 4 * (lane >> 5);
                Pack<float, 4> b;
                if (c + 4 <= a.N) {
                    b = *reinterpret_cast<const Pack<float, 4>*>(bias + c);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) b.v[e] = c + e < a.N ? bias[c + e] : 0.f;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc[0][2 * w + j][4 * q + e] += b.v[e];
                    acc[1][2 * w + j][4 * q + e] += b.v[e];
                }
            }
    }
}
template <class T>
__device__ __forceinline__ void finish_gated_wave(const GemmArgs& a, int z, int64_t m0, int64_t n0, int lane, f32x16 (&acc)[2][4]) {
    float v[16];
    if (a.part) {   // (uniform) rows of the splits' sums: gate's, then up's, each of whole eights
        const int64_t up = a.pitch / 2;
        float* s = a.part + (int64_t)z * a.M * a.pitch;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                block_of(acc[i][j], v);
                store_block_f32(s + (j >> 1) * up, a.pitch, m0 + 32 * i, n0 + 32 * (j & 1), a.M, up, lane, v);
            }
        return;
    }
    // One output after the other: with the three in turn for every 16 columns, 8192 x 1536 -> 6144 with g and u took 428 us, not 301.
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int w = 0; w < 3; ++w) {
            void* C = w == 0 ? a.Z : w == 1 ? a.Z2 : a.C;
            if (!C) continue;   // (uniform)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                block_of(acc[i][w == 1 ? j + 2 : j], v);
                if (w == 2) {
                    act_values(v, a.act);
#pragma unroll
                    for (int e = 0; e < 16; ++e) v[e] *= acc[i][j + 2][e];
                }
                store_block<T>(C, w == 2 ? a.ldc : a.ldz, m0 + 32 * i, n0 + 32 * j, a.M, a.N, lane, v);
            }
        }
}

template <class T, int P, int EDGE, int NT, int EROW>
struct FinishOf {
    typedef Finish<T, P, EDGE, NT, EROW> type;
};
template <class T, int EDGE, int NT, int EROW>
struct FinishOf<T, kGatedForward, EDGE, NT, EROW> {
    typedef FinishGated<T, EDGE, NT, EROW> type;
};

// Tiles of 256 x 256: eight waves of 64 x 128, one workgroup a CU. Measured on MI355X: 8192^3 bf16 872 us (1260 TFLOP/s),
// 8191 x 4096 x 8192 bf16 460 us, f16 486 and with gelu_tanh and z stored 510 to 518 (in the first calls after a pause 575). Bound by
// the operand loads and LDS reads beside the MFMAs (busy for 58% of the time; without the loads 8192^3 took 800 us against 925, as they
// were then). Not kept (f16, each against the kernel of its
// time): four waves of 128 x 128, 579 us against 530 (its epilogue stalls the only wave of a SIMD); fragments read a step
// ahead, 519 against 512; steps of 32 of K, 527 against 512.
template <class T, int P>
__device__ __forceinline__ void big_body(const GemmArgs& a, int L, char* lds) {
    typedef typename Vec<T>::x8 x8;
    constexpr int EDGE = 256, NT = 512, FM = 2, FN = 4, OPB = EDGE * 128, STAGE = 2 * OPB, EROW = EDGE + 8;
    static_assert(64 * EROW * 4 <= 2 * STAGE, "staged rows fit the stages' memory");
    const TilePlace tp = tile_place<EDGE, Is<P>::gated_fwd ? EDGE / 2 : EDGE>(a, L);
    if (tp.none) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm0 = (wave & 3) * 64, wn0 = (wave >> 2) * 128;
    typedef OperandA<T, P, EDGE, NT> OpA;
    typedef OperandB<T, P, EDGE, NT> OpB;
    OpA A;
    OpB B;
    A.init(a.A, nullptr, a.lda, tp.m0, a.M, 0, 0, tid);
    B.init(a.B, a.B2, a.ldb, tp.n0, a.N, a.half, a.each, tid);
    const int64_t KT = (a.K + 63) / 64, t0 = (int64_t)tp.z * a.per, t1 = min(KT, t0 + a.per);
    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
    auto issue = [&](int st, int64_t t) {
        A.issue(t, a.K - t * 64, lds0 + st * STAGE, wave);
        B.issue(t, a.K - t * 64, lds0 + st * STAGE + OPB, wave);
    };
    // Two groups of four waves, one of each on a SIMD, half a step apart: while one multiplies, the other reads its
    // fragments. A step is 16 of K: fragments | barrier | eight products | barrier; the second group is one barrier late. The
    // loads of tile t + 1 go out during the first steps of t, when both groups have read the last of t - 1, and have landed before
    // the last step's first barrier, which comes before either group's first read of t + 1.
    const bool late = wave >= 4;
    if (t0 < t1) issue(0, t0);
    if constexpr (Is<P>::gated_fwd) {
        if (!a.part) gated_biases(a, tp.n0 + wn0 / 2, lane, acc);
    }
    wait_vmcnt<0>();
    asm volatile("s_barrier" ::: "memory");
    if (late) asm volatile("s_barrier" ::: "memory");
    for (int64_t t = t0; t < t1; ++t) {
        const int stage = (int)(t - t0) & 1;
        const char* As = lds + stage * STAGE;
        const char* Bs = As + OPB;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            x8 af[FM], bf[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) bf[j] = OpB::frag(Bs, wn0 + 32 * j, ks, lane);
#pragma unroll
            for (int i = 0; i < FM; ++i) af[i] = OpA::frag(As, wm0 + 32 * i, ks, lane);
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < t1) {
                if (ks == 0) A.issue(t + 1, a.K - (t + 1) * 64, lds0 + (stage ^ 1) * STAGE, wave);
                if (ks == 1) B.issue(t + 1, a.K - (t + 1) * 64, lds0 + (stage ^ 1) * STAGE + OPB, wave);
            }
            if (ks == 3) wait_vmcnt<0>();
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = Is<P>::gated_fwd ? Vec<T>::mfma(bf[j], af[i], acc[i][j]) : Vec<T>::mfma(af[i], bf[j], acc[i][j]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_barrier" ::: "memory");
        }
    }
    if (!late) asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < FM; ++i) wattn::settle(acc[i]);
    if constexpr (Is<P>::gated_fwd) {
        if (a.part || rows_whole<T>(a)) {   // (uniform)
            finish_gated_wave<T>(a, tp.z, tp.m0 + wm0, tp.n0 + wn0 / 2, lane, acc);
            return;
        }
    }
    float* st = reinterpret_cast<float*>(lds);
    typename FinishOf<T, P, EDGE, NT, EROW>::type fin;
    fin.init(a, tp, tid, true);
    __syncthreads();
#pragma unroll 1
    for (int rb = 0; rb < EDGE; rb += 64) {
        fin.fetch(a, rb);
        if (wm0 == rb) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        const int b = 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3), c = lane & 31;   // of A's block and of B's
                        st[(32 * i + (Is<P>::gated_fwd ? c : b)) * EROW + wn0 + 32 * j + (Is<P>::gated_fwd ? b : c)] = acc[i][j][v];
                    }
        }
        __syncthreads();
        fin.rows(a, tp.z, st, rb);
        __syncthreads();
    }
}

constexpr int kBigLds = 2 * 2 * 256 * 128;   // two stages of both operands
template <class T, int P>
__global__ __launch_bounds__(512, 2) void prod_big_kernel(GemmArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[kBigLds];
    big_body<T, P>(a, blockIdx.x, lds);
}
// dX and dW in one launch of these tiles: the CUs that dX's last round leaves take dW's (gated_pair has the sizes and figures)
template <class T, int PX, int PW>
__global__ __launch_bounds__(512, 2) void prod_pair_big_kernel(GemmArgs x, GemmArgs w, int x_wgs) {
    __shared__ __attribute__((aligned(1024))) char lds[kBigLds];
    if ((int)blockIdx.x < x_wgs) big_body<T, PX>(x, blockIdx.x, lds);
    else big_body<T, PW>(w, (int)blockIdx.x - x_wgs, lds);
}

// Tiles of 128 x 128: four waves of 64 x 64. STAGES 2: 64 KB of LDS, two workgroups a CU; STAGES 4: one. A wave keeps its MFMAs
// fed by itself: the fragments of K step ks + 1 are read between the products of ks. Before the last step's products every wave
// has read the last of tile t and tile t + 1 has landed; the one barrier a tile is there, and behind it the first fragments of
// t + 1 are read and the loads of tile t + STAGES begin to go out into t's piece, a quarter of them a K step. (Loads of tiles past
// the end give zeros and touch no memory, so that every round has the same number under way.) Measured on MI355X: 2176 x 6144
// x 1536 with bias and residual 54.1 us (759 TFLOP/s). A CU takes 0.55 us a tile and 64 of K, 0.42 with the loads left out; MFMA
// busy for 40% of the time.
template <class T, int STAGES, int P>
__device__ __forceinline__ void tile_body(const GemmArgs& a, int L, char* lds) {
    typedef typename Vec<T>::x8 x8;
    constexpr int EDGE = 128, NT = 256, F = 2, OPB = EDGE * 128, STAGE = 2 * OPB, EROW = EDGE + 8;
    typedef OperandA<T, P, EDGE, NT> OpA;
    typedef OperandB<T, P, EDGE, NT> OpB;
    constexpr int LOADS = OpA::PER + OpB::PER;
    static_assert(64 * EROW * 4 <= STAGES * STAGE, "staged rows fit the stages' memory");
    const TilePlace tp = tile_place<EDGE, Is<P>::gated_fwd ? EDGE / 2 : EDGE>(a, L);
    if (tp.none) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm0 = (wave & 1) * 64, wn0 = (wave >> 1) * 64;
    OpA A;
    OpB B;
    A.init(a.A, nullptr, a.lda, tp.m0, a.M, 0, 0, tid);
    B.init(a.B, a.B2, a.ldb, tp.n0, a.N, a.half, a.each, tid);
    const int64_t KT = (a.K + 63) / 64, t0 = (int64_t)tp.z * a.per, t1 = min(KT, t0 + a.per);
    f32x16 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
    // K left at tile t: none past this split's end
    auto left = [&](int64_t t) { return t < t1 ? a.K - t * 64 : (int64_t)0; };
    x8 f[2][2 * F];   // two sets of fragments: A's, then B's
    auto read = [&](const char* s, int ks, int n, x8& to) {
        if (n < F) to = OpA::frag(s, wm0 + 32 * n, ks, lane);
        else to = OpB::frag(s + OPB, wn0 + 32 * (n - F), ks, lane);
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        A.issue(t0 + s, left(t0 + s), lds0 + s * STAGE, wave);
        B.issue(t0 + s, left(t0 + s), lds0 + s * STAGE + OPB, wave);
    }
    // the tile whose loads are going out: its descriptors, its K, its place
    int64_t lp = left(t0 + STAGES - 1);
    auto ra = A.tile(t0 + STAGES - 1, lp);
    auto rb = B.tile(t0 + STAGES - 1, lp);
    uint32_t dst = lds0 + (STAGES - 1) * STAGE;
    auto load = [&](int q) {
        A.load(ra, q, lp, dst, wave);
        B.load(rb, q, lp, dst + OPB, wave);
    };
    static_assert(OpA::PER == 4 && OpB::PER == 4, "a load of each operand a K step");
    load(0);
    wait_vmcnt<(STAGES - 2) * LOADS + 2>();   // tile t0
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int n = 0; n < 2 * F; ++n) read(lds, 0, n, f[0][n]);
    int stage = 0;
    for (int64_t t = t0; t < t1; ++t) {
        const int after = stage + 1 < STAGES ? stage + 1 : 0;
        const char* now = lds + stage * STAGE;
        const char* next = lds + after * STAGE;
#pragma unroll
        for (int ks = 0; ks < 3; ++ks)
#pragma unroll
            for (int n = 0; n < F * F; ++n) {
                acc[n / F][n % F] = Vec<T>::mfma(f[ks & 1][n / F], f[ks & 1][F + n % F], acc[n / F][n % F]);
                read(now, ks + 1, n, f[(ks & 1) ^ 1][n]);
                if (n == F) load(ks + 1);
                __builtin_amdgcn_sched_barrier(0);
            }
        lp = left(t + STAGES);
        ra = A.tile(t + STAGES, lp);
        rb = B.tile(t + STAGES, lp);
        dst = lds0 + stage * STAGE;
        wait_vmcnt<(STAGES - 2) * LOADS>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int n = 0; n < F * F; ++n) {
            acc[n / F][n % F] = Vec<T>::mfma(f[1][n / F], f[1][F + n % F], acc[n / F][n % F]);
            read(next, 0, n, f[0][n]);
            if (n == F) load(0);
            __builtin_amdgcn_sched_barrier(0);
        }
        stage = after;
    }
#pragma unroll
    for (int i = 0; i < F; ++i) wattn::settle(acc[i]);
    wait_vmcnt<0>();   // (loads past the end: zeros, but into this memory)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    float* st = reinterpret_cast<float*>(lds);
    typename FinishOf<T, P, EDGE, NT, EROW>::type fin;
    fin.init(a, tp, tid, false);
    __syncthreads();
#pragma unroll 1
    for (int rb = 0; rb < EDGE; rb += 64) {
        fin.fetch(a, rb);
        if (wm0 == rb) {
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        st[(32 * i + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3)) * EROW + wn0 + 32 * j + (lane & 31)] =
                            acc[i][j][v];
        }
        __syncthreads();
        fin.rows(a, tp.z, st, rb);
        __syncthreads();
    }
}

template <class T, int STAGES, int P>
__global__ __launch_bounds__(256, STAGES == 2 ? 2 : 1) void prod_tile_kernel(GemmArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[STAGES * 2 * 128 * 128];
    tile_body<T, STAGES, P>(a, blockIdx.x, lds);
}

// dX (x_wgs workgroups, a multiple of 8) and dW in one launch: each alone leaves CUs empty in its last turn. Measured on MI355X:
// 2176 x 1536 -> 6144 bf16 103 us (797 TFLOP/s) against 113 one after the other; prod_pair has more shapes. Large ones run on the 256 x
// 256 tiles' two launches (4096 x 4096 -> 4096 236 us, 1163 TFLOP/s).
template <class T, int PX, int PW>
__global__ __launch_bounds__(256, 2) void prod_pair_kernel(GemmArgs x, GemmArgs w, int x_wgs) {
    __shared__ __attribute__((aligned(1024))) char lds[2 * 2 * 128 * 128];
    if ((int)blockIdx.x < x_wgs) tile_body<T, 2, PX>(x, blockIdx.x, lds);
    else tile_body<T, 2, PW>(w, (int)blockIdx.x - x_wgs, lds);
}

// the K splits' sums in their order, then the epilogue
template <class T, int P>
__device__ __forceinline__ void sum_body(const GemmArgs& a, int64_t block) {
    const int64_t chunks = a.pitch / 8, i = block * 256 + threadIdx.x, m = i / chunks, n = (i - m * chunks) * 8;
    if (m >= a.M) return;
    float v[8], b[8];
    Pack<T, 8> r;
    if constexpr (Is<P>::fwd) {
        bias8(a, a.bias, n, b);
        if (a.R) residual8<T>(a, m, n, r);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    const float* p = a.part + m * a.pitch + n;
    for (int z = 0; z < a.splits; ++z, p += a.M * a.pitch)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const float4 x = *reinterpret_cast<const float4*>(p + e);
            v[e] += x.x;
            v[e + 1] += x.y;
            v[e + 2] += x.z;
            v[e + 3] += x.w;
        }
    finish8<T, P>(a, m, n, v, b, r, true);
}
template <class T, int P>
__global__ __launch_bounds__(256) void prod_sum_kernel(GemmArgs a) {
    sum_body<T, P>(a, blockIdx.x);
}
template <class T>
__global__ __launch_bounds__(256) void gated_sum_kernel(GemmArgs a) {
    const int64_t up = a.pitch / 2, chunks = up / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / chunks, n = (i - m * chunks) * 8;
    if (m >= a.M) return;
    float v[2][8], bg[8], bu[8];
    bias8(a, a.bias, n, bg);
    bias8(a, a.bias2, n, bu);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[0][e] = v[1][e] = 0.f;
    const float* p = a.part + m * a.pitch + n;
    for (int z = 0; z < a.splits; ++z, p += a.M * a.pitch)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 x = *reinterpret_cast<const float4*>(p + w * up + e);
                v[w][e] += x.x;
                v[w][e + 1] += x.y;
                v[w][e + 2] += x.z;
                v[w][e + 3] += x.w;
            }
    finish_gated8<T>(a, m, n, v[0], v[1], bg, bu, true);
}

// rows [rows][cols] into rows of cols rounded up to a multiple of 8, zeros behind them; up to three operands in one launch (each may
// have no rows)
struct PadArgs {
    const void* src[3];
    int64_t ld[3], rows[3], cols;
    void* dst[3];
};
inline int64_t pad_chunks(const PadArgs& a) { return (a.rows[0] + a.rows[1] + a.rows[2]) * ((a.cols + 7) / 8); }
template <class T>
__device__ __forceinline__ void pad_body(const PadArgs& a, int64_t block, int64_t blocks) {
    const int64_t chunks = (a.cols + 7) / 8, n0 = a.rows[0] * chunks, n1 = n0 + a.rows[1] * chunks, n = n1 + a.rows[2] * chunks;
    for (int64_t i = block * 256 + threadIdx.x; i < n; i += blocks * 256) {
        const int w = i >= n1 ? 2 : i >= n0 ? 1 : 0;
        const int64_t j = i - (w == 2 ? n1 : w == 1 ? n0 : 0), r = j / chunks, c = (j - r * chunks) * 8;
        const void* src = w == 2 ? a.src[2] : w == 1 ? a.src[1] : a.src[0];
        void* dst = w == 2 ? a.dst[2] : w == 1 ? a.dst[1] : a.dst[0];
        float v[8];
        load8(static_cast<const T*>(src) + r * (w == 2 ? a.ld[2] : w == 1 ? a.ld[1] : a.ld[0]), c, a.cols, v);
        store8(static_cast<T*>(dst) + r * chunks * 8, c, chunks * 8, v);
    }
}
template <class T>
__global__ __launch_bounds__(256) void prod_pad_kernel(PadArgs a) {
    pad_body<T>(a, blockIdx.x, gridDim.x);
}

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// whether the tile kernel's 16-byte loads can take rows of `cols` elements
bool loads16(const void* p, int64_t ld, int64_t cols) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && cols % 8 == 0;
}

// The context's scratch, cut into pieces: first their sizes are added up, then the one allocation is handed out.
struct Scratch {
    size_t need = 0;
    size_t take(size_t bytes) {
        const size_t at = need;
        need += up256(bytes);
        return at;
    }
};

inline int64_t pad_blocks(const PadArgs& a) { return std::min<int64_t>(ceil_div(pad_chunks(a), 256), 65536); }
template <class T>
void pad(sa3k_ctx* ctx, const PadArgs& a, const char* name) {
    if (pad_chunks(a) == 0) return;
    KernelScope ks(ctx, name);
    launch_k(ctx, false, prod_pad_kernel<T>, dim3((unsigned)pad_blocks(a)), dim3(256), 0, a);
    SA3K_LAUNCHED();
}

// bytes of the splits' sums of M rows, `pitch` apart
size_t split_bytes(const ProdPlan& p, int64_t M, int64_t pitch) {
    return p.splits > 1 ? (size_t)p.splits * (size_t)M * (size_t)pitch * sizeof(float) : 0;
}

// the plan's numbers into the arguments; the workgroups of the launch
template <int P>
int64_t plan_into(GemmArgs& a, const ProdPlan& p, float* part) {
    constexpr int W = Is<P>::gated_fwd ? 2 : 1;   // weights whose columns a tile holds
    a.splits = p.splits;
    a.per = p.per;
    a.part = p.splits > 1 ? part : nullptr;
    a.pitch = W * up8(a.N);
    return ceil_div(ceil_div(a.M, p.edge) * ceil_div(a.N, p.edge / W), 8) * 8 * p.splits;
}
template <class T, int P>
void sum_splits(sa3k_ctx* ctx, const GemmArgs& a, const char* name) {
    if (a.splits == 1) return;
    KernelScope ks(ctx, name);
    if constexpr (Is<P>::gated_fwd)
        launch_k(ctx, true, gated_sum_kernel<T>, dim3((unsigned)ceil_div(a.M * (a.pitch / 16), 256)), dim3(256), 0, a);
    else launch_k(ctx, true, prod_sum_kernel<T, P>, dim3((unsigned)ceil_div(a.M * (a.pitch / 8), 256)), dim3(256), 0, a);
    SA3K_LAUNCHED();
}
// the products alone, splits not added up
template <class T, int P>
void tile_launch(sa3k_ctx* ctx, GemmArgs& a, const ProdPlan& p, float* part, const char* name) {
    const int64_t wgs = plan_into<P>(a, p, part);
    const dim3 grid((unsigned)wgs);
    KernelScope ks(ctx, name, (Is<P>::gated_fwd ? 4.0 : 2.0) * (double)a.M * (double)a.N * (double)a.K);
    if (p.edge == 256) launch_k(ctx, a.splits == 1, prod_big_kernel<T, P>, grid, dim3(512), 0, a);
    else if (wgs <= 256)   // one workgroup a CU at the most: deeper stages
        launch_k(ctx, a.splits == 1, prod_tile_kernel<T, 4, P>, grid, dim3(256), 0, a);
    else launch_k(ctx, a.splits == 1, prod_tile_kernel<T, 2, P>, grid, dim3(256), 0, a);
    SA3K_LAUNCHED();
}
template <class T, int P>
void tile_run(sa3k_ctx* ctx, GemmArgs& a, const ProdPlan& p, float* part, const char* name, const char* sum_name) {
    tile_launch<T, P>(ctx, a, p, part, name);
    sum_splits<T, P>(ctx, a, sum_name);
}

}  // namespace
