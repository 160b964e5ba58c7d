// Products with bias, activation and residual in the epilogue, and their backward:
//   z = X W^T + b, Y = act(z) + R;   dz = dY act'(z), dX = dz W, dW = dz^T X, db = sum over rows dz
//
// One tile kernel does the three products C[m][n] = sum_k A(m, k) B(n, k), on v_mfma_f32_32x32x16 with f32 sums. An operand
// lies K-contiguous ([rows][K]: X, W and dz of dX) or K-major ([K][rows]: W of dX, both of dW); a K-major tile is staged as
// it lies, as sub-tiles of [64 k][64 rows], and read transposed (ds_read_b64_tr_b16), so no operand is ever transposed
// in memory. Tiles of 64 along K go straight into LDS (buffer_load ... lds) through a descriptor that ends where the
// operand does: rows and K past the end are zeros. Two stages; the loads of tile t + 1 run while t is computed.
//
// These loads take 16 bytes: operands whose rows are not 16-byte aligned, or not a multiple of 8 long, are copied once into
// padded rows first (a copy of M K + N K elements against M N K multiply-adds).
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
__device__ __forceinline__ void bias8(const GemmArgs& a, int64_t n, float (&b)[8]) {
    if (a.bias) {
        load8(a.bias, n, a.N, b);
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
template <class T, bool FWD>
__device__ __forceinline__ void finish8(const GemmArgs& a, int64_t m, int64_t n, float (&v)[8], const float (&b)[8],
                                        const Pack<T, 8>& r, bool in) {
    if constexpr (FWD) {
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
        if (a.c_f32) {
            float* c = static_cast<float*>(a.C) + m * a.ldc;
            if (a.accumulate) {
                float o[8];
                load8(c, n, a.N, o);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += o[e];
            }
            store8(c, n, a.N, v);
        } else {
            store8(static_cast<T*>(a.C) + m * a.ldc, n, a.N, v);
        }
    }
}

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

// One operand's tile: ROWS rows x 64 of K. KMAJOR: stored [K][rows], staged as sub-tiles of [64 k][64 rows].
template <class T, int ROWS, int NT, bool KMAJOR>
struct Operand {
    typedef typename Vec<T>::x8 x8;
    static constexpr int PER = ROWS * 8 / NT;   // loads a thread makes for a tile
    const char* base;                           // of the tile's first row at K = 0
    int64_t step;                               // bytes from one tile of K to the next
    uint32_t row_bytes, off[PER];
    int rows, kc;                               // rows in range; this thread's chunk of K (K-contiguous)

    __device__ __forceinline__ void init(const void* p, int64_t ld, int64_t row0, int64_t n, int tid) {
        row_bytes = (uint32_t)(ld * 2);
        rows = (int)min((int64_t)ROWS, n - row0);
        base = static_cast<const char*>(p) + (KMAJOR ? row0 * 2 : row0 * ld * 2);
        step = KMAJOR ? 64 * ld * 2 : 128;
        // slot s = q NT + tid of an LDS row of eight 16-byte chunks holds chunk (s % 8) ^ swz(row); NT / 8 is a multiple of 16,
        // so a thread's chunk is the same in every round
        kc = (tid & 7) ^ swz(tid >> 3);
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int s = q * NT + tid;
            if constexpr (KMAJOR)
                off[q] = (uint32_t)((s & 511) >> 3) * row_bytes + (uint32_t)((s >> 9) * 128 + kc * 16);
            else
                off[q] = (uint32_t)(s >> 3) * row_bytes + (uint32_t)(kc * 16);
        }
    }
    // the descriptor of tile t of K, `left` of K in range from its start on (none: every load gives zeros)
    __device__ __forceinline__ u32x4 tile(int64_t t, int64_t left) const {
        const int k = (int)max((int64_t)0, min((int64_t)64, left));
        // The last row in range ends the descriptor: rows past it are zeros. Rows are whole chunks of 8 elements, or padded to
        // that with zeros (a descriptor that ended inside a chunk would drop the dword that crosses its end).
        const uint32_t bytes = k == 0 ? 0u
                               : KMAJOR ? (uint32_t)(k - 1) * row_bytes + (uint32_t)((rows + 7) & ~7) * 2
                                        : (uint32_t)(rows - 1) * row_bytes + (uint32_t)((k + 7) & ~7) * 2;
        return buffer_rsrc(base + t * step, bytes);
    }
    // load q of tile t into the LDS piece at lds_addr
    __device__ __forceinline__ void load(const u32x4& rs, int q, int64_t left, uint32_t lds_addr, int wave) const {
        const bool none = !KMAJOR && kc * 8 >= left;   // a chunk past K lies in the next row: kept out
        dma16(rs, none ? 0xFFFFFFF0u : off[q], __builtin_amdgcn_readfirstlane(lds_addr + (uint32_t)((q * NT + wave * 64) * 16)));
    }
    __device__ __forceinline__ void issue(int64_t t, int64_t left, uint32_t lds_addr, int wave) const {
        const u32x4 rs = tile(t, left);
#pragma unroll
        for (int q = 0; q < PER; ++q) load(rs, q, left, lds_addr, wave);
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

// Which tile a workgroup takes, in tiles of EDGE: workgroups go out to the 8 XCDs in turn; XCD c takes the run
// [c n / 8, (c + 1) n / 8) of the items in (split, raster) order, in groups of eight rows of tiles, so that tiles that share
// operands run on one XCD and share its L2.
struct TilePlace {
    int z;
    int64_t m0, n0;
    bool none;
};
template <int EDGE>
__device__ __forceinline__ TilePlace tile_place(const GemmArgs& a, int L) {   // L: the workgroup's number among this product's
    const int tiles_m = (int)((a.M + EDGE - 1) / EDGE), tiles_n = (int)((a.N + EDGE - 1) / EDGE);
    const int nwg = (tiles_m * tiles_n + 7) & ~7;   // a split's workgroups
    const int item = (L & 7) * ((nwg * a.splits) >> 3) + (L >> 3);
    TilePlace p;
    p.z = __builtin_amdgcn_readfirstlane(item / nwg);
    const int bid = __builtin_amdgcn_readfirstlane(item - p.z * nwg);
    p.none = bid >= tiles_m * tiles_n;
    const int group = bid / (8 * tiles_n), gsz = min(tiles_m - group * 8, 8), in_g = bid - group * 8 * tiles_n;
    p.m0 = p.none ? 0 : (int64_t)(group * 8 + in_g % gsz) * EDGE;
    p.n0 = p.none ? 0 : (int64_t)(in_g / gsz) * EDGE;
    return p;
}

// The end of a tile: 64 rows of its sums at a time, staged in LDS as f32; a thread finishes 8 columns, the same in every
// round, of four of the rows. The bias is read once, a round's residual before its sums are staged, so that the rounds do
// not wait for memory one after the other (with both read in place and the activation branched on for each value, 8191 x 4096 x
// 8192 f16 gelu_tanh with z took 546 us against 513, 2176 x 1536 x 6144 gelu with z 62.5 against 56.2, in turn on one card).
template <class T, bool FWD, int EDGE, int NT, int EROW>
struct Finish {
    static constexpr int CPR = EDGE / 8, STEP = NT / CPR, ROUNDS = 64 / STEP;   // threads a row; rows a round
    int64_t m0, n;
    int r0, cq;
    float b[8];
    Pack<T, 8> res[ROUNDS];

    __device__ __forceinline__ void init(const GemmArgs& a, const TilePlace& tp, int tid) {
        cq = (tid % CPR) * 8;
        r0 = tid / CPR;
        m0 = tp.m0;
        n = tp.n0 + cq;
        if (FWD && !a.part) bias8(a, n, b);
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
            if (!a.part) finish8<T, FWD>(a, m, n, v, b, res[i], in);
            else if (in) store8(a.part + ((int64_t)z * a.M + m) * a.pitch, n, a.pitch, v);
        }
    }
};

// Tiles of 256 x 256: eight waves of 64 x 128, one workgroup a CU. Measured on MI355X: 8192^3 bf16 872 us (1260 TFLOP/s),
// 8191 x 4096 x 8192 bf16 460 us, f16 486 and with gelu_tanh and z stored 510 to 518 (in the first calls after a pause 575). Bound by
// the operand loads and LDS reads beside the MFMAs (busy for 58% of the time; without the loads 8192^3 took 800 us against 925, as they
// were then). Not kept (f16, each against the kernel of its
// time): four waves of 128 x 128, 579 us against 530 (its epilogue stalls the only wave of a SIMD); fragments read a step
// ahead, 519 against 512; steps of 32 of K, 527 against 512.
template <class T, bool AK, bool BK, bool FWD>
__global__ __launch_bounds__(512, 2) void prod_big_kernel(GemmArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int EDGE = 256, NT = 512, FM = 2, FN = 4, OPB = EDGE * 128, STAGE = 2 * OPB, EROW = EDGE + 8;
    static_assert(64 * EROW * 4 <= 2 * STAGE, "staged rows fit the stages' memory");
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
    const TilePlace tp = tile_place<EDGE>(a, blockIdx.x);
    if (tp.none) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm0 = (wave & 3) * 64, wn0 = (wave >> 2) * 128;
    Operand<T, EDGE, NT, AK> A;
    Operand<T, EDGE, NT, BK> B;
    A.init(a.A, a.lda, tp.m0, a.M, tid);
    B.init(a.B, a.ldb, tp.n0, a.N, tid);
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
            for (int j = 0; j < FN; ++j) bf[j] = Operand<T, EDGE, NT, BK>::frag(Bs, wn0 + 32 * j, ks, lane);
#pragma unroll
            for (int i = 0; i < FM; ++i) af[i] = Operand<T, EDGE, NT, AK>::frag(As, wm0 + 32 * i, ks, lane);
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
                for (int j = 0; j < FN; ++j) acc[i][j] = Vec<T>::mfma(af[i], bf[j], acc[i][j]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_barrier" ::: "memory");
        }
    }
    if (!late) asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < FM; ++i) wattn::settle(acc[i]);
    float* st = reinterpret_cast<float*>(lds);
    Finish<T, FWD, EDGE, NT, EROW> fin;
    fin.init(a, tp, tid);
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
                    for (int v = 0; v < 16; ++v)
                        st[(32 * i + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3)) * EROW + wn0 + 32 * j + (lane & 31)] =
                            acc[i][j][v];
        }
        __syncthreads();
        fin.rows(a, tp.z, st, rb);
        __syncthreads();
    }
}

// Tiles of 128 x 128: four waves of 64 x 64. STAGES 2: 64 KB of LDS, two workgroups a CU; STAGES 4: one. A wave keeps its MFMAs
// fed by itself: the fragments of K step ks + 1 are read between the products of ks. Before the last step's products every wave
// has read the last of tile t and tile t + 1 has landed; the one barrier a tile is there, and behind it the first fragments of
// t + 1 are read and the loads of tile t + STAGES begin to go out into t's piece, a quarter of them a K step. (Loads of tiles past
// the end give zeros and touch no memory, so that every round has the same number under way.) Measured on MI355X: 2176 x 6144
// x 1536 with bias and residual 54.1 us (759 TFLOP/s). A CU takes 0.55 us a tile and 64 of K, 0.42 with the loads left out; MFMA
// busy for 40% of the time.
template <class T, int STAGES, bool AK, bool BK, bool FWD>
__device__ __forceinline__ void tile_body(const GemmArgs& a, int L, char* lds) {
    typedef typename Vec<T>::x8 x8;
    constexpr int EDGE = 128, NT = 256, F = 2, OPB = EDGE * 128, STAGE = 2 * OPB, EROW = EDGE + 8;
    typedef Operand<T, EDGE, NT, AK> OpA;
    typedef Operand<T, EDGE, NT, BK> OpB;
    constexpr int LOADS = OpA::PER + OpB::PER;
    static_assert(64 * EROW * 4 <= STAGES * STAGE, "staged rows fit the stages' memory");
    const TilePlace tp = tile_place<EDGE>(a, L);
    if (tp.none) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm0 = (wave & 1) * 64, wn0 = (wave >> 1) * 64;
    OpA A;
    OpB B;
    A.init(a.A, a.lda, tp.m0, a.M, tid);
    B.init(a.B, a.ldb, tp.n0, a.N, tid);
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
    u32x4 ra = A.tile(t0 + STAGES - 1, lp), rb = B.tile(t0 + STAGES - 1, lp);
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
    Finish<T, FWD, EDGE, NT, EROW> fin;
    fin.init(a, tp, tid);
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

template <class T, int STAGES, bool AK, bool BK, bool FWD>
__global__ __launch_bounds__(256, STAGES == 2 ? 2 : 1) void prod_tile_kernel(GemmArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[STAGES * 2 * 128 * 128];
    tile_body<T, STAGES, AK, BK, FWD>(a, blockIdx.x, lds);
}

// dX (x_wgs workgroups, a multiple of 8) and dW in one launch: each alone leaves CUs empty in its last turn. Measured on MI355X:
// 2176 x 1536 -> 6144 bf16 103 us (797 TFLOP/s) against 113 one after the other; prod_pair has more shapes. Large ones run on the 256 x
// 256 tiles' two launches (4096 x 4096 -> 4096 236 us, 1163 TFLOP/s).
template <class T>
__global__ __launch_bounds__(256, 2) void prod_pair_kernel(GemmArgs x, GemmArgs w, int x_wgs) {
    __shared__ __attribute__((aligned(1024))) char lds[2 * 2 * 128 * 128];
    if ((int)blockIdx.x < x_wgs) tile_body<T, 2, false, true, false>(x, blockIdx.x, lds);
    else tile_body<T, 2, true, true, false>(w, (int)blockIdx.x - x_wgs, lds);
}

// the K splits' sums in their order, then the epilogue
template <class T, bool FWD>
__global__ __launch_bounds__(256) void prod_sum_kernel(GemmArgs a) {
    const int64_t chunks = a.pitch / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / chunks, n = (i - m * chunks) * 8;
    if (m >= a.M) return;
    float v[8], b[8];
    Pack<T, 8> r;
    if constexpr (FWD) {
        bias8(a, n, b);
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
    finish8<T, FWD>(a, m, n, v, b, r, true);
}

// Few rows (at most 16): 16 columns of the output a workgroup, whose eight waves split K in steps of 32 and read W
// straight from memory into the MFMA's registers (each element once); the waves' sums are joined in LDS. Bound by the latency
// of a launch and a few rounds of loads: 1 x 1536 x 6144 bf16 7.2 us, 19 MB of W.
template <class T>
__global__ __launch_bounds__(512) void prod_few_kernel(GemmArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int W = 8, U = 8;
    __shared__ float red[W][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15;
    const int64_t n0 = (int64_t)blockIdx.x * 16, wn = n0 + r;
    const int64_t steps = (a.K + 31) / 32;
    const T* wp = static_cast<const T*>(a.B) + min(wn, a.N - 1) * a.ldb;
    const T* xp = static_cast<const T*>(a.A) + min((int64_t)r, a.M - 1) * a.lda;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    // eight of K at k, zeros past its end (rows and columns past theirs repeat the last one: never stored)
    auto ld = [&](const T* p, int64_t k) {
        x8 v;
        if (k + 8 <= a.K) {
            const Pack<T, 8> q = *reinterpret_cast<const Pack<T, 8>*>(p + k);
            v = __builtin_bit_cast(x8, q);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = k + e < a.K ? p[k + e] : (T)0.f;
        }
        return v;
    };
    for (int64_t s0 = wave; s0 < steps; s0 += W * U) {
        x8 w[U], x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = (s0 + u * W) * 32 + 8 * (lane >> 4);
            w[u] = ld(wp, k);
            x[u] = ld(xp, k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (__is_same(T, bf16)) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[u], x[u], acc, 0, 0, 0);
            else acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[u], x[u], acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) red[wave][r][4 * (lane >> 4) + v] = acc[v];
    __syncthreads();
    if (tid < 256) {
        const int64_t m = tid >> 4, n = n0 + (tid & 15);
        if (m >= a.M || n >= a.N) return;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += red[w][m][tid & 15];
        if (a.bias) v += a.bias[n];
        if (a.Z) static_cast<T*>(a.Z)[m * a.ldz + n] = (T)v;
        float y[1] = {v};
        act_values(y, a.act);
        v = y[0];
        if (a.R) v += (float)static_cast<const T*>(a.R)[m * a.ldr + n];
        static_cast<T*>(a.C)[m * a.ldc + n] = (T)v;
    }
}

// rows [rows][cols] into rows of cols rounded up to a multiple of 8, zeros behind them; two operands in one launch (either may
// have no rows)
struct PadArgs {
    const void* src[2];
    int64_t ld[2], rows[2], cols;
    void* dst[2];
};
template <class T>
__global__ __launch_bounds__(256) void prod_pad_kernel(PadArgs a) {
    const int64_t chunks = (a.cols + 7) / 8, n0 = a.rows[0] * chunks, n = n0 + a.rows[1] * chunks;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int w = i >= n0;
        const int64_t j = w ? i - n0 : i, r = j / chunks, c = (j - r * chunks) * 8;
        float v[8];
        load8(static_cast<const T*>(w ? a.src[1] : a.src[0]) + r * (w ? a.ld[1] : a.ld[0]), c, a.cols, v);
        store8(static_cast<T*>(w ? a.dst[1] : a.dst[0]) + r * chunks * 8, c, chunks * 8, v);
    }
}

// dz = dY act'(z) [M][pitch] (null: not stored) and its column sums over this workgroup's rows, part [gridDim.y][N] (null:
// none; a single row of workgroups writes db itself). A workgroup takes 256 columns, 8 a thread, eight rows at a time.
// dz is rounded to the tensors' type, as the matrix units read 16 bits; db is of dz before that. Against 64 bits dX and dW are off by
// 2.3e-3 of their norm in bf16, where their own rounding alone gives 1.7e-3.
// Bound by HBM: 2176 x 6144 bf16 gelu 17.2 us, 80 MB, 4.7 TB/s.
template <class T>
__global__ __launch_bounds__(256) void prod_dz_kernel(const T* dY, int64_t lddy, const T* Z, int64_t ldz, int64_t M, int64_t N,
                                                      int act, T* dz, int64_t pitch, float* part, int accumulate) {
    __shared__ float red[8][256 + 8];
    const int c = (threadIdx.x & 31) * 8, rl = threadIdx.x >> 5;
    const int64_t n = (int64_t)blockIdx.x * 256 + c;
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = 0.f;
    // (lanes past the last column go along, as zeros: see finish8)
    for (int64_t m = (int64_t)blockIdx.y * 8 + rl; m < M; m += (int64_t)gridDim.y * 8) {
        float d[8];
        load8(dY + m * lddy, n, N, d);
        if (act) {   // (uniform)
            float z[8];
            load8(Z + m * ldz, n, N, z);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] *= act_slope(z[e], act);
        }
        if (dz) store8(dz + m * pitch, n, pitch, d);   // (columns past N: 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += d[e];
    }
    if (!part) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) red[rl][c + e] = s[e];
    __syncthreads();
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= N) return;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += red[w][threadIdx.x];
    if (gridDim.y == 1 && accumulate) t += part[j];
    part[(int64_t)blockIdx.y * N + j] = t;
}

// db (+)= the workgroups' sums
__global__ __launch_bounds__(kColumnSumThreads) void prod_db_kernel(const float* __restrict__ part, int parts, int64_t N,
                                                                    float* db, int accumulate) {
    column_sums(part, parts, N, [&](int64_t i, float t) { db[i] = accumulate ? db[i] + t : t; });
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

template <class T>
void pad(sa3k_ctx* ctx, const PadArgs& a) {
    const int64_t n = (a.rows[0] + a.rows[1]) * (up8(a.cols) / 8);
    if (n == 0) return;
    KernelScope ks(ctx, "linear_act_pad");
    launch_k(ctx, false, prod_pad_kernel<T>, dim3((unsigned)std::min<int64_t>(ceil_div(n, 256), 65536)), dim3(256), 0, a);
    SA3K_LAUNCHED();
}

size_t split_bytes(const ProdPlan& p, int64_t M, int64_t N) {
    return p.splits > 1 ? (size_t)p.splits * (size_t)M * (size_t)up8(N) * sizeof(float) : 0;
}

// the plan's numbers into the arguments; the workgroups of the launch
int64_t plan_into(GemmArgs& a, const ProdPlan& p, float* part) {
    a.splits = p.splits;
    a.per = p.per;
    a.part = p.splits > 1 ? part : nullptr;
    a.pitch = up8(a.N);
    return ceil_div(ceil_div(a.M, p.edge) * ceil_div(a.N, p.edge), 8) * 8 * p.splits;
}
template <class T, bool FWD>
void sum_splits(sa3k_ctx* ctx, const GemmArgs& a) {
    if (a.splits == 1) return;
    KernelScope ks(ctx, "linear_act_sum");
    launch_k(ctx, true, prod_sum_kernel<T, FWD>, dim3((unsigned)ceil_div(a.M * (a.pitch / 8), 256)), dim3(256), 0, a);
    SA3K_LAUNCHED();
}
template <class T, bool AK, bool BK, bool FWD>
void tile_run(sa3k_ctx* ctx, GemmArgs& a, const ProdPlan& p, float* part, const char* name) {
    const int64_t wgs = plan_into(a, p, part);
    {
        const dim3 grid((unsigned)wgs);
        KernelScope ks(ctx, name, 2.0 * (double)a.M * (double)a.N * (double)a.K);
        if (p.edge == 256) launch_k(ctx, a.splits == 1, prod_big_kernel<T, AK, BK, FWD>, grid, dim3(512), 0, a);
        else if (wgs <= 256)   // one workgroup a CU at the most: deeper stages
            launch_k(ctx, a.splits == 1, prod_tile_kernel<T, 4, AK, BK, FWD>, grid, dim3(256), 0, a);
        else launch_k(ctx, a.splits == 1, prod_tile_kernel<T, 2, AK, BK, FWD>, grid, dim3(256), 0, a);
        SA3K_LAUNCHED();
    }
    sum_splits<T, FWD>(ctx, a);
}

template <class T>
void fwd_run(sa3k_ctx* ctx, const ProdArgs& p) {
    GemmArgs a{};
    a.A = p.X; a.lda = p.ldx; a.B = p.W; a.ldb = p.ldw;
    a.M = p.M; a.N = p.N; a.K = p.K;
    a.C = p.Y; a.ldc = p.ldy; a.act = p.act; a.bias = p.bias; a.R = p.R; a.ldr = p.ldr; a.Z = p.Zo; a.ldz = p.ldz;
    if (p.M <= kFewRows) {
        KernelScope ks(ctx, "linear_act_few", 2.0 * (double)a.M * (double)a.N * (double)a.K);
        launch_k(ctx, true, prod_few_kernel<T>, dim3((unsigned)ceil_div(a.N, 16)), dim3(512), 0, a);
        SA3K_LAUNCHED();
        return;
    }
    const bool px = !loads16(p.X, p.ldx, p.K), pw = !loads16(p.W, p.ldw, p.K);
    const int64_t Kp = px || pw ? up8(p.K) : p.K;
    const ProdPlan plan = prod_plan(p.M, p.N, Kp);
    Scratch s;
    // (if one operand is padded, both are: they share K)
    const size_t ox = s.take(px || pw ? (size_t)p.M * Kp * 2 : 0), ow = s.take(px || pw ? (size_t)p.N * Kp * 2 : 0);
    const size_t os = s.take(split_bytes(plan, p.M, p.N));
    char* ws = s.need ? reinterpret_cast<char*>(layer_workspace(ctx, s.need)) : nullptr;
    if (px || pw) {
        pad<T>(ctx, PadArgs{{p.X, p.W}, {p.ldx, p.ldw}, {p.M, p.N}, p.K, {ws + ox, ws + ow}});
        a.A = ws + ox;
        a.B = ws + ow;
        a.lda = a.ldb = a.K = Kp;
    }
    tile_run<T, false, false, true>(ctx, a, plan, reinterpret_cast<float*>(ws + os), "linear_act_fwd");
}

// Row shares of the pass over dY and z: one for up to 64 rows (which saves the launch that adds up shares), else about 128, each
// of the same number of rounds of eight rows.
int dz_parts(int64_t M) {
    if (M <= 64) return 1;
    const int64_t groups = std::max<int64_t>(1, ceil_div(M, 8)), rounds = ceil_div(groups, 128);
    return (int)ceil_div(groups, rounds);
}

template <class T>
void bwd_run(sa3k_ctx* ctx, const ProdArgs& p) {
    const int64_t M = p.M, N = p.N, K = p.K, Np = up8(N), Kp = up8(K);
    const bool products = p.dX || p.dW;
    // dz as the products read it: dY itself, or its own rows
    const bool own_dz = products && M > 0 && (p.act != SA3K_ACT_NONE || !loads16(p.dY, p.lddy, N));
    const bool px = p.dW && M > 0 && !loads16(p.X, p.ldx, K), pw = p.dX && M > 0 && !loads16(p.W, p.ldw, K);
    const bool do_x = p.dX && M > 0, do_w = p.dW != nullptr;
    ProdPair plan{false, prod_plan(M > 0 ? M : 1, K, N), prod_plan(N, K, M > 0 ? M : 1)};
    if (do_x && do_w) plan = prod_pair({M, K, N}, {N, K, M});
    const int parts = dz_parts(M);
    Scratch s;
    const size_t oz = s.take(own_dz ? (size_t)M * Np * 2 : 0), ox = s.take(px ? (size_t)M * Kp * 2 : 0);
    const size_t ow = s.take(pw ? (size_t)N * Kp * 2 : 0), ob = s.take(p.db && parts > 1 ? (size_t)parts * N * 4 : 0);
    const size_t sx = do_x ? split_bytes(plan.a, M, K) : 0, sw = do_w ? split_bytes(plan.b, N, K) : 0;
    const size_t osx = s.take(plan.together ? sx : std::max(sx, sw)), osw = plan.together ? s.take(sw) : osx;
    char* ws = s.need ? reinterpret_cast<char*>(layer_workspace(ctx, s.need)) : nullptr;
    T* dz = own_dz ? reinterpret_cast<T*>(ws + oz) : nullptr;
    float* part = !p.db ? nullptr : parts > 1 ? reinterpret_cast<float*>(ws + ob) : p.db;
    if (own_dz || p.db) {
        KernelScope ks(ctx, "linear_act_dz");
        launch_k(ctx, !products && parts == 1, prod_dz_kernel<T>, dim3((unsigned)ceil_div(N, 256), (unsigned)parts), dim3(256), 0,
                 static_cast<const T*>(p.dY), p.lddy, static_cast<const T*>(p.Z), p.ldz, M, N, p.act, dz, Np, part, p.accumulate);
        SA3K_LAUNCHED();
    }
    if (p.db && parts > 1) {
        KernelScope ks(ctx, "linear_act_db");
        launch_k(ctx, !products, prod_db_kernel, dim3((unsigned)ceil_div(N, 64)), dim3(kColumnSumThreads), 0, part, parts, N, p.db,
                 p.accumulate);
        SA3K_LAUNCHED();
    }
    const void* g = own_dz ? dz : p.dY;
    const int64_t ldg = own_dz ? Np : p.lddy;
    GemmArgs x{}, w{};
    pad<T>(ctx, PadArgs{{p.W, p.X}, {p.ldw, p.ldx}, {pw ? N : 0, px ? M : 0}, K, {ws + ow, ws + ox}});
    if (do_x) {   // [M][K] = dz [M][N] . W [N][K]
        x.A = g; x.lda = ldg;
        x.B = pw ? ws + ow : p.W;
        x.ldb = pw ? Kp : p.ldw;
        x.M = M; x.N = K; x.K = N;
        x.C = p.dX; x.ldc = p.lddx;
    }
    if (do_w) {   // [N][K] = dz^T [N][M] . X [M][K]
        w.A = g; w.lda = ldg;
        w.B = px ? ws + ox : p.X;
        w.ldb = px ? Kp : p.ldx;
        w.M = N; w.N = K; w.K = M;
        w.C = p.dW; w.ldc = p.lddw;
        w.c_f32 = p.dw_type == SA3K_TYPE_F32;
        w.accumulate = p.accumulate;
    }
    float *part_x = reinterpret_cast<float*>(ws + osx), *part_w = reinterpret_cast<float*>(ws + osw);
    if (plan.together) {
        const int64_t nx = plan_into(x, plan.a, part_x), nw = plan_into(w, plan.b, part_w);
        {
            KernelScope ks(ctx, "linear_act_dx_dw", 4.0 * (double)M * (double)N * (double)K);
            launch_k(ctx, x.splits == 1 && w.splits == 1, prod_pair_kernel<T>, dim3((unsigned)(nx + nw)), dim3(256), 0, x, w,
                     (int)nx);
            SA3K_LAUNCHED();
        }
        sum_splits<T, false>(ctx, x);
        sum_splits<T, false>(ctx, w);
        return;
    }
    if (do_x) tile_run<T, false, true, false>(ctx, x, plan.a, part_x, "linear_act_dx");
    if (do_w) tile_run<T, true, true, false>(ctx, w, plan.b, part_w, "linear_act_dw");
}

}  // namespace

extern "C" {

SA3K_API int sa3k_linear_act_fwd(sa3k_ctx* ctx, int type, int act, const void* X, int64_t ldx, const void* W, int64_t ldw,
                                 const float* bias, const void* residual, int64_t ldr, int64_t M, int64_t N, int64_t K,
                                 void* Y, int64_t ldy, void* Z, int64_t ldz) {
    return sa3k_guard(ctx, "sa3k_linear_act_fwd", [&] {
        ProdArgs p;
        p.type = type; p.act = act; p.M = M; p.N = N; p.K = K;
        p.X = X; p.ldx = ldx; p.W = W; p.ldw = ldw; p.bias = bias; p.R = residual; p.ldr = ldr;
        p.Y = Y; p.ldy = ldy; p.Zo = Z; p.ldz = ldz;
        int code;
        const char* msg = prod_check(p, false, &code);
        require_ok(msg, code);
        if (M == 0) return;
        DeviceScope dev(ctx);
        if (type == SA3K_TYPE_BF16) fwd_run<bf16>(ctx, p);
        else fwd_run<f16>(ctx, p);
    });
}

SA3K_API int sa3k_linear_act_bwd(sa3k_ctx* ctx, int type, int act, const void* dY, int64_t lddy, const void* Z, int64_t ldz,
                                 const void* X, int64_t ldx, const void* W, int64_t ldw, int64_t M, int64_t N, int64_t K,
                                 void* dX, int64_t lddx, void* dW, int dw_type, int64_t lddw, float* db, int accumulate) {
    return sa3k_guard(ctx, "sa3k_linear_act_bwd", [&] {
        ProdArgs p;
        p.type = type; p.act = act; p.M = M; p.N = N; p.K = K;
        p.dY = dY; p.lddy = lddy; p.Z = Z; p.ldz = ldz; p.X = X; p.ldx = ldx; p.W = W; p.ldw = ldw;
        p.dX = dX; p.lddx = lddx; p.dW = dW; p.dw_type = dw_type; p.lddw = lddw; p.db = db; p.accumulate = accumulate;
        int code;
        const char* msg = prod_check(p, true, &code);
        require_ok(msg, code);
        DeviceScope dev(ctx);
        if (type == SA3K_TYPE_BF16) bwd_run<bf16>(ctx, p);
        else bwd_run<f16>(ctx, p);
    });
}

}  // extern "C"
