// What the windowed attention kernels share (wattn.hip: forward; wattn_bwd.hip: backward): element types, the
// LDS tile layout and its loads.
//
// A tile is R rows (keys or queries) of D elements as D / 64 sub-tiles of [R][64], 128-byte LDS rows whose
// eight 16-byte chunks are XOR-swizzled by swz(row), so that row reads (16 bytes of row lane % 32) and transposed
// reads (ds_read_b64_tr_b16) meet no bank conflicts. Tiles are filled by buffer_load ... lds through a descriptor
// that ends at the sample's last row: rows past it read as zeros, whatever lies there in memory.
#pragma once

#include "layer_ops_dev.h"

namespace sa3k {
namespace wattn {

constexpr int BLK = 64;                    // rows of a workgroup's tiles
constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

typedef float f32x16 __attribute__((__vector_size__(16 * sizeof(float))));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

template <class T>
struct Vec;
template <>
struct Vec<bf16> {
    typedef bf16 x8 __attribute__((__vector_size__(16)));
    typedef bf16 x4 __attribute__((__vector_size__(8)));
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Vec<f16> {
    typedef f16 x8 __attribute__((__vector_size__(16)));
    typedef f16 x4 __attribute__((__vector_size__(8)));
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

__device__ __forceinline__ int swz(int r) {
    const int a = (r >> 1) & 7;
    return ((a >> 2) & 1) | ((((a >> 1) ^ (a >> 2)) & 1) << 1) | ((a & 1) << 2);
}
// chunk c (8 dims) of row r of a tile of R rows
template <class T, int R = BLK>
__device__ __forceinline__ typename Vec<T>::x8 ld_row(const char* t, int r, int c) {
    return *reinterpret_cast<const typename Vec<T>::x8*>(t + (c >> 3) * (R * 128) + r * 128 + (((c & 7) ^ swz(r)) << 4));
}
// lane j of a 16-lane group gets rows k0 .. k0 + 3 of column n0 + j (n0 a multiple of 16)
template <class T, int R = BLK>
__device__ __forceinline__ typename Vec<T>::x4 ld_tr(const char* t, int k0, int n0, int lane) {
    const int j = lane & 15, row = k0 + (j >> 2), n = (n0 & 63) + 4 * (j & 3);
    const char* a = t + (n0 >> 6) * (R * 128) + row * 128 + (((n >> 3) ^ swz(row)) << 4) + (n & 7) * 2;
    return __builtin_bit_cast(typename Vec<T>::x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                       (__attribute__((address_space(3))) v4s*)(lds_ptr_t)a));
}
// A lane's places in a tile, the same in every tile: eight addresses that a kernel works out once; the rest of a read's
// address is a constant.
//   row  chunk 2 (ks % 4) + lane / 32 of row lane % 32: eight dims of the row, for K step ks of a product
//   tr   transposed: lane j of a 16-lane group gets four rows' column n0 + j; rows 4 (lane / 32) + 8 u .. + 3, u = 0, 1,
//        are the rows that a 32 x 32 product's result holds; columns 32 i + 16 ((lane / 16) % 2) .. + 15
struct LaneOff {
    uint32_t row[4], tr[2][2];
    __device__ __forceinline__ void init(int lane) {
        const int c32 = lane & 31, hl = lane >> 5, j = lane & 15;
#pragma unroll
        for (int k = 0; k < 4; ++k) row[k] = (uint32_t)(c32 * 128 + (((2 * k + hl) ^ swz(c32)) << 4));
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int r = 4 * hl + 8 * u + (j >> 2), n = 32 * i + 16 * ((lane >> 4) & 1) + 4 * (j & 3);
                tr[i][u] = (uint32_t)(r * 128 + (((n >> 3) ^ swz(r)) << 4) + (n & 7) * 2);
            }
    }
};
// the fragment of rows 32 h .. 32 h + 31 and K step ks of the tile of R rows at LDS address t
template <class T, int R>
__device__ __forceinline__ typename Vec<T>::x8 rd_row(uint32_t t, const LaneOff& o, int h, int ks) {
    return *(const __attribute__((address_space(3))) typename Vec<T>::x8*)(uintptr_t)(t + o.row[ks & 3] +
                                                                                    (uint32_t)((ks >> 2) * R * 128 + h * 4096));
}
// the transposed fragment of rows 16 m .. 16 m + 15 and columns 32 i .. 32 i + 31
template <class T, int R>
__device__ __forceinline__ typename Vec<T>::x8 rd_tr(uint32_t t, const LaneOff& o, int m, int i) {
    typename Vec<T>::x4 q[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
        q[u] = __builtin_bit_cast(typename Vec<T>::x4,
                                  __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(uintptr_t)(
                                      t + o.tr[i & 1][u] + (uint32_t)((i >> 1) * R * 128 + m * 2048))));
    return typename Vec<T>::x8{q[0][0], q[0][1], q[0][2], q[0][3], q[1][0], q[1][1], q[1][2], q[1][3]};
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(lds_ptr_t)p; }

__device__ __forceinline__ u32x4 buffer_rsrc(const void* base, uint32_t bytes) {
    const unsigned long long a = (unsigned long long)(uintptr_t)base;
    u32x4 r;
    // the descriptor lives in SGPRs: its words are made provably uniform
    r.x = __builtin_amdgcn_readfirstlane((unsigned)a);
    r.y = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32) & 0xffffu);
    r.z = __builtin_amdgcn_readfirstlane(bytes);
    r.w = 0x00020000u;
    return r;
}
// 16 bytes a lane at rs + voff into LDS at lds_addr + 16 lane. Inline asm so that the compiler's waits do not
// drain these loads before unrelated LDS reads; the kernels order them with vmcnt waits and barriers.
__device__ __forceinline__ void dma16(const u32x4& rs, uint32_t voff, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds_addr), "v"(voff), "s"(rs)
                 : "memory");
}
// ROWS rows from row0 on of a tensor of n rows `pitch` elements apart, D elements each, into a tile, by NT threads
// (thread tid of wave `wave` of them). Slot s of a sub-tile is row s / 8, chunk (s % 8) ^ swz(row).
template <int D, int ROWS, int NT>
__device__ __forceinline__ void tile_dma(const void* base, int64_t pitch, int n, int row0, uint32_t tile, int tid,
                                         int wave) {
    constexpr int SUBS = D / 64, PER = ROWS * 8 / NT;   // loads a thread makes for a sub-tile
    static_assert(ROWS * 8 % NT == 0, "whole rounds of loads");
    const int valid = max(0, min(ROWS, n - row0));
    const u32x4 rs = buffer_rsrc(static_cast<const char*>(base) + (int64_t)row0 * pitch * 2,
                                 valid > 0 ? (uint32_t)(((valid - 1) * pitch + D) * 2) : 0u);
#pragma unroll
    for (int u = 0; u < SUBS; ++u)
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int sl = q * NT + tid, row = sl >> 3, kc = (sl & 7) ^ swz(row);
            const uint32_t voff = (uint32_t)row * (uint32_t)(pitch * 2) + (uint32_t)(u * 128 + kc * 16);
            dma16(rs, voff, __builtin_amdgcn_readfirstlane(tile + (uint32_t)(u * ROWS * 128 + (q * NT + wave * 64) * 16)));
        }
}
// 64 floats v[i0 .. i0 + 63] (zeros past n) into LDS, by one wave
__device__ __forceinline__ void vec_dma(const float* v, int n, int i0, const float* lds_vec, int lane) {
    const int valid = max(0, min(BLK, n - i0));
    const u32x4 rs = buffer_rsrc(v + i0, (uint32_t)valid * 4);
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr_t)lds_vec);
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(m0), "v"((uint32_t)lane * 4), "s"(rs)
                 : "memory");
}
// all but the last N of this wave's loads have landed, and its earlier LDS reads have returned: memory that only this
// wave uses is ordered by this alone
template <int N>
__device__ __forceinline__ void wait_own_loads() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (0 << 8) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}
// The tiles of a workgroup run through STAGES pieces of LDS, LOADS loads a wave and tile. Before tile i is used: its loads
// have landed, `later` tiles' (at most STAGES - 2) that were issued after it may be under way; then a barrier makes
// every wave's visible, and says that every wave is done with the tile before, whose piece the next loads overwrite.
template <int LATER, int LOADS>
__device__ __forceinline__ void wait_tile(int later) {
    static_assert(LATER * LOADS < 64, "vmcnt range");
    if constexpr (LATER > 0) {
        if (later < LATER) return wait_tile<LATER - 1, LOADS>(later);
    }
    constexpr int N = LATER * LOADS;
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
    asm volatile("s_barrier" ::: "memory");
}

// The sums of a loop, after it, as the registers that the loop used. Without this the compiler takes the vectors apart for
// the code behind the loop and copies every element to a register of its own in every round.
template <int N>
__device__ __forceinline__ void settle(f32x16 (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// 2^x on the hardware's exp unit: results below 2^-126 flush to zero
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// Visible bits. A lane holds rows 8 (v / 4) + 4 (lane / 32) + v % 4, v = 0 .. 15, of each 32 rows of a tile: bit
// 8 (v / 4) + v % 4 of a 32-bit word once that is shifted by 4 (lane / 32). Two instructions an element: the bit spread over a
// word, and a select by it.
__device__ __forceinline__ unsigned long long bits_below(int n) {
    return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
}
struct Bits {
    uint32_t w[2];
    // rows r0 .. r0 + 63: those of lo .. lo + n - 1, and those below first
    __device__ __forceinline__ void set(int r0, int lo, int n, int first, int lane) {
        const unsigned long long m = (bits_below(lo + n - r0) & ~bits_below(lo - r0)) | bits_below(first - r0);
        const int sh = 4 * (lane >> 5);
        w[0] = (uint32_t)m >> sh;
        w[1] = (uint32_t)(m >> 32) >> sh;
    }
    __device__ __forceinline__ uint32_t spread(int h, int v) const {   // all ones where visible
        return (uint32_t)__builtin_amdgcn_sbfe((int)w[h], 8 * (v >> 2) + (v & 3), 1);
    }
};
__device__ __forceinline__ float keep(float x, uint32_t m) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & m); }
__device__ __forceinline__ float keep_or_none(float x, uint32_t m) {   // -inf where hidden
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & m) | (~m & 0xFF800000u));
}

// a sample's lengths, in range
__device__ __forceinline__ int clamp_len(const int32_t* len, int b, int most) {
    return len ? min(max(len[b], 0), most) : most;
}

// 16 bytes of a row as 8 elements, zeros where there is no row
template <class T>
__device__ __forceinline__ typename Vec<T>::x8 ld_global(const T* p, bool ok) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (ok) u = *reinterpret_cast<const uint4*>(p);
    return __builtin_bit_cast(typename Vec<T>::x8, u);
}

// Which (sample, key/value head, member of the group) and which block a workgroup takes. Workgroups go out to the 8
// XCDs in turn: consecutive ones differ in (sample, key/value head) first, so with a multiple of 8 of those the query
// heads that share keys and values run on one XCD and share its L2. The last blocks, which see the most
// keys when causal, go first.
struct Place {
    int b, kh, h, blk;
};
__device__ __forceinline__ Place place(const AttnShape& a, int blocks, int index) {
    const int L = index, BH = a.B * a.H, BK = a.B * a.K;
    const int i = L % BH, bk = i % BK, g = i / BK;
    Place p;
    p.b = bk / a.K;
    p.kh = bk - p.b * a.K;
    p.h = p.kh * a.G + g;
    p.blk = blocks - 1 - L / BH;
    return p;
}

}  // namespace wattn
}  // namespace sa3k
