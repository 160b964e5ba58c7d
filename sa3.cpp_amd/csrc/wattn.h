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
// rows k0 .. + 3 and k0 + 8 .. + 11: the eight rows that a 32 x 32 product's result holds in two groups of four
template <class T, int R = BLK>
__device__ __forceinline__ typename Vec<T>::x8 ld_tr8(const char* t, int k0, int n0, int lane) {
    const typename Vec<T>::x4 a = ld_tr<T, R>(t, k0, n0, lane), b = ld_tr<T, R>(t, k0 + 8, n0, lane);
    return typename Vec<T>::x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

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
__device__ __forceinline__ void tile_dma(const void* base, int64_t pitch, int n, int row0, const char* tile, int tid,
                                         int wave) {
    constexpr int SUBS = D / 64, PER = ROWS * 8 / NT;   // loads a thread makes for a sub-tile
    static_assert(ROWS * 8 % NT == 0, "whole rounds of loads");
    const int valid = max(0, min(ROWS, n - row0));
    const u32x4 rs = buffer_rsrc(static_cast<const char*>(base) + (int64_t)row0 * pitch * 2,
                                 valid > 0 ? (uint32_t)(((valid - 1) * pitch + D) * 2) : 0u);
    const uint32_t dst = (uint32_t)(uintptr_t)(lds_ptr_t)tile;
#pragma unroll
    for (int u = 0; u < SUBS; ++u)
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int sl = q * NT + tid, row = sl >> 3, kc = (sl & 7) ^ swz(row);
            const uint32_t voff = (uint32_t)row * (uint32_t)(pitch * 2) + (uint32_t)(u * 128 + kc * 16);
            dma16(rs, voff, __builtin_amdgcn_readfirstlane(dst + (uint32_t)(u * ROWS * 128 + (q * NT + wave * 64) * 16)));
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
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }   // vmcnt(0)
// all but the last N of this wave's loads have landed, and its earlier LDS reads have returned: memory that only this
// wave uses is ordered by this alone
template <int N>
__device__ __forceinline__ void wait_own_loads() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (0 << 8) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}
// this wave's loads have landed; then a barrier makes every wave's visible
__device__ __forceinline__ void wait_loads_all() {
    wait_loads();
    asm volatile("s_barrier" ::: "memory");
}

// 2^x on the hardware's exp unit: results below 2^-126 flush to zero
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

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
__device__ __forceinline__ Place place(const AttnShape& a, int blocks) {
    const int L = blockIdx.x, BH = a.B * a.H, BK = a.B * a.K;
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
