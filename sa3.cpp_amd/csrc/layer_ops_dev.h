// Device helpers shared by the layer operators (lnorm.hip, wattn*.hip, linact.hip).
#pragma once

#include "layer_ops.h"
#include "sa3k_internal.h"

namespace sa3k {

typedef __bf16 bf16;
typedef _Float16 f16;

// The calling thread's current device is the context's while this lives, and what it was afterwards.
struct DeviceScope {
    int before = -1;
    explicit DeviceScope(const sa3k_ctx* ctx) {
        int now = -1;
        SA3K_HIP(hipGetDevice(&now));
        if (now == ctx->device) return;
        SA3K_HIP(hipSetDevice(ctx->device));
        before = now;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
};

// throws what a check of layer_ops.h found
inline void require_ok(const char* msg, int code) {
    if (msg) sa3k_throw(code, msg);
}

// The layer operators' scratch, at least `bytes` of it, used in turn on the context's stream. Not the products' workspace: that
// one's address is in the DiT's captured steps, and these calls, whose needs are larger, would move it by growing it.
inline float* layer_workspace(sa3k_ctx* ctx, size_t bytes) {
    if (bytes > ctx->layer_ws_bytes) {
        SA3K_REQUIRE(!ctx->capturing, "the layer operators' scratch cannot grow while a graph is being captured");
        if (ctx->layer_ws) {
            SA3K_HIP(hipStreamSynchronize(ctx->stream));
            SA3K_HIP(hipFree(ctx->layer_ws));
            ctx->layer_ws = nullptr;
            ctx->layer_ws_bytes = 0;
        }
        SA3K_HIP(hipMalloc(&ctx->layer_ws, bytes));
        ctx->layer_ws_bytes = bytes;
    }
    return static_cast<float*>(ctx->layer_ws);
}

// N elements at p, which need only be aligned to their size: global memory takes wide accesses at any
// address, so a row that starts at an odd element costs one more cache line and no second code path
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[N];
};

// Where addresses come from memory, the compiler has to be told that they are of global memory. 16 bytes at a time, at an address
// that is aligned to an element (elements of T, two or four bytes); store16_past goes past the caches.
#define SA3K_GLOBAL __attribute__((address_space(1)))
typedef unsigned u32x4a __attribute__((ext_vector_type(4)));
typedef unsigned u32x4at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x4at4 __attribute__((ext_vector_type(4), aligned(4)));
template <class T>
__device__ __forceinline__ u32x4a load16(const SA3K_GLOBAL T* p) {
    if constexpr (sizeof(T) == 4) return *(const SA3K_GLOBAL u32x4at4*)p;
    else return *(const SA3K_GLOBAL u32x4at2*)p;
}
template <class T>
__device__ __forceinline__ void store16(SA3K_GLOBAL T* p, u32x4a v) {
    if constexpr (sizeof(T) == 4) *(SA3K_GLOBAL u32x4at4*)p = u32x4at4(v);
    else *(SA3K_GLOBAL u32x4at2*)p = u32x4at2(v);
}
template <class T>
__device__ __forceinline__ void store16_past(SA3K_GLOBAL T* p, u32x4a v) {
    if constexpr (sizeof(T) == 4) __builtin_nontemporal_store(u32x4at4(v), (SA3K_GLOBAL u32x4at4*)p);
    else __builtin_nontemporal_store(u32x4at2(v), (SA3K_GLOBAL u32x4at2*)p);
}

// The sums of `parts` workspace rows of n floats each: a workgroup takes 64 columns, a sixteenth of the rows a wave, eight
// rows in flight; added in row order within a wave, then wave by wave. Calls store(i, sum) for column i. (With four waves a
// workgroup 512 rows of 2050 columns took 9.4 us.)
constexpr int kColumnSumThreads = 1024;
template <class F>
__device__ __forceinline__ void column_sums(const float* __restrict__ part, int parts, int64_t n, F&& store) {
    __shared__ float s[16][64];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * 64 + lane;
    const int per = (parts + 15) / 16, lo = min(parts, w * per), hi = min(parts, lo + per);
    float t = 0.f;
    if (i < n)
        for (int k = lo; k < hi; k += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = part[(int64_t)min(k + u, hi - 1) * n + i];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (k + u < hi) t += v[u];
        }
    s[w][lane] = t;
    __syncthreads();
    if (w || i >= n) return;
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += s[k][lane];
    store(i, t);
}

}  // namespace sa3k
