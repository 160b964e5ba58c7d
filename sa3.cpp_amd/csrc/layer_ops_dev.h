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

// N elements at p, which need only be aligned to their size: global memory takes wide accesses at any
// address, so a row that starts at an odd element costs one more cache line and no second code path
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[N];
};

}  // namespace sa3k
