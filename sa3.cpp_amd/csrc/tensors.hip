// Global norm and clip over many gradient tensors of several types.
//   s = g / count, norm = sqrt(sum s^2), out = s min(1, clip / (norm + 1e-6))
// Two launches, bound by HBM: every gradient is read once for the norm and once for the result, which is written once.
//   pass 1  sums of squares in f64, one a workgroup, in a fixed order
//   pass 2  every workgroup adds those up in the same order, so that all agree on the factor without a third launch, then
//           scales its pieces
// The list lies on the device as pieces of at most 32 KB, each of one tensor; a workgroup takes every gridDim-th. Pass 2
// takes them in the opposite order, so that what pass 1 read last is still in the memory-side cache, and writes past it.
// Measured on MI355X: 288 f32 tensors of 26.5M elements 16.9 and 34.6 us (6.2 TB/s), 108 tensors of 453M in bf16 and f32 147 and 328 us
// (6.2 and 5.5 TB/s). Eight workgroups a CU; the pass that scales loads a piece whole before it stores it, in 60 registers (with the
// first piece's loads ahead of the sums it took more than 128 and spilled).
#include <algorithm>
#include <memory>

#include "layer_ops_dev.h"
#include "tensors.h"

struct sa3k_tensors {
    const sa3k_ctx* ctx = nullptr;   // that made it
    sa3k::TensorPiece* pieces = nullptr;
    double* partials = nullptr;   // [grid], then the norm and the factor of the last call
    int64_t n = 0;
    int grid = 0;
};

namespace {
using namespace sa3k;

constexpr int kThreads = 256, kLoads = kPieceBytes / 16 / kThreads;   // of 16 bytes, a thread's of a piece
constexpr int kMostGroups = 2048;                         // eight workgroups a CU

template <class T>
constexpr int kVec = 16 / (int)sizeof(T);

// Whole pieces keep all of a thread's loads in registers, kThreads apart; shorter ones go load by load.
template <class T>
__device__ __forceinline__ bool whole(const TensorPiece& p) { return p.n == kPieceBytes / (int)sizeof(T); }
__device__ __forceinline__ void load_whole(const TensorPiece& p, u32x4a (&raw)[kLoads]) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) raw[u] = load16((const SA3K_GLOBAL f16*)p.grad + (u * kThreads + (int)threadIdx.x) * 8);
}
// elements i .. of a piece, zeros past its end
template <class T>
__device__ __forceinline__ u32x4a load_part(const TensorPiece& p, int i) {
    const SA3K_GLOBAL T* g = (const SA3K_GLOBAL T*)p.grad;
    if (i + kVec<T> <= p.n) return load16(g + i);
    Pack<T, kVec<T>> q;
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) q.v[e] = i + e < p.n ? g[i + e] : (T)0.f;
    return __builtin_bit_cast(u32x4a, q);
}

template <class T>
__device__ __forceinline__ void add_squares(u32x4a raw, float inv, double& acc) {
    const Pack<T, kVec<T>> q = __builtin_bit_cast(Pack<T, kVec<T>>, raw);
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) {
        const float s = (float)q.v[e] * inv;   // (by 1 without an average)
        acc = __builtin_fma((double)s, (double)s, acc);
    }
}
template <class T>
__device__ __forceinline__ void add_piece(const TensorPiece& p, float inv, double& acc) {
    if (whole<T>(p)) {
        u32x4a raw[kLoads];
        load_whole(p, raw);
#pragma unroll
        for (int u = 0; u < kLoads; ++u) add_squares<T>(raw[u], inv, acc);
    } else {
#pragma unroll 1
        for (int i = (int)threadIdx.x * kVec<T>; i < p.n; i += kThreads * kVec<T>) add_squares<T>(load_part<T>(p, i), inv, acc);
    }
}

struct Factors {
    float inv, scale;
};
template <class T, class O, bool WHOLE>
__device__ __forceinline__ void scale_store(const TensorPiece& p, int i, u32x4a raw, const Factors& f) {
    constexpr int V = kVec<T>, W = kVec<O>;
    SA3K_GLOBAL O* o = (SA3K_GLOBAL O*)p.out;
    const Pack<T, V> q = __builtin_bit_cast(Pack<T, V>, raw);
    Pack<O, W> r[V / W];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        r[e / W].v[e % W] = (O)((float)q.v[e] * f.inv * f.scale);   // (by 1 where there is no average, or no clip)
    }
    if (WHOLE || i + V <= p.n) {
#pragma unroll
        for (int w = 0; w < V / W; ++w) store16_past(o + i + w * W, __builtin_bit_cast(u32x4a, r[w]));
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (i + e < p.n) o[i + e] = r[e / W].v[e % W];
    }
}
template <class T, class O>
__device__ __forceinline__ void scale_piece(const TensorPiece& p, const Factors& f) {
    constexpr int V = kVec<T>;
    if (whole<T>(p)) {
        u32x4a raw[kLoads];
        load_whole(p, raw);
#pragma unroll
        for (int u = 0; u < kLoads; ++u) scale_store<T, O, true>(p, (u * kThreads + (int)threadIdx.x) * V, raw[u], f);
    } else {
#pragma unroll 1
        for (int i = (int)threadIdx.x * V; i < p.n; i += kThreads * V) scale_store<T, O, false>(p, i, load_part<T>(p, i), f);
    }
}
// (the kind is uniform)
__device__ __forceinline__ void scale_any(const TensorPiece& p, const Factors& f) {
    if ((p.kind & 3) == 0) scale_piece<float, float>(p, f);
    else if (p.kind == 1) scale_piece<f16, f16>(p, f);
    else if (p.kind == 2) scale_piece<bf16, bf16>(p, f);
    else if (p.kind == 5) scale_piece<f16, float>(p, f);
    else scale_piece<bf16, float>(p, f);
}

// the same bits in every thread
__device__ __forceinline__ double group_sum(double v) {
    __shared__ double sh[kThreads / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) t += sh[w];
    return t;
}

__global__ __launch_bounds__(kThreads, 4) void tensors_norm_kernel(const TensorPiece* __restrict__ pieces, int64_t n, float inv,
                                                                double* __restrict__ partials) {
    double acc = 0.0;
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        const TensorPiece p = pieces[i];
        if ((p.kind & 3) == 0) add_piece<float>(p, inv, acc);
        else if ((p.kind & 3) == 1) add_piece<f16>(p, inv, acc);
        else add_piece<bf16>(p, inv, acc);
    }
    const double t = group_sum(acc);
    if (threadIdx.x == 0) partials[blockIdx.x] = t;
}

__global__ __launch_bounds__(kThreads, 4) void tensors_clip_kernel(const TensorPiece* __restrict__ pieces, int64_t n, float inv, int avg,
                                                                float most, const double* __restrict__ partials, int parts,
                                                                double* __restrict__ stat) {
    double acc = 0.0;
    for (int k = threadIdx.x; k < parts; k += kThreads) acc += partials[k];
    const double norm = sqrt(group_sum(acc));
    const bool clip = most > 0.f && norm > (double)most;
    const float scale = clip ? (float)((double)most / (norm + 1e-6)) : 1.f;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        stat[0] = norm;
        stat[1] = (double)scale;
    }
    for (int64_t i = n - 1 - (int64_t)blockIdx.x; i >= 0; i -= gridDim.x) {
        const TensorPiece p = pieces[i];
        // (in place, with nothing to change: the gradient is its own result)
        if (avg || clip || p.out != p.grad) scale_any(p, Factors{inv, scale});
    }
}

void tensors_free(sa3k_tensors* t) {
    if (!t) return;
    if (t->pieces) (void)hipFree(t->pieces);
    if (t->partials) (void)hipFree(t->partials);
    delete t;
}

}  // namespace

extern "C" {

SA3K_API int sa3k_tensors_create(sa3k_ctx* ctx, const sa3k_tensor* tensors, int64_t count, sa3k_tensors** out) {
    return sa3k_guard(ctx, "sa3k_tensors_create", [&] {
        SA3K_REQUIRE(out != nullptr, "out is null");
        *out = nullptr;
        int code;
        const char* msg = tensors_check(tensors, count, &code);
        require_ok(msg, code);
        DeviceScope dev(ctx);
        const std::vector<TensorPiece> pieces = tensor_pieces(tensors, count);
        std::unique_ptr<sa3k_tensors, void (*)(sa3k_tensors*)> t(new sa3k_tensors(), tensors_free);
        t->ctx = ctx;
        t->n = (int64_t)pieces.size();
        t->grid = (int)std::max<int64_t>(1, std::min<int64_t>(t->n, kMostGroups));
        SA3K_HIP(hipMalloc(&t->partials, sizeof(double) * (size_t)(t->grid + 2)));
        if (t->n > 0) {
            const size_t bytes = sizeof(TensorPiece) * pieces.size();
            SA3K_HIP(hipMalloc(&t->pieces, bytes));
            SA3K_HIP(hipMemcpyAsync(t->pieces, pieces.data(), bytes, hipMemcpyHostToDevice, ctx->stream));
            sa3k_note_main(ctx);
            SA3K_HIP(hipStreamSynchronize(ctx->stream));
        }
        *out = t.release();
    });
}

SA3K_API int sa3k_tensors_destroy(sa3k_ctx* ctx, sa3k_tensors* t) {
    return sa3k_guard(ctx, "sa3k_tensors_destroy", [&] {
        if (!t) return;
        SA3K_REQUIRE(t->ctx == ctx, "the list belongs to another context");
        DeviceScope dev(ctx);
        SA3K_HIP(hipStreamSynchronize(ctx->stream));
        tensors_free(t);
    });
}

SA3K_API int sa3k_tensors_clip(sa3k_ctx* ctx, sa3k_tensors* t, int count, float max_norm, double* stat, double* norm_out) {
    return sa3k_guard(ctx, "sa3k_tensors_clip", [&] {
        SA3K_REQUIRE(t != nullptr, "null list");
        SA3K_REQUIRE(t->ctx == ctx, "the list belongs to another context");
        int code;
        const char* msg = clip_check(count, max_norm, stat, &code);
        require_ok(msg, code);
        DeviceScope dev(ctx);
        const int avg = count > 1 ? 1 : 0;
        const float inv = 1.0f / (float)count;
        double* st = stat ? stat : t->partials + t->grid;
        {
            KernelScope ks(ctx, "tensors_norm");
            launch_k(ctx, false, tensors_norm_kernel, dim3((unsigned)t->grid), dim3(kThreads), 0, t->pieces, t->n, inv, t->partials);
            SA3K_LAUNCHED();
        }
        {
            KernelScope ks(ctx, "tensors_clip");
            launch_k(ctx, true, tensors_clip_kernel, dim3((unsigned)t->grid), dim3(kThreads), 0, t->pieces, t->n, inv, avg, max_norm,
                     t->partials, t->grid, st);
            SA3K_LAUNCHED();
        }
        if (norm_out) {
            double r[2];
            SA3K_HIP(hipMemcpyAsync(r, st, sizeof r, hipMemcpyDeviceToHost, ctx->stream));
            sa3k_note_main(ctx);
            SA3K_HIP(hipStreamSynchronize(ctx->stream));
            *norm_out = r[0];
        }
    });
}

}  // extern "C"
