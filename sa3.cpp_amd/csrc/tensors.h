// Host-side arithmetic of the calls over many gradient tensors: the checks of their arguments and the cut into pieces. No
// HIP in here: compiled with g++ in the CPU tests too.
#pragma once

#include <algorithm>
#include <vector>

#include "layer_ops.h"

namespace sa3k {

constexpr int64_t kTensorMost = (int64_t)1 << 40;   // elements of one tensor stay below this

inline bool grad_type(int t) { return t == SA3K_TYPE_F32 || t == SA3K_TYPE_F16 || t == SA3K_TYPE_BF16; }

// Whether no output meets another tensor's gradient or output, nor its own gradient but in place: such elements would be
// scaled twice, or read after they were written.
inline bool outputs_apart(const sa3k_tensor* t, int64_t n) {
    struct Range {
        uintptr_t lo, hi;
        int64_t of;
    };
    std::vector<Range> out;
    auto range = [](const void* p, int64_t k, int type, int64_t of) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(p);
        return Range{a, a + (uintptr_t)k * (uintptr_t)elem_bytes(type), of};
    };
    for (int64_t i = 0; i < n; ++i)
        if (t[i].n > 0) out.push_back(range(t[i].out ? t[i].out : t[i].grad, t[i].n, t[i].out ? t[i].out_type : t[i].type, i));
    std::sort(out.begin(), out.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
    for (size_t i = 1; i < out.size(); ++i)
        if (out[i].lo < out[i - 1].hi) return false;
    for (int64_t i = 0; i < n; ++i) {
        if (t[i].n == 0) continue;
        const Range g = range(t[i].grad, t[i].n, t[i].type, i);
        // outputs lie apart and in order: those that meet g are the last that begins at or before it, and those that begin within
        auto o = std::upper_bound(out.begin(), out.end(), g.lo, [](uintptr_t a, const Range& b) { return a < b.lo; });
        if (o != out.begin()) --o;
        for (; o != out.end() && o->lo < g.hi; ++o)
            if (o->hi > g.lo && !(o->of == i && o->lo == g.lo && o->hi == g.hi)) return false;
    }
    return true;
}

inline const char* tensors_check(const sa3k_tensor* t, int64_t n, int* code) {
    *code = SA3K_ERR_INVALID;
    if (n < 0 || n > ((int64_t)1 << 24)) return "the number of tensors is out of range";
    if (n > 0 && !t) return "null list";
    for (int64_t i = 0; i < n; ++i) {
        const sa3k_tensor& x = t[i];
        if (!grad_type(x.type) || !grad_type(x.out_type)) {
            *code = SA3K_ERR_UNSUPPORTED;
            return "types must be f32, f16 or bf16";
        }
        if (x.out_type != x.type && x.out_type != SA3K_TYPE_F32) {
            *code = SA3K_ERR_UNSUPPORTED;
            return "out_type must be f32 or type";
        }
        if (x.n < 0 || x.n >= kTensorMost) return "a tensor's number of elements is out of range";
        if (x.n > 0 && !x.grad) return "a gradient is null";
        if (!elem_aligned(x.grad, elem_bytes(x.type)) || !elem_aligned(x.out, elem_bytes(x.out_type)))
            return "a tensor is not aligned to its elements";
        if ((!x.out || x.out == x.grad) && x.out_type != x.type) return "a gradient written in place keeps its type";
    }
    if (!outputs_apart(t, n)) return "an output meets another tensor, or its own gradient but in place";
    return nullptr;
}
inline const char* clip_check(int count, float max_norm, const void* stat, int* code) {
    *code = SA3K_ERR_INVALID;
    if (count <= 0) return "cannot apply empty gradient batch";
    if (max_norm != max_norm) return "the largest norm must be a number";
    if (!elem_aligned(stat, 8)) return "the norm's place is not 8-byte aligned";
    return nullptr;
}

// A piece of a tensor: what a workgroup reads at a time. kind: 2 bits of the gradient's type (0 f32, 1 f16, 2 bf16), bit 2: the
// output is f32 all the same.
struct TensorPiece {
    const void* grad;
    void* out;
    int32_t n, kind;
};
// Bytes of a piece: eight loads of 16 bytes for each of 256 threads. (A tensor's last piece is shorter, so a list of many small
// tensors has as many pieces as tensors.)
constexpr int kPieceBytes = 32768;

inline int piece_kind(const sa3k_tensor& t) {
    const int k = t.type == SA3K_TYPE_F32 ? 0 : t.type == SA3K_TYPE_F16 ? 1 : 2;
    return k | (t.out_type == SA3K_TYPE_F32 ? 4 : 0);
}
inline std::vector<TensorPiece> tensor_pieces(const sa3k_tensor* t, int64_t n) {
    std::vector<TensorPiece> p;
    for (int64_t i = 0; i < n; ++i) {
        const char* g = static_cast<const char*>(t[i].grad);
        char* o = static_cast<char*>(t[i].out ? t[i].out : const_cast<void*>(t[i].grad));
        const int64_t most = kPieceBytes / elem_bytes(t[i].type);
        for (int64_t at = 0; at < t[i].n; at += most) {
            const int64_t left = t[i].n - at;
            p.push_back(TensorPiece{g + at * elem_bytes(t[i].type), o + at * elem_bytes(t[i].out_type),
                                    (int32_t)(left < most ? left : most), piece_kind(t[i])});
        }
    }
    return p;
}

}  // namespace sa3k
