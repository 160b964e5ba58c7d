// The tensor lists' checks and pieces (csrc/tensors.h) for the CPU tests.
#include "tensors.h"

using namespace sa3k;

extern "C" {

int tensors(const sa3k_tensor* t, int64_t n) {
    int code = -1;
    return tensors_check(t, n, &code) ? code : 0;
}
int clip(int count, float most, int64_t stat) {
    int code = -1;
    return clip_check(count, most, reinterpret_cast<const void*>((uintptr_t)stat), &code) ? code : 0;
}
// gradient, output, elements and kind of each piece, at most `most` of them
int64_t pieces(const sa3k_tensor* t, int64_t n, int64_t* out, int64_t most) {
    const std::vector<TensorPiece> p = tensor_pieces(t, n);
    for (size_t i = 0; i < p.size() && (int64_t)i < most; ++i) {
        out[4 * i] = (int64_t)(uintptr_t)p[i].grad;
        out[4 * i + 1] = (int64_t)(uintptr_t)p[i].out;
        out[4 * i + 2] = p[i].n;
        out[4 * i + 3] = p[i].kind;
    }
    return (int64_t)p.size();
}

}  // extern "C"
