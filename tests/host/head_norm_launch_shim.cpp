// The head norms' angles and the heads a wave takes (csrc/head_norm.h) for the CPU tests.
#include "head_norm.h"

using namespace sa3k;

extern "C" {

void turns(int dims, float base, uint64_t* out) { head_turns(dims, base, out); }
int parts(int heads, int dim) { return head_parts(heads, dim); }
int lanes(int dim) { return head_lanes(dim); }
int groups() { return kGroups; }

}  // extern "C"
