// Layers of up to 256 inputs and outputs over many rows (mx_narrow.hip).
#pragma once
#include "mx_finish.h"

namespace mxk {

constexpr int kNarrow = 256;            // inputs and outputs
constexpr int64_t kNarrowRows = 4096;   // from here on the rows' bytes count, not the launches

struct NarrowFwd {
    const void* x;
    int64_t ldx, M;
    int K, N;
    const uint8_t *wc, *ws;
    uint8_t *xc, *xs;       // the rounded x for the backward pass, or NULL
    bool vec, whole;        // four values of x, of y at a time (set by the launch)
    Finish f;
};
int launch_narrow_fwd(const char* fn, const NarrowFwd& a, int dtype, int act, hipStream_t st);

}  // namespace mxk
