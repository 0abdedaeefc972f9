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
    Finish f;
};
int launch_narrow_fwd(const char* fn, const NarrowFwd& a, int dtype, int act, hipStream_t st);

struct NarrowBwd {
    const void* dy;
    int64_t lddy;
    const float* slope;     // [M][N], or NULL
    const uint16_t* mask;   // [M][ceil(N / 16)], or NULL
    float factor;
    const uint8_t *xc, *xs, *wc, *ws;
    int64_t M;
    int K, N;
    void* dx;               // each NULL to skip
    int64_t lddx;
    void* dw;
    float* slab;            // dw: [groups][C][C], C = 128 or 256
    float* colsum;          // [groups][N], or NULL
};
// workgroups of the backward kernel: 32 rows at a time, four times at least
static inline int narrow_groups(int64_t M) {
    const int64_t g = (M + 127) / 128;
    return g < 256 ? (int)g : 256;
}
static inline int narrow_columns(int64_t K, int64_t N) { return K > 128 || N > 128 ? 256 : 128; }
// what the kernel's loads of whole 16-byte pieces ask of the layout
static inline bool narrow_bwd_ok(const void* dy, int64_t lddy, int size, int64_t M, int64_t K, int64_t N, bool slope) {
    return M >= kNarrowRows && K <= kNarrow && N <= kNarrow && (uintptr_t)dy % 16 == 0 && lddy * size % 16 == 0 && N * size % 16 == 0 &&
           (!slope || N % 4 == 0) && lddy <= (1 << 20);
}
int launch_narrow_bwd(const char* fn, const NarrowBwd& a, int dtype, hipStream_t st);

}  // namespace mxk
