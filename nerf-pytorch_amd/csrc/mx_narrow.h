// Layers of up to 256 inputs and outputs over many rows (mx_narrow.hip).
#pragma once
#include "mx_finish.h"

namespace mxk {

constexpr int kNarrow = 256;            // inputs and outputs
// Rows from which the fixed cost (weights read back, partial sums) is less than the bytes and launches that are saved.
// Against the general way, us: forward 256 -> 256 relu fp32 with 8192 rows 11.3 : 8.1, 16384 13.3 : 14.1; sin fp32 with 12288
// 16.2 : 10.7, 16384 16.7 : 17.2, 32768 21.4 : 22.5; 64 -> 64 sin fp32 with 32768 8.6 : 15.5.  Backward 256 -> 256 sin fp32 with
// 4096 39.9 : 40.1, 8192 44.4 : 48.6, 32768 57 : 117, relu bf16 with 4096 31.0 : 28.3, 8192 36.0 : 35.3, 32768 47 : 63; 64 -> 64
// sin fp32 with 4096 18.0 : 23.2.  The borders are those of 256 columns; narrower layers cross earlier, as the figures of 64 show,
// and take the general way for longer than they need.
constexpr int64_t kNarrowRowsFwd = 16384, kNarrowRowsBwd = 4096;

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
static inline int narrow_columns(int64_t K, int64_t N) { return K > 128 || N > 128 ? 256 : 128; }
// workgroups of the backward kernel: 32 rows at a time, four times at least; one fits a compute unit, or two of 128 columns
// (131072 x 128 x 128 fp32 sin 45 -> 41 us, and one more for the sums)
static inline int narrow_groups(int64_t M, int columns) {
    const int64_t g = (M + 127) / 128, most = columns == 256 ? 256 : 512;
    return (int)(g < most ? g : most);
}
// what the kernel's loads of whole 16-byte pieces ask of the layout
static inline bool narrow_bwd_ok(const void* dy, int64_t lddy, int size, int64_t M, int64_t K, int64_t N, const float* slope) {
    return M >= kNarrowRowsBwd && K <= kNarrow && N <= kNarrow && (uintptr_t)dy % 16 == 0 && lddy * size % 16 == 0 && N * size % 16 == 0 &&
           (!slope || (N % 4 == 0 && (uintptr_t)slope % 16 == 0)) && lddy <= (1 << 20);
}
int launch_narrow_bwd(const char* fn, const NarrowBwd& a, int dtype, hipStream_t st);

}  // namespace mxk
