// Where the large tile of mx_gemm.hip keeps what it has staged in LDS.  Plain arithmetic, so that a host program can follow
// every read (tests/host/mx_large_lds.cpp).
#pragma once

namespace mxk {

struct LargeLds {
    static constexpr int ROWS = 512;              // the tile's 256 rows of W, then its 256 of X
    static constexpr int STAGE = ROWS * 128;      // two of them
    static constexpr int SCALES = ROWS * 16;      // two windows of scales, of two stages each, behind the stages (packed rows)
    // A lane reads two scale bytes at its fixed place whatever its stage is.  Behind the last stage, and for the half of it
    // that does not exist where the steps are odd, that place lies up to twelve bytes behind the row's sixteen: what is read
    // there is not used, but the last row's has to lie in LDS as well.
    static constexpr int SPARE = 16;

    static constexpr int bytes(bool packed) { return 2 * STAGE + (packed ? 2 * SCALES + SPARE : 0); }
    // the two scale bytes of lane group q in row `row` of the first window
    static constexpr int scale_place(int row, int q) { return 2 * STAGE + row * 16 + 2 * q; }
    // where stage d's scales lie from there: their window, and inside it (moved back by what the last window was)
    static constexpr int scales_of(int steps, int d) {
        const int window = (d >> 1) * 16, end = steps * 4 - 16;
        return (d >> 1 & 1) * SCALES + (d & 1) * 8 + (window > end ? window - end : 0);
    }
};

}  // namespace mxk
