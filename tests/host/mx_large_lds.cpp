// Every scale that the large packed tile (csrc/mx_gemm.hip) reads from LDS, for all lengths of its rows: inside the memory it
// asks for, and where it is used, the byte that the request for its window put there.
#include <cstdio>

#include "../../nerf-pytorch_amd/csrc/mx_large.h"

using L = mxk::LargeLds;

int main() {
    int farthest = 0;
    for (int steps = 4; steps <= 64; ++steps) {
        const int stages = (steps + 1) / 2;
        for (int d = 0; d <= stages; ++d)          // the kernel reads one stage ahead, behind the last one too
            for (int row = 0; row < L::ROWS; ++row)
                for (int q = 0; q < 4; ++q) {
                    const int at = L::scale_place(row, q) + L::scales_of(steps, d);
                    if (at + 2 > farthest) farthest = at + 2;
                    if (at < 2 * L::STAGE || at + 2 > L::bytes(true)) {
                        printf("steps %d stage %d row %d group %d reads byte %d of %d\n", steps, d, row, q, at, L::bytes(true));
                        return 1;
                    }
                    // lane group q of stage d multiplies blocks 8 d + 2 q and 8 d + 2 q + 1 of its row
                    const int block = 8 * d + 2 * q;
                    if (d == stages || block >= 4 * steps) continue;
                    const int window = d / 2 * 16, end = 4 * steps - 16, first = window < end ? window : end;
                    const int want = 2 * L::STAGE + (d / 2 % 2) * L::SCALES + row * 16 + (block - first);
                    if (at != want || block - first > 14) {
                        printf("steps %d stage %d row %d group %d reads byte %d instead of %d\n", steps, d, row, q, at, want);
                        return 2;
                    }
                }
    }
    printf("farthest %d of %d\n", farthest, L::bytes(true));
    return 0;
}
