// Products with few rows: y = post * f(pre * (Q(x) W^T + b)) for up to 64 rows of x, W packed.
//
// Bound by W's bytes: every code is read once, by the one wave that multiplies it, straight into registers.  A workgroup
// owns 16 rows of W; its waves share the reduction, 512 values at a time (a chunk), and join their sums in LDS in the
// order of the waves.  Four steps of the 16x16x128 instruction make a chunk, and which blocks a step takes is free as long as
// both operands agree: lane group q takes blocks 4q .. 4q+3 of the sixteen, one after the other.  A lane then reads 64
// neighbouring bytes of a row per chunk, 256 per row and wave, and the four scale bytes it needs are one word, out of which
// the instruction picks its byte.
//
// FUSED: the rows of x are rounded here, by every workgroup, into LDS while the first codes of W are under way -- for a few
// rows that costs less than a launch of its own (4096 x 4096, one bf16 row: 4.6 us against 5.9).
#include "mx_finish.h"

namespace mxk {
namespace {

constexpr int kAhead = 4;      // chunks of W a wave has under way

struct WFrag {
    i32x4 c[4];
    int s;
};

// the 64 bytes of codes and the scale word of lane group q in chunk `chunk` of a row; nothing behind the row's last step
__device__ __forceinline__ void load_chunk(WFrag& f, const uint8_t* codes, const uint8_t* scales, int chunk, int q, int steps) {
    const bool in = chunk * 4 + q < steps;
    const i32x4* p = reinterpret_cast<const i32x4*>(codes + (int64_t)(chunk * 4 + q) * 64);
#pragma unroll
    for (int h = 0; h < 4; ++h) f.c[h] = in ? p[h] : i32x4{0, 0, 0, 0};
    f.s = in ? *reinterpret_cast<const int*>(scales + (int64_t)(chunk * 4 + q) * 4) : 0;
}

__device__ __forceinline__ i32x8 wide8(i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }
template <int H>
__device__ __forceinline__ f32x4 step(const WFrag& w, const WFrag& x, f32x4 acc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide8(w.c[H]), wide8(x.c[H]), acc, 4, 4, H, w.s, H, x.s);
}

template <typename T, int ACT, int MT, bool FUSED>
__global__ __launch_bounds__(MT == 1 ? 1024 : 512) void mx_few_kernel(FewArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6, r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int chunks = (a.steps + 3) / 4;
    const int64_t cp = a.steps * 64ll, sp = a.steps * 4ll;
    const int64_t row = n0 + r < a.N ? n0 + r : a.N - 1;    // rows behind the last one repeat it (never stored)
    const uint8_t *wc = a.wc + row * cp, *ws = a.ws + row * sp;

    WFrag w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load_chunk(w[i], wc, ws, wave + i * waves, q, a.steps);

    const uint8_t *xc = a.xc, *xs = a.xs;
    if constexpr (FUSED) {
        uint8_t* lc = smem;
        uint8_t* ls = smem + a.M * cp;
        const int groups = a.steps * 16;        // of eight values, per row
        for (int i = threadIdx.x; i < a.M * groups; i += blockDim.x) {    // whole quads: groups is a multiple of 16
            const int m = i / groups, k = (i - m * groups) * 8;
            const T* p = (const T*)a.x + m * a.ldx + k;
            float v[8];
            if (k + 8 <= a.K) load8(p, v);
            else load8_tail(p, (int64_t)a.K - k, v);
            const unsigned s = scale_byte(quad_max(amax8(v)));
            reinterpret_cast<unsigned*>(lc)[i] = encode8(v, s);
            if ((threadIdx.x & 3) == 0) ls[i >> 2] = (uint8_t)s;
        }
        __syncthreads();
        xc = lc;
        xs = ls;
    }

    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c0 = wave; c0 < chunks; c0 += kAhead * waves) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int c = c0 + i * waves;
            if (c >= chunks) break;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int m = t * 16 + r < a.M ? t * 16 + r : a.M - 1;
                WFrag x;
                load_chunk(x, xc + m * cp, xs + m * sp, c, q, a.steps);
                acc[t] = step<0>(w[i], x, acc[t]);
                acc[t] = step<1>(w[i], x, acc[t]);
                acc[t] = step<2>(w[i], x, acc[t]);
                acc[t] = step<3>(w[i], x, acc[t]);
            }
            if (c + kAhead * waves < chunks) load_chunk(w[i], wc, ws, c + kAhead * waves, q, a.steps);
        }
    }

    // sums of the waves, [wave][m][n]: lane holds n = 4q .. 4q+3 of row m = r
    if constexpr (FUSED) __syncthreads();     // everybody has read its x
    f32x4* part = reinterpret_cast<f32x4*>(smem);
#pragma unroll
    for (int t = 0; t < MT; ++t) part[(wave * MT + t) * 64 + r * 4 + q] = acc[t];
    __syncthreads();
    if ((int)threadIdx.x < MT * 64) {
        const int m = threadIdx.x >> 2, n = n0 + (threadIdx.x & 3) * 4;
        f32x4 v = part[threadIdx.x];
        for (int i = 1; i < waves; ++i) v += part[i * MT * 64 + threadIdx.x];
        finish4<T, ACT, false>(a.f, v, m, n, a.N, m < a.M, load_bias<T>(a.f.bias, n, a.N));
    }
}

template <typename T, int ACT, int MT>
int launch(const char* fn, const FewArgs& a, hipStream_t st) {
    const int chunks = (a.steps + 3) / 4;
    // one chunk per wave where there are that many, in whole SIMDs; the last step needs a thread per four outputs
    const int waves = chunks >= 12 && MT == 1 ? 16 : chunks >= 6 ? 8 : 4;
    const unsigned grid = (unsigned)((a.N + 15) / 16);
    size_t lds = (size_t)waves * MT * 1024;
    if (a.x) {
        const size_t x = (size_t)a.M * a.steps * 68;
        lds = x > lds ? x : lds;
        mx_few_kernel<T, ACT, MT, true><<<grid, waves * 64, lds, st>>>(a);
    } else {
        mx_few_kernel<T, ACT, MT, false><<<grid, waves * 64, lds, st>>>(a);
    }
    return nerf_check_launch(fn);
}

template <typename T, int ACT>
int by_rows(const char* fn, const FewArgs& a, hipStream_t st) {
    if (a.M <= 16) return launch<T, ACT, 1>(fn, a, st);
    if (a.M <= 32) return launch<T, ACT, 2>(fn, a, st);
    return launch<T, ACT, 4>(fn, a, st);
}

template <typename T>
int by_act(const char* fn, const FewArgs& a, int act, hipStream_t st) {
    if (act == NERF_ACT_NONE) return by_rows<T, NERF_ACT_NONE>(fn, a, st);
    if (act == NERF_ACT_RELU) return by_rows<T, NERF_ACT_RELU>(fn, a, st);
    if (act == NERF_ACT_SIN) return by_rows<T, NERF_ACT_SIN>(fn, a, st);
    return by_rows<T, NERF_ACT_SIGMOID>(fn, a, st);
}

}  // namespace

int launch_few(const char* fn, const FewArgs& a, int dtype, int act, hipStream_t st) {
    if (dtype == NERF_F32) return by_act<float>(fn, a, act, st);
    if (dtype == NERF_BF16) return by_act<__bf16>(fn, a, act, st);
    return by_act<_Float16>(fn, a, act, st);
}

}  // namespace mxk
