// How the sums of the MXFP4 products leave: bias, activation, what the backward pass needs, type (mx_gemm.hip, mx_few.hip).
#pragma once
#include "mx_common.h"
#include "sincos.h"

namespace mxk {

// What happens to a sum on its way out.  slab != NULL: fp32 partial sums [split][M][N], finished by mx_finish_kernel.
struct Finish {
    void* out;
    int64_t ldo;
    const void* bias;       // type of out, or NULL
    float pre, post;
    float* slope;           // sin, sigmoid: d y / d z [M][N] for the gradient, or NULL
    uint16_t* mask;         // relu: decisions [M][ceil(N / 16)], or NULL
    float* slab;
};

template <int ACT>
__device__ __forceinline__ void activate(float z, const Finish& f, float& y, float& slope) {
    if constexpr (ACT == NERF_ACT_NONE) {
        y = f.post * f.pre * z;
        slope = 0.0f;
    } else if constexpr (ACT == NERF_ACT_RELU) {
        const float t = f.pre * z;
        y = f.post * (t <= 0.0f ? 0.0f : t);   // a NaN stays one
        slope = t > 0.0f ? 1.0f : 0.0f;
    } else {
        static_assert(ACT == NERF_ACT_SIGMOID, "");
        // exp(-|t|) cannot overflow, and 1 - s would cancel: s and 1 - s are both formed from it
        const float t = f.pre * z, e = expf(-fabsf(t)), r = 1.0f / (1.0f + e);
        const float s = t >= 0.0f ? r : e * r;
        y = f.post * (t != t ? t : s);
        slope = f.post * f.pre * r * (e * r);
    }
}

// Sines and cosines of four values.  The library's path for large arguments stands once, outside of the four, for the waves
// that need it: inlined behind each of the four it filled the registers (training forward 262144 x 256 -> 256 fp32 213 -> 196 us).
__device__ __forceinline__ void sincos4(const f32x4& t, f32x4& sn, f32x4& cs) {
    bool near = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) near = near && fabsf(t[i]) <= 1.0e5f;     // a NaN is not
    if (__all(near)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a, b;
            nerf_sincosf_bounded(t[i], &a, &b);
            sn[i] = a;
            cs[i] = b;
        }
    } else {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            float a, b;
            nerf_sincosf(i == 0 ? t[0] : i == 1 ? t[1] : i == 2 ? t[2] : t[3], &a, &b);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sn[j] = i == j ? a : sn[j];
                cs[j] = i == j ? b : cs[j];
            }
        }
    }
}

// Four neighbouring outputs of one row (n .. n+3, those below N).  The four lanes that hold
// sixteen neighbours of one row are a quad, or (ACROSS) sixteen lanes apart.
template <typename T, int ACT, bool ACROSS>
__device__ __forceinline__ void finish4(const Finish& f, f32x4 acc, int64_t m, int n, int N, bool row_ok, const f32x4& bias) {
    f32x4 y = {}, sl = {};
    if constexpr (ACT == NERF_ACT_SIN) {
        f32x4 t;
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = f.pre * (acc[i] + bias[i]);
        sincos4(t, y, sl);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] *= f.post;
            sl[i] *= f.post * f.pre;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a, b;
            activate<ACT>(acc[i] + bias[i], f, a, b);
            y[i] = a;
            sl[i] = b;
        }
    }
    if constexpr (ACT == NERF_ACT_RELU) {
        if (f.mask) {   // uniform
            unsigned bits = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) bits |= (sl[i] > 0.0f && n + i < N ? 1u : 0u) << i;
            bits <<= 4 * (n / 4 & 3);
            if constexpr (ACROSS) {
                bits |= __shfl_xor(bits, 16);
                bits |= __shfl_xor(bits, 32);
            } else {
                bits = quad_or(bits);
            }
            if (n % 16 == 0 && row_ok && n < N) f.mask[m * ((N + 15) / 16) + n / 16] = (uint16_t)bits;
        }
    }
    if (!row_ok) return;
    T* o = (T*)f.out + m * f.ldo + n;
    typedef typename Loose<T, 4>::type x4;
    x4 t;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = (T)y[i];
    if (n + 4 <= N) {
        *reinterpret_cast<x4*>(o) = t;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < N) o[i] = t[i];
    }
    if constexpr (ACT == NERF_ACT_SIN || ACT == NERF_ACT_SIGMOID) {
        if (f.slope) {
            float* s = f.slope + m * N + n;
            if (n + 4 <= N) {
                *reinterpret_cast<typename Loose<float, 4>::type*>(s) = sl;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < N) s[i] = sl[i];
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ f32x4 load_bias(const void* bias, int n, int N) {
    f32x4 b = {0.f, 0.f, 0.f, 0.f};
    if (bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < N) b[i] = (float)((const T*)bias)[n + i];
    }
    return b;
}

// A value as bf16 terms, v = t0 + t1 + ..: each the rounding of what the previous ones left.
template <int TERMS>
__device__ __forceinline__ void split_terms(float v, __bf16 (&t)[TERMS]) {
    const float top = __builtin_bit_cast(float, 0x7f7f0000u);   // largest bf16: fp32 values above it would round to infinity
    const bool finite = fabsf(v) < __builtin_inff();
    t[0] = (__bf16)(finite ? fminf(fmaxf(v, -top), top) : v);
#pragma unroll
    for (int i = 1; i < TERMS; ++i) {
        v = finite ? v - (float)t[i - 1] : 0.0f;                // exact
        t[i] = (__bf16)v;
    }
}

// Products with few rows (mx_few.hip).  x != NULL: rounded in the kernel (few_fused() says whether that is the way), else
// xc / xs hold it packed.
struct FewArgs {
    const uint8_t *wc, *ws;
    const void* x;
    int64_t ldx;
    const uint8_t *xc, *xs;
    int M, K, N;
    int steps;              // of 128 values
    Finish f;
};
constexpr int kFewRows = 64;
// Rows up to which a workgroup per sixteen columns, which reads x from the L2 each time, beats the tiles, which share it:
// sixteen (one tile row), or by what the workgroups read of x together and what a workgroup of the split product has to
// join.  Against the tiles, us, K -> N: 4096 -> 4096 with 64 rows 10.4 : 12.0; 8192 -> 4096 with 32 11.7 : 12.6, with 48 15.2 : 13.3; 8192 -> 8192 with 16
// 15.9 : 17.3, with 24 18.2 : 17.6, with 64 29.7 : 19.0; 1024 -> 16384 with 8 6.2 : 6.8, with 64 11.4 : 7.9.
static inline bool few_rows(int64_t M, int64_t K, int64_t N) {
    return M <= 16 || (M <= kFewRows && M * (K > N ? K : N) <= 1 << 18 && M * K * N <= 1 << 30);
}
// One launch for both where every workgroup's rounding of x is short; a row has a cost of its own.  Against two launches,
// us: 4096 -> 4096 with 1 row 4.6 : 5.9, with 4 5.7 : 6.2; 256 -> 256 with 24 4.3 : 5.1, with 64 6.3 : 5.6; 1024 -> 4096
// with 8 4.5 : 5.2, with 16 5.9 : 5.4.
static inline bool few_fused(int64_t M, int64_t K) { return M * (K + 512) <= 18432; }
int launch_few(const char* fn, const FewArgs& a, int dtype, int act, hipStream_t st);

}  // namespace mxk
