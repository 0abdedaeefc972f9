// Layers of up to 256 inputs and outputs over many rows -- the hidden layers of a NeRF, where a row is a sample: bound by the
// rows' bytes, so each pass reads and writes them once.
//
// Forward: W stays in LDS; a wave takes 16 rows of x, rounds them in registers, multiplies and finishes one output tile after
// the other; the next rows are requested before the products.  No barrier in the loop.  262144 x 256 -> 256 fp32: one launch
// that reads x and writes y, 109 us = 4.9 TB/s (ReLU), against a rounding pass (75 us) and a product (84 us); four waves per
// SIMD in workgroups of eight that share W, three in workgroups of four took 121 us.
#include "mx_narrow.h"

namespace mxk {
namespace {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// eight lanes (half a DPP row) hold a block: four values each
__device__ __forceinline__ unsigned max8(unsigned m) {
    m = quad_max(m);
    const unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true);   // lane i of eight <- lane 7 - i
    return o > m ? o : m;
}
__device__ __forceinline__ i32x8 wide8(i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

constexpr int XPITCH(int steps) { return steps * 64 + 16; }   // LDS rows of codes: 16 bytes of padding spread them over the banks

// STEPS: K <= 128 STEPS.  A row of x is 32 STEPS lanes of four values; lane group q takes blocks STEPS q .. of a row.
template <typename T, int ACT, int STEPS>
__global__ __launch_bounds__(512, 4) void mx_narrow_fwd_kernel(NarrowFwd a) {
    constexpr int LANES = 32 * STEPS, RPL = 64 / LANES, LOADS = 16 / RPL;   // lanes of a row, rows and requests
    typedef T x4 __attribute__((ext_vector_type(4)));
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int ntiles = (a.N + 15) / 16;
    uint8_t* wl = smem;                                             // [n][16-byte pieces, swapped by row]
    uint8_t* wsl = wl + 256 * 64 * STEPS;                           // [n][4 STEPS]
    float* bl = reinterpret_cast<float*>(wsl + 256 * 4 * STEPS);    // [n]
    uint8_t* xl = reinterpret_cast<uint8_t*>(bl + 256) + wave * (16 * XPITCH(STEPS) + 64 * STEPS);
    uint8_t* xsl = xl + 16 * XPITCH(STEPS);                         // [row][4 STEPS]

    constexpr int PIECES = 4 * STEPS;
    for (int i = tid; i < ntiles * 16 * PIECES; i += 512) {
        const int row = i / PIECES, c = i % PIECES;
        const i32x4 v = row < a.N ? reinterpret_cast<const i32x4*>(a.wc)[i] : i32x4{0, 0, 0, 0};
        *reinterpret_cast<i32x4*>(wl + row * (64 * STEPS) + ((c ^ (row & (PIECES - 1))) * 16)) = v;
        wsl[i] = row < a.N ? a.ws[i] : 0;
    }
    if (tid < 256) bl[tid] = a.f.bias && tid < a.N ? (float)((const T*)a.f.bias)[tid] : 0.0f;
    __syncthreads();

    const int k = (lane % LANES) * 4, lrow = lane / LANES;
    const int64_t tiles = (a.M + 15) / 16, stride = (int64_t)gridDim.x * 8;
    x4 v[LOADS];
    auto request = [&](int64_t tile) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int64_t m = tile * 16 + i * RPL + lrow;
            v[i] = x4{};
            if (tile < tiles && m < a.M) {
                const T* p = (const T*)a.x + m * a.ldx + k;
                if (a.vec) {
                    // vec: K is a multiple of four.  Non-temporal, x passes through once: 131 -> 121 us (ReLU); such stores of
                    // y, whose rows leave 64 bytes at a time, were slower (143 us).
                    if (k < a.K) v[i] = __builtin_nontemporal_load(reinterpret_cast<const x4*>(p));
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (k + j < a.K) v[i][j] = p[j];
                }
            }
        }
    };
    int64_t tile = (int64_t)blockIdx.x * 8 + wave;
    request(tile);
    for (; tile < tiles; tile += stride) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            unsigned m = 0;
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[j] = (float)v[i][j];
                const unsigned b = __builtin_bit_cast(unsigned, f[j]) & 0x7fffffffu;
                m = b > m ? b : m;
            }
            const unsigned s = scale_byte(max8(m));
            const float sc = scale_arg(s);
            unsigned c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[0], f[1], sc, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], sc, 1);
            c = s == 255u ? 0u : c;
            const int row = i * RPL + lrow;
            *reinterpret_cast<uint16_t*>(xl + row * XPITCH(STEPS) + k / 2) = (uint16_t)c;
            if (lane % 8 == 0) xsl[row * (4 * STEPS) + k / 32] = (uint8_t)s;
        }
        asm volatile("" ::: "memory");      // one wave: LDS answers in order, the compiler has to ask in order
        __builtin_amdgcn_wave_barrier();
        i32x4 xf[STEPS];
#pragma unroll
        for (int h = 0; h < STEPS; ++h) xf[h] = *reinterpret_cast<const i32x4*>(xl + r * XPITCH(STEPS) + (STEPS * q + h) * 16);
        const int xs = STEPS == 2 ? *reinterpret_cast<const uint16_t*>(xsl + r * 8 + 2 * q) : xsl[r * 4 + q];
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        const int64_t m = tile * 16 + r;
        const bool ok = m < a.M;
        if (a.xc && ok) {
#pragma unroll
            for (int h = 0; h < STEPS; ++h)
                *reinterpret_cast<i32x4*>(a.xc + m * (64 * STEPS) + (STEPS * q + h) * 16) = xf[h];
            if constexpr (STEPS == 2) *reinterpret_cast<uint16_t*>(a.xs + m * 8 + 2 * q) = (uint16_t)xs;
            else a.xs[m * 4 + q] = (uint8_t)xs;
        }
        request(tile + stride);
        constexpr int U = ACT == NERF_ACT_SIN || ACT == NERF_ACT_SIGMOID ? 2 : 4;
#pragma unroll U
        for (int t = 0; t < ntiles; ++t) {
            const int row = t * 16 + r, n = t * 16 + q * 4;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            const int ws = STEPS == 2 ? *reinterpret_cast<const uint16_t*>(wsl + row * 8 + 2 * q) : wsl[row * 4 + q];
            const uint8_t* w = wl + row * (64 * STEPS);
            const i32x4 w0 = *reinterpret_cast<const i32x4*>(w + (((STEPS * q) ^ (row & (PIECES - 1))) * 16));
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide8(w0), wide8(xf[0]), acc, 4, 4, 0, ws, 0, xs);
            if constexpr (STEPS == 2) {
                const i32x4 w1 = *reinterpret_cast<const i32x4*>(w + (((STEPS * q + 1) ^ (row & (PIECES - 1))) * 16));
                acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide8(w1), wide8(xf[1]), acc, 4, 4, 1, ws, 1, xs);
            }
            const f32x4 bias = *reinterpret_cast<const f32x4*>(bl + n);
            finish4<T, ACT, true>(a.f, acc, m, n, a.N, ok, bias, a.whole && n + 4 <= a.N);
        }
    }
}

template <typename T, int ACT, int STEPS>
int launch_fwd(const char* fn, const NarrowFwd& a, hipStream_t st) {
    constexpr int lds = 256 * 68 * STEPS + 1024 + 8 * (16 * XPITCH(STEPS) + 64 * STEPS);
    const int64_t groups = (a.M + 127) / 128;
    const unsigned grid = (unsigned)(groups < 512 ? groups : 512);      // two workgroups of eight waves on each of 256 compute units
    mx_narrow_fwd_kernel<T, ACT, STEPS><<<grid, 512, lds, st>>>(a);
    return nerf_check_launch(fn);
}
template <typename T, int ACT>
int by_steps(const char* fn, const NarrowFwd& a, hipStream_t st) {
    return a.K > 128 ? launch_fwd<T, ACT, 2>(fn, a, st) : launch_fwd<T, ACT, 1>(fn, a, st);
}
template <typename T>
int by_act(const char* fn, NarrowFwd a, int act, hipStream_t st) {
    a.vec = a.K % 4 == 0 && (uintptr_t)a.x % (4 * sizeof(T)) == 0 && a.ldx * sizeof(T) % (4 * sizeof(T)) == 0;
    a.whole = (uintptr_t)a.f.out % (4 * sizeof(T)) == 0 && a.f.ldo * sizeof(T) % (4 * sizeof(T)) == 0;
    if (act == NERF_ACT_NONE) return by_steps<T, NERF_ACT_NONE>(fn, a, st);
    if (act == NERF_ACT_RELU) return by_steps<T, NERF_ACT_RELU>(fn, a, st);
    if (act == NERF_ACT_SIN) return by_steps<T, NERF_ACT_SIN>(fn, a, st);
    return by_steps<T, NERF_ACT_SIGMOID>(fn, a, st);
}

}  // namespace

int launch_narrow_fwd(const char* fn, const NarrowFwd& a, int dtype, int act, hipStream_t st) {
    if (dtype == NERF_F32) return by_act<float>(fn, a, act, st);
    if (dtype == NERF_BF16) return by_act<__bf16>(fn, a, act, st);
    return by_act<_Float16>(fn, a, act, st);
}

}  // namespace mxk
