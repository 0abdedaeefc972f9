// Shared pieces of the microscaled 4-bit (MXFP4) operators: mx.hip (quantise, read back), mx_few.hip (products with few rows),
// mx_narrow.hip (narrow layers over many rows, forward and backward), mx_gemm.hip (tiled products, the other gradients).
//
// The format.  A row is cut into blocks of 32 values.  A block holds one scale byte s, standing for 2^(s - 127), and 32
// codes of 4 bits (sign, two exponent bits, one mantissa bit): 0 .5 1 1.5 2 3 4 6.  With E the biased fp32 exponent
// field of the block's largest magnitude, s = max(E - 2, 0), so that the largest value lands in [4, 8) -- the code 6 is
// the last one, values above it saturate -- and every code is x / 2^(s - 127) rounded to nearest, ties to even.  A block
// that holds a NaN or an infinity gets s = 255 and codes 0: it stands for NaN as a whole, here and in the matrix pipe.
// Packed rows are padded to 128 values with zeros (64 bytes of codes, four of scales; low nibble = even index): one
// 16x16x128 matrix instruction reads 64 bytes of a row, 16 of them -- one block -- per lane.
#pragma once
#include "common.h"

#include <utility>

namespace mxk {

// f(integral_constant<int, 0>) ... f(integral_constant<int, N-1>)
template <int... I, typename F>
__device__ __forceinline__ void unrolled_impl(std::integer_sequence<int, I...>, F&& f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
    unrolled_impl(std::make_integer_sequence<int, N>{}, f);
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// bytes of a packed row
__host__ __device__ inline int64_t code_pitch(int64_t K) { return (K + 127) / 128 * 64; }
__host__ __device__ inline int64_t scale_pitch(int64_t K) { return (K + 127) / 128 * 4; }

// scale byte of a block from the largest magnitude's fp32 bits.  The magnitudes are compared as integers: the order of
// non-negative floats, with NaN above infinity, so neither can be lost (a float maximum would drop a NaN).
__device__ __forceinline__ unsigned scale_byte(unsigned amax_bits) {
    const unsigned e = amax_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// The conversion instructions take the scale as a float and use its exponent field alone: s << 23, also for s = 0
// (2^-127, which as a float would be a subnormal) and s = 255 (NaN on reading back).
__device__ __forceinline__ float scale_arg(unsigned s) { return __builtin_bit_cast(float, s << 23); }

// eight values -> eight codes
__device__ __forceinline__ unsigned encode8(const float (&v)[8], unsigned s) {
    const float sc = scale_arg(s);
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], sc, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], sc, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], sc, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], sc, 3);
    return s == 255u ? 0u : c;
}

// eight codes -> eight values, rounded once to T (exact in fp32 and bf16)
__device__ __forceinline__ void decode8(unsigned c, unsigned s, float (&v)[8]) {
    const float sc = scale_arg(s);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sc, 1),
                d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sc, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sc, 3);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = d.x; v[5] = d.y; v[6] = e.x; v[7] = e.y;
}
__device__ __forceinline__ bf16x8 decode8_bf16(unsigned c, unsigned s) {
    const float sc = scale_arg(s);
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 1),
                 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 2), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 3);
    return bf16x8{a.x, a.y, b.x, b.y, d.x, d.y, e.x, e.y};
}
__device__ __forceinline__ f16x8 decode8_f16(unsigned c, unsigned s) {
    const float sc = scale_arg(s);
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 1),
                d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, sc, 3);
    return f16x8{a.x, a.y, b.x, b.y, d.x, d.y, e.x, e.y};
}

// Vectors in global memory at the alignment of their elements: the hardware takes a vector access at any address, so rows
// of odd length or pitch need no path of their own, only their tails do.
template <typename T, int N> struct Loose { typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };

// eight consecutive values of a row as floats
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        typedef typename Loose<float, 4>::type x4;
        const x4 a = *reinterpret_cast<const x4*>(p), b = *reinterpret_cast<const x4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else {
        typedef typename Loose<T, 8>::type x8;
        const x8 a = *reinterpret_cast<const x8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    }
}
template <typename T>
__device__ __forceinline__ void load8_tail(const T* p, int64_t n, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
}

__device__ __forceinline__ unsigned amax8(const float (&v)[8]) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned b = __builtin_bit_cast(unsigned, v[i]) & 0x7fffffffu;
        m = b > m ? b : m;
    }
    return m;
}
// maximum over the four lanes of a quad
__device__ __forceinline__ unsigned quad_max(unsigned m) {
    unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true);   // lanes 1 0 3 2
    m = o > m ? o : m;
    o = (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true);            // lanes 2 3 0 1
    return o > m ? o : m;
}
__device__ __forceinline__ unsigned quad_or(unsigned m) {
    m |= (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true);
    return m | (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true);
}

// The transposing LDS read (ds_read_b64_tr_b16): sixteen lanes name four rows of sixteen 16-bit values (lane i: row i / 4,
// values 4 (i % 4) ..), lane j gets value j of the four rows.
// eight rows of a column: `at` is this lane's place for four of them, the other four lie `four` bytes on.  (Without __restrict__
// the compiler takes the read for one of whatever is on its way from global memory to LDS, and waits for all of that.)
__device__ __forceinline__ bf16x8 read_turned(const uint8_t* __restrict__ at, int four) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + four));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}


// What every entry point checks of its sizes.  K up to 2^22: 32-bit offsets inside a tile of 256 rows.  A thread for every eight
// values of the padded rows, whole workgroups of them below 2^32 in a launch: with K <= 128 that is fewer than 2^28 rows.
static inline bool sizes_ok(int64_t rows, int64_t K) {
    return rows >= 0 && K >= 1 && K <= (1 << 22) && rows <= 0xffffff00ll / (code_pitch(K) / 4);
}

// launches shared between the files
int launch_quantize(const char* fn, const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales,
                    hipStream_t st);
int launch_dequantize(const char* fn, const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, int dtype, void* out, int64_t ldo,
                      hipStream_t st);

}  // namespace mxk
