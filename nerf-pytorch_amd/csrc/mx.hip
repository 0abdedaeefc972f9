// Microscaled 4-bit (MXFP4) rows: quantise and read back.  The format is described in mx_common.h.
//
// Both kernels are bound by HBM: a thread owns eight consecutive values (16 bytes of a 16-bit type, 32 of fp32), the four
// threads of a quad one block.  The block's maximum takes two DPP steps, the rounding is the conversion instruction's
// (v_cvt_scalef32_pk_fp4_f32: to nearest even, saturating).  Packed rows are back to back, so thread i writes code word i and
// block i / 4's scale whatever the row's length; only the unpacked side needs the row, hence a division, and not even that
// where rows are whole multiples of 128 values and back to back (FLAT).
#include "mx_common.h"

namespace mxk {
namespace {

// One group of eight values per thread: two and four with all loads in flight together were slower, for small tensors (13 x
// 8000 fp16: 2.6 against 3.4 us with four, compute units without a workgroup) as for large ones (reading 8192 x 8192 bf16: 61
// against 68 us with four; rounding 262144 x 256 fp32: 50 against 52).
template <typename T, bool FLAT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t total, int64_t K, int groups,
                                                         unsigned* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;   // below 2^32
    if (i >= total) return;   // whole quads: a row is a multiple of sixteen groups
    float v[8];
    if constexpr (FLAT) {
        load8(x + i * 8, v);
    } else {
        const int64_t row = (unsigned)i / (unsigned)groups, k = (i - row * groups) * 8;
        if (k + 8 <= K) load8(x + row * ldx + k, v);
        else load8_tail(x + row * ldx + k, K - k, v);
    }
    const unsigned s = scale_byte(quad_max(amax8(v)));
    codes[i] = encode8(v, s);
    if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)s;
}

template <typename T, bool FLAT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const unsigned* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                           int64_t total, int64_t K, int groups, T* __restrict__ out, int64_t ldo) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const unsigned c = codes[i], s = scales[i >> 2];
    int64_t k = 0;
    T* p;
    if constexpr (FLAT) {
        p = out + i * 8;
    } else {
        const int64_t row = (unsigned)i / (unsigned)groups;
        k = (i - row * groups) * 8;
        if (k >= K) return;
        p = out + row * ldo + k;
    }
    T t[8];
    if constexpr (sizeof(T) == 4) {
        decode8(c, s, t);
    } else if constexpr (__is_same(T, __bf16)) {
        const bf16x8 v = decode8_bf16(c, s);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = v[j];
    } else {
        const f16x8 v = decode8_f16(c, s);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = v[j];
    }
    if (FLAT || k + 8 <= K) {
        typedef T t4 __attribute__((ext_vector_type(sizeof(T) == 4 ? 4 : 8)));
        constexpr int L = sizeof(T) == 4 ? 4 : 8;
#pragma unroll
        for (int h = 0; h < 8 / L; ++h) {
            t4 w;
#pragma unroll
            for (int j = 0; j < L; ++j) w[j] = t[h * L + j];
            *reinterpret_cast<typename Loose<T, L>::type*>(p + h * L) = w;
        }
    } else {
        const int n = (int)(K - k);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) p[j] = t[j];
    }
}

template <typename T>
void quantize_as(const void* xv, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales, hipStream_t st) {
    const T* x = (const T*)xv;
    const int64_t groups = code_pitch(K) / 4, total = M * groups;
    const bool flat = K % 128 == 0 && ldx == K;
    const unsigned grid = (unsigned)ceil_div64(total, 256);
    const auto launch = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(x, ldx, total, K, (int)groups, (unsigned*)codes, scales); };
    if (flat) launch(mx_quantize_kernel<T, true>);
    else launch(mx_quantize_kernel<T, false>);
}

template <typename T>
void dequantize_as(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* ov, int64_t ldo, hipStream_t st) {
    T* out = (T*)ov;
    const int64_t groups = code_pitch(K) / 4, total = M * groups;
    const bool flat = K % 128 == 0 && ldo == K;
    const unsigned grid = (unsigned)ceil_div64(total, 256);
    const unsigned* c = (const unsigned*)codes;
    const auto launch = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(c, scales, total, K, (int)groups, out, ldo); };
    if (flat) launch(mx_dequantize_kernel<T, true>);
    else launch(mx_dequantize_kernel<T, false>);
}

}  // namespace

int launch_quantize(const char* fn, const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales,
                    hipStream_t st) {
    if (dtype == NERF_F32) quantize_as<float>(x, ldx, M, K, codes, scales, st);
    else if (dtype == NERF_BF16) quantize_as<__bf16>(x, ldx, M, K, codes, scales, st);
    else quantize_as<_Float16>(x, ldx, M, K, codes, scales, st);
    return nerf_check_launch(fn);
}

int launch_dequantize(const char* fn, const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, int dtype, void* out, int64_t ldo,
                      hipStream_t st) {
    if (dtype == NERF_F32) dequantize_as<float>(codes, scales, M, K, out, ldo, st);
    else if (dtype == NERF_BF16) dequantize_as<__bf16>(codes, scales, M, K, out, ldo, st);
    else dequantize_as<_Float16>(codes, scales, M, K, out, ldo, st);
    return nerf_check_launch(fn);
}

}  // namespace mxk

extern "C" size_t nerf_mx_codes_bytes(int64_t rows, int64_t K) {
    return mxk::sizes_ok(rows, K) ? (size_t)(rows * mxk::code_pitch(K)) : 0;
}
extern "C" size_t nerf_mx_scales_bytes(int64_t rows, int64_t K) {
    return mxk::sizes_ok(rows, K) ? (size_t)(rows * mxk::scale_pitch(K)) : 0;
}

extern "C" int nerf_mx_quantize(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales,
                                void* stream) {
    NERF_REQUIRE(mxk::sizes_ok(M, K) && ldx >= K, "nerf_mx_quantize: bad shape M=%lld K=%lld ldx=%lld", (long long)M, (long long)K,
                 (long long)ldx);
    NERF_REQUIRE(dtype >= NERF_F32 && dtype <= NERF_F16, "nerf_mx_quantize: unknown type %d", dtype);
    if (M == 0) return NERF_OK;
    NERF_REQUIRE_PTR(x);
    NERF_REQUIRE_PTR(codes);
    NERF_REQUIRE_PTR(scales);
    NERF_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 4 == 0, "nerf_mx_quantize: codes must be 16-byte, scales 4-byte aligned");
    return mxk::launch_quantize("nerf_mx_quantize", x, dtype, ldx, M, K, codes, scales, (hipStream_t)stream);
}

extern "C" int nerf_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, int dtype, void* out, int64_t ldo,
                                  void* stream) {
    NERF_REQUIRE(mxk::sizes_ok(M, K) && ldo >= K, "nerf_mx_dequantize: bad shape M=%lld K=%lld ldo=%lld", (long long)M, (long long)K,
                 (long long)ldo);
    NERF_REQUIRE(dtype >= NERF_F32 && dtype <= NERF_F16, "nerf_mx_dequantize: unknown type %d", dtype);
    if (M == 0) return NERF_OK;
    NERF_REQUIRE_PTR(codes);
    NERF_REQUIRE_PTR(scales);
    NERF_REQUIRE_PTR(out);
    NERF_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 4 == 0,
                 "nerf_mx_dequantize: codes must be 16-byte, scales 4-byte aligned");
    return mxk::launch_dequantize("nerf_mx_dequantize", codes, scales, M, K, dtype, out, ldo, (hipStream_t)stream);
}
