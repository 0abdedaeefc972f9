// Layers of up to 256 inputs and outputs over many rows -- the hidden layers of a NeRF, where a row is a sample: bound by the
// rows' bytes, so each pass reads and writes them once.
//
// Forward: W stays in LDS; a wave takes 16 rows of x, rounds them in registers, multiplies and finishes one output tile after
// the other; the next rows are requested before the products.  No barrier in the loop.  262144 x 256 -> 256 fp32: one launch
// that reads x and writes y, 0.54 GB in 97 us over the same x again and again (half of it is still in the last-level cache), 112
// us a call with another x each time (ReLU), against a rounding pass (75 us) and a product (84 us); four waves per SIMD in
// workgroups of eight that share W (three in workgroups of four took 121 us where this took 109).
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
                if (k + 4 <= a.K) {
                    // Non-temporal, x passes through once: 131 -> 121 us (ReLU); such stores of
                    // y, whose rows leave 64 bytes at a time, were slower (143 us).
                    v[i] = __builtin_nontemporal_load(reinterpret_cast<const typename Loose<T, 4>::type*>(p));
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
        constexpr int U = ACT == NERF_ACT_SIN || ACT == NERF_ACT_SIGMOID ? 1 : 4;
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
            finish4<T, ACT, true>(a.f, acc, m, n, a.N, ok, bias);
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
int by_act(const char* fn, const NarrowFwd& a, int act, hipStream_t st) {
    if (act == NERF_ACT_NONE) return by_steps<T, NERF_ACT_NONE>(fn, a, st);
    if (act == NERF_ACT_RELU) return by_steps<T, NERF_ACT_RELU>(fn, a, st);
    if (act == NERF_ACT_SIN) return by_steps<T, NERF_ACT_SIN>(fn, a, st);
    return by_steps<T, NERF_ACT_SIGMOID>(fn, a, st);
}

// ------------------------------------------------------------------------------------------------------- backward
// All three gradients in one pass over dy, the slopes and the packed x.  A workgroup of eight waves walks its 32-row pieces:
//   * dz = dy * slope, out of LDS, where dy and the slopes came by themselves; as soon as a wave has read its rows the next
//     piece's are requested into their place;
//   * dz is split into bf16 terms, x is decoded, both as rows in LDS;
//   * dx: the 32 rows times W, whose fragments every wave keeps in registers (an eighth of the columns each);
//   * dW += dz^T x: each wave keeps a quarter by a half of the whole C x C result in accumulators to the end; the operands
//     run along the rows here, so they are read with the transposing LDS read (ds_read_b64_tr_b16: lane j of sixteen gets
//     column j of four rows);
//   * db: column sums in registers.
// In the end every workgroup writes its dW and db sums, two small kernels add them in order.
//
// 262144 x 256 x 256 fp32 moves 0.84 GB in 270 us (sin; ReLU 0.58 GB in 236, bf16 ReLU 0.31 GB in 114), and 12 + 7 us for the
// sums.  With nothing to load the three phases take 200 us, splitting 78, dx 59, dW 63: two waves on a SIMD (the sums fill its
// registers) hide little of each other's waits for LDS, and what is loaded and stored meets them only in part.  What brought
// it from 297: operands read slots ahead of their matrix instructions (286); the transposing reads marked as apart from the
// requests, for which the compiler had them wait (281); requests in front of the splitting instead of behind it, W's codes
// loaded at once (267).  27 % of the LDS cycles are bank conflicts (10.1 of 37.8 M): rows are 32 bytes longer than 512, so the rows
// eight apart that the lane groups of a transposing read name start on the same bank.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const void* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000);   // addresses are clamped by hand
}
__device__ __forceinline__ void to_lds16(__amdgpu_buffer_rsrc_t b, uint8_t* dst, int voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void*)dst, 16, voff, 0, 0, 0);
}
// Sums over the four 16-lane rows of a wave of four values each: row i of the result holds value i's sum.
__device__ __forceinline__ float rows_sum(float a, float b, float c, float d) {
    const auto add = [](unsigned x, unsigned y) { return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y); };
    const auto bits = [](float v) { return __builtin_bit_cast(unsigned, v); };
    const auto p = __builtin_amdgcn_permlane16_swap(bits(a), bits(b), false, false);    // rows 0, 2 of the sum: a, rows 1, 3: b
    const auto s = __builtin_amdgcn_permlane16_swap(bits(c), bits(d), false, false);
    const unsigned ab = bits(add(p[0], p[1])), cd = bits(add(s[0], s[1]));
    const auto v = __builtin_amdgcn_permlane32_swap(ab, cd, false, false);
    return add(v[0], v[1]);
}

template <typename T, int TERMS, int C>
struct NarrowLds {
    static constexpr int PITCH = C * 2 + 32;                  // bytes of a row of bf16; 32 of padding spread rows over the banks
    static constexpr int PLANE = 32 * PITCH;
    static constexpr int X = TERMS * PLANE;                   // decoded x behind the terms of dz
    static constexpr int DY = X + PLANE, SLOPE = DY + 32 * C * (int)sizeof(T);
    static constexpr int BYTES = SLOPE + 32 * C * 4;
};

// SLOPE: 0 none, 1 slopes, 2 decisions of a ReLU.
template <typename T, int TERMS, int C, int SLOPE>
__global__ __launch_bounds__(512, 2) void mx_narrow_bwd_kernel(NarrowBwd a) {
    using L = NarrowLds<T, TERMS, C>;
    constexpr int PITCH = L::PITCH, STEPS = C / 128;
    constexpr int NT = C / 64, KT = C / 32, XT = C / 128;     // tiles of a wave: dW (NT of n, KT of k), dx (XT of k)
    constexpr int CHUNKS = C / 64;                            // groups of four columns a thread converts
    constexpr int CODES = C / 16;                             // codes a thread decodes
    typedef T x4 __attribute__((ext_vector_type(4)));
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int steps = (a.K + 127) / 128;
    const int row = tid >> 4, l16 = tid & 15;                 // what this thread converts
    const int64_t pieces = (a.M + 31) / 32;
    const int turned = (q * 8 + (r >> 2)) * PITCH + (r & 3) * 8;   // this lane's place in a 32 x 16 block read turned

    // codes of one row -> bf16 values in LDS
    auto decode = [&](const unsigned (&c)[CODES / 8], unsigned s, bool in) {
        uint8_t* o = smem + L::X + row * PITCH + l16 * (CODES * 2);
#pragma unroll
        for (int i = 0; i < CODES / 8; ++i)
            *reinterpret_cast<bf16x8*>(o + i * 16) = in ? decode8_bf16(c[i], s) : decode8_bf16(0u, 0u);
    };

    unsigned wcodes[C / 32][CODES / 8], wscale[C / 32];       // 32 rows of W at a time
    if (a.dx) {
#pragma unroll
        for (int s = 0; s < C / 32; ++s) {
            const int n = s * 32 + row, k = l16 * CODES;
            const int64_t at = n < a.N && k < steps * 128 ? (int64_t)n * (steps * 128) + k : 0;    // values from the first code
#pragma unroll
            for (int i = 0; i < CODES / 8; ++i) wcodes[s][i] = reinterpret_cast<const unsigned*>(a.wc + at / 2)[i];
            wscale[s] = a.ws[at / 32];
        }
    }

    constexpr int DYB = C * (int)sizeof(T);
    const unsigned xpitch = a.dw ? steps * 128 : 0;
    const uint8_t* xc = a.dw ? a.xc : (const uint8_t*)a.dy;
    const uint8_t* xs = a.dw ? a.xs : (const uint8_t*)a.dy;
    [[maybe_unused]] uint16_t bits[CHUNKS];
    unsigned codes[CODES / 8], scale;
    // What wave w converts, rows 4w .. 4w + 3 of the piece, it also loads: no other wave is waited for.
    auto request = [&](int64_t piece) {
        // (hidden from the compiler, which would keep every lane's offsets in registers across the loop)
        int lane = threadIdx.x & 63, row = threadIdx.x >> 4, l16 = threadIdx.x & 15;
        asm volatile("" : "+v"(lane), "+v"(row), "+v"(l16));
        const int64_t m0 = piece * 32;
        const int rows = a.M - m0 < 32 ? (int)(a.M - m0) : 32;
        auto clamp = [&](int v) { return v < rows ? v : rows - 1; };
        const auto dy = rows_of((const T*)a.dy + m0 * a.lddy);
#pragma unroll
        for (int i = 0; i < 4 * DYB / 1024; ++i) {
            const int c = lane * 16 % DYB, at = wave * 4 + (i * 1024 + lane * 16) / DYB;
            to_lds16(dy, smem + L::DY + wave * (4 * DYB) + i * 1024,
                     clamp(at) * (int)a.lddy * (int)sizeof(T) + (c < a.N * (int)sizeof(T) ? c : 0));
        }
        if constexpr (SLOPE == 1) {
            const auto sl = rows_of(a.slope + m0 * a.N);
#pragma unroll
            for (int i = 0; i < 4 * C * 4 / 1024; ++i) {
                const int c = lane * 16 % (C * 4), at = wave * 4 + (i * 1024 + lane * 16) / (C * 4);
                to_lds16(sl, smem + L::SLOPE + wave * (16 * C) + i * 1024, clamp(at) * a.N * 4 + (c < a.N * 4 ? c : 0));
            }
        }
        // (without dW the first bytes of dy: a branch around would make the compiler wait for these behind it)
        const unsigned k = l16 * CODES < xpitch ? l16 * CODES : 0;
        const uint64_t at = (uint64_t)(m0 + clamp(row)) * xpitch + k;    // values from the first code
#pragma unroll
        for (int i = 0; i < CODES / 8; ++i) codes[i] = reinterpret_cast<const unsigned*>(xc + at / 2)[i];
        scale = xs[at / 32];
        if constexpr (SLOPE == 2) {
            const int words = (a.N + 15) / 16;
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) {
                const int w = i * 4 + l16 / 4;
                bits[i] = a.mask[(m0 + clamp(row)) * words + (w < words ? w : 0)];
            }
        }
    };

    int64_t piece = blockIdx.x;
    if (piece < pieces) request(piece);

    // this wave's columns of W, as the A operand of dx = dz W: through LDS (where the requests do not go).  Its tiles take
    // turns in groups of four columns: a lane's results are then neighbours.
    const int wcolumns = (q * 8 + (r >> 2)) * PITCH + wave * (XT * 32) + (r & 3) * (XT * 8);
    bf16x8 wf[XT][C / 32];
    if (a.dx) {
#pragma unroll
        for (int s = 0; s < C / 32; ++s) {
            decode(wcodes[s], wscale[s], s * 32 + row < a.N && l16 * CODES < steps * 128);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
#pragma unroll
            for (int t = 0; t < XT; ++t) wf[t][s] = read_turned(smem + L::X + wcolumns + t * 8, 4 * PITCH);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
        }
    }

    f32x4 acc[KT][NT];
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 db = {0.f, 0.f, 0.f, 0.f};     // lane row q: columns 64 q + 4 l16 ..
    const int wn = wave >> 1, wk = wave & 1;

    for (; piece < pieces; piece += gridDim.x) {
        // the piece has landed, and everybody is done with the rows of the previous one
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        int row = threadIdx.x >> 4, l16 = threadIdx.x & 15, r = lane & 15, q = lane >> 4;    // (hidden as above)
        asm volatile("" : "+v"(row), "+v"(l16), "+v"(r), "+v"(q));
        const int64_t m0 = piece * 32;
        const bool in_row = m0 + row < a.M;
        if (a.dw) decode(codes, scale, in_row && l16 * CODES < steps * 128);
        f32x4 dz[4] = {};
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const int n = i * 64 + l16 * 4;
            const bool in = in_row && n < a.N;      // N is a multiple of four
            const x4 d = *reinterpret_cast<const x4*>(smem + L::DY + row * DYB + n * (int)sizeof(T));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v = (float)d[j];
                if constexpr (SLOPE == 1) v *= reinterpret_cast<const float*>(smem + L::SLOPE + row * (C * 4) + n * 4)[j];
                if constexpr (SLOPE == 2) v = bits[i] >> (4 * (l16 & 3) + j) & 1 ? v : 0.0f;
                v = in ? v : 0.0f;
                const unsigned b = __builtin_bit_cast(unsigned, v) & 0x7fffffffu;
                top = b > top ? b : top;
                dz[i][j] = v;
            }
        }
        // this wave has read its rows: the next ones come while these are split
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (piece + gridDim.x < pieces) request(piece + gridDim.x);
        __builtin_amdgcn_sched_barrier(0);
        const bool careful = __any(top >= 0x7f7f8000u);     // not finite, or infinite as bf16
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            bf16x4 t[TERMS];
            if (careful) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    __bf16 u[TERMS];
                    split_terms<TERMS>(dz[i][j], u);
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) t[k][j] = u[k];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x = dz[i][j];
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) {
                        const __bf16 u = (__bf16)x;
                        t[k][j] = u;
                        x -= (float)u;
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < TERMS; ++k)
                *reinterpret_cast<bf16x4*>(smem + k * L::PLANE + row * PITCH + (i * 64 + l16 * 4) * 2) = t[k];
            __builtin_amdgcn_sched_barrier(0);      // registers are short: one group at a time
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) db[j] += rows_sum(dz[0][j], dz[1][j], dz[2][j], dz[3][j]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                           // (not __syncthreads(): the requests stay under way)
        asm volatile("" ::: "memory");

        // Both products: an operand of dz is read AHEAD slots before its matrix instructions, into the place of one just used.
        if (a.dx) {
            constexpr int AHEAD = SLOPE == 2 ? 3 : 4, LEN = C / 32 * TERMS;      // slots of a row tile
            bf16x8 z[AHEAD];
            auto read_z = [&](auto I) {
                constexpr int i = decltype(I)::value, mt = i / LEN, s = i / TERMS % (C / 32), k = i % TERMS;
                if constexpr (i < 2 * LEN)
                    z[i % AHEAD] = *reinterpret_cast<const bf16x8*>(smem + k * L::PLANE + (mt * 16 + r) * PITCH + s * 64 + q * 16);
            };
            unrolled<AHEAD>(read_z);
            f32x4 o[XT];
            unrolled<2 * LEN>([&](auto I) {
                constexpr int i = decltype(I)::value, mt = i / LEN, s = i / TERMS % (C / 32);
                if constexpr (i % LEN == 0) {
#pragma unroll
                    for (int t = 0; t < XT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int t = 0; t < XT; ++t) o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[t][s], z[i % AHEAD], o[t], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
                read_z(std::integral_constant<int, i + AHEAD>{});
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (i % LEN == LEN - 1) {
                    const int64_t m = m0 + mt * 16 + r;
                    if (m < a.M) {
                        constexpr int VALUES = sizeof(T) == 2 ? 4 * XT : 4;     // of a store
                        const int k0 = (wave * 4 + q) * (4 * XT);
                        T* p = (T*)a.dx + m * a.lddx + k0;
#pragma unroll
                        for (int h = 0; h < 4 * XT; h += VALUES) {
                            typename Loose<T, VALUES>::type v;
#pragma unroll
                            for (int j = 0; j < VALUES; ++j) v[j] = (T)(o[(h + j) / 4][(h + j) % 4] * a.factor);
                            if (k0 + h + VALUES <= a.K) {
                                *reinterpret_cast<typename Loose<T, VALUES>::type*>(p + h) = v;
                            } else {
#pragma unroll
                                for (int j = 0; j < VALUES; ++j)
                                    if (k0 + h + j < a.K) p[h + j] = v[j];
                            }
                        }
                    }
                }
            });
        }
        if (a.dw) {
            constexpr int AHEAD = 2, LEN = NT * TERMS, HALF = KT / 2;    // slots of half the columns of x
            const uint8_t* zl = smem + turned + wn * (NT * 32);
            const uint8_t* xl = smem + L::X + turned + wk * (KT * 32);
            bf16x8 x[HALF], z[AHEAD];
            auto read_z = [&](auto I) {
                constexpr int i = decltype(I)::value, j = i / TERMS % NT, k = i % TERMS;
                if constexpr (i < 2 * LEN) z[i % AHEAD] = read_turned(zl + k * L::PLANE + j * 32, 4 * PITCH);
            };
            unrolled<HALF>([&](auto I) { x[decltype(I)::value] = read_turned(xl + decltype(I)::value * 32, 4 * PITCH); });
            unrolled<AHEAD>(read_z);
            unrolled<2 * LEN>([&](auto I) {
                constexpr int i = decltype(I)::value, half = i / LEN, j = i / TERMS % NT;
#pragma unroll
                for (int t = 0; t < HALF; ++t) {
                    f32x4& sum = acc[half * HALF + t][j];
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[t], z[i % AHEAD], sum, 0, 0, 0);
                    if constexpr (i == LEN - 1) x[t] = read_turned(xl + (HALF + t) * 32, 4 * PITCH);
                }
                __builtin_amdgcn_sched_barrier(0);
                read_z(std::integral_constant<int, i + AHEAD>{});
                __builtin_amdgcn_sched_barrier(0);
            });
        }
    }

    if (a.dw) {     // this workgroup's sums: lane holds four k of one n
        float* s = a.slab + (int64_t)blockIdx.x * (C * C);
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                *reinterpret_cast<f32x4*>(s + ((wn * NT + j) * 16 + r) * C + (wk * KT + i) * 16 + q * 4) = acc[i][j];
    }
    if (a.colsum) {
        __syncthreads();
        float* s = reinterpret_cast<float*>(smem);      // [wave][256]
        *reinterpret_cast<f32x4*>(s + wave * 256 + q * 64 + l16 * 4) = db;
        __syncthreads();
        if (tid < a.N) {
            float v = 0.0f;
            for (int i = 0; i < 8; ++i) v += s[i * 256 + tid];
            a.colsum[(int64_t)blockIdx.x * a.N + tid] = v * a.factor;
        }
    }
}

// dW = factor * sum of the workgroups' parts, in their order: sixteen threads walk the parts of four neighbours, joined in order
template <typename T, int C>
__global__ __launch_bounds__(256) void mx_narrow_join_kernel(const float* __restrict__ slab, int groups, int N, int K, float factor,
                                                            T* __restrict__ dw) {
    __shared__ f32x4 part[16][16];
    const int c = threadIdx.x & 15, w = threadIdx.x >> 4;
    const int at = (blockIdx.x * 16 + c) * 4, n = at / C, k = at % C;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (n < N && k < K) {
#pragma unroll 4
        for (int g = w; g < groups; g += 16) v += *reinterpret_cast<const f32x4*>(slab + (int64_t)g * (C * C) + at);
    }
    part[w][c] = v;
    __syncthreads();
    if (w == 0 && n < N) {
        f32x4 s = part[0][c];
        for (int i = 1; i < 16; ++i) s += part[i][c];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < K) dw[(int64_t)n * K + k + j] = (T)(s[j] * factor);
    }
}

template <typename T, int TERMS, int C, int SLOPE>
int launch_bwd(const char* fn, const NarrowBwd& a, hipStream_t st) {
    constexpr int lds = NarrowLds<T, TERMS, C>::BYTES;
    static_assert(lds <= 160 * 1024 && 32 * C * 4 <= lds, "LDS");
    int rc = nerf_set_lds(mx_narrow_bwd_kernel<T, TERMS, C, SLOPE>, lds);
    if (rc) return rc;
    const int groups = narrow_groups(a.M, C);
    mx_narrow_bwd_kernel<T, TERMS, C, SLOPE><<<(unsigned)groups, 512, lds, st>>>(a);
    if ((rc = nerf_check_launch(fn)) || !a.dw) return rc;
    mx_narrow_join_kernel<T, C><<<(unsigned)((a.N * C + 63) / 64), 256, 0, st>>>(a.slab, groups, a.N, a.K, a.factor, (T*)a.dw);
    return nerf_check_launch(fn);
}
template <typename T, int TERMS, int SLOPE>
int by_columns(const char* fn, const NarrowBwd& a, hipStream_t st) {
    return narrow_columns(a.K, a.N) == 256 ? launch_bwd<T, TERMS, 256, SLOPE>(fn, a, st) : launch_bwd<T, TERMS, 128, SLOPE>(fn, a, st);
}
// terms without and with slopes (a ReLU's decisions need no more than none)
template <typename T, int TERMS, int SMOOTH>
int by_slope(const char* fn, const NarrowBwd& a, hipStream_t st) {
    if (a.slope) return by_columns<T, SMOOTH, 1>(fn, a, st);
    return a.mask ? by_columns<T, TERMS, 2>(fn, a, st) : by_columns<T, TERMS, 0>(fn, a, st);
}

}  // namespace

int launch_narrow_bwd(const char* fn, const NarrowBwd& a, int dtype, hipStream_t st) {
    if (dtype == NERF_F32) return by_slope<float, 3, 3>(fn, a, st);
    if (dtype == NERF_F16) return by_slope<_Float16, 2, 2>(fn, a, st);
    return by_slope<__bf16, 1, 2>(fn, a, st);
}

int launch_narrow_fwd(const char* fn, const NarrowFwd& a, int dtype, int act, hipStream_t st) {
    if (dtype == NERF_F32) return by_act<float>(fn, a, act, st);
    if (dtype == NERF_BF16) return by_act<__bf16>(fn, a, act, st);
    return by_act<_Float16>(fn, a, act, st);
}

}  // namespace mxk
