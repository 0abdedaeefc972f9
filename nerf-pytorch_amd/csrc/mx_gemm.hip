// Products of the microscaled 4-bit (MXFP4) operators (format: mx_common.h): one tiled kernel for
//     forward        y  = post * f(pre * (X W^T + b))     X, W packed     v_mfma_scale_f32_16x16x128_f8f6f4
//     data gradient  dx = dZ W                            bf16 operands   v_mfma_f32_16x16x32_bf16
//     weight grad.   dW = dZ^T X                          bf16 operands
// Both matrix instructions take 64 bytes of a row per step and 16 of them per lane at the same place (row = lane & 15, bytes
// 16 (lane >> 4) .. +16), and both issue every 16 cycles: staging, LDS image and loop are the same for the two types, only
// the packed type has scales next to its rows and four times the values per byte.
//
// The gradients are those of the product at the rounded operands (straight through the rounding).  X and W as they were
// rounded are exact in bf16 (a code times a power of two); dz goes in as `terms` bf16 terms (dz = t0 + t1 + t2, each the
// rounding of what the previous ones left): one for bf16 dy without a smooth activation (exact), two for fp16 dy (11 bits:
// exact) and for 16-bit dy through sin / sigmoid (2^-17, far under the output's own rounding), three for fp32 (exact up to
// 2^-25).  Sums are fp32 throughout; a split reduction writes fp32 slabs that a second kernel adds in a fixed order.
#include "mx_large.h"
#include "mx_narrow.h"

namespace mxk {
namespace {

enum Kind { PACKED = 0, BF16 = 1 };

struct Operand {
    const uint8_t* p;       // rows of 64-byte steps
    int64_t pitch;          // bytes between rows
    const uint8_t* sc;      // PACKED: four scale bytes per step
    int64_t sc_pitch;
    int64_t rows;
    int64_t plane;          // BF16: bytes between the terms of the operand (0: the same for all terms)
};

struct GemmArgs {
    Operand w, x;           // out[m][n] = sum over steps of x[m] . w[n]
    int64_t M;
    int N;
    int steps;              // 64-byte steps per row
    int terms;
    int per_split;          // stages (two steps) per grid.z slice
    int tiles_m, tiles_n;
    Finish f;
};

__device__ __forceinline__ i32x8 wide(i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// Rows of an operand as a buffer; global memory -> LDS, 16 (4) bytes per lane one after the other behind dst.  Every
// address lies in [base, base + size).  (The size must be a literal for the builtin.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const uint8_t* base, int size) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, size, 0x00020000);
}
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t b, uint8_t* dst, int voff, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void*)dst, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void load_lds4(__amdgpu_buffer_rsrc_t b, uint8_t* dst, int voff, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void*)dst, 4, voff, soff, 0, 0);
}

// Tile of workgroup `t`.  Workgroups go round the eight XCDs; each XCD gets a contiguous run of tiles, walked in groups of
// eight tile rows, so that what shares an L2 shares operand rows.
__device__ __forceinline__ void tile_of(const GemmArgs& a, int t, int tm, int tn, int64_t& m0, int& n0) {
    const int tiles = a.tiles_m * a.tiles_n;
    const int per = tiles / 8, extra = tiles % 8, xcd = t & 7, i = t >> 3;
    t = xcd * per + (xcd < extra ? xcd : extra) + i;
    constexpr int GROUP = 8;
    const int group = t / (GROUP * a.tiles_n), first = group * GROUP;
    const int height = a.tiles_m - first < GROUP ? a.tiles_m - first : GROUP;
    const int in_group = t - group * GROUP * a.tiles_n;
    m0 = (int64_t)(first + in_group % height) * tm;
    n0 = in_group / height * tn;
}

// A wave's sums on their way out as they lie in the registers, four n of one m per lane: rows of 64 bytes (fp32) or 32 at a
// time, joined in the L2.  For the light activations: half the instructions of the way through LDS, and those are what the
// end of a tile takes.
template <int NI, int MI, typename T, int ACT>
__device__ __forceinline__ void store_direct(const GemmArgs& a, const f32x4 (&acc)[NI][MI], int64_t m_first, int n_first) {
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    f32x4 bias[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) bias[i] = load_bias<T>(a.f.bias, n_first + i * 16 + q * 4, a.N);
#pragma unroll
    for (int j = 0; j < MI; ++j)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int64_t m = m_first + j * 16 + r;
            finish4<T, ACT, true>(a.f, acc[i][j], m, n_first + i * 16 + q * 4, a.N, m < a.M, bias[i]);
            __builtin_amdgcn_sched_barrier(0);   // one group of registers at a time
        }
}

// The same through LDS (32 rows of `lds` at a time): the stores take whole rows of the wave's tile, and the activation's
// code stands once in a loop.  m, n: the wave tile's place.
template <int NI, int MI, typename T, int ACT>
__device__ __forceinline__ void store_tile(const GemmArgs& a, const f32x4 (&acc)[NI][MI], float* lds, int64_t m_first, int n_first) {
    constexpr int WNN = NI * 16, PITCH = WNN + 4;      // floats; 16 bytes of padding spread the rows over the banks
    constexpr int LPR = WNN / 4, RPI = 64 / LPR;       // lanes per row, rows per instruction
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int n = n_first + (lane % LPR) * 4;
    const f32x4 bias = a.f.slab ? f32x4{0.f, 0.f, 0.f, 0.f} : load_bias<T>(a.f.bias, n, a.N);
    constexpr int U = ACT == NERF_ACT_SIN || ACT == NERF_ACT_SIGMOID ? 2 : 8;   // rows in flight
#pragma unroll
    for (int jj = 0; jj < MI; jj += 2) {
#pragma unroll
        for (int j = jj; j < jj + 2; ++j)
#pragma unroll
            for (int i = 0; i < NI; ++i) *reinterpret_cast<f32x4*>(lds + ((j - jj) * 16 + r) * PITCH + i * 16 + q * 4) = acc[i][j];
        __builtin_amdgcn_wave_barrier();
#pragma unroll U
        for (int row = 0; row < 32; row += RPI) {
            const int lr = row + lane / LPR;
            const f32x4 v = *reinterpret_cast<const f32x4*>(lds + lr * PITCH + (lane % LPR) * 4);
            const int64_t m = m_first + jj * 16 + lr;
            if (a.f.slab) {
                float* s = a.f.slab + ((int64_t)blockIdx.z * a.M + m) * a.N + n;
                if (m < a.M) {
                    if (n + 4 <= a.N) {
                        *reinterpret_cast<typename Loose<float, 4>::type*>(s) = v;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (n + i < a.N) s[i] = v[i];
                    }
                }
            } else {
                finish4<T, ACT, false>(a.f, v, m, n, a.N, m < a.M, bias);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}
template <int NI>
constexpr int store_tile_floats() { return 32 * (NI * 16 + 4); }

// Tile of TM rows x TN columns of the output, WM x WN waves, two LDS stages of 128 bytes a row.
//
// LDS image of a stage: rows of 128 bytes, the 16-byte piece c of row r at place c ^ (r & 7), so that the fragment reads of
// eight neighbouring rows (ds_read_b128, the same piece of each) touch all banks once.  The loads go straight to LDS
// (buffer_load ... lds writes lane after lane, so the permutation is applied to the global address; a row's 128 bytes stay
// one contiguous request).  W is the A operand: a lane then holds four neighbouring n of one m.
//
// Order of a stage's two halves: [read the second half's fragments | multiply the first's], then wait for the next stage's
// loads, barrier, [request the stage after it, read its first fragments | multiply the second half's].  One barrier a stage;
// loads have a whole stage to arrive.
template <int KIND, int TM, int TN, int WM, int WN, typename T, int ACT>
__global__ __launch_bounds__(64 * WM * WN, TM == 128 ? 2 : 4) void mx_gemm_kernel(GemmArgs a) {
    constexpr int NW = WM * WN, MI = TM / WM / 16, NI = TN / WN / 16, R = TM + TN;
    constexpr int ROWS = R / NW;            // rows a wave stages: all of one operand
    constexpr int PIECES = ROWS / 8;        // 1 KiB requests: eight rows each
    constexpr int SPIECES = ROWS * 2 / 64;  // PACKED: requests of 64 scale words, two per row
    static_assert(TN % ROWS == 0 && ROWS % 32 == 0, "a wave stages rows of one operand");
    constexpr int STAGE = R * 128 + (KIND == PACKED ? R * 8 : 0);
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;

    int64_t m0;
    int n0;
    tile_of(a, (int)blockIdx.x, TM, TN, m0, n0);

    // what this wave stages
    const bool is_w = wave * ROWS < TN;
    const Operand& op = is_w ? a.w : a.x;
    const int64_t row0 = is_w ? (int64_t)n0 + wave * ROWS : m0 + (wave * ROWS - TN);
    const int64_t left = op.rows - row0;
    const int valid = left > ROWS ? ROWS : left < 1 ? 1 : (int)left;   // rows behind the last one repeat it (never stored)
    const uint8_t* base = op.p + (left < 1 ? op.rows - 1 : row0) * op.pitch;
    const int col = (lane & 7) ^ (lane >> 3);
    int voff[PIECES], svoff[SPIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int row = i * 8 + (lane >> 3);
        voff[i] = (row < valid ? row : valid - 1) * (int)op.pitch + col * 16;
    }
    const uint8_t* sbase = nullptr;
    if constexpr (KIND == PACKED) {
        sbase = op.sc + (left < 1 ? op.rows - 1 : row0) * op.sc_pitch;
#pragma unroll
        for (int i = 0; i < SPIECES; ++i) {
            const int row = i * 32 + (lane >> 1);
            svoff[i] = (row < valid ? row : valid - 1) * (int)op.sc_pitch + (lane & 1) * 4;
        }
    }
    const int stages = (a.steps + 1) / 2;
    const bool odd = a.steps & 1;
    const int total = stages * a.terms;
    const int g0 = (int)blockIdx.z * a.per_split, g1 = g0 + a.per_split < total ? g0 + a.per_split : total;

    int load_term = g0 / stages, load_st = g0 - load_term * stages;   // stage to request next
    auto request = [&](int buf) {
        uint8_t* dst = smem + buf * STAGE + wave * (ROWS * 128);
        // an odd number of steps: the last stage's second half does not exist; it is read from the first (and not used)
        const bool half = odd && load_st == stages - 1;
        const int back = half && col >= 4 ? 64 : 0;
        const auto rows = buffer_of(base + load_term * op.plane, valid * (int)op.pitch);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) load_lds16(rows, dst + i * 1024, voff[i] - back, load_st * 128);
        if constexpr (KIND == PACKED) {
            uint8_t* sdst = smem + buf * STAGE + R * 128 + wave * (ROWS * 8);
            const int sback = half && (lane & 1) ? 4 : 0;
            const auto scales = buffer_of(sbase, valid * (int)op.sc_pitch);
#pragma unroll
            for (int i = 0; i < SPIECES; ++i) load_lds4(scales, sdst + i * 256, svoff[i] - sback, load_st * 8);
        }
        if (++load_st == stages) { load_st = 0; ++load_term; }
    };

    const int wm = wave / WN, wn = wave % WN;
    f32x4 acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Frags {
        i32x4 w[NI], x[MI];
        int sw[NI], sx[MI];
    } fr[2];
    const int place[2] = {r * 128 + ((q ^ (r & 7)) * 16), r * 128 + (((4 + q) ^ (r & 7)) * 16)};
    auto read = [&](Frags& f, int buf, int half) {
        const uint8_t* wl = smem + buf * STAGE + wn * (NI * 2048) + place[half];
        const uint8_t* xl = smem + buf * STAGE + TN * 128 + wm * (MI * 2048) + place[half];
#pragma unroll
        for (int i = 0; i < NI; ++i) f.w[i] = *reinterpret_cast<const i32x4*>(wl + i * 2048);
#pragma unroll
        for (int j = 0; j < MI; ++j) f.x[j] = *reinterpret_cast<const i32x4*>(xl + j * 2048);
        if constexpr (KIND == PACKED) {
            const uint8_t* ws = smem + buf * STAGE + R * 128 + wn * (NI * 128) + r * 8 + half * 4 + q;
            const uint8_t* xs = smem + buf * STAGE + R * 128 + TN * 8 + wm * (MI * 128) + r * 8 + half * 4 + q;
#pragma unroll
            for (int i = 0; i < NI; ++i) f.sw[i] = ws[i * 128];
#pragma unroll
            for (int j = 0; j < MI; ++j) f.sx[j] = xs[j * 128];
        }
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int j = 0; j < MI; ++j)
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                if constexpr (KIND == PACKED)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(f.w[i]), wide(f.x[j]), acc[i][j], 4, 4, 0, f.sw[i],
                                                                                0, f.sx[j]);
                else
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, f.w[i]),
                                                                        __builtin_bit_cast(bf16x8, f.x[j]), acc[i][j], 0, 0, 0);
            }
    };
    auto publish = [&] {   // every wave's requests have landed, every wave has read what it needs of the previous stage
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    int st = load_st;   // stage being multiplied, within its term
    request(0);
    publish();
    if (g0 + 1 < g1) request(1);
    read(fr[0], 0, 0);
    for (int g = g0; g < g1; ++g) {
        const int buf = (g - g0) & 1;
        const bool two = !(odd && st == stages - 1);
        if (++st == stages) st = 0;
        if (two) read(fr[1], buf, 1);
        multiply(fr[0]);
        if (g + 1 < g1) {
            publish();
            if (g + 2 < g1) request(buf);
            read(fr[0], buf ^ 1, 0);
        }
        if (two) multiply(fr[1]);
    }

    // no request is in flight; the barrier lets the last readers finish
    static_assert(NW * store_tile_floats<NI>() * 4 <= 2 * STAGE, "the way out fits the stages");
    __syncthreads();
    store_tile<NI, MI, T, ACT>(a, acc, reinterpret_cast<float*>(smem) + wave * store_tile_floats<NI>(), m0 + wm * (MI * 16),
                               n0 + wn * (NI * 16));
}

// One matrix instruction of the large tile, accumulating IN PLACE.  With the builtin the compiler
// takes the result for a new value: it moved the large tile's accumulators between register files and spilled.
// What it no longer sees is the result's latency; settle_all() covers that where the sums are read.
// BYTE: where in their registers the scales are.
template <int KIND, int BYTE>
__device__ __forceinline__ void mfma_in_place(f32x4& acc, const i32x4& w, const i32x4& x, int sw, int sx) {
    static_assert(BYTE < 2, "");
    if constexpr (KIND == PACKED && BYTE == 0)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+v"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx));
    else if constexpr (KIND == PACKED)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+v"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx));
    else
        asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(w), "v"(x));
}
// The wait between the last matrix instructions and the first reads of their results (at most 16 passes of 4 cycles); every
// accumulator passes through an empty statement behind it, so that no read moves in front.
template <int NI, int MI>
__device__ __forceinline__ void settle_all(f32x4 (&acc)[NI][MI]) {
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) asm volatile("" : "+v"(acc[i][j]));
}

// The large tile: 256 x 256, eight waves of 128 (m) x 64 (n), two on each SIMD: what one wave waits for to issue -- a request,
// a fragment read -- the other's matrix instructions hide.  (Four waves of 128 x 128 read a third less LDS, but alone on their
// SIMDs took 51 us where these took 47, packed 4096 x 4096 x 4096, and 146 where they took 141, 4096 x 8192 x 8192.)  Stages as
// above, 128 bytes of each of the 512 rows, in two buffers.  Now 44 and 135 us (4.1 PFLOP/s): 1.7 us a stage and 15 a tile, 10
// of those its stores, which leave all compute units together; bf16 4096 x 4096 x 4096 98 us (1.4 PFLOP/s).
//
// A stage's two halves are eight slots of four matrix instructions: slot j multiplies row fragment x[j] with the half's four
// column fragments.  As soon as slot j is done, x[j] of the next half is read into its place, eight slots ahead; the column
// fragments have two sets.  At the start of the second half everybody holds all it needs of the stage: there is the stage's
// one barrier, behind it the stage after next is requested into the buffer, one piece a slot, and the reads go to the next
// stage, which had a whole stage to arrive.
//
// PACKED: the order of the blocks inside a stage is free as long as both operands agree, and lane group q takes blocks
// 2q and 2q + 1 of the eight in its two halves: their two scale bytes are neighbours, one 16-bit read per row and stage,
// and the matrix instruction picks the byte.  Scales are requested for two stages at a time, 16 bytes a row (8-byte
// requests of 512 rows cost the L2 as much as the codes did); the last window of a row is moved back to end with it.  LDS serves
// sixteen lanes at a time, of two neighbouring groups: with q and q + 1 in places 2q and 2q + 2 the permutation of a row is
// another than for bf16 (half of the LDS cycles were conflicts before, 138 -> 135 us; 17 % are left, 2.0 of 12.1 M; bf16 has none).
//
// Rows of 64 bytes a stage in a ring of four were slower: requests of half a cache line halve what the L2 delivers.
template <int KIND, typename T, int ACT>
__global__ __launch_bounds__(512, 2) void mx_gemm_large_kernel(GemmArgs a) {
    constexpr int TILE = 256, NI = 4, MI = 8;
    constexpr int PIECES = 8;               // requests of a wave per stage
    constexpr int STAGE = LargeLds::STAGE, SCALES = LargeLds::SCALES;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];   // two stages; PACKED: and two windows of scales

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const auto swizzle = [](int row) { return KIND == PACKED ? (row >> 1 & 1) | (row & 4) : row; };
    const int r = lane & 15, q = lane >> 4;
    int64_t m0;
    int n0;
    tile_of(a, (int)blockIdx.x, TILE, TILE, m0, n0);

    // waves 0 to 3 stage the tile's 256 rows of W, 4 to 7 those of X; rows behind the last one repeat it (never stored)
    const bool is_w = wave < 4;
    const Operand& op = is_w ? a.w : a.x;
    const int64_t row0 = (is_w ? (int64_t)n0 : m0) + (wave & 3) * 64;
    const int64_t left = op.rows - row0;
    const int valid = left > 64 ? 64 : left < 1 ? 1 : (int)left;
    const int64_t first = left < 1 ? op.rows - 1 : row0;
    const uint8_t* from = op.p + first * op.pitch;
    const int size = valid * (int)op.pitch, ssize = valid * (int)op.sc_pitch;
    const uint8_t* sfrom = KIND == PACKED ? op.sc + first * op.sc_pitch : nullptr;
    const int col = (lane & 7) ^ swizzle(lane >> 3);
    int voff[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int row = i * 8 + (lane >> 3);
        voff[i] = (row < valid ? row : valid - 1) * (int)op.pitch + col * 16;
    }
    const int svoff = (lane < valid ? lane : valid - 1) * (int)op.sc_pitch;
    const int stages = (a.steps + 1) / 2;
    const bool odd = a.steps & 1;     // PACKED, one term: the last stage holds four blocks of eight
    const int D = stages * a.terms;   // the large tile does not split the reduction

    int load_st = 0;             // stage to request next
    struct Request {
        __amdgpu_buffer_rsrc_t rows;
        uint8_t* dst;
        int soff;
    };
    auto request = [&](int d) {
        const Request rq{buffer_of(from, size), smem + (d & 1) * STAGE + wave * 8192, load_st * 128};
        if constexpr (KIND == PACKED) {
            if ((d & 1) == 0) {
                const int window = d * 8, end = a.steps * 4 - 16;   // a.steps >= 4
                load_lds16(buffer_of(sfrom, ssize), smem + 2 * STAGE + (d >> 1 & 1) * SCALES + wave * 1024, svoff, window < end ? window : end);
            }
            if (odd && d == stages - 1) {   // read from the first four blocks instead, and not used (once per tile)
#pragma unroll
                for (int i = 0; i < PIECES; ++i) voff[i] -= col >= 4 ? 64 : 0;
            }
        }
        if (++load_st == stages) {
            load_st = 0;
            from += op.plane;
        }
        return rq;
    };
    auto issue = [&](auto I, const Request& rq) { load_lds16(rq.rows, rq.dst + decltype(I)::value * 1024, voff[decltype(I)::value], rq.soff); };

    const int wm = wave >> 2, wn = wave & 3;
    f32x4 acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    i32x4 w0[NI], w1[NI], x[MI];
    struct Scales {
        int w[NI], x[MI];
    } scales, next_scales;   // both halves' of a stage
    const int piece0 = KIND == PACKED ? 2 * q : q, piece1 = KIND == PACKED ? 2 * q + 1 : 4 + q;
    const int place[2] = {r * 128 + ((piece0 ^ swizzle(r & 7)) * 16), r * 128 + ((piece1 ^ swizzle(r & 7)) * 16)};
    const int splace = LargeLds::scale_place(r, q);
    auto read_w = [&](auto I, auto HALF, i32x4 (&w)[NI], const uint8_t* stage) {
        w[decltype(I)::value] = *reinterpret_cast<const i32x4*>(stage + wn * 8192 + place[decltype(HALF)::value] + decltype(I)::value * 2048);
    };
    auto read_x = [&](auto J, auto HALF, const uint8_t* stage) {
        x[decltype(J)::value] =
            *reinterpret_cast<const i32x4*>(stage + 32768 + wm * 16384 + place[decltype(HALF)::value] + decltype(J)::value * 2048);
    };
    auto read_scale = [&](auto I, Scales& sc, int scale_at) {   // I of 12: columns, then rows
        constexpr int i = decltype(I)::value;
        if constexpr (KIND == PACKED) {
            if constexpr (i < NI) sc.w[i] = *reinterpret_cast<const uint16_t*>(smem + splace + scale_at + wn * 1024 + i * 256);
            else sc.x[i - NI] = *reinterpret_cast<const uint16_t*>(smem + splace + scale_at + 4096 + wm * 2048 + (i - NI) * 256);
        }
    };
    auto slot = [&](auto J, auto HALF, const i32x4 (&w)[NI]) {
        constexpr int j = decltype(J)::value, half = decltype(HALF)::value;
#pragma unroll
        for (int i = 0; i < NI; ++i)
            mfma_in_place<KIND, half>(acc[i][j], w[i], x[j], KIND == PACKED ? scales.w[i] : 0, KIND == PACKED ? scales.x[j] : 0);
    };
    // the last stage of an odd row: lane groups 2 and 3 multiply zeros (a branch around would put copies of the sums at its end)
    auto blank = [&](i32x4 (&w)[NI]) {
#pragma unroll
        for (int i = 0; i < NI; ++i) w[i] = q < 2 ? w[i] : i32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < MI; ++j) x[j] = q < 2 ? x[j] : i32x4{0, 0, 0, 0};
    };
    auto publish = [&] {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    constexpr std::integral_constant<int, 0> H0{};
    constexpr std::integral_constant<int, 1> H1{};
    // One stage: x and w0 hold its first half's fragments, and in the end the next stage's.
    auto stage_body = [&](auto REQUEST, int d) {
        const uint8_t* here = smem + (d & 1) * STAGE;
        const uint8_t* next = smem + ((d & 1) ^ 1) * STAGE;
        if constexpr (!REQUEST)
            if (KIND == PACKED && odd && d == D - 1) {
                blank(w0);
#pragma unroll
                for (int i = 0; i < NI; ++i) scales.w[i] = q < 2 ? scales.w[i] : 0;
#pragma unroll
                for (int j = 0; j < MI; ++j) scales.x[j] = q < 2 ? scales.x[j] : 0;
            }
        __builtin_amdgcn_sched_barrier(0);
        unrolled<MI>([&](auto J) {
            constexpr int j = decltype(J)::value;
            slot(J, H0, w0);
            __builtin_amdgcn_sched_barrier(0);
            read_x(J, H1, here);
            if constexpr (j < NI) read_w(J, H1, w1, here);
            __builtin_amdgcn_sched_barrier(0);
        });
        publish();
        if constexpr (!REQUEST)
            if (KIND == PACKED && odd && d == D - 1) blank(w1);
        Request rq;
        if constexpr (REQUEST) rq = request(d + 2);
        const int scale_at = LargeLds::scales_of(a.steps, d + 1);
        __builtin_amdgcn_sched_barrier(0);
        unrolled<MI>([&](auto J) {
            constexpr int j = decltype(J)::value;
            if constexpr (REQUEST) issue(J, rq);
            __builtin_amdgcn_sched_barrier(0);
            slot(J, H1, w1);
            __builtin_amdgcn_sched_barrier(0);
            read_x(J, H0, next);
            if constexpr (j < NI) {
                read_w(J, H0, w0, next);
                read_scale(std::integral_constant<int, 3 * j>{}, next_scales, scale_at);
                read_scale(std::integral_constant<int, 3 * j + 1>{}, next_scales, scale_at);
                read_scale(std::integral_constant<int, 3 * j + 2>{}, next_scales, scale_at);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        scales = next_scales;
    };

    {
        const Request rq = request(0);
        unrolled<PIECES>([&](auto I) { issue(I, rq); });
    }
    publish();
    if (D > 1) {
        const Request rq = request(1);
        unrolled<PIECES>([&](auto I) { issue(I, rq); });
    }
    unrolled<NI>([&](auto I) { read_w(I, H0, w0, smem); });
    unrolled<MI>([&](auto J) { read_x(J, H0, smem); });
    unrolled<NI + MI>([&](auto I) { read_scale(I, scales, LargeLds::scales_of(a.steps, 0)); });
    int d = 0;   // (behind the last stage old contents are read, and not used)
    for (; d + 2 < D; ++d) stage_body(std::true_type{}, d);
    for (; d < D; ++d) stage_body(std::false_type{}, d);
    settle_all(acc);
    // nothing is under way; the barrier lets the last readers finish
    static_assert(8 * store_tile_floats<NI>() * 4 <= 2 * STAGE, "the way out fits the stages");
    __syncthreads();
    if constexpr (ACT == NERF_ACT_NONE || ACT == NERF_ACT_RELU)
        store_direct<NI, MI, T, ACT>(a, acc, m0 + wm * 128, n0 + wn * 64);
    else
        store_tile<NI, MI, T, ACT>(a, acc, reinterpret_cast<float*>(smem) + wave * store_tile_floats<NI>(), m0 + wm * 128, n0 + wn * 64);
}

// out = finish(sum of the slabs): Z threads walk the slabs of four neighbours, joined in order.  A workgroup takes 1024 / Z
// neighbours of one row's groups of sixteen.
template <typename T, int ACT, int Z>
__global__ __launch_bounds__(256) void mx_finish_kernel(Finish f, int64_t M, int N, int splits) {
    constexpr int G = 256 / Z;
    __shared__ f32x4 part[Z][G];
    const int c = threadIdx.x % G, w = threadIdx.x / G;
    const int quads = (N + 15) / 16 * 4;    // groups of four, whole quads of lanes inside a row
    const int64_t i = (int64_t)blockIdx.x * G + c;
    const int64_t m = i / quads;
    const int n = (int)(i - m * quads) * 4;
    const bool ok = m < M;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (ok && n < N) {
        const float* s = f.slab + m * N + n;
        const int64_t step = M * N;
        if (n + 4 <= N) {
#pragma unroll 4
            for (int z = w; z < splits; z += Z) v += *reinterpret_cast<const typename Loose<float, 4>::type*>(s + z * step);
        } else {
            for (int z = w; z < splits; z += Z)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + j < N) v[j] += s[z * step + j];
        }
    }
    if constexpr (Z > 1) {
        part[w][c] = v;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int z = 1; z < Z; ++z) v += part[z][c];
    }
    finish4<T, ACT, false>(f, v, m, n, N, ok, load_bias<T>(f.bias, n, N));
}

// ---------------------------------------------------------------------------------------------- gradients: operands
// dz = dy * (d y / d z), split into bf16 terms: rows [term][M][Np] for the data gradient and, turned, [term][N][Mp] for
// the weight gradient (either may be NULL); Np, Mp: rounded up to 64, zeros behind the end.  colsum: partial column sums
// of dz [grid.y][N], or NULL.  Tiles of 64 x 64, `deep` of them one under the other per workgroup; the terms go through LDS
// as rows and are read out turned.  Bound by bytes, and by launch and latency where there are few: 4096 x 4096 bf16, whose rows
// the product reads in place, 67 MB in 18 us; 6000 x 257 fp32 with slopes 33 MB in 13 us.  16 to 20 % of the LDS cycles are bank
// conflicts.
struct DzArgs {
    const void* dy;
    int64_t lddy;
    const float* slope;
    const uint16_t* mask;
    float factor;
    int64_t M;
    int N;
    int64_t Np, Mp;
    __bf16* rows;
    __bf16* turned;
    float* colsum;
    int deep;
};

template <typename T, int TERMS>
__global__ __launch_bounds__(256) void mx_dz_kernel(DzArgs a) {
    constexpr int PITCH = 160, PLANE = 64 * PITCH;          // bytes: 64 bf16 and 32 of padding
    __shared__ __attribute__((aligned(16))) uint8_t tile[TERMS * PLANE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n0 = blockIdx.x * 64;
    const int lr = tid >> 2, lc = (tid & 3) * 16;           // reading: a row, sixteen columns
    const int r = lane & 15, q = lane >> 4;
    const uint8_t* turned = tile + (q * 8 + (r >> 2)) * PITCH + wave * 32 + (r & 3) * 8;    // writing: sixteen columns a wave
    float csum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) csum[i] = 0.0f;
    for (int d = 0; d < a.deep; ++d) {
        const int64_t m0 = ((int64_t)blockIdx.y * a.deep + d) * 64;
        if (m0 >= a.Mp) break;
        const int64_t m = m0 + lr;
        float v[16];
        const T* p = (const T*)a.dy + m * a.lddy + n0 + lc;
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.0f;
        if (m < a.M) {
            if (n0 + lc + 16 <= a.N) {
#pragma unroll
                for (int i = 0; i < 16; i += 8) {
                    float t[8];
                    load8(p + i, t);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[i + j] = t[j];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (n0 + lc + i < a.N) v[i] = (float)p[i];
            }
            if (a.mask) {
                unsigned bits = n0 + lc < a.N ? a.mask[m * ((a.N + 15) / 16) + (n0 + lc) / 16] : 0u;
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = (bits >> i) & 1u ? v[i] : 0.0f;
            }
            if (a.slope) {
                const float* s = a.slope + m * a.N + n0 + lc;
                if (n0 + lc + 16 <= a.N) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const f32x4 t = *reinterpret_cast<const typename Loose<float, 4>::type*>(s + i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[i + j] *= t[j];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (n0 + lc + i < a.N) v[i] *= s[i];
                }
            }
        }
        __bf16 t[16][TERMS];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            csum[i] += v[i];
            split_terms<TERMS>(v[i], t[i]);
        }
        if (a.turned) __syncthreads();      // the previous tile has been read
#pragma unroll
        for (int k = 0; k < TERMS; ++k) {
            bf16x8 lo, hi;
#pragma unroll
            for (int i = 0; i < 8; ++i) { lo[i] = t[i][k]; hi[i] = t[8 + i][k]; }
            if (a.rows && m < a.M) {
                __bf16* o = a.rows + ((int64_t)k * a.M + m) * a.Np + n0 + lc;
                *reinterpret_cast<bf16x8*>(o) = lo;
                *reinterpret_cast<bf16x8*>(o + 8) = hi;
            }
            if (a.turned) {
                *reinterpret_cast<bf16x8*>(tile + k * PLANE + lr * PITCH + lc * 2) = lo;
                *reinterpret_cast<bf16x8*>(tile + k * PLANE + lr * PITCH + lc * 2 + 16) = hi;
            }
        }
        if (a.turned) {
            __syncthreads();
            const int n = n0 + wave * 16 + r;
#pragma unroll
            for (int k = 0; k < TERMS; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bf16x8 c = read_turned(turned + k * PLANE + h * (32 * PITCH), 4 * PITCH);
                    if (n < a.N) *reinterpret_cast<bf16x8*>(a.turned + ((int64_t)k * a.N + n) * a.Mp + m0 + h * 32 + q * 8) = c;
                }
        }
    }
    if (a.colsum) {     // the sixteen rows of a wave, then the four waves, always in the same order
        float* part = reinterpret_cast<float*>(tile);       // [wave][64]
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = csum[i];
            s += __shfl_xor(s, 4);
            s += __shfl_xor(s, 8);
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            if (lane < 4) part[wave * 64 + lane * 16 + i] = s;
        }
        __syncthreads();
        if (tid < 64 && n0 + tid < a.N)
            a.colsum[(int64_t)blockIdx.y * a.N + n0 + tid] = (((part[tid] + part[64 + tid]) + part[128 + tid]) + part[192 + tid]) * a.factor;
    }
}

// db[n] = sum of the partial column sums: a workgroup takes 16 columns, sixteen threads walk each, joined in order
template <typename T>
__global__ __launch_bounds__(256) void mx_colsum_kernel(const float* __restrict__ part, int parts, int N, T* __restrict__ db) {
    __shared__ float s[16][17];
    const int c = threadIdx.x & 15, w = threadIdx.x >> 4, n = blockIdx.x * 16 + c;
    float v = 0.0f;
    if (n < N)
        for (int i = w; i < parts; i += 16) v += part[(int64_t)i * N + n];
    s[w][c] = v;
    __syncthreads();
    if (w == 0 && n < N) {
        float sum = 0.0f;
        for (int i = 0; i < 16; ++i) sum += s[i][c];
        db[n] = (T)sum;
    }
}

// Packed rows [rows][K] -> turned bf16 values [K][rows_p], zeros behind the last row.  Tiles of 64 rows x 128 values; W and x
// in one launch, neighbouring workgroups write neighbours.  Bound by bytes: 4096 x 4096 both, 86 MB in 16 us; half of its LDS
// cycles are bank conflicts, of rows eight apart that start on the same bank.
struct Turn {
    const uint8_t *codes, *scales;
    int64_t rows, rows_p;       // rows_p: 0 where there is nothing to turn
    __bf16* out;
};
__global__ __launch_bounds__(256) void mx_turn_kernel(Turn first, Turn second, int64_t K) {
    constexpr int PITCH = 288;                              // bytes: 128 bf16 and 32 of padding
    __shared__ __attribute__((aligned(16))) uint8_t tile[64 * PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4;
    const bool is_first = blockIdx.x < first.rows_p / 64;
    const Turn& t = is_first ? first : second;
    const int64_t m0 = ((int64_t)blockIdx.x - (is_first ? 0 : first.rows_p / 64)) * 64, k0 = (int64_t)blockIdx.y * 128;
    const int64_t m = m0 + (tid >> 2);
    u32x4 c = {0u, 0u, 0u, 0u};
    unsigned s = 0;
    if (m < t.rows) {
        const int64_t block = m * scale_pitch(K) + k0 / 32 + (tid & 3);
        c = *reinterpret_cast<const u32x4*>(t.codes + block * 16);
        s = t.scales[block];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *reinterpret_cast<bf16x8*>(tile + (tid >> 2) * PITCH + (tid & 3) * 64 + i * 16) = decode8_bf16(c[i], s);
    __syncthreads();
    const uint8_t* turned = tile + (q * 8 + (r >> 2)) * PITCH + wave * 64 + (r & 3) * 8;    // 32 values of the row a wave
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bf16x8 v = read_turned(turned + j * 32 + h * (32 * PITCH), 4 * PITCH);
            const int64_t k = k0 + wave * 32 + j * 16 + r;
            if (k < K) *reinterpret_cast<bf16x8*>(t.out + k * t.rows_p + m0 + h * 32 + q * 8) = v;
        }
}

// ------------------------------------------------------------------------------------------------ launches
constexpr int kTargetGroups = 256;   // compute units

struct Plan {
    int tile;
    int tiles_m, tiles_n, splits, per_split;
    size_t slab_floats;
};

// Tile and split of an M x N product over rows of `steps` times 64 bytes.
//
// The largest tile of which there are three for every four compute units, counting tiles at the edges as whole ones: a tile of
// 256 x 256 reads half of what 128 x 128 does for each product, and a quarter of idle units is less than that (rounding and packed
// product in bf16, tiles of 128 against 256: 4096 x 4096 -> 4096 70 : 54 us, 4096 x 8192 -> 8192 198 : 150, 3328 x 4096 -> 4096, 208
// tiles, 60 : 47, 16384 x 1024 -> 1024 34 : 30).  Little is lost where tiles are wide of what they cover or start a second
// round: tiles of 64 : 128 : 256, rounding and product in bf16, 50000 x 1000 -> 16 31 : 35 : 37 us, -> 64 32 : 35 : 38, -> 130 40 : 44 :
// 38, 32768 x 4096 -> 257 111 : 104 : 103, 4096 x 4096 -> 4352, 272 tiles, 92 : 78 : 77, -> 4608 99 : 78 : 77; fp32 data gradient of
// 32 -> 2000 over 50000 rows 406 : 397 : 420, of 130 -> 2000 504 : 475 : 427.  Below
// 256 tiles of 128 the work goes to tiles of 64 (1024^3 training in bf16 66 -> 53 us, 512 x 4096 -> 4096 32 -> 23.6 us, rows of
// 319 -> 257 over 6000 in fp32 86 -> 74 us), and where those are too few the reduction is split.
Plan plan_for(int64_t M, int64_t N, int64_t steps, int terms) {
    Plan p{};
    const int64_t total = (steps + 1) / 2 * terms;
    const auto tiles_of = [&](int64_t t) { return ceil_div64(M, t) * ceil_div64(N, t); };
    p.tile = tiles_of(256) >= kTargetGroups * 3 / 4 && steps >= 4 ? 256 : tiles_of(128) >= kTargetGroups ? 128 : 64;   // (a window of scales is four steps)
    p.tiles_m = (int)ceil_div64(M, p.tile);
    p.tiles_n = (int)ceil_div64(N, p.tile);
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    int64_t splits = 1;
    if (p.tile != 256 && tiles < kTargetGroups) {
        splits = kTargetGroups / tiles;
        const int64_t most = total / 4 < 1 ? 1 : total / 4;    // at least four stages a slice
        if (splits > most) splits = most;
        if (splits > 256) splits = 256;
    }
    p.per_split = (int)ceil_div64(total, splits);
    p.splits = (int)ceil_div64(total, p.per_split);
    p.slab_floats = p.splits > 1 ? (size_t)p.splits * M * N : 0;
    return p;
}

template <int KIND, int TILE, typename T, int ACT>
int launch_gemm_tile(const char* fn, const GemmArgs& a, int splits, hipStream_t st) {
    constexpr int lds = 2 * (2 * TILE * 128 + (KIND == PACKED ? 2 * TILE * 8 : 0));
    int rc = nerf_set_lds(mx_gemm_kernel<KIND, TILE, TILE, 2, 2, T, ACT>, lds);
    if (rc) return rc;
    mx_gemm_kernel<KIND, TILE, TILE, 2, 2, T, ACT><<<dim3((unsigned)(a.tiles_m * a.tiles_n), 1, (unsigned)splits), 256, lds, st>>>(a);
    return nerf_check_launch(fn);
}

template <int KIND, typename T, int ACT>
int launch_gemm_large(const char* fn, const GemmArgs& a, int splits, hipStream_t st) {
    constexpr int lds = LargeLds::bytes(KIND == PACKED);
    int rc = nerf_set_lds(mx_gemm_large_kernel<KIND, T, ACT>, lds);
    if (rc) return rc;
    mx_gemm_large_kernel<KIND, T, ACT><<<dim3((unsigned)(a.tiles_m * a.tiles_n), 1, (unsigned)splits), 512, lds, st>>>(a);
    return nerf_check_launch(fn);
}

template <int KIND, typename T, int ACT>
int launch_gemm(const char* fn, GemmArgs a, const Plan& p, hipStream_t st) {
    a.tiles_m = p.tiles_m;
    a.tiles_n = p.tiles_n;
    a.per_split = p.per_split;
    if (p.splits == 1) a.f.slab = nullptr;
    int rc = p.tile == 256   ? launch_gemm_large<KIND, T, ACT>(fn, a, p.splits, st)
             : p.tile == 128 ? launch_gemm_tile<KIND, 128, T, ACT>(fn, a, p.splits, st)
                             : launch_gemm_tile<KIND, 64, T, ACT>(fn, a, p.splits, st);
    if (rc || p.splits == 1) return rc;
    const int64_t items = a.M * ((a.N + 15) / 16 * 4);
    if (p.splits >= 8) mx_finish_kernel<T, ACT, 16><<<(unsigned)ceil_div64(items, 16), 256, 0, st>>>(a.f, a.M, a.N, p.splits);
    else mx_finish_kernel<T, ACT, 1><<<(unsigned)ceil_div64(items, 256), 256, 0, st>>>(a.f, a.M, a.N, p.splits);
    return nerf_check_launch(fn);
}

template <typename T>
int launch_forward(const char* fn, const GemmArgs& a, const Plan& p, int act, hipStream_t st) {
    if (act == NERF_ACT_NONE) return launch_gemm<PACKED, T, NERF_ACT_NONE>(fn, a, p, st);
    if (act == NERF_ACT_RELU) return launch_gemm<PACKED, T, NERF_ACT_RELU>(fn, a, p, st);
    if (act == NERF_ACT_SIN) return launch_gemm<PACKED, T, NERF_ACT_SIN>(fn, a, p, st);
    return launch_gemm<PACKED, T, NERF_ACT_SIGMOID>(fn, a, p, st);
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

int terms_for(int dtype, int act) {
    if (dtype == NERF_F32) return 3;
    if (dtype == NERF_F16) return 2;
    return act == NERF_ACT_SIN || act == NERF_ACT_SIGMOID ? 2 : 1;
}

struct FwdLayout {
    bool few, narrow, fused;      // fused: x is rounded by the product's own kernel
    Plan plan;
    size_t scales, slab, bytes;   // offsets (codes at 0): the quantised x where the caller keeps none, partial sums
};
FwdLayout fwd_layout(int64_t M, int64_t K, int64_t N, bool keeps_x) {
    FwdLayout l{};
    l.few = few_rows(M, K, N);
    l.narrow = M >= kNarrowRowsFwd && K <= kNarrow && N <= kNarrow;
    l.fused = (l.few && !keeps_x && few_fused(M, K)) || l.narrow;
    if (!l.few && !l.narrow) l.plan = plan_for(M, N, ceil_div64(K, 128), 1);
    if (!keeps_x && !l.fused) {
        l.scales = up256((size_t)(M * code_pitch(K)));
        l.slab = l.scales + up256((size_t)(M * scale_pitch(K)));
    }
    l.bytes = l.slab + l.plan.slab_floats * 4;
    return l;
}

struct BwdLayout {
    bool narrow;
    int terms, deep;
    int64_t Np, Mp, parts;
    Plan dx, dw;
    size_t rows, turned, part, wt, xt, slab, bytes;
};
// `narrow`: whether the layout of dy allows that path; the size that callers ask for covers both ways.
BwdLayout bwd_layout(int dtype, int act, int64_t M, int64_t K, int64_t N, bool need_dx, bool need_dw, bool need_db, bool narrow) {
    BwdLayout l{};
    if (narrow) {
        l.narrow = true;
        const int c = narrow_columns(K, N), groups = narrow_groups(M, c);
        if (need_dw) l.bytes = (size_t)groups * c * c * 4;
        l.part = l.bytes;
        if (need_db) l.bytes += up256((size_t)groups * N * 4);
        return l;
    }
    l.terms = terms_for(dtype, act);
    l.Np = ceil_div64(N, 64) * 64;
    l.Mp = ceil_div64(M, 64) * 64;
    const int64_t tiles = (l.Np / 64) * (l.Mp / 64);
    l.deep = tiles >= 8192 ? 8 : tiles >= 2048 ? 2 : 1;
    l.parts = ceil_div64(l.Mp / 64, l.deep);
    l.dx = plan_for(M, K, l.Np / 32, l.terms);
    l.dw = plan_for(N, K, l.Mp / 32, l.terms);
    size_t at = 0;
    l.rows = at;
    if (need_dx) at += up256((size_t)l.terms * M * l.Np * 2);
    l.turned = at;
    if (need_dw) at += up256((size_t)l.terms * N * l.Mp * 2);
    l.part = at;
    if (need_db) at += up256((size_t)l.parts * N * 4);
    l.wt = at;
    if (need_dx) at += up256((size_t)K * l.Np * 2);
    l.xt = at;
    if (need_dw) at += up256((size_t)K * l.Mp * 2);
    l.slab = at;
    const size_t s1 = need_dx ? l.dx.slab_floats : 0, s2 = need_dw ? l.dw.slab_floats : 0;
    at += (s1 > s2 ? s1 : s2) * 4;   // one after the other on one stream
    l.bytes = at;
    return l;
}

template <typename T>
int launch_dz(const char* fn, const DzArgs& a, int terms, hipStream_t st) {
    const dim3 grid((unsigned)(a.Np / 64), (unsigned)ceil_div64(a.Mp / 64, a.deep));
    if (terms == 1) mx_dz_kernel<T, 1><<<grid, 256, 0, st>>>(a);
    else if (terms == 2) mx_dz_kernel<T, 2><<<grid, 256, 0, st>>>(a);
    else mx_dz_kernel<T, 3><<<grid, 256, 0, st>>>(a);
    return nerf_check_launch(fn);
}

int launch_colsum(const char* fn, const float* part, int parts, int N, int dtype, void* db, hipStream_t st) {
    const unsigned grid = (unsigned)ceil_div64(N, 16);
    if (dtype == NERF_F32) mx_colsum_kernel<float><<<grid, 256, 0, st>>>(part, parts, N, (float*)db);
    else if (dtype == NERF_BF16) mx_colsum_kernel<__bf16><<<grid, 256, 0, st>>>(part, parts, N, (__bf16*)db);
    else mx_colsum_kernel<_Float16><<<grid, 256, 0, st>>>(part, parts, N, (_Float16*)db);
    return nerf_check_launch(fn);
}

template <typename T>
int backward(const char* fn, const BwdLayout& l, DzArgs dz, const uint8_t* xcodes, const uint8_t* xscales, const uint8_t* wcodes,
             const uint8_t* wscales, int64_t M, int64_t K, int64_t N, uint8_t* ws, void* dx, int64_t lddx, void* dw, void* db,
             hipStream_t st) {
    // bf16 without a slope, in rows that the product can take: dy is its own one term
    const bool direct = __is_same(T, __bf16) && !dz.slope && !dz.mask && N % 64 == 0 && (uintptr_t)dz.dy % 16 == 0 && dz.lddy % 8 == 0 &&
                        dz.lddy < (1 << 22);
    dz.rows = dx && !direct ? (__bf16*)(ws + l.rows) : nullptr;
    dz.turned = dw ? (__bf16*)(ws + l.turned) : nullptr;
    dz.colsum = db ? (float*)(ws + l.part) : nullptr;
    int rc = NERF_OK;
    if ((dz.rows || dz.turned || dz.colsum) && (rc = launch_dz<T>(fn, dz, l.terms, st))) return rc;
    constexpr int dtype = sizeof(T) == 4 ? NERF_F32 : __is_same(T, __bf16) ? NERF_BF16 : NERF_F16;
    if (db && (rc = launch_colsum(fn, dz.colsum, (int)l.parts, (int)N, dtype, db, st))) return rc;
    const Turn w{wcodes, wscales, N, dx ? l.Np : 0, (__bf16*)(ws + l.wt)}, x{xcodes, xscales, M, dw ? l.Mp : 0, (__bf16*)(ws + l.xt)};
    if (w.rows_p + x.rows_p) {
        mx_turn_kernel<<<dim3((unsigned)((w.rows_p + x.rows_p) / 64), (unsigned)ceil_div64(K, 128)), 256, 0, st>>>(w, x, K);
        if ((rc = nerf_check_launch(fn))) return rc;
    }
    if (dx) {   // dx[m][k] = sum over n of dz[m][n] W[n][k]
        GemmArgs a{};
        a.w = Operand{ws + l.wt, l.Np * 2, nullptr, 0, K, 0};
        a.x = direct ? Operand{(const uint8_t*)dz.dy, dz.lddy * 2, nullptr, 0, M, 0} : Operand{ws + l.rows, l.Np * 2, nullptr, 0, M, M * l.Np * 2};
        a.M = M;
        a.N = (int)K;
        a.steps = (int)(l.Np / 32);
        a.terms = l.terms;
        a.f = Finish{dx, lddx, nullptr, 1.0f, dz.factor, nullptr, nullptr, (float*)(ws + l.slab)};
        if ((rc = launch_gemm<BF16, T, NERF_ACT_NONE>(fn, a, l.dx, st))) return rc;
    }
    if (dw) {   // dW[n][k] = sum over m of dz[m][n] X[m][k]
        GemmArgs a{};
        a.w = Operand{ws + l.xt, l.Mp * 2, nullptr, 0, K, 0};
        a.x = Operand{ws + l.turned, l.Mp * 2, nullptr, 0, N, N * l.Mp * 2};
        a.M = N;
        a.N = (int)K;
        a.steps = (int)(l.Mp / 32);
        a.terms = l.terms;
        a.f = Finish{dw, K, nullptr, 1.0f, dz.factor, nullptr, nullptr, (float*)(ws + l.slab)};
        if ((rc = launch_gemm<BF16, T, NERF_ACT_NONE>(fn, a, l.dw, st))) return rc;
    }
    return NERF_OK;
}

}  // namespace
}  // namespace mxk

using namespace mxk;

// On top of what the packed rows ask (fewer than 2^28 of them): an int N that 32-bit offsets reach, and a launch of fewer than
// 2^32 threads
static bool linear_sizes_ok(int64_t M, int64_t K, int64_t N) {
    return sizes_ok(M, K) && N >= 1 && N <= (1 << 22) && sizes_ok(N, K) && ceil_div64(M, 128) * ceil_div64(N, 128) < (1 << 24);
}

constexpr int64_t kTrainRows = 65535ll * 64;   // of a backward pass: grid.y; 32-bit offsets inside a turned tile

extern "C" size_t nerf_mx_linear_fwd_workspace_bytes(int64_t M, int64_t K, int64_t N, int keeps_x) {
    return linear_sizes_ok(M, K, N) && M > 0 ? fwd_layout(M, K, N, keeps_x).bytes : 0;
}

extern "C" int nerf_mx_linear_fwd(const void* x, int dtype, int64_t ldx, const uint8_t* wcodes, const uint8_t* wscales, const void* bias,
                                  int64_t M, int64_t K, int64_t N, int act, double pre, double post, void* y, int64_t ldy, float* slope,
                                  uint16_t* mask, uint8_t* xcodes, uint8_t* xscales, void* workspace, void* stream) {
    const char* fn = "nerf_mx_linear_fwd";
    NERF_REQUIRE(linear_sizes_ok(M, K, N) && ldx >= K && ldy >= N, "%s: bad shape M=%lld K=%lld N=%lld ldx=%lld ldy=%lld", fn, (long long)M,
                 (long long)K, (long long)N, (long long)ldx, (long long)ldy);
    NERF_REQUIRE(dtype >= NERF_F32 && dtype <= NERF_F16, "%s: unknown type %d", fn, dtype);
    NERF_REQUIRE(act >= NERF_ACT_NONE && act <= NERF_ACT_SIGMOID, "%s: unknown activation %d", fn, act);
    NERF_REQUIRE(!xcodes || (M <= kTrainRows && N <= kTrainRows), "%s: more than 65535*64 rows of x or W kept for a backward pass", fn);
    if (M == 0) return NERF_OK;
    NERF_REQUIRE_PTR(x);
    NERF_REQUIRE_PTR(wcodes);
    NERF_REQUIRE_PTR(wscales);
    NERF_REQUIRE_PTR(y);
    const FwdLayout l = fwd_layout(M, K, N, xcodes != nullptr);
    if (l.bytes) NERF_REQUIRE_PTR(workspace);
    NERF_REQUIRE((xcodes == nullptr) == (xscales == nullptr), "%s: xcodes and xscales go together", fn);
    NERF_REQUIRE((uintptr_t)wcodes % 16 == 0 && (uintptr_t)wscales % 4 == 0 && (uintptr_t)xcodes % 16 == 0 && (uintptr_t)xscales % 4 == 0 &&
                     (uintptr_t)workspace % 16 == 0,
                 "%s: codes and workspace must be 16-byte, scales 4-byte aligned", fn);
    const hipStream_t st = (hipStream_t)stream;
    uint8_t* ws = (uint8_t*)workspace;
    uint8_t* xc = xcodes ? xcodes : ws;
    uint8_t* xs = xscales ? xscales : ws + l.scales;
    const Finish f{y, ldy, bias, (float)pre, (float)post, act == NERF_ACT_SIN || act == NERF_ACT_SIGMOID ? slope : nullptr,
                   act == NERF_ACT_RELU ? mask : nullptr, (float*)(ws + l.slab)};
    if (l.narrow) {
        const NarrowFwd a{x, ldx, M, (int)K, (int)N, wcodes, wscales, xcodes, xscales, f};
        return launch_narrow_fwd(fn, a, dtype, act, st);
    }
    if (!l.fused) {
        int rc = launch_quantize(fn, x, dtype, ldx, M, K, xc, xs, st);
        if (rc) return rc;
    }
    if (l.few) {
        const FewArgs a{wcodes, wscales, l.fused ? x : nullptr, ldx, xc, xs, (int)M, (int)K, (int)N, (int)ceil_div64(K, 128), f};
        return launch_few(fn, a, dtype, act, st);
    }
    GemmArgs a{};
    a.w = Operand{wcodes, code_pitch(K), wscales, scale_pitch(K), N, 0};
    a.x = Operand{xc, code_pitch(K), xs, scale_pitch(K), M, 0};
    a.M = M;
    a.N = (int)N;
    a.steps = (int)ceil_div64(K, 128);
    a.terms = 1;
    a.f = f;
    if (dtype == NERF_F32) return launch_forward<float>(fn, a, l.plan, act, st);
    if (dtype == NERF_BF16) return launch_forward<__bf16>(fn, a, l.plan, act, st);
    return launch_forward<_Float16>(fn, a, l.plan, act, st);
}

extern "C" size_t nerf_mx_linear_bwd_workspace_bytes(int dtype, int act, int64_t M, int64_t K, int64_t N, int need_dx, int need_dw,
                                                     int need_db) {
    if (!linear_sizes_ok(M, K, N) || M < 1 || dtype < NERF_F32 || dtype > NERF_F16) return 0;
    const size_t general = bwd_layout(dtype, act, M, K, N, need_dx, need_dw, need_db, false).bytes;
    if (M < kNarrowRowsBwd || K > kNarrow || N > kNarrow) return general;
    const size_t narrow = bwd_layout(dtype, act, M, K, N, need_dx, need_dw, need_db, true).bytes;
    return narrow > general ? narrow : general;
}

extern "C" int nerf_mx_linear_bwd(const void* dy, int dtype, int64_t lddy, const float* slope, const uint16_t* mask, int act, double pre,
                                  double post, const uint8_t* xcodes, const uint8_t* xscales, const uint8_t* wcodes,
                                  const uint8_t* wscales, int64_t M, int64_t K, int64_t N, void* workspace, void* dx, int64_t lddx,
                                  void* dw, void* db, void* stream) {
    const char* fn = "nerf_mx_linear_bwd";
    NERF_REQUIRE(linear_sizes_ok(M, K, N) && M >= 1 && lddy >= N && (!dx || lddx >= K), "%s: bad shape M=%lld K=%lld N=%lld", fn,
                 (long long)M, (long long)K, (long long)N);
    NERF_REQUIRE(dtype >= NERF_F32 && dtype <= NERF_F16, "%s: unknown type %d", fn, dtype);
    NERF_REQUIRE(act >= NERF_ACT_NONE && act <= NERF_ACT_SIGMOID, "%s: unknown activation %d", fn, act);
    NERF_REQUIRE(M <= kTrainRows && N <= kTrainRows, "%s: more than 65535*64 rows of x or W per call", fn);
    if (!dx && !dw && !db) return NERF_OK;
    NERF_REQUIRE_PTR(dy);
    NERF_REQUIRE_PTR(workspace);
    if (act == NERF_ACT_RELU) NERF_REQUIRE_PTR(mask);
    if (act == NERF_ACT_SIN || act == NERF_ACT_SIGMOID) NERF_REQUIRE_PTR(slope);
    if (dx) { NERF_REQUIRE_PTR(wcodes); NERF_REQUIRE_PTR(wscales); }
    if (dw) { NERF_REQUIRE_PTR(xcodes); NERF_REQUIRE_PTR(xscales); }
    NERF_REQUIRE((uintptr_t)wcodes % 16 == 0 && (uintptr_t)xcodes % 16 == 0 && (uintptr_t)workspace % 16 == 0,
                 "%s: codes and workspace must be 16-byte aligned", fn);
    const bool smooth = act == NERF_ACT_SIN || act == NERF_ACT_SIGMOID;
    const int size = dtype == NERF_F32 ? 4 : 2;
    const BwdLayout l = bwd_layout(dtype, act, M, K, N, dx != nullptr, dw != nullptr, db != nullptr,
                                   narrow_bwd_ok(dy, lddy, size, M, K, N, smooth ? slope : nullptr));
    DzArgs dz{};
    dz.dy = dy;
    dz.lddy = lddy;
    dz.slope = smooth ? slope : nullptr;
    dz.mask = act == NERF_ACT_RELU ? mask : nullptr;
    // the constant factor of dz stays out of the terms (they are exact without it) and is applied to the sums
    dz.factor = dz.slope ? 1.0f : (float)(pre * post);
    dz.M = M;
    dz.N = (int)N;
    dz.Np = l.Np;
    dz.Mp = l.Mp;
    dz.deep = l.deep;
    const hipStream_t st = (hipStream_t)stream;
    uint8_t* ws = (uint8_t*)workspace;
    if (l.narrow) {
        float* part = db ? (float*)(ws + l.part) : nullptr;
        const NarrowBwd a{dy, lddy, dz.slope, dz.mask, dz.factor, xcodes, xscales, wcodes, wscales, M, (int)K, (int)N, dx, lddx, dw, (float*)ws, part};
        int rc = launch_narrow_bwd(fn, a, dtype, st);
        return rc || !db ? rc : launch_colsum(fn, part, narrow_groups(M, narrow_columns(K, N)), (int)N, dtype, db, st);
    }
    if (dtype == NERF_F32)
        return backward<float>(fn, l, dz, xcodes, xscales, wcodes, wscales, M, K, N, ws, dx, lddx, dw, db, st);
    if (dtype == NERF_BF16)
        return backward<__bf16>(fn, l, dz, xcodes, xscales, wcodes, wscales, M, K, N, ws, dx, lddx, dw, db, st);
    return backward<_Float16>(fn, l, dz, xcodes, xscales, wcodes, wscales, M, K, N, ws, dx, lddx, dw, db, st);
}
