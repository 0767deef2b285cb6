// Linear layer on operands of 8 bits: out = act(x W^T + bias) + residual, x [n][ci] and W [co][ci] as e4m3 codes with a
// power of two for every 32 channels (mx.hpp).
//
// Two forms of the product, by what the output keeps. 16-bit outputs take the scaled matrix instruction
// (v_mfma_scale_f32_16x16x128_f8f6f4), which multiplies the codes and applies the powers itself; within an
// instruction it adds products to some 16 bits below the largest (measured: 1.5e-5 of the result in the 2-norm, a
// hundredth of bf16's rounding and a twentieth of fp16's). An fp32 output would show that, so there codes become bf16
// with their powers, which is exact, and v_mfma_f32_16x16x32_bf16 adds in fp32 (6e-8), at half the rate.
//
// The roles are turned: W is the first operand, so that a lane holds four consecutive outputs of one row.
//
// Figures here and below are of a captured graph's replays on one set of inputs. Large products are bound by the matrix cores at
// the clock that the chip's power leaves, and by how tiles reach them: 8,192^3 takes 467-471 us in bf16 (2,340 TFLOP/s; the
// library's 8-bit product 388-419) and 855-862 in fp32 (1,290; its bf16 product 763-782). 35,001 x 4,096 -> 1,024 in fp32 with
// a residual takes 304 us (321 with input sets that take turns), the matrix cores 39 % busy at 2.1 GHz: half of a wave's time
// goes into waiting for loads (tiles of 256 x 256 in cache, no residual: 323 us, 268 without the loop's loads, 229 without its
// LDS reads), and a tile's rows leave at the memory's rate with nothing beside them, since a CU holds one such workgroup. Few rows
// are bound by the latency of W: 5 rows, 1,024 -> 4,096, 4.0 us. No product is split along its channels: what has few tiles leaves
// the device part empty (64 rows, 4,096 -> 1,024: 10 us on 16 workgroups; 2,606 x 8,192 -> 27: 19 on 41).
// Tried and taken back: widening a step's codes while the products of the one before run (fp32; no faster, 40 registers more);
// loads through registers to LDS (442 us where direct ones into buffers of their own took 295).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "mx.hpp"

namespace tsp {
namespace {

constexpr int LM_K = 128;      // channels of a step

typedef int i32x8_t __attribute__((ext_vector_type(8)));

struct LinearArgs {
    const uint8_t *x, *xp, *w, *wp;      // codes and powers
    const float *bias, *residual;
    void* out;
    int64_t n;
    int ci, co, act, out_dtype;
    int vec;       // outputs of a row in whole aligned pieces of 8 (co a multiple of it), of 4, or 0
    int tiles;
};

__device__ __forceinline__ f32x4_t scaled_product(u32x4_t a0, u32x4_t a1, uint32_t ap, u32x4_t b0, u32x4_t b1, uint32_t bp, f32x4_t c) {
    i32x8_t a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = a0[i], a[4 + i] = a1[i], b[i] = b0[i], b[4 + i] = b1[i];
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)ap, 0, (int)bp);
}

// Sixteen codes of one block as bf16 with their power.
__device__ __forceinline__ void widen(u32x4_t codes, uint32_t power, u32x4_t& lo, u32x4_t& hi) {
    const float s = mx_scale(power);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[i], s, false));
        const uint32_t b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[i], s, true));
        if (i < 2) lo[2 * i] = a, lo[2 * i + 1] = b;
        else hi[2 * i - 4] = a, hi[2 * i - 3] = b;
    }
}
__device__ __forceinline__ f32x4_t exact_product(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// The piece of 16 codes that lane group g holds as the first or second half of its operand. The scaled instruction
// wants channels 16 g and 64 + 16 g, and applies the power of block g of four; in the other form a lane takes its own
// block, 32 g and 32 g + 16.
template <bool EXACT>
__device__ __forceinline__ constexpr int operand_piece(int g, int half) { return EXACT ? 2 * g + half : g + 4 * half; }

__device__ __forceinline__ f32x4_t silu4(f32x4_t y) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = y[i] / (1.f + __expf(-y[i]));
    return y;
}

// An output, its bias and activation applied.
__device__ __forceinline__ void finish1(const LinearArgs& a, int64_t row, int o, float y) {
    const int64_t at = row * a.co + o;
    if (a.residual) y += a.residual[at];
    if (a.out_dtype == TSP_F32) static_cast<float*>(a.out)[at] = y;
    else static_cast<uint16_t*>(a.out)[at] = a.out_dtype == TSP_BF16 ? f32_to_bf16_bits(y) : f32_to_f16_bits(y);
}
// EACH pieces of four consecutive outputs of a row, which begin on a boundary of their size (co is a multiple of four): the residual's
// (zeros without one), and the outputs, the residual added.
template <int EACH>
__device__ __forceinline__ void residual4(const LinearArgs& a, int64_t row, int o, f32x4_t (&r)[EACH]) {
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        r[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (a.residual && row < a.n && o + 4 * k < a.co) r[k] = *reinterpret_cast<const f32x4_t*>(a.residual + row * a.co + o + 4 * k);
    }
}
template <int EACH>
__device__ __forceinline__ void finish4(const LinearArgs& a, int64_t row, int o, const f32x4_t (&y)[EACH]) {
    if (o >= a.co) return;
    const int64_t at = row * a.co + o;
    if (a.out_dtype == TSP_F32) {
#pragma unroll
        for (int k = 0; k < EACH; ++k)
            if (o + 4 * k < a.co) *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + at + 4 * k) = y[k];
        return;
    }
    uint2 p[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        if (a.out_dtype == TSP_BF16) p[k] = uint2{f32x2_to_bf16x2_bits(y[k][0], y[k][1]), f32x2_to_bf16x2_bits(y[k][2], y[k][3])};
        else p[k] = uint2{f32_to_f16_bits(y[k][0]) | ((uint32_t)f32_to_f16_bits(y[k][1]) << 16), f32_to_f16_bits(y[k][2]) | ((uint32_t)f32_to_f16_bits(y[k][3]) << 16)};
    }
    uint16_t* out = static_cast<uint16_t*>(a.out) + at;
    if constexpr (EACH == 2) {
        if (a.vec == 8) {       // (rows of whole 16-byte pieces)
            *reinterpret_cast<u32x4_t*>(out) = u32x4_t{p[0].x, p[0].y, p[1].x, p[1].y};
            return;
        }
    }
#pragma unroll
    for (int k = 0; k < EACH; ++k)
        if (o + 4 * k < a.co) *reinterpret_cast<uint2*>(out + 4 * k) = p[k];
}

// Waits for all but the last N of this wave's loads and for its LDS reads, and then for the workgroup. (A plain barrier
// waits for every load.)
template <int N>
__device__ __forceinline__ void loads_and_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A tile of TX rows x TW outputs by WX x WW waves, in steps of 128 channels that STAGES buffers hold, so that STAGES - 1 of them
// are on their way. Codes go straight from memory to LDS, 16 bytes a lane, each from the piece that belongs in its place:
// piece p of row r lies in slot p ^ (r % 8), so that eight rows cover all banks. Powers go there too, a row's four of a step
// at once, or with ANY (channels that are no whole steps) one a load. Rows and channels past the ends read as zeros (out of the
// buffer's range), and so do steps past the last, which keep the count of loads that are on their way. Each buffer is
// an array of its own: of one array the compiler would have every load land before any of it is read.
template <int TX, int TW, int WX, int WW, int STAGES, bool EXACT, bool ANY>
__global__ __launch_bounds__(WX * WW * 64) void k_linear_mx(LinearArgs a) {
#ifdef __HIP_DEVICE_COMPILE__       // (the host pass does not know the loads)
    constexpr int NW = WX * WW, NT = NW * 64, RX = TX / WX / 16, RW = TW / WW / 16, ROWS = TX + TW;
    constexpr int LOADS_X = TX * LM_K / 1024 / NW, LOADS_W = TW * LM_K / 1024 / NW, PARTS = ANY ? 4 : 1;
    constexpr int PROWS = (ROWS + NT - 1) / NT * NT, LOADS = LOADS_X + LOADS_W + PARTS * PROWS / NT;      // (every wave has as many)
    static_assert(TX % 64 == 0 && LOADS_X > 0 && LOADS_W > 0 && STAGES >= 2 && STAGES <= 4, "whole loads a wave");
    static_assert(TX * LM_K % (1024 * NW) == 0 && TW * LM_K % (1024 * NW) == 0, "whole loads a wave");
    __shared__ __attribute__((aligned(16))) uint8_t sC0[ROWS * LM_K], sC1[ROWS * LM_K], sC2[STAGES > 2 ? ROWS * LM_K : 16], sC3[STAGES > 3 ? ROWS * LM_K : 16];
    __shared__ uint32_t sP0[PARTS * PROWS], sP1[PARTS * PROWS], sP2[STAGES > 2 ? PARTS * PROWS : 1], sP3[STAGES > 3 ? PARTS * PROWS : 1];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    // An eighth of the tiles each XCD, which takes every eighth workgroup and has an L2 of its own: bands of BAND tiles of
    // rows, column by column, so that what runs on it at once is a patch of about as many rows as outputs.
    constexpr int BAND = 8;
    const int tiles_w = (a.co + TW - 1) / TW, tiles_x = a.tiles / tiles_w;
    const int tile = (int)(blockIdx.x % 8) * (int)(gridDim.x / 8) + (int)(blockIdx.x / 8);
    if (tile >= a.tiles) return;
    const int band = tile / (BAND * tiles_w), in = tile - band * BAND * tiles_w, high = min(BAND, tiles_x - band * BAND);
    const int64_t x0 = (int64_t)(band * BAND + in % high) * TX;
    const int w0 = in / high * TW, blocks = a.ci / MX_BLOCK;
    const int rows_x = (int)min((int64_t)TX, a.n - x0), rows_w = min(TW, a.co - w0);
    auto buffer = [](const uint8_t* p, int bytes) __attribute__((always_inline)) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, bytes, 0x00027000); };
    const auto rx = buffer(a.x + x0 * a.ci, rows_x * a.ci), rw = buffer(a.w + (int64_t)w0 * a.ci, rows_w * a.ci);
    const auto rxp = buffer(a.xp + x0 * blocks, rows_x * blocks), rwp = buffer(a.wp + (int64_t)w0 * blocks, rows_w * blocks);
    constexpr int NOWHERE = 1 << 30;      // past every tile's bytes
    const int row8 = lane >> 3, piece8 = ((lane & 7) ^ (row8 & 7)) * 16;
    using lds = __attribute__((address_space(3))) void*;
    auto stage = [&](int k0, uint8_t* sC, uint32_t* sP) __attribute__((always_inline)) {
        const int at = k0 + piece8 < a.ci ? row8 * a.ci + k0 + piece8 : NOWHERE;
#pragma unroll
        for (int i = 0; i < LOADS_X; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds)(sC + (i * NW + wave) * 1024), 16, at + (i * NW + wave) * 8 * a.ci, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < LOADS_W; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds)(sC + TX * LM_K + (i * NW + wave) * 1024), 16, at + (i * NW + wave) * 8 * a.ci, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < PROWS / NT; ++i)
#pragma unroll
            for (int j = 0; j < PARTS; ++j) {
                const int r0 = (i * NW + wave) * 64, b = k0 / MX_BLOCK + j;      // 64 rows of x, or of W
                const int from = b < blocks && r0 < ROWS ? ((r0 < TX ? r0 : r0 - TX) + lane) * blocks + b : NOWHERE;
                if (r0 < TX) __builtin_amdgcn_raw_ptr_buffer_load_lds(rxp, (lds)(sP + j * PROWS + r0), ANY ? 1 : 4, from, 0, 0, 0);
                else __builtin_amdgcn_raw_ptr_buffer_load_lds(rwp, (lds)(sP + j * PROWS + r0), ANY ? 1 : 4, from, 0, 0, 0);
            }
    };
    const int wx = wave / WW * RX * 16, ww = wave % WW * RW * 16;      // the wave's first rows of the tile
    f32x4_t acc[RW][RX];
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int j = 0; j < RX; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // Rows of W follow x's. The second half of an operand is the piece whose number differs in one bit.
    constexpr int flip = (operand_piece<EXACT>(0, 0) ^ operand_piece<EXACT>(0, 1)) * 16;
    const int swizzled = (operand_piece<EXACT>(g, 0) ^ (r16 & 7)) * 16;
    const int x_at = (wx + r16) * LM_K + swizzled, w_at = (TX + ww + r16) * LM_K + swizzled;
    const int xp_at = (wx + r16) * 4 + (ANY ? g * PROWS * 4 : g), wp_at = xp_at + (TX + ww - wx) * 4;
    auto multiply = [&](const uint8_t* sC, const uint32_t* sP) __attribute__((always_inline)) {
        // (rows 16 apart have one swizzle, and places that differ by a constant)
        auto piece = [&](bool of_w, int i, int half) __attribute__((always_inline)) {
            return *reinterpret_cast<const u32x4_t*>(sC + ((of_w ? w_at : x_at) ^ (half ? flip : 0)) + i * 16 * LM_K);
        };
        auto power = [&](bool of_w, int i) __attribute__((always_inline)) {
            return (uint32_t) reinterpret_cast<const uint8_t*>(sP)[(of_w ? wp_at : xp_at) + i * 64];
        };
        // (the smaller side is held, the other comes by)
        if constexpr (EXACT) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                u32x4_t w[RW][2];
#pragma unroll
                for (int i = 0; i < RW; ++i) widen(piece(true, i, half), power(true, i), w[i][0], w[i][1]);
#pragma unroll
                for (int j = 0; j < RX; ++j) {
                    u32x4_t x[2];
                    widen(piece(false, j, half), power(false, j), x[0], x[1]);
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int i = 0; i < RW; ++i) acc[i][j] = exact_product(w[i][s], x[s], acc[i][j]);
                }
            }
        } else {
            u32x4_t w[RW][2];
            uint32_t wp[RW];
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                wp[i] = power(true, i);
                w[i][0] = piece(true, i, 0);
                w[i][1] = piece(true, i, 1);
            }
#pragma unroll
            for (int j = 0; j < RX; ++j) {
                const uint32_t xp = power(false, j);
                const u32x4_t x0 = piece(false, j, 0), x1 = piece(false, j, 1);
#pragma unroll
                for (int i = 0; i < RW; ++i) acc[i][j] = scaled_product(w[i][0], w[i][1], wp[i], x0, x1, xp, acc[i][j]);
            }
        }
    };
    auto codes = [&](auto i) __attribute__((always_inline)) -> uint8_t* {
        constexpr int I = decltype(i)::value;
        if constexpr (I == 0) return sC0;
        else if constexpr (I == 1) return sC1;
        else if constexpr (I == 2) return sC2;
        else return sC3;
    };
    auto powers = [&](auto i) __attribute__((always_inline)) -> uint32_t* {
        constexpr int I = decltype(i)::value;
        if constexpr (I == 0) return sP0;
        else if constexpr (I == 1) return sP1;
        else if constexpr (I == 2) return sP2;
        else return sP3;
    };
    // The step at k0 in buffer I; the one STAGES - 1 later takes the place of the step before.
    auto step = [&](int k0, auto i) __attribute__((always_inline)) {
        constexpr int I = decltype(i)::value, LAST = (I + STAGES - 1) % STAGES;
        using Last = std::integral_constant<int, LAST>;
        if (k0 >= a.ci) return;
        loads_and_barrier<LOADS * (STAGES - 2)>();
        stage(k0 + (STAGES - 1) * LM_K, codes(Last{}), powers(Last{}));
        multiply(codes(i), powers(i));
    };
    using std::integral_constant;
    stage(0, sC0, sP0);
    if constexpr (STAGES > 2) stage(LM_K, sC1, sP1);
    if constexpr (STAGES > 3) stage(2 * LM_K, sC2, sP2);
    for (int k0 = 0; k0 < a.ci; k0 += STAGES * LM_K) {
        step(k0, integral_constant<int, 0>{});
        step(k0 + LM_K, integral_constant<int, 1>{});
        if constexpr (STAGES > 2) step(k0 + 2 * LM_K, integral_constant<int, 2>{});
        if constexpr (STAGES > 3) step(k0 + 3 * LM_K, integral_constant<int, 3>{});
    }
    loads_and_barrier<0>();      // (no load is on its way to LDS any more, and none of it is read)
    // Rows leave in whole pieces: 16 of them at a time go through the wave's own part of LDS, 16-byte piece p of row r in
    // place p ^ r.
    constexpr int PIECES = RW * 4;
    static_assert(NW * 16 * PIECES * 16 <= ROWS * LM_K && (PIECES == 16 || PIECES == 8), "the waves' parts fit a buffer");
    char* s = reinterpret_cast<char*>(sC0) + wave * (16 * PIECES * 16);
    // (two pieces of four outputs a lane where they leave in 16 bits, one in 32, whose residual's are read 16 rows
    // ahead: 35,001 x 4,096 -> 1,024 337 us, 319 so. In 16 bits that took 4 % where there is none)
    constexpr int EACH = EXACT ? 1 : 2, LANES = PIECES / EACH, TURNS = 16 * LANES / 64;
    f32x4_t ahead[EXACT ? 2 : 1][TURNS][EACH];
    auto fetch = [&](int j, f32x4_t (&r)[TURNS][EACH]) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < TURNS; ++q)
            residual4<EACH>(a, x0 + wx + j * 16 + (q * 64 + lane) / LANES, w0 + ww + (q * 64 + lane) % LANES * EACH * 4, r[q]);
    };
    const bool adds = a.residual && a.vec;
    if (EXACT && adds) fetch(0, ahead[0]);
    f32x4_t bias[RW];
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int o = w0 + ww + i * 16 + 4 * g + e;
            bias[i][e] = a.bias && o < a.co ? a.bias[o] : 0.f;
        }
#pragma unroll
    for (int j = 0; j < RX; ++j) {
        if constexpr (EXACT)
            if (adds && j + 1 < RX) fetch(j + 1, ahead[(j + 1) % 2]);
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            f32x4_t y = acc[i][j] + bias[i];
            if (a.act) y = silu4(y);
            *reinterpret_cast<f32x4_t*>(s + (r16 * PIECES + ((i * 4 + g) ^ (r16 & (PIECES - 1)))) * 16) = y;
        }
        asm volatile("" ::: "memory");      // (the wave's own writes; LDS takes them in order)
        const int64_t row0 = x0 + wx + j * 16;
        if (a.vec == 0) {
            for (int at = lane; at < 16 * PIECES * 4; at += 64) {
                const int r = at / (PIECES * 4), e = at % (PIECES * 4);
                const float y = *reinterpret_cast<const float*>(s + (r * PIECES + ((e / 4) ^ (r & (PIECES - 1)))) * 16 + e % 4 * 4);
                if (row0 + r < a.n && w0 + ww + e < a.co) finish1(a, row0 + r, w0 + ww + e, y);
            }
        } else {
            if (!EXACT && adds) fetch(j, ahead[0]);
#pragma unroll
            for (int q = 0; q < TURNS; ++q) {
                const int r = (q * 64 + lane) / LANES, p = (q * 64 + lane) % LANES * EACH;
                f32x4_t y[EACH];
#pragma unroll
                for (int k = 0; k < EACH; ++k) {
                    y[k] = *reinterpret_cast<const f32x4_t*>(s + (r * PIECES + ((p + k) ^ (r & (PIECES - 1)))) * 16);
                    if (adds) y[k] += ahead[EXACT ? j % 2 : 0][q][k];
                }
                if (row0 + r < a.n) finish4<EACH>(a, row0 + r, w0 + ww + p * 4, y);
            }
        }
        asm volatile("" ::: "memory");
    }
#endif
}

// Up to RT * 16 rows: W is all there is to read. Eight waves take WT * 16 outputs, every eighth step of 128 channels each,
// straight from memory to the operands; their sums meet in LDS, in the waves' order.
constexpr int LF_NW = 8;
template <int RT, int WT, bool EXACT>
__global__ __launch_bounds__(LF_NW * 64) void k_linear_mx_few(LinearArgs a) {
    __shared__ f32x4_t sAcc[LF_NW][WT * RT][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int o0 = blockIdx.x * (WT * 16), blocks = a.ci / MX_BLOCK;
    f32x4_t acc[WT][RT];
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    struct Operand {
        u32x4_t c[2];
        uint32_t p;
    };
    auto load = [&](const uint8_t* codes, const uint8_t* powers, int row, bool there, int k0) __attribute__((always_inline)) {
        Operand x{{{0, 0, 0, 0}, {0, 0, 0, 0}}, 0};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = k0 + operand_piece<EXACT>(g, half) * 16;
            if (there && k < a.ci) x.c[half] = *reinterpret_cast<const u32x4_t*>(codes + (int64_t)row * a.ci + k);
        }
        if (there && k0 / MX_BLOCK + g < blocks) x.p = powers[(int64_t)row * blocks + k0 / MX_BLOCK + g];
        return x;
    };
    auto multiply = [&](const Operand (&w)[WT], const Operand (&x)[RT]) __attribute__((always_inline)) {
        if constexpr (EXACT) {
            u32x4_t wf[WT][4];
#pragma unroll
            for (int i = 0; i < WT; ++i) {
                widen(w[i].c[0], w[i].p, wf[i][0], wf[i][1]);
                widen(w[i].c[1], w[i].p, wf[i][2], wf[i][3]);
            }
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                u32x4_t xf[4];
                widen(x[j].c[0], x[j].p, xf[0], xf[1]);
                widen(x[j].c[1], x[j].p, xf[2], xf[3]);
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int i = 0; i < WT; ++i) acc[i][j] = exact_product(wf[i][s], xf[s], acc[i][j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int i = 0; i < WT; ++i) acc[i][j] = scaled_product(w[i].c[0], w[i].c[1], w[i].p, x[j].c[0], x[j].c[1], x[j].p, acc[i][j]);
        }
    };
    constexpr int AHEAD = RT * WT <= 2 ? 4 : 2, STEP = LF_NW * LM_K;      // steps on their way
    for (int k0 = wave * LM_K; k0 < a.ci; k0 += AHEAD * STEP) {
        Operand w[AHEAD][WT], x[AHEAD][RT];
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) {
            const int k = k0 + s * STEP;
#pragma unroll
            for (int i = 0; i < WT; ++i) w[s][i] = load(a.w, a.wp, o0 + i * 16 + r16, o0 + i * 16 + r16 < a.co && k < a.ci, k);
#pragma unroll
            for (int j = 0; j < RT; ++j) x[s][j] = load(a.x, a.xp, j * 16 + r16, j * 16 + r16 < a.n && k < a.ci, k);
        }
#pragma unroll
        for (int s = 0; s < AHEAD; ++s)
            if (k0 + s * STEP < a.ci) multiply(w[s], x[s]);
    }
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j) sAcc[wave][i * RT + j][lane] = acc[i][j];
    __syncthreads();
    if (wave >= WT * RT) return;
    f32x4_t y = sAcc[0][wave][lane];
#pragma unroll
    for (int w = 1; w < LF_NW; ++w) y += sAcc[w][wave][lane];
    const int64_t row = wave % RT * 16 + r16;
    const int o = o0 + wave / RT * 16 + 4 * g;
    if (row >= a.n) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (a.bias && o + e < a.co) y[e] += a.bias[o + e];
    if (a.act) y = silu4(y);
    if (a.vec) {
        f32x4_t one[1];
        residual4<1>(a, row, o, one);
        one[0] += y;
        finish4<1>(a, row, o, one);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (o + e < a.co) finish1(a, row, o + e, y[e]);
    }
}

// The tile with the least time of its rounds. A step of 128 channels takes a workgroup so many us where the device is full
// (8,192 rows and outputs of 8,192 channels) and where it has a CU to itself (1,000 rows, 4,096 -> 1,024); a tile's first loads
// and its rows' way out some more, twice that where a residual is read. (The numbers were fitted while bf16's 256 x 256 tile had
// eight waves, and with input sets that took turns: they say 549 us for 8,192^3 in bf16. For all of what follows they still name
// the fastest tile.) us by tiles of 256 x 256, 192 x 256 (fp32 out alone), 128 x 128, 128 x 64 and 64 x 64, bf16 out / fp32 out with a
// residual: 35,001 rows, 4,096 -> 1,024: 185, -, 204, 264, 311 / 368, 304, 323, 377, 430; 1,024 -> 4,096: 172, -, 205, 247, 363 /
// 427, 406, 403, 451, 540; 12,345 rows, 1,024 -> 1,024: 21, -, 24, 28, 35 / 45, 62, 43, 44, 49; 8,192 rows, 8,192 -> 8,192, no
// residual: 467, -, 654, 893, 1,157 / 857, 953, 992, 1,240, 1,358; 1,000 rows, 4,096 -> 1,024: 47, -, 36, 20, 12 / 98, 84, 45, 25, 18.
// (More waves a tile than its products need hide the loads of what lies in memory: 128 x 128 by eight takes 351 where four take
// 363. 256 x 128 with two steps on their way: no faster than the best.)
int linear_shape(int64_t n, int ci, int co, bool exact, bool residual) {
    struct Times { double full, alone, rest; };
    struct Shape { int x, w, slots; Times by[2]; };
    static const Shape shapes[5] = {{256, 256, 256, {{2.05, 1.56, 6.}, {3.4, 2.7, 10.}}}, {192, 256, 256, {{}, {2.6, 2.2, 9.}}},
                                    {128, 128, 512, {{1.4, 1., 3.}, {1.95, 1.3, 3.2}}}, {128, 64, 512, {{0.95, 0.55, 2.5}, {1.23, 0.74, 2.}}},
                                    {64, 64, 512, {{0.55, 0.42, 2.}, {0.74, 0.55, 1.5}}}};
    int best = 0;
    double least = 1e30;
    for (int i = 0; i < 5; ++i) {
        if (i == 1 && !exact) continue;
        const Shape& s = shapes[i];
        const Times& t = s.by[exact];
        const int64_t tiles = ceil_div(n, s.x) * ceil_div(co, s.w), last = tiles % s.slots, steps = ceil_div(ci, LM_K);
        const double out = t.rest * (residual ? 2. : 1.), full = steps * t.full + out, alone = steps * t.alone + out;
        // (a round of at most a workgroup a CU is as long as one alone; one of nearly 256 large ones is not)
        const double time = (double)(tiles / s.slots) * full + (last == 0 ? 0. : last <= (s.slots == 256 ? 128 : 256) ? alone : full);
        if (time < least) least = time, best = i;
    }
    return best;
}

}  // namespace
}  // namespace tsp

using namespace tsp;

extern "C" size_t tsp_linear_mx_workspace_bytes(int64_t n, int ci, int co) {
    (void)n, (void)ci, (void)co;
    return 0;
}

extern "C" int tsp_linear_mx(const void* d_x, const uint8_t* d_x_powers, int64_t n, int ci, const void* d_w, const uint8_t* d_w_powers,
                             const float* d_bias, int co, int act, const float* d_residual, void* d_out, int out_dtype, void* d_workspace,
                             size_t workspace_bytes, void* stream) {
    clear_error();
    (void)d_workspace, (void)workspace_bytes;      // (none is needed)
    TSP_REQUIRE(n >= 0 && n < (1ll << 31) && ci > 0 && ci <= (1 << 20) && co > 0 && co <= (1 << 24), TSP_ERR_INVALID,
                "tsp_linear_mx: n=%lld ci=%d co=%d out of range", (long long)n, ci, co);
    TSP_REQUIRE(dtype_valid(out_dtype) && (act == 0 || act == 1), TSP_ERR_INVALID, "tsp_linear_mx: bad dtype or act");
    TSP_REQUIRE(ci % MX_BLOCK == 0, TSP_ERR_UNSUPPORTED, "tsp_linear_mx: ci=%d (need a multiple of %d)", ci, MX_BLOCK);
    if (n == 0) return TSP_OK;
    TSP_REQUIRE(d_x && d_x_powers && d_w && d_w_powers && d_out, TSP_ERR_INVALID, "tsp_linear_mx: null pointer");
    TSP_REQUIRE(reinterpret_cast<uintptr_t>(d_x) % 16 == 0 && reinterpret_cast<uintptr_t>(d_w) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(d_x_powers) % 4 == 0 && reinterpret_cast<uintptr_t>(d_w_powers) % 4 == 0,
                TSP_ERR_INVALID, "tsp_linear_mx: codes must be 16-byte aligned, powers 4-byte aligned");
    const size_t out_bytes = (size_t)n * co * dtype_size(out_dtype), blocks = ci / MX_BLOCK;
    TSP_REQUIRE(!overlap(d_out, out_bytes, d_x, (size_t)n * ci) && !overlap(d_out, out_bytes, d_w, (size_t)co * ci) &&
                    !overlap(d_out, out_bytes, d_x_powers, n * blocks) && !overlap(d_out, out_bytes, d_w_powers, co * blocks) &&
                    !overlap(d_out, out_bytes, d_bias, (size_t)co * 4) &&
                    (!overlap(d_out, out_bytes, d_residual, (size_t)n * co * 4) || (d_out == d_residual && out_dtype == TSP_F32)),
                TSP_ERR_INVALID, "tsp_linear_mx: out overlaps an input (it may be an f32 residual, or apart)");
    const int vec = co % 4 || reinterpret_cast<uintptr_t>(d_out) % 16 || reinterpret_cast<uintptr_t>(d_residual) % 16 ? 0 : co % 8 ? 4 : 8;
    LinearArgs a{static_cast<const uint8_t*>(d_x), d_x_powers, static_cast<const uint8_t*>(d_w), d_w_powers, d_bias, d_residual,
                       d_out, n, ci, co, act, out_dtype, vec, 0};
    hipStream_t s = as_stream(stream);
    using std::integral_constant;
    auto by_form = [&](auto&& go) {
        if (out_dtype == TSP_F32) go(std::true_type{});
        else go(std::false_type{});
    };
    // Few rows by the other kernel, with two tiles of outputs a workgroup where there are many: us, by it (one tile, two) and by
    // tiles, in bf16 / fp32. 5 rows, 1,024 -> 4,096: 3.9 (4.1) and 4.9 / 4.2 (5.0) and 6.1; 4,096 -> 5,000: 10.1 (9.1) and 9.8 / 11.0
    // (10.2) and 15.3, -> 8,192: 10.3 (9.3) and 13.1 / 11.0 (10.2) and 16.0, -> 16,384: 18.1 (17.7) and 14.8 / 22.0 (20.3) and 17.6.
    // 32 rows, 1,024 -> 1,024: 4.4 (5.2) and 5.2 / 5.4 (5.9) and 6.8; 4,096 -> 1,024: 10.3 (13.1) and 9.9 / 10.8 (13.3) and 15.3,
    // -> 8,192: 19.9 (14.0) and 13.5 / 21.0 (14.3) and 16.6. 64 rows, 1,024 -> 1,024: 6.0 (6.8) and 5.0 / 6.5 (7.6) and 6.4.
    const bool wide = co > 4096;
    if (co <= 8192 && n <= (out_dtype == TSP_F32 ? (wide ? 32 : 48) : wide ? 16 : 32)) {
        by_form([&](auto exact) {
            constexpr bool EXACT = decltype(exact)::value;
            auto few = [&](auto rt, auto wt) {
                constexpr int RT = decltype(rt)::value, WT = decltype(wt)::value;
                hipLaunchKernelGGL((k_linear_mx_few<RT, WT, EXACT>), dim3((unsigned)ceil_div(co, 16 * WT)), dim3(LF_NW * 64), 0, s, a);
            };
            auto by_rows = [&](auto wt) {
                if (n <= 16) few(integral_constant<int, 1>{}, wt);
                else if constexpr (EXACT || decltype(wt)::value == 1) {
                    if (n <= 32) few(integral_constant<int, 2>{}, wt);
                    else if constexpr (EXACT && decltype(wt)::value == 1) few(integral_constant<int, 4>{}, wt);
                }
            };
            if (wide) by_rows(integral_constant<int, 2>{});
            else by_rows(integral_constant<int, 1>{});
        });
        TSP_CHECK_LAUNCH();
        return TSP_OK;
    }
    auto go = [&](auto tx, auto tw, auto wx, auto ww, auto stages, auto exact, auto any) -> int {
        constexpr int TX = decltype(tx)::value, TW = decltype(tw)::value, WX = decltype(wx)::value, WW = decltype(ww)::value, ST = decltype(stages)::value;
        const int64_t tiles = ceil_div(n, TX) * ceil_div(co, TW);
        TSP_REQUIRE(tiles * WX * WW * 64 < (1ll << 31), TSP_ERR_INVALID, "tsp_linear_mx: too many rows and outputs");
        a.tiles = (int)tiles;
        hipLaunchKernelGGL((k_linear_mx<TX, TW, WX, WW, ST, decltype(exact)::value, decltype(any)::value>), dim3((unsigned)ceil_div(tiles, 8) * 8),
                           dim3(WX * WW * 64), 0, s, a);
        return TSP_OK;
    };
    const int shape = linear_shape(n, ci, co, out_dtype == TSP_F32, d_residual != nullptr);
    int rc = TSP_OK;
    by_form([&](auto exact) {
        auto by_steps = [&](auto any) {
            // (16 waves of 64 x 64 where 16-bit outputs' products are short; eight of 128 x 64 for fp32's, or channels that are
            // no whole steps, whose powers would take more LDS by 16: 8,192^3 in bf16 467 and 512 us, in fp32 1,092 and 857)
            constexpr int WX = decltype(exact)::value || decltype(any)::value ? 2 : 4;
            const integral_constant<int, 64> c64;
            const integral_constant<int, 128> c128;
            const integral_constant<int, 256> c256;
            const integral_constant<int, 2> c2;
            const integral_constant<int, 3> c3;
            const integral_constant<int, 4> c4;
            if (shape == 0) rc = go(c256, c256, integral_constant<int, WX>{}, c4, c2, exact, any);
            else if (shape == 2) rc = go(c128, c128, c2, c4, c2, exact, any);
            else if (shape == 3) rc = go(c128, c64, c4, c2, c3, exact, any);
            else if (shape == 4) rc = go(c64, c64, c2, c2, c4, exact, any);
            else if constexpr (decltype(exact)::value) rc = go(integral_constant<int, 192>{}, c256, c2, c4, c2, exact, any);
        };
        if (ci % LM_K == 0) by_steps(std::false_type{});
        else by_steps(std::true_type{});
    });
    if (rc != TSP_OK) return rc;
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
