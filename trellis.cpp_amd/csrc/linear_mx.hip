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
    int vec;       // rows of out and residual in whole pieces of four
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
__device__ __forceinline__ int operand_piece(int g, int half) { return EXACT ? 2 * g + half : g + 4 * half; }

// Four consecutive outputs of a row.
__device__ __forceinline__ void finish(const LinearArgs& a, int64_t row, int o, f32x4_t y) {
    if (row >= a.n || o >= a.co) return;
    const int64_t at = row * a.co + o;
    const int count = min(4, a.co - o);
    if (a.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < count) y[i] += a.bias[o + i];
    }
    if (a.act) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = y[i] / (1.f + __expf(-y[i]));
    }
    if (a.vec) {
        if (a.residual) y += *reinterpret_cast<const f32x4_t*>(a.residual + at);
        if (a.out_dtype == TSP_F32) {
            *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + at) = y;
        } else {
            uint2 p;
            if (a.out_dtype == TSP_BF16) p = uint2{f32x2_to_bf16x2_bits(y[0], y[1]), f32x2_to_bf16x2_bits(y[2], y[3])};
            else p = uint2{f32_to_f16_bits(y[0]) | ((uint32_t)f32_to_f16_bits(y[1]) << 16), f32_to_f16_bits(y[2]) | ((uint32_t)f32_to_f16_bits(y[3]) << 16)};
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = p;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= count) break;
        const float v = y[i] + (a.residual ? a.residual[at + i] : 0.f);
        if (a.out_dtype == TSP_F32) static_cast<float*>(a.out)[at + i] = v;
        else static_cast<uint16_t*>(a.out)[at + i] = a.out_dtype == TSP_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
    }
}

// A tile of TX rows x TW outputs by WX x WW waves. Codes go straight from memory to LDS, 16 bytes a lane, each from the
// piece that belongs in its place: piece p of row r lies in slot p ^ (r % 8), so that eight rows cover all banks.
// Rows and channels past the ends read as zeros (out of the buffer's range).
template <int TX, int TW, int WX, int WW, bool EXACT>
__global__ __launch_bounds__(WX * WW * 64) void k_linear_mx(LinearArgs a) {
    constexpr int NW = WX * WW, NT = NW * 64, RX = TX / WX / 16, RW = TW / WW / 16;
    constexpr int LOADS_X = TX * LM_K / 1024 / NW, LOADS_W = TW * LM_K / 1024 / NW;
    static_assert((TX + TW) % NT == 0 && LOADS_X > 0 && LOADS_W > 0, "whole loads a wave");
    __shared__ __attribute__((aligned(16))) uint8_t sX[2][TX * LM_K], sW[2][TW * LM_K];
    __shared__ uint32_t sP[2][TX + TW];      // the rows' four powers of a step, x's first
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int tiles_w = (a.co + TW - 1) / TW;
    const int64_t x0 = (int64_t)(blockIdx.x / tiles_w) * TX;
    const int w0 = (int)(blockIdx.x % tiles_w) * TW;
    const int rows_x = (int)min((int64_t)TX, a.n - x0), rows_w = min(TW, a.co - w0);
    const auto rx = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x + x0 * a.ci), (short)0, rows_x * a.ci, 0x00027000);
    const auto rw = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + (int64_t)w0 * a.ci), (short)0, rows_w * a.ci, 0x00027000);
    constexpr int NOWHERE = 1 << 30;      // past every tile's bytes
    auto stage = [&](int k0, int buf) __attribute__((always_inline)) {
        const int row = lane >> 3, k = k0 + ((lane & 7) ^ (row & 7)) * 16;
        const int at = k < a.ci ? row * a.ci + k : NOWHERE;
#pragma unroll
        for (int i = 0; i < LOADS_X; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (__attribute__((address_space(3))) void*)(sX[buf] + (i * NW + wave) * 1024), 16,
                                                     at + (i * NW + wave) * 8 * a.ci, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < LOADS_W; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (__attribute__((address_space(3))) void*)(sW[buf] + (i * NW + wave) * 1024), 16,
                                                     at + (i * NW + wave) * 8 * a.ci, 0, 0, 0);
    };
    const int blocks = a.ci / MX_BLOCK;
    constexpr int EACH = (TX + TW) / NT;      // rows of powers a thread
    auto powers = [&](int k0, uint32_t (&p)[EACH]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int r = i * NT + threadIdx.x, row = r < TX ? r : r - TX, b = k0 / MX_BLOCK;
            const bool there = row < (r < TX ? rows_x : rows_w);
            const uint8_t* from = (r < TX ? a.xp + (x0 + row) * blocks : a.wp + (int64_t)(w0 + row) * blocks) + b;
            p[i] = 0;
            if (!there) continue;
            if (blocks % 4 == 0) {
                p[i] = *reinterpret_cast<const uint32_t*>(from);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (b + j < blocks) p[i] |= (uint32_t)from[j] << (8 * j);
            }
        }
    };
    auto put_powers = [&](int buf, const uint32_t (&p)[EACH]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) sP[buf][i * NT + threadIdx.x] = p[i];
    };
    const int wx = wave / WW * RX * 16, ww = wave % WW * RW * 16;      // the wave's first rows of the tile
    f32x4_t acc[RW][RX];
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int j = 0; j < RX; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto piece = [&](const uint8_t* s, int row, int half) __attribute__((always_inline)) {
        return *reinterpret_cast<const u32x4_t*>(s + row * LM_K + ((operand_piece<EXACT>(g, half) ^ (row & 7)) * 16));
    };
    uint32_t p[EACH];
    stage(0, 0);
    powers(0, p);
    put_powers(0, p);
    int buf = 0;
    for (int k0 = 0; k0 < a.ci; k0 += LM_K, buf ^= 1) {
        __builtin_amdgcn_s_waitcnt(0x0f70);      // this wave's own loads; the barrier says that every wave's have landed
        __syncthreads();
        const bool more = k0 + LM_K < a.ci;
        if (more) {
            stage(k0 + LM_K, buf ^ 1);
            powers(k0 + LM_K, p);
        }
        const uint8_t *px = reinterpret_cast<const uint8_t*>(sP[buf]) + g, *pw = px + TX * 4;
        if constexpr (EXACT) {
            u32x4_t x[RX][4];
#pragma unroll
            for (int j = 0; j < RX; ++j) {
                const int row = wx + j * 16 + r16;
                const uint32_t power = px[row * 4];
                widen(piece(sX[buf], row, 0), power, x[j][0], x[j][1]);
                widen(piece(sX[buf], row, 1), power, x[j][2], x[j][3]);
            }
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                const int row = ww + i * 16 + r16;
                const uint32_t power = pw[row * 4];
                u32x4_t w[4];
                widen(piece(sW[buf], row, 0), power, w[0], w[1]);
                widen(piece(sW[buf], row, 1), power, w[2], w[3]);
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int j = 0; j < RX; ++j) acc[i][j] = exact_product(w[s], x[j][s], acc[i][j]);
            }
        } else {
            u32x4_t x[RX][2];
            uint32_t xp[RX];
#pragma unroll
            for (int j = 0; j < RX; ++j) {
                const int row = wx + j * 16 + r16;
                xp[j] = px[row * 4];
                x[j][0] = piece(sX[buf], row, 0);
                x[j][1] = piece(sX[buf], row, 1);
            }
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                const int row = ww + i * 16 + r16;
                const uint32_t wp = pw[row * 4];
                const u32x4_t w0 = piece(sW[buf], row, 0), w1 = piece(sW[buf], row, 1);
#pragma unroll
                for (int j = 0; j < RX; ++j) acc[i][j] = scaled_product(w0, w1, wp, x[j][0], x[j][1], xp[j], acc[i][j]);
            }
        }
        if (more) put_powers(buf ^ 1, p);
    }
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int j = 0; j < RX; ++j) finish(a, x0 + wx + j * 16 + r16, w0 + ww + i * 16 + 4 * g, acc[i][j]);
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
    TSP_REQUIRE(n >= 0 && n < (1ll << 31) && ci > 0 && ci <= (1 << 20) && co > 0 && co <= (1 << 24), TSP_ERR_INVALID,
                "tsp_linear_mx: n=%lld ci=%d co=%d out of range", (long long)n, ci, co);
    TSP_REQUIRE(dtype_valid(out_dtype) && (act == 0 || act == 1), TSP_ERR_INVALID, "tsp_linear_mx: bad dtype or act");
    TSP_REQUIRE(ci % MX_BLOCK == 0, TSP_ERR_UNSUPPORTED, "tsp_linear_mx: ci=%d (need a multiple of %d)", ci, MX_BLOCK);
    if (n == 0) return TSP_OK;
    TSP_REQUIRE(d_x && d_x_powers && d_w && d_w_powers && d_out, TSP_ERR_INVALID, "tsp_linear_mx: null pointer");
    TSP_REQUIRE(reinterpret_cast<uintptr_t>(d_x) % 16 == 0 && reinterpret_cast<uintptr_t>(d_w) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(d_x_powers) % 4 == 0 && reinterpret_cast<uintptr_t>(d_w_powers) % 4 == 0,
                TSP_ERR_INVALID, "tsp_linear_mx: codes must be 16-byte aligned, powers 4-byte aligned");
    const size_t need = tsp_linear_mx_workspace_bytes(n, ci, co);
    TSP_REQUIRE(need == 0 || d_workspace, TSP_ERR_INVALID, "tsp_linear_mx: null workspace");
    TSP_REQUIRE(workspace_bytes >= need, TSP_ERR_WORKSPACE, "tsp_linear_mx: workspace of %zu bytes, needs %zu", workspace_bytes, need);
    const size_t out_bytes = (size_t)n * co * dtype_size(out_dtype), blocks = ci / MX_BLOCK;
    TSP_REQUIRE(!overlap(d_out, out_bytes, d_x, (size_t)n * ci) && !overlap(d_out, out_bytes, d_w, (size_t)co * ci) &&
                    !overlap(d_out, out_bytes, d_x_powers, n * blocks) && !overlap(d_out, out_bytes, d_w_powers, co * blocks) &&
                    !overlap(d_out, out_bytes, d_bias, (size_t)co * 4) &&
                    (!overlap(d_out, out_bytes, d_residual, (size_t)n * co * 4) || (d_out == d_residual && out_dtype == TSP_F32)),
                TSP_ERR_INVALID, "tsp_linear_mx: out overlaps an input (it may be an f32 residual, or apart)");
    const bool vec = co % 4 == 0 && !(reinterpret_cast<uintptr_t>(d_out) % 16 || reinterpret_cast<uintptr_t>(d_residual) % 16);
    const LinearArgs a{static_cast<const uint8_t*>(d_x), d_x_powers, static_cast<const uint8_t*>(d_w), d_w_powers, d_bias, d_residual,
                       d_out, n, ci, co, act, out_dtype, vec};
    hipStream_t s = as_stream(stream);
    const int64_t tiles = ceil_div(n, 128) * ceil_div(co, 128);
    TSP_REQUIRE(tiles < (1ll << 24), TSP_ERR_INVALID, "tsp_linear_mx: too many rows and outputs");
    if (out_dtype == TSP_F32) hipLaunchKernelGGL((k_linear_mx<128, 128, 2, 2, true>), dim3((unsigned)tiles), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_linear_mx<128, 128, 2, 2, false>), dim3((unsigned)tiles), dim3(256), 0, s, a);
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
