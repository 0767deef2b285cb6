// Root-mean-square norm of rows with the residual's addition before it and, where asked, an 8-bit output:
//   h = x + residual,  y = h / sqrt(mean(h^2) + eps) * gamma,  residual_out = h
// in fp32; the norm is of the sum before residual_out rounds it. In 8 bits y leaves as e4m3 codes and a power of two
// for every 32 channels (mx.hpp), the operands of tsp_linear_mx. tsp_mx_quantize rounds rows without a norm.
//
// Bound by memory: one read, one write. 35,001 rows of 1,024 (bf16 x, fp32 residual in and out, 8 bits out) take 76 us, 5.2 TB/s
// with part of it in the memory-side cache; 60,013 of 2,048 in bf16 187 us, 5.3 TB/s; the vector units are 15 % busy, and
// 5 rows take 2.6 us. A wave holds a row of up to 2,048 channels in registers, eight consecutive
// ones a lane and piece, four waves one of up to 8,192; gamma stays in registers while the wave goes over its
// rows. Four neighbouring lanes hold a block of 32, so that its largest value is two lane moves. Rows of no whole
// pieces are held in smaller ones up to 4,096 channels; longer ones, and whole pieces past 8,192 channels, are read twice, value by
// value, by a workgroup each: 8,000 rows of 8,192 in bf16 with a residual take 98 us (5.3 TB/s), of 12,288 565 and of 16,384 760 (1.4).
// tsp_mx_quantize: 35,001 rows of 1,024 bf16 17 us and 12,345 of 2,048 12.5 (6.2-6.4 TB/s, in part from the cache), of 35,001 x 4,096
// 79 (5.5).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "inverse_root.hpp"
#include "mx.hpp"

namespace tsp {
namespace {

constexpr int RN_NT = 256;
constexpr int RN_NONE = -1;      // no residual

struct RmsArgs {
    const void *x, *residual;
    const float* gamma;
    void *out, *residual_out;
    uint8_t* powers;
    int64_t n;
    int c, out_dtype;
    float eps, inv_c;
};

// One value; a block of 32 channels is 32 neighbouring threads'.
__device__ __forceinline__ float load1(const void* p, int dt, int64_t i) {
    return dt == TSP_F32 ? static_cast<const float*>(p)[i]
           : dt == TSP_BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]) : f16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}
__device__ __forceinline__ void store1(void* p, int dt, int64_t i, float v) {
    if (dt == TSP_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = dt == TSP_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
}
__device__ __forceinline__ void store_mx8(void* codes, uint8_t* powers, int64_t i, float v) {
    uint32_t m = abs_bits(v);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 32));
    const uint32_t power = mx_power<MX_E4M3>(m);
    s16x2_t c{0, 0};
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v, 0.f, mx_scale(power), false);
    static_cast<uint8_t*>(codes)[i] = (uint8_t)__builtin_bit_cast(uint32_t, c);
    if ((threadIdx.x & 31) == 0) powers[i / MX_BLOCK] = (uint8_t)power;
}
// A piece of V channels, 8, 4 or 1.
template <int DT, int V>
__device__ __forceinline__ void load_piece(const void* p, int64_t i, float (&v)[V]) {
    if constexpr (V == 8) {
        load8<DT>(p, i, v);
    } else if constexpr (V == 1) {
        v[0] = load1(p, DT, i);
    } else if constexpr (DT == TSP_F32) {
        const f32x4_t a = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = a[k];
    } else {
        const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        auto f = [](uint32_t w) { return DT == TSP_BF16 ? bf16_bits_to_f32((uint16_t)w) : f16_bits_to_f32((uint16_t)w); };
        v[0] = f(a.x), v[1] = f(a.x >> 16), v[2] = f(a.y), v[3] = f(a.y >> 16);
    }
}
template <int DT, int V>
__device__ __forceinline__ void store_piece(void* p, int64_t i, const float (&v)[V]) {
    if constexpr (V == 8) {
        store8<DT>(p, i, v);
    } else if constexpr (V == 1) {
        store1(p, DT, i, v[0]);
    } else if constexpr (DT == TSP_F32) {
        *reinterpret_cast<f32x4_t*>(static_cast<float*>(p) + i) = f32x4_t{v[0], v[1], v[2], v[3]};
    } else {
        auto two = [](float a, float b) {
            return DT == TSP_BF16 ? f32x2_to_bf16x2_bits(a, b) : f32_to_f16_bits(a) | ((uint32_t)f32_to_f16_bits(b) << 16);
        };
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = uint2{two(v[0], v[1]), two(v[2], v[3])};
    }
}

// A row by NW waves (1: four rows a workgroup), CHUNKS pieces of V channels a lane. (Pieces of 4 for rows of no
// whole 8, single values for others and tensors that are not aligned.)
template <int XDT, int RDT, int NW, int CHUNKS, int V>
__global__ __launch_bounds__(RN_NT) void k_rms_norm(RmsArgs a) {
    __shared__ float sum_of[2][4];
    const int lane = threadIdx.x % (NW * 64), wave = threadIdx.x / 64, pieces = a.c / V;
    float gamma[CHUNKS][V];
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
        const int piece = k * NW * 64 + lane;
#pragma unroll
        for (int e = 0; e < V; ++e) gamma[k][e] = 1.f;
        if (a.gamma && piece < pieces) load_piece<TSP_F32, V>(a.gamma, piece * V, gamma[k]);
    }
    int turn = 0;
    // (with NW = 4 the whole workgroup has one row, and leaves together)
    for (int64_t row = NW == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x; row < a.n; row += (int64_t)gridDim.x * (NW == 1 ? 4 : 1), turn ^= 1) {
        const int64_t base = row * a.c;
        float h[CHUNKS][V], q = 0.f;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int piece = k * NW * 64 + lane;
#pragma unroll
            for (int e = 0; e < V; ++e) h[k][e] = 0.f;
            if (piece < pieces) {
                load_piece<XDT, V>(a.x, base + piece * V, h[k]);
                if constexpr (RDT != RN_NONE) {
                    float r[V];
                    load_piece<RDT, V>(a.residual, base + piece * V, r);
#pragma unroll
                    for (int e = 0; e < V; ++e) h[k][e] += r[e];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
#pragma unroll
            for (int e = 0; e < V; ++e) q += h[k][e] * h[k][e];
        }
        q = group_sum<64>(q);
        if constexpr (NW > 1) {     // (two places taken in turn: one barrier a row)
            if ((threadIdx.x & 63) == 0) sum_of[turn][wave] = q;
            __syncthreads();
            q = (sum_of[turn][0] + sum_of[turn][1]) + (sum_of[turn][2] + sum_of[turn][3]);
        }
        const float scale = inverse_root(fmaf(q, a.inv_c, a.eps));
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int piece = k * NW * 64 + lane;
            if (piece >= pieces) break;      // (whole blocks' lanes, where blocks of 32 are asked for)
            const int64_t at = base + piece * V;
            if constexpr (RDT != RN_NONE) {
                if (a.residual_out) store_piece<RDT, V>(a.residual_out, at, h[k]);
            }
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = h[k][e] * scale * gamma[k][e];
            if (V != 4 && a.out_dtype == TSP_MX8) {
                if constexpr (V == 1) store_mx8(a.out, a.powers, at, y[0]);
                if constexpr (V == 8) {
                    const uint32_t power = mx_power_of<MX_E4M3>(y);
                    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.out) + at) = mx_codes8(y, power);
                    if ((lane & 3) == 0) a.powers[at / MX_BLOCK] = (uint8_t)power;
                }
            } else if (a.out_dtype == TSP_BF16) {
                store_piece<TSP_BF16, V>(a.out, at, y);
            } else if (a.out_dtype == TSP_F16) {
                store_piece<TSP_F16, V>(a.out, at, y);
            } else {
                store_piece<TSP_F32, V>(a.out, at, y);
            }
        }
    }
}

// Any row, twice, value by value.
__global__ __launch_bounds__(RN_NT) void k_rms_norm_any(RmsArgs a, int x_dtype, int residual_dtype) {
    __shared__ float sum_of[RN_NT / 64];
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
        const int64_t base = row * a.c;
        float q = 0.f;
        for (int i = threadIdx.x; i < a.c; i += RN_NT) {
            float h = load1(a.x, x_dtype, base + i);
            if (a.residual) h += load1(a.residual, residual_dtype, base + i);
            q += h * h;
        }
        q = group_sum<64>(q);
        if ((threadIdx.x & 63) == 0) sum_of[threadIdx.x / 64] = q;
        __syncthreads();
        q = (sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]);
        __syncthreads();
        const float scale = inverse_root(fmaf(q, a.inv_c, a.eps));
        for (int i = threadIdx.x; i < a.c; i += RN_NT) {
            float h = load1(a.x, x_dtype, base + i);
            if (a.residual) h += load1(a.residual, residual_dtype, base + i);
            if (a.residual_out) store1(a.residual_out, residual_dtype, base + i, h);
            const float y = h * scale * (a.gamma ? a.gamma[i] : 1.f);
            if (a.out_dtype == TSP_MX8) store_mx8(a.out, a.powers, base + i, y);
            else store1(a.out, a.out_dtype, base + i, y);
        }
    }
}

// Rows' values as they follow each other in memory; a block of 32 never spans two rows.
template <int XDT>
__global__ __launch_bounds__(RN_NT) void k_mx_quantize(const void* x, int64_t pieces, uint8_t* codes, uint8_t* powers) {
    for (int64_t p = (int64_t)blockIdx.x * RN_NT + threadIdx.x; p < pieces; p += (int64_t)gridDim.x * RN_NT) {
        float v[8];
        load8<XDT>(x, p * 8, v);
        const uint32_t power = mx_power_of<MX_E4M3>(v);
        *reinterpret_cast<uint2*>(codes + p * 8) = mx_codes8(v, power);
        if ((threadIdx.x & 3) == 0) powers[p / 4] = (uint8_t)power;
    }
}

template <class F>
void dt_switch(int dt, F&& f) {
    switch (dt) {
        case TSP_F32: f(std::integral_constant<int, TSP_F32>{}); break;
        case TSP_F16: f(std::integral_constant<int, TSP_F16>{}); break;
        default: f(std::integral_constant<int, TSP_BF16>{}); break;
    }
}

}  // namespace
}  // namespace tsp

using namespace tsp;

extern "C" int tsp_rms_norm(const void* d_x, int x_dtype, int64_t n, int c, const void* d_residual, int residual_dtype,
                            const float* d_gamma, float eps, void* d_out, int out_dtype, uint8_t* d_powers, void* d_residual_out,
                            void* stream) {
    clear_error();
    TSP_REQUIRE(n >= 0 && n < (1ll << 31) && c > 0 && c <= (1 << 20), TSP_ERR_INVALID, "tsp_rms_norm: n=%lld c=%d out of range", (long long)n, c);
    TSP_REQUIRE(dtype_valid(x_dtype) && (dtype_valid(out_dtype) || out_dtype == TSP_MX8) && (!d_residual || dtype_valid(residual_dtype)),
                TSP_ERR_INVALID, "tsp_rms_norm: bad dtype");
    TSP_REQUIRE(eps >= 0.f && std::isfinite(eps), TSP_ERR_INVALID, "tsp_rms_norm: eps=%g", eps);
    TSP_REQUIRE(out_dtype != TSP_MX8 || c % MX_BLOCK == 0, TSP_ERR_UNSUPPORTED, "tsp_rms_norm: 8-bit rows of %d channels (need a multiple of %d)",
                c, MX_BLOCK);
    TSP_REQUIRE(d_residual || !d_residual_out, TSP_ERR_INVALID, "tsp_rms_norm: residual_out without a residual");
    if (n == 0) return TSP_OK;
    TSP_REQUIRE(d_x && d_out && (out_dtype != TSP_MX8 || d_powers), TSP_ERR_INVALID, "tsp_rms_norm: null pointer");
    const size_t elems = (size_t)n * c;
    auto bytes = [&](int dt) { return dt == TSP_MX8 ? elems : elems * dtype_size(dt); };
    // a value is read by the thread that writes it, and before: an output may be an input where both are the same values
    struct Part { const void* p; size_t bytes; int dt; };
    const Part in[2] = {{d_x, bytes(x_dtype), x_dtype}, {d_residual, d_residual ? bytes(residual_dtype) : 0, residual_dtype}};
    const Part out[3] = {{d_out, bytes(out_dtype), out_dtype},
                         {d_residual_out, d_residual_out ? bytes(residual_dtype) : 0, residual_dtype},
                         {out_dtype == TSP_MX8 ? d_powers : nullptr, elems / MX_BLOCK, -1}};
    for (const Part& o : out)
        for (const Part& i : in)
            TSP_REQUIRE(!overlap(o.p, o.bytes, i.p, i.bytes) || (o.p == i.p && o.dt == i.dt), TSP_ERR_INVALID,
                        "tsp_rms_norm: an output overlaps an input (it may be one of the same dtype, or apart)");
    TSP_REQUIRE(!overlap(out[0].p, out[0].bytes, out[1].p, out[1].bytes) && !overlap(out[0].p, out[0].bytes, out[2].p, out[2].bytes) &&
                    !overlap(out[1].p, out[1].bytes, out[2].p, out[2].bytes) &&
                    !(d_gamma && (overlap(out[0].p, out[0].bytes, d_gamma, (size_t)c * 4) || overlap(out[1].p, out[1].bytes, d_gamma, (size_t)c * 4) ||
                                  overlap(out[2].p, out[2].bytes, d_gamma, (size_t)c * 4))),
                TSP_ERR_INVALID, "tsp_rms_norm: the outputs overlap each other or gamma");
    const RmsArgs a{d_x, d_residual, d_gamma, d_out, d_residual_out, d_powers, n, c, out_dtype, eps, 1.f / (float)c};
    auto off16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
    hipStream_t s = as_stream(stream);
    const dim3 block(RN_NT);
    const bool aligned = !(off16(d_x) || off16(d_residual) || off16(d_gamma) || off16(d_out) || off16(d_residual_out));
    // (35,001 rows of 500 in bf16 with a residual: 23 us in pieces of four, 28 value by value, 86 twice)
    const int v = aligned && c % 8 == 0 ? (c <= 8192 ? 8 : 0) : c > 4096 ? 0 : aligned && c % 4 == 0 ? 4 : 1;
    if (v == 0) {
        hipLaunchKernelGGL(k_rms_norm_any, dim3((unsigned)std::min<int64_t>(n, 16384)), block, 0, s, a, x_dtype, residual_dtype);
        TSP_CHECK_LAUNCH();
        return TSP_OK;
    }
    dt_switch(x_dtype, [&](auto xd) {
        auto go = [&](auto rd) {
            constexpr int XD = decltype(xd)::value, RD = decltype(rd)::value;
            const dim3 by_wave((unsigned)std::min<int64_t>(ceil_div(n, 4), 2048)), by_group((unsigned)std::min<int64_t>(n, 4096));
            if (v == 1) {
                if (c <= 512) hipLaunchKernelGGL((k_rms_norm<XD, RD, 1, 8, 1>), by_wave, block, 0, s, a);
                else if (c <= 1024) hipLaunchKernelGGL((k_rms_norm<XD, RD, 1, 16, 1>), by_wave, block, 0, s, a);
                else hipLaunchKernelGGL((k_rms_norm<XD, RD, 4, 16, 1>), by_group, block, 0, s, a);
            } else if (v == 4) {
                if (c <= 512) hipLaunchKernelGGL((k_rms_norm<XD, RD, 1, 2, 4>), by_wave, block, 0, s, a);
                else if (c <= 1024) hipLaunchKernelGGL((k_rms_norm<XD, RD, 1, 4, 4>), by_wave, block, 0, s, a);
                else hipLaunchKernelGGL((k_rms_norm<XD, RD, 4, 4, 4>), by_group, block, 0, s, a);
            } else if (c <= 512) hipLaunchKernelGGL((k_rms_norm<XD, RD, 1, 1, 8>), by_wave, block, 0, s, a);
            else if (c <= 1024) hipLaunchKernelGGL((k_rms_norm<XD, RD, 1, 2, 8>), by_wave, block, 0, s, a);
            else if (c <= 2048) hipLaunchKernelGGL((k_rms_norm<XD, RD, 1, 4, 8>), by_wave, block, 0, s, a);
            else if (c <= 4096) hipLaunchKernelGGL((k_rms_norm<XD, RD, 4, 2, 8>), by_group, block, 0, s, a);
            else hipLaunchKernelGGL((k_rms_norm<XD, RD, 4, 4, 8>), by_group, block, 0, s, a);
        };
        if (d_residual) dt_switch(residual_dtype, go);
        else go(std::integral_constant<int, RN_NONE>{});
    });
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}

extern "C" int tsp_mx_quantize(const void* d_x, int x_dtype, int64_t n, int c, void* d_codes, uint8_t* d_powers, void* stream) {
    clear_error();
    TSP_REQUIRE(n >= 0 && n < (1ll << 31) && c > 0 && c <= (1 << 20), TSP_ERR_INVALID, "tsp_mx_quantize: n=%lld c=%d out of range", (long long)n, c);
    TSP_REQUIRE(dtype_valid(x_dtype), TSP_ERR_INVALID, "tsp_mx_quantize: bad dtype");
    TSP_REQUIRE(c % MX_BLOCK == 0, TSP_ERR_UNSUPPORTED, "tsp_mx_quantize: rows of %d channels (need a multiple of %d)", c, MX_BLOCK);
    if (n == 0) return TSP_OK;
    TSP_REQUIRE(d_x && d_codes && d_powers, TSP_ERR_INVALID, "tsp_mx_quantize: null pointer");
    TSP_REQUIRE(reinterpret_cast<uintptr_t>(d_x) % 16 == 0 && reinterpret_cast<uintptr_t>(d_codes) % 16 == 0, TSP_ERR_INVALID,
                "tsp_mx_quantize: x and codes must be 16-byte aligned");
    const size_t elems = (size_t)n * c;
    TSP_REQUIRE(!overlap(d_x, elems * dtype_size(x_dtype), d_codes, elems) && !overlap(d_x, elems * dtype_size(x_dtype), d_powers, elems / MX_BLOCK) &&
                    !overlap(d_codes, elems, d_powers, elems / MX_BLOCK),
                TSP_ERR_INVALID, "tsp_mx_quantize: x, codes and powers must not overlap");
    const int64_t pieces = (int64_t)(elems / 8);
    dt_switch(x_dtype, [&](auto xd) {
        hipLaunchKernelGGL((k_mx_quantize<decltype(xd)::value>), dim3((unsigned)std::min<int64_t>(ceil_div(pieces, RN_NT), 8192)), dim3(RN_NT), 0,
                           as_stream(stream), d_x, pieces, static_cast<uint8_t*>(d_codes), d_powers);
    });
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
