// Numbers of few bits with a power of two for every 32 channels, as CDNA4's conversions and scaled matrix products
// take them: e4m3 codes (8 bits) or e2m1 codes (4 bits: 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) times
// 2^(power - 127), power a byte (e8m0; 255: NaN).
//
// The power is the least with which the largest of the 32 fits the codes' range, 448 = 1.75 * 2^8 or 6 = 1.5 * 2^2, so
// that no value is cut. A block that holds an Inf or a NaN has power 255: all of it stands for NaN.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "overlap.hpp"

namespace tsp {

constexpr int MX_BLOCK = 32;

enum { MX_E4M3 = 8, MX_E2M1 = 4 };

// The power byte of a block by the bits of its largest |value| (the largest bits where a value is Inf or NaN): the
// exponent goes up by one where the mantissa is past that of the codes' largest value.
template <int BITS>
__device__ __forceinline__ uint32_t mx_power(uint32_t amax_bits) {
    constexpr uint32_t kPast = BITS == MX_E4M3 ? 0x7fffff - 0x600000 : 0x7fffff - 0x400000;
    constexpr int kTop = BITS == MX_E4M3 ? 8 : 2;
    const int e = (int)((amax_bits + kPast) >> 23) - kTop;
    return amax_bits >= 0x7f800000u ? 255u : (uint32_t)max(e, 0);
}

// 2^(power - 127) as the conversions take it, which read the exponent's bits alone (0: 2^-127; 255: NaN).
__device__ __forceinline__ float mx_scale(uint32_t power) { return __uint_as_float(power << 23); }

// The largest of a value over aligned groups of four lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));    // quad_perm [1, 0, 3, 2]
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false)); // quad_perm [2, 3, 0, 1]
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The power byte of the block whose 32 channels four neighbouring lanes hold, eight each.
template <int BITS>
__device__ __forceinline__ uint32_t mx_power_of(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
    return mx_power<BITS>(quad_max(m));
}

// Eight values as e4m3 codes of that power, rounded to nearest even.
typedef short s16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint2 mx_codes8(const float (&v)[8], uint32_t power) {
    const float s = mx_scale(power);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        s16x2_t c{0, 0};
        c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v[4 * i], v[4 * i + 1], s, false);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v[4 * i + 2], v[4 * i + 3], s, true);
        w[i] = __builtin_bit_cast(uint32_t, c);
    }
    return uint2{w[0], w[1]};
}
// ... as e2m1 codes, the first in the lowest four bits.
__device__ __forceinline__ uint32_t mx_codes4(const float (&v)[8], uint32_t power) {
    const float s = mx_scale(power);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
    return c;
}

// Eight values of a tensor of type DT at element i (16-byte aligned pieces), and back.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
    if constexpr (DT == TSP_F32) {
        const f32x4_t* x = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + i);
        const f32x4_t a = x[0], b = x[1];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = a[k], v[4 + k] = b[k];
    } else {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[2 * k] = DT == TSP_BF16 ? __uint_as_float(a[k] << 16) : f16_bits_to_f32((uint16_t)a[k]);
            v[2 * k + 1] = DT == TSP_BF16 ? __uint_as_float(a[k] & 0xffff0000u) : f16_bits_to_f32((uint16_t)(a[k] >> 16));
        }
    }
}
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&v)[8]) {
    if constexpr (DT == TSP_F32) {
        f32x4_t* y = reinterpret_cast<f32x4_t*>(static_cast<float*>(p) + i);
        y[0] = f32x4_t{v[0], v[1], v[2], v[3]};
        y[1] = f32x4_t{v[4], v[5], v[6], v[7]};
    } else {
        u32x4_t a;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            a[k] = DT == TSP_BF16 ? f32x2_to_bf16x2_bits(v[2 * k], v[2 * k + 1])
                                  : f32_to_f16_bits(v[2 * k]) | ((uint32_t)f32_to_f16_bits(v[2 * k + 1]) << 16);
        *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(p) + i) = a;
    }
}

}  // namespace tsp
