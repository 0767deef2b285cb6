// Packed samples: rows of several samples one after another, sample s on rows [offsets[s],
// offsets[s + 1]) (device int32 [samples + 1], non-decreasing). Kernels cut every sample into units of
// at most `per` rows; a launch has as many workgroups as there can be units (ceil(n / per) + samples:
// the host does not know the lengths) and each finds its own unit here.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace tsp {

struct PackedUnit {
    int sample;        // -1: there are fewer units
    int first, count;  // the sample's first unit, how many it has
    int row0, rows;    // the sample's rows
    int other0, others;   // the sample's rows in a second packed tensor, where one is asked for
};

// x / d for 0 <= x < 2^31 by a multiplication: with s = ceil(log2 d) and mul = floor(2^(31 + s) / d) + 1,
// mul * d exceeds 2^(31 + s) by at most d <= 2^s, so that (x * mul) >> (31 + s) is exact. (The compiler's
// own division is some thirty instructions.)
struct FastDiv {
    uint32_t mul;
    int shift;
};
inline FastDiv fast_div(uint32_t d) {
    int s = 0;
    while ((1ull << s) < d) ++s;
    return FastDiv{(uint32_t)((1ull << (31 + s)) / d + 1), s};
}
__device__ __forceinline__ int operator/(int x, FastDiv d) { return (int)(((uint64_t)(uint32_t)x * d.mul) >> (31 + d.shift)); }

// Rows of sample s of n < 2^31; bounds outside [0, n] or out of order are cut to it, so that no row
// outside the tensor is touched. offsets NULL: one sample of all n rows.
__device__ __forceinline__ void packed_rows(const int32_t* offsets, int s, int n, int& row0, int& rows) {
    row0 = offsets ? min(max(offsets[s], 0), n) : 0;
    rows = offsets ? max(min(offsets[s + 1], n), row0) - row0 : n;
}

// The unit-th unit of `per` rows (each row counted `mult` times; n * mult + per < 2^31), called by whole
// waves with a uniform unit: 64 samples a step, their unit counts summed across the wave. With SECOND also
// the sample's rows in a second tensor of n2 rows, and up to 16 samples in the order of their lengths there,
// the longest first: units that take longest then start first, and the device is not left waiting for a
// long one that began last. (A packed causal batch of 7 samples, 12,345 tokens: 158 us so, 182 in the
// samples' own order; 128 samples of 64: 26 us in their own order, 51 when all are ordered.)
constexpr int kOrderedSamples = 16;
template <bool SECOND = false>
__device__ __forceinline__ PackedUnit packed_unit(const int32_t* offsets, int samples, int n, int mult, int per, int unit,
                                                  const int32_t* offsets2 = nullptr, int n2 = 0) {
    PackedUnit u{-1, 0, 0, 0, 0, 0, 0};
    if (samples == 1) {
        packed_rows(offsets, 0, n, u.row0, u.rows);
        if constexpr (SECOND) packed_rows(offsets2, 0, n2, u.other0, u.others);
        u.count = (int)((unsigned)(u.rows * mult + per - 1) / (unsigned)per);
        if (unit < u.count) u.sample = 0;
        return u;
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 < samples; s0 += 64) {
        const int s = s0 + lane;
        int row0 = 0, rows = 0, other0 = 0, others = -1;
        if (s < samples) {
            packed_rows(offsets, s, n, row0, rows);
            if constexpr (SECOND) packed_rows(offsets2, s, n2, other0, others);
        }
        const int cnt = (int)((unsigned)(rows * mult + per - 1) / (unsigned)per);
        int end = cnt;      // units up to this sample's last
        if (SECOND && samples <= kOrderedSamples) {
            for (int j = 0; j < samples; ++j) {
                const int v = __builtin_amdgcn_readlane(others, j), c = __builtin_amdgcn_readlane(cnt, j);
                if (v > others || (v == others && j < lane)) end += c;
            }
        } else {
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(end, o, 64);
                if (lane >= o) end += v;
            }
        }
        const int first = before + end - cnt;
        const uint64_t mine = __ballot(unit >= first && unit < first + cnt);
        if (mine) {
            const int l = __builtin_ctzll(mine);
            u.sample = s0 + l;
            u.count = __builtin_amdgcn_readlane(cnt, l);
            u.first = __builtin_amdgcn_readlane(first, l);
            u.row0 = __builtin_amdgcn_readlane(row0, l);
            u.rows = __builtin_amdgcn_readlane(rows, l);
            if constexpr (SECOND) {
                u.other0 = __builtin_amdgcn_readlane(other0, l);
                u.others = __builtin_amdgcn_readlane(others, l);
            }
            return u;
        }
        before += __builtin_amdgcn_readlane(end, 63);      // (one step alone where they are ordered)
    }
    return u;
}

// Sample `sample` and its units (uniform, by whole waves).
__device__ __forceinline__ PackedUnit packed_sample(const int32_t* offsets, int n, int mult, int per, int sample) {
    PackedUnit u{sample, 0, 0, 0, 0, 0, 0};
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s = lane; s < sample; s += 64) {
        int row0, rows;
        packed_rows(offsets, s, n, row0, rows);
        before += (int)((unsigned)(rows * mult + per - 1) / (unsigned)per);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64);
    u.first = __builtin_amdgcn_readfirstlane(before);
    packed_rows(offsets, sample, n, u.row0, u.rows);
    u.count = (int)((unsigned)(u.rows * mult + per - 1) / (unsigned)per);
    return u;
}

// Rows of heads as the transformer pieces take them: 16-byte aligned, strides multiples of 8 elements (a
// row's below 2^20, so that a tile of rows spans less than 2^31 bytes).
inline bool heads_aligned(const tsp_heads& t) {
    return t.row_stride >= 0 && t.head_stride >= 0 && t.row_stride <= (1ll << 20) && t.head_stride <= (1ll << 40) &&
           t.row_stride % 8 == 0 && t.head_stride % 8 == 0 && reinterpret_cast<uintptr_t>(t.data) % 16 == 0;
}
// ... that can be written: no two heads of d elements share one.
inline bool heads_apart(const tsp_heads& t, int64_t n, int heads, int d) {
    const int64_t r = t.row_stride, h = t.head_stride;
    if (n <= 1 && heads <= 1) return true;
    if (heads <= 1) return r >= d;
    if (n <= 1) return h >= d;
    return (h >= d && r >= (heads - 1) * h + d) || (r >= d && h >= (n - 1) * r + d);
}

}  // namespace tsp
