// Rotary positions on several axes, for q and k together: pair j of axis a is turned by the angle
// pos[i][a] * theta^(-j / pairs[a]); the pairs of axis 0 come first, pairs after the last axis's stay as
// they are. With gamma, each head's row is RMS-normalised before: x / sqrt(mean(x^2) + eps) * gamma.
//
// An angle is formed in turns (pos * theta^(-j/P) / 2 pi) in 64 bits and only its fraction is rounded to
// 32, so that a position of 10^9 turns as exactly as one of 10.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "packed.hpp"

namespace tsp {
namespace {

constexpr int RP_NT = 256;
constexpr int RP_MAX_AXES = 4, RP_MAX_PAIRS = 128;

struct RopeSide {
    const void* x;
    void* y;
    int64_t x_row, x_head, y_row, y_head;   // strides in elements
    const float* gamma;                     // [heads][d], or NULL
};

struct RopeArgs {
    RopeSide side[2];
    const int32_t* pos;
    int64_t n;
    int hq, heads, d, axes, halves, parts;
    float eps;
    double turns[RP_MAX_PAIRS];             // theta^(-j/P) / (2 pi) of each pair
    int8_t axis[RP_MAX_PAIRS];              // its axis, -1: not turned
};

// Four pairs of a head, as the lane that turns them holds them: elements 8 u .. 8 u + 7, or with halves 4 u
// .. 4 u + 3 of each half.
template <int DT>
__device__ __forceinline__ void load_pairs(const void* p, int unit, int d, bool halves, float (&u)[4], float (&v)[4]) {
    if constexpr (DT == TSP_F32) {
        const float* x = static_cast<const float*>(p);
        const f32x4_t a = *reinterpret_cast<const f32x4_t*>(x + (halves ? 4 * unit : 8 * unit));
        const f32x4_t b = *reinterpret_cast<const f32x4_t*>(x + (halves ? 4 * unit + d / 2 : 8 * unit + 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = halves ? a[i] : i < 2 ? a[2 * i] : b[2 * i - 4];
            v[i] = halves ? b[i] : i < 2 ? a[2 * i + 1] : b[2 * i - 3];
        }
    } else {
        const uint16_t* x = static_cast<const uint16_t*>(p);
        auto f = [](uint32_t b) { return DT == TSP_BF16 ? bf16_bits_to_f32((uint16_t)b) : f16_bits_to_f32((uint16_t)b); };
        if (halves) {
            const uint2 a = *reinterpret_cast<const uint2*>(x + 4 * unit), b = *reinterpret_cast<const uint2*>(x + 4 * unit + d / 2);
            u[0] = f(a.x & 0xffff), u[1] = f(a.x >> 16), u[2] = f(a.y & 0xffff), u[3] = f(a.y >> 16);
            v[0] = f(b.x & 0xffff), v[1] = f(b.x >> 16), v[2] = f(b.y & 0xffff), v[3] = f(b.y >> 16);
        } else {
            const u32x4_t a = *reinterpret_cast<const u32x4_t*>(x + 8 * unit);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = f(a[i] & 0xffff), v[i] = f(a[i] >> 16);
        }
    }
}
template <int DT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    return DT == TSP_BF16 ? f32x2_to_bf16x2_bits(lo, hi) : f32_to_f16_bits(lo) | ((uint32_t)f32_to_f16_bits(hi) << 16);
}
template <int DT>
__device__ __forceinline__ void store_pairs(void* p, int unit, int d, bool halves, const float (&u)[4], const float (&v)[4]) {
    if constexpr (DT == TSP_F32) {
        float* y = static_cast<float*>(p);
        *reinterpret_cast<f32x4_t*>(y + (halves ? 4 * unit : 8 * unit)) =
            halves ? f32x4_t{u[0], u[1], u[2], u[3]} : f32x4_t{u[0], v[0], u[1], v[1]};
        *reinterpret_cast<f32x4_t*>(y + (halves ? 4 * unit + d / 2 : 8 * unit + 4)) =
            halves ? f32x4_t{v[0], v[1], v[2], v[3]} : f32x4_t{u[2], v[2], u[3], v[3]};
    } else {
        uint16_t* y = static_cast<uint16_t*>(p);
        if (halves) {
            *reinterpret_cast<uint2*>(y + 4 * unit) = uint2{pack16<DT>(u[0], u[1]), pack16<DT>(u[2], u[3])};
            *reinterpret_cast<uint2*>(y + 4 * unit + d / 2) = uint2{pack16<DT>(v[0], v[1]), pack16<DT>(v[2], v[3])};
        } else {
            *reinterpret_cast<u32x4_t*>(y + 8 * unit) =
                u32x4_t{pack16<DT>(u[0], v[0]), pack16<DT>(u[1], v[1]), pack16<DT>(u[2], v[2]), pack16<DT>(u[3], v[3])};
        }
    }
}

// A group of L lanes takes one row and every `part`-th of its heads, four pairs a lane: the row's sines
// and cosines are formed once for all of them. The heads' loads go out BATCH at a time.
template <int XDT, int ODT, int L>
__global__ __launch_bounds__(RP_NT) void k_rope(RopeArgs a) {
    constexpr int BATCH = 4, XS = XDT == TSP_F32 ? 4 : 2, OS = ODT == TSP_F32 ? 4 : 2;
    const int unit = threadIdx.x % L;
    const bool live = unit * 8 < a.d, halves = a.halves;
    double turns[4];
    int axis[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        axis[i] = live ? a.axis[4 * unit + i] : -1;
        turns[i] = axis[i] < 0 ? 0. : a.turns[4 * unit + i];
    }
    const unsigned items = (unsigned)(a.n * a.parts);      // (below 2^31)
    // (whole groups of lanes leave together)
    for (unsigned item = (blockIdx.x * RP_NT + threadIdx.x) / L; item < items; item += gridDim.x * (RP_NT / L)) {
        const int row = (int)(item / (unsigned)a.parts), part = (int)(item - (unsigned)row * a.parts);
        float cs[4], sn[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cs[i] = 1.f, sn[i] = 0.f;
            if (axis[i] >= 0) {
                const double t = (double)a.pos[(int64_t)row * a.axes + axis[i]] * turns[i];
                sincospif(2.f * (float)(t - rint(t)), &sn[i], &cs[i]);
            }
        }
        for (int h0 = part; h0 < a.heads; h0 += BATCH * a.parts) {
            float u[BATCH][4] = {}, v[BATCH][4] = {};
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const int h = h0 + b * a.parts;
                if (!live || h >= a.heads) continue;
                const RopeSide& s = a.side[h >= a.hq];
                load_pairs<XDT>(static_cast<const char*>(s.x) + ((int64_t)row * s.x_row + (h >= a.hq ? h - a.hq : h) * s.x_head) * XS,
                                unit, a.d, halves, u[b], v[b]);
            }
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const int h = h0 + b * a.parts;
                if (h >= a.heads) break;
                const RopeSide& s = a.side[h >= a.hq];
                const int hh = h >= a.hq ? h - a.hq : h;
                if (s.gamma) {
                    float q = 0.f, gu[4] = {}, gv[4] = {};
                    if (live) {
                        load_pairs<TSP_F32>(s.gamma + hh * a.d, unit, a.d, halves, gu, gv);
#pragma unroll
                        for (int i = 0; i < 4; ++i) q += u[b][i] * u[b][i] + v[b][i] * v[b][i];
                    }
                    const float scale = 1.0f / sqrtf(group_sum<L>(q) / (float)a.d + a.eps);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        u[b][i] *= scale * gu[i];
                        v[b][i] *= scale * gv[i];
                    }
                }
                if (!live) continue;
                float x[4], y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = u[b][i] * cs[i] - v[b][i] * sn[i];
                    y[i] = v[b][i] * cs[i] + u[b][i] * sn[i];
                    if (axis[i] < 0) x[i] = u[b][i], y[i] = v[b][i];     // (not 0 * Inf)
                }
                store_pairs<ODT>(static_cast<char*>(s.y) + ((int64_t)row * s.y_row + hh * s.y_head) * OS, unit, a.d, halves, x, y);
            }
        }
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

extern "C" int tsp_rope_axes(const tsp_heads* q, int hq, const tsp_heads* k, int hk, int dtype, int64_t n, int d,
                             const int32_t* d_pos, int axes, const int* pairs, double theta, int flags,
                             const float* d_q_gamma, const float* d_k_gamma, float eps, const tsp_heads* q_out,
                             const tsp_heads* k_out, int out_dtype, void* stream) {
    clear_error();
    TSP_REQUIRE(n >= 0 && n < (1ll << 31), TSP_ERR_INVALID, "tsp_rope_axes: n=%lld out of range", (long long)n);
    TSP_REQUIRE(dtype_valid(dtype) && dtype_valid(out_dtype), TSP_ERR_INVALID, "tsp_rope_axes: bad dtype");
    TSP_REQUIRE(flags == 0 || flags == TSP_ROPE_HALVES, TSP_ERR_INVALID, "tsp_rope_axes: bad flags %d", flags);
    TSP_REQUIRE(hq > 0 && hk >= 0 && hq + hk <= 4096 && (k != nullptr) == (hk > 0), TSP_ERR_INVALID,
                "tsp_rope_axes: hq=%d hk=%d (k %s)", hq, hk, k ? "given" : "NULL");
    TSP_REQUIRE(d > 0 && d % 8 == 0 && d <= 2 * RP_MAX_PAIRS, TSP_ERR_UNSUPPORTED,
                "tsp_rope_axes: heads of %d (need a multiple of 8 up to %d)", d, 2 * RP_MAX_PAIRS);
    TSP_REQUIRE(axes > 0 && axes <= RP_MAX_AXES && pairs, TSP_ERR_INVALID, "tsp_rope_axes: %d axes (1 to %d)", axes, RP_MAX_AXES);
    TSP_REQUIRE(theta > 0 && std::isfinite(theta) && eps >= 0.f, TSP_ERR_INVALID, "tsp_rope_axes: theta=%g eps=%g", theta, eps);
    int64_t total = 0;
    for (int i = 0; i < axes; ++i) {
        TSP_REQUIRE(pairs[i] >= 0 && pairs[i] <= d / 2, TSP_ERR_INVALID, "tsp_rope_axes: %d pairs on axis %d", pairs[i], i);
        total += pairs[i];
    }
    TSP_REQUIRE(total <= d / 2, TSP_ERR_INVALID, "tsp_rope_axes: %lld pairs, a head of %d has %d", (long long)total, d, d / 2);
    if (n == 0) return TSP_OK;
    TSP_REQUIRE(q && q_out && q->data && q_out->data && d_pos && (hk == 0 || (k_out && k->data && k_out->data)), TSP_ERR_INVALID,
                "tsp_rope_axes: null pointer");
    TSP_REQUIRE(heads_aligned(*q) && heads_aligned(*q_out) && (hk == 0 || (heads_aligned(*k) && heads_aligned(*k_out))), TSP_ERR_INVALID,
                "tsp_rope_axes: data must be 16-byte aligned, strides multiples of 8 (a row's up to 2^20)");
    TSP_REQUIRE(heads_apart(*q_out, n, hq, d) && (hk == 0 || heads_apart(*k_out, n, hk, d)), TSP_ERR_INVALID,
                "tsp_rope_axes: the output's heads overlap");
    RopeArgs a{};
    auto side = [](const tsp_heads& x, const tsp_heads& y, const float* g) {
        return RopeSide{x.data, y.data, x.row_stride, x.head_stride, y.row_stride, y.head_stride, g};
    };
    a.side[0] = side(*q, *q_out, d_q_gamma);
    if (hk) a.side[1] = side(*k, *k_out, d_k_gamma);
    a.pos = d_pos;
    a.n = n;
    a.hq = hq;
    a.heads = hq + hk;
    a.d = d;
    a.axes = axes;
    a.halves = flags & TSP_ROPE_HALVES ? 1 : 0;
    a.eps = eps;
    for (int p = 0; p < d / 2; ++p) a.axis[p] = -1;
    int p = 0;
    for (int ax = 0; ax < axes; ++ax)
        for (int j = 0; j < pairs[ax]; ++j, ++p) {
            a.axis[p] = (int8_t)ax;
            a.turns[p] = std::pow(theta, -(double)j / pairs[ax]) / (2 * M_PI);
        }
    // Lanes of a group: a head's units of 8 elements and, where they are no power of two, some that idle. A row
    // is shared by as many groups as it takes to give the device some 2048 workgroups, at most one a head.
    const int lanes = d <= 64 ? 8 : d <= 128 ? 16 : 32, groups = RP_NT / lanes;
    a.parts = (int)std::min<int64_t>(a.heads, std::max<int64_t>(1, 2048ll * groups / n));
    const int64_t blocks = std::min<int64_t>(ceil_div(n * a.parts, groups), 8192);
    dt_switch(dtype, [&](auto xd) {
        dt_switch(out_dtype, [&](auto od) {
            constexpr int XD = decltype(xd)::value, OD = decltype(od)::value;
            const dim3 grid((unsigned)blocks), block(RP_NT);
            hipStream_t s = as_stream(stream);
            if (lanes == 8) hipLaunchKernelGGL((k_rope<XD, OD, 8>), grid, block, 0, s, a);
            else if (lanes == 16) hipLaunchKernelGGL((k_rope<XD, OD, 16>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((k_rope<XD, OD, 32>), grid, block, 0, s, a);
        });
    });
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
