// Rotary positions on several axes, for q and k together: pair j of axis a is turned by the angle
// pos[i][a] * theta^(-j / pairs[a]); the pairs of axis 0 come first, pairs after the last axis's stay as
// they are. With gamma, each head's row is RMS-normalised before: x / sqrt(mean(x^2) + eps) * gamma.
//
// An angle is formed in turns (pos * theta^(-j/P) / 2 pi) in 64 bits and only its fraction is rounded to
// 32, so that a far position turns as exactly as a near one (to 2^-22 up to 2^28).
//
// Bound by memory: one read and one write. A row's sines and cosines (some 400 instructions for four pairs)
// are formed once for all its heads; the heads' rows are loaded four at a time and kept packed until they
// are turned. q and k of 35,001 rows x 8 heads of 128 with norms, bf16: 56 us, 5.1 TB/s; 117,343 x (16 + 4) heads
// of 64, f16: 120 us, 5.0 TB/s (a copy of 4 GiB: 4.7).
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "inverse_root.hpp"
#include "overlap.hpp"
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
    int heads;
};

struct RopeArgs {
    RopeSide side[2];
    const int32_t* pos;
    int64_t n;
    int d, axes, parts;
    float eps, inv_d;
    double turns[RP_MAX_PAIRS];             // theta^(-j/P) / (2 pi) of each pair
    int8_t axis[RP_MAX_PAIRS];              // its axis, -1: not turned
};

// Four pairs of a head, as the lane that turns them holds them: elements 8 u .. 8 u + 7, or with halves 4 u
// .. 4 u + 3 of each half.
template <int DT> struct Raw { u32x4_t a; };
template <> struct Raw<TSP_F32> { f32x4_t a, b; };
template <int DT, bool HALVES>
__device__ __forceinline__ Raw<DT> load_raw(const void* p, int unit, int d) {
    Raw<DT> r;
    if constexpr (DT == TSP_F32) {
        const float* x = static_cast<const float*>(p);
        r.a = *reinterpret_cast<const f32x4_t*>(x + (HALVES ? 4 * unit : 8 * unit));
        r.b = *reinterpret_cast<const f32x4_t*>(x + (HALVES ? 4 * unit + d / 2 : 8 * unit + 4));
    } else if constexpr (HALVES) {
        const uint16_t* x = static_cast<const uint16_t*>(p);
        const uint2 a = *reinterpret_cast<const uint2*>(x + 4 * unit), b = *reinterpret_cast<const uint2*>(x + 4 * unit + d / 2);
        r.a = u32x4_t{a.x, a.y, b.x, b.y};
    } else {
        r.a = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(p) + 8 * unit);
    }
    return r;
}
template <int DT, bool HALVES>
__device__ __forceinline__ void pairs_of(const Raw<DT>& r, float (&u)[4], float (&v)[4]) {
    if constexpr (DT == TSP_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = HALVES ? r.a[i] : i < 2 ? r.a[2 * i] : r.b[2 * i - 4];
            v[i] = HALVES ? r.b[i] : i < 2 ? r.a[2 * i + 1] : r.b[2 * i - 3];
        }
    } else {
        auto f = [](uint32_t b) { return DT == TSP_BF16 ? bf16_bits_to_f32((uint16_t)b) : f16_bits_to_f32((uint16_t)b); };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = HALVES ? f(i & 1 ? r.a[i / 2] >> 16 : r.a[i / 2] & 0xffff) : f(r.a[i] & 0xffff);
            v[i] = HALVES ? f(i & 1 ? r.a[2 + i / 2] >> 16 : r.a[2 + i / 2] & 0xffff) : f(r.a[i] >> 16);
        }
    }
}
template <int DT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    return DT == TSP_BF16 ? f32x2_to_bf16x2_bits(lo, hi) : f32_to_f16_bits(lo) | ((uint32_t)f32_to_f16_bits(hi) << 16);
}
template <int DT, bool halves>
__device__ __forceinline__ void store_pairs(void* p, int unit, int d, const float (&u)[4], const float (&v)[4]) {
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
template <int XDT, int ODT, int L, bool HALVES>
__global__ __launch_bounds__(RP_NT, 4) void k_rope(RopeArgs a) {
    constexpr int BATCH = 4, XS = XDT == TSP_F32 ? 4 : 2, OS = ODT == TSP_F32 ? 4 : 2;
    const int unit = threadIdx.x % L;
    const bool live = unit * 8 < a.d;
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
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {
            const RopeSide& s = a.side[side];
            const char* x = static_cast<const char*>(s.x) + ((int64_t)row * s.x_row + part * s.x_head) * XS;
            char* y = static_cast<char*>(s.y) + ((int64_t)row * s.y_row + part * s.y_head) * OS;
            const int64_t x_step = a.parts * s.x_head * XS, y_step = a.parts * s.y_head * OS;
            const float* gamma = s.gamma + part * a.d;
            for (int h0 = part; h0 < s.heads; h0 += BATCH * a.parts) {
                Raw<XDT> raw[BATCH] = {};
#pragma unroll
                for (int b = 0; b < BATCH; ++b)
                    if (live && h0 + b * a.parts < s.heads) raw[b] = load_raw<XDT, HALVES>(x + b * x_step, unit, a.d);
                x += BATCH * x_step;
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    if (h0 + b * a.parts >= s.heads) break;
                    float u[4], v[4];
                    pairs_of<XDT, HALVES>(raw[b], u, v);
                    if (s.gamma) {
                        float q = 0.f, gu[4], gv[4];
                        Raw<TSP_F32> g{};
                        if (live) g = load_raw<TSP_F32, HALVES>(gamma, unit, a.d);
                        pairs_of<TSP_F32, HALVES>(g, gu, gv);
#pragma unroll
                        for (int i = 0; i < 4; ++i) q += u[i] * u[i] + v[i] * v[i];
                        const float scale = inverse_root(fmaf(group_sum<L>(q), a.inv_d, a.eps));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            u[i] *= scale * gu[i];
                            v[i] *= scale * gv[i];
                        }
                        gamma += a.parts * a.d;
                    }
                    if (live) {
                        float p[4], r[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[i] = u[i] * cs[i] - v[i] * sn[i];
                            r[i] = v[i] * cs[i] + u[i] * sn[i];
                            if (axis[i] < 0) p[i] = u[i], r[i] = v[i];     // (not 0 * Inf)
                        }
                        store_pairs<ODT, HALVES>(y, unit, a.d, p, r);
                    }
                    y += y_step;
                }
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
    TSP_REQUIRE(!(reinterpret_cast<uintptr_t>(d_q_gamma) % 16 || reinterpret_cast<uintptr_t>(d_k_gamma) % 16), TSP_ERR_INVALID,
                "tsp_rope_axes: gamma must be 16-byte aligned");
    TSP_REQUIRE(heads_apart(*q_out, n, hq, d) && (hk == 0 || heads_apart(*k_out, n, hk, d)), TSP_ERR_INVALID,
                "tsp_rope_axes: the output's heads overlap");
    // in place a group of lanes has read its heads before it writes them: they must be the same ones
    auto other = [&](const tsp_heads& x, const tsp_heads& y, int heads) {
        return x.data == y.data && (dtype != out_dtype || (n > 1 && x.row_stride != y.row_stride) || (heads > 1 && x.head_stride != y.head_stride));
    };
    TSP_REQUIRE(!other(*q, *q_out, hq) && (hk == 0 || (!other(*k, *k_out, hk) && q->data != k_out->data && k->data != q_out->data &&
                                                       q_out->data != k_out->data)),
                TSP_ERR_INVALID, "tsp_rope_axes: an output may be its own input, with one dtype and the same strides, and no other");
    const Runs none = runs_of(nullptr, 0);
    auto runs = [&](const tsp_heads* t, int heads, int dt) { return heads ? runs_of(*t, n, heads, d, dtype_size(dt)) : none; };
    const Runs out[2] = {runs(q_out, hq, out_dtype), runs(k_out, hk, out_dtype)}, in[2] = {runs(q, hq, dtype), runs(k, hk, dtype)};
    const Runs read[3] = {runs_of(d_pos, 4ll * n * axes), runs_of(d_q_gamma, 4ll * hq * d), runs_of(d_k_gamma, 4ll * hk * d)};
    bool over = meet(out[0], out[1]) || meet(out[0], in[1]) || meet(out[1], in[0]) || (q_out->data != q->data && meet(out[0], in[0])) ||
                (hk && k_out->data != k->data && meet(out[1], in[1]));
    for (const Runs& r : read) over |= meet(out[0], r) || meet(out[1], r);
    TSP_REQUIRE(!over, TSP_ERR_INVALID, "tsp_rope_axes: an output overlaps another tensor of the call (it may be its own input)");
    RopeArgs a{};
    auto side = [](const tsp_heads& x, const tsp_heads& y, const float* g, int heads) {
        return RopeSide{x.data, y.data, x.row_stride, x.head_stride, y.row_stride, y.head_stride, g, heads};
    };
    a.side[0] = side(*q, *q_out, d_q_gamma, hq);
    if (hk) a.side[1] = side(*k, *k_out, d_k_gamma, hk);
    a.pos = d_pos;
    a.n = n;
    a.d = d;
    a.axes = axes;
    a.eps = eps;
    a.inv_d = 1.f / (float)d;
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
    a.parts = (int)std::min<int64_t>(std::max(hq, hk), std::max<int64_t>(1, 2048ll * groups / n));
    const int64_t blocks = std::min<int64_t>(ceil_div(n * a.parts, groups), 8192);
    dt_switch(dtype, [&](auto xd) {
        dt_switch(out_dtype, [&](auto od) {
            constexpr int XD = decltype(xd)::value, OD = decltype(od)::value;
            const dim3 grid((unsigned)blocks), block(RP_NT);
            hipStream_t s = as_stream(stream);
            auto go = [&](auto l, auto halves) {
                hipLaunchKernelGGL((k_rope<XD, OD, decltype(l)::value, decltype(halves)::value>), grid, block, 0, s, a);
            };
            auto by_pairing = [&](auto l) {
                if (flags & TSP_ROPE_HALVES) go(l, std::true_type{});
                else go(l, std::false_type{});
            };
            if (lanes == 8) by_pairing(std::integral_constant<int, 8>{});
            else if (lanes == 16) by_pairing(std::integral_constant<int, 16>{});
            else by_pairing(std::integral_constant<int, 32>{});
        });
    });
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
