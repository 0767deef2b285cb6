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
    int hq, heads, d, axes, halves;
    float eps;
    double turns[RP_MAX_PAIRS];             // theta^(-j/P) / (2 pi) of each pair
    int8_t axis[RP_MAX_PAIRS];              // its axis, -1: not turned
};

// One (row, head) a group of L lanes; each lane takes whole pairs.
template <int XDT, int ODT, int L>
__global__ __launch_bounds__(RP_NT) void k_rope(RopeArgs a) {
    const int lane = threadIdx.x % L;
    const int64_t item = ((int64_t)blockIdx.x * RP_NT + threadIdx.x) / L;
    const bool live = item < a.n * a.heads;
    const int64_t row = live ? item / a.heads : 0;
    const int head = live ? (int)(item - row * a.heads) : 0;
    const RopeSide& s = a.side[head >= a.hq];
    const int h = head >= a.hq ? head - a.hq : head;
    const auto* x = reinterpret_cast<const typename Elem<XDT>::storage*>(s.x) + row * s.x_row + h * s.x_head;
    auto* y = reinterpret_cast<typename Elem<ODT>::storage*>(s.y) + row * s.y_row + h * s.y_head;
    const float* gamma = s.gamma ? s.gamma + h * a.d : nullptr;
    float scale = 1.f;
    if (gamma) {
        float q = 0.f;
        for (int e = lane; e < a.d; e += L) {
            const float v = Elem<XDT>::load(x, e);
            q += v * v;
        }
        scale = 1.0f / sqrtf(group_sum<L>(q) / (float)a.d + a.eps);
    }
    if (!live) return;
    for (int p = lane; p < a.d / 2; p += L) {
        const int i = a.halves ? p : 2 * p, j = a.halves ? p + a.d / 2 : 2 * p + 1;
        float u = Elem<XDT>::load(x, i) * scale, v = Elem<XDT>::load(x, j) * scale;
        if (gamma) {
            u *= gamma[i];
            v *= gamma[j];
        }
        const int ax = a.axis[p];
        if (ax >= 0) {
            const double t = (double)a.pos[row * a.axes + ax] * a.turns[p];
            float sn, cs;
            sincospif(2.f * (float)(t - rint(t)), &sn, &cs);
            const float w = u * cs - v * sn;
            v = v * cs + u * sn;
            u = w;
        }
        Elem<ODT>::store(y, i, u);
        Elem<ODT>::store(y, j, v);
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
    constexpr int L = 16;
    const int64_t blocks = ceil_div(n * a.heads * L, RP_NT);
    TSP_REQUIRE(blocks * RP_NT < (1ll << 32), TSP_ERR_INVALID, "tsp_rope_axes: too many rows");
    dt_switch(dtype, [&](auto xd) {
        dt_switch(out_dtype, [&](auto od) {
            hipLaunchKernelGGL((k_rope<decltype(xd)::value, decltype(od)::value, L>), dim3((unsigned)blocks), dim3(RP_NT), 0,
                               as_stream(stream), a);
        });
    });
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
