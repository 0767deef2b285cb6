// Group norm over packed samples, channels last: for sample s and group g of C / G channels,
//   y = (x - mean) / sqrt(var + eps) * gamma[c] + beta[c], then y * sigmoid(y) where asked,
// mean and (biased) var over the sample's rows and the group's channels.
//
// Two launches over the same units of rows. The first leaves each unit's mean and sum of squared
// deviations per group in the workspace, the second joins a sample's units (in the order of the units,
// whatever the order in which they ran) and normalises its rows.
#include <algorithm>

#include "common.hpp"
#include "packed.hpp"

namespace tsp {
namespace {

constexpr int GN_NT = 512;              // threads of a workgroup
constexpr int GN_MAX_GROUPS = 4096;     // statistics a workgroup holds in LDS

struct GnArgs {
    const void* x;
    void* out;
    const int32_t* offsets;
    const float *gamma, *beta;
    float2* part;          // [unit][group]: mean, sum of squared deviations
    int64_t n;
    int c, groups, samples, per;
    float eps;
    int silu;
};

__device__ __forceinline__ int unit_rows(const PackedUnit& u, int unit, int per, int64_t& row) {
    const int lo = (unit - u.first) * per;
    row = u.row0 + lo;
    return min(u.rows - lo, per);
}

__device__ __forceinline__ float act(float y, int silu) { return silu ? y / (1.0f + expf(-y)) : y; }

// One group of one unit a workgroup. Sums are of x minus the group's first value, so that a mean far
// from zero does not swallow the variance.
template <int XDT>
__global__ __launch_bounds__(GN_NT) void k_gn_stats(GnArgs a) {
    __shared__ float2 sPart[GN_NT / 64];
    const PackedUnit u = packed_unit(a.offsets, a.samples, (int)a.n, 1, a.per, blockIdx.x);
    if (u.sample < 0) return;
    int64_t row;
    const int rows = unit_rows(u, blockIdx.x, a.per, row);
    const int cg = a.c / a.groups, g = blockIdx.y;
    const auto* x = reinterpret_cast<const typename Elem<XDT>::storage*>(a.x) + row * a.c + g * cg;
    const int64_t cnt = (int64_t)rows * cg;
    const float shift = Elem<XDT>::load(x, 0);
    float s = 0.f, q = 0.f;
    for (int64_t e = threadIdx.x; e < cnt; e += GN_NT) {
        const int64_t r = e / cg;
        const float d = Elem<XDT>::load(x, r * a.c + (e - r * cg)) - shift;
        s += d;
        q += d * d;
    }
    s = group_sum<64>(s);
    q = group_sum<64>(q);
    if ((threadIdx.x & 63) == 0) sPart[threadIdx.x >> 6] = float2{s, q};
    __syncthreads();
    if (threadIdx.x == 0) {
        float S = 0.f, Q = 0.f;
        for (int w = 0; w < GN_NT / 64; ++w) {
            S += sPart[w].x;
            Q += sPart[w].y;
        }
        const float m = S / (float)cnt;
        a.part[(int64_t)blockIdx.x * a.groups + g] = float2{shift + m, fmaxf(Q - S * m, 0.f)};
    }
}

// Mean and 1 / sqrt(var + eps) of every group of the unit's sample, into LDS.
__device__ __forceinline__ void join_units(const GnArgs& a, const PackedUnit& u, float* sMean, float* sRstd) {
    const int cg = a.c / a.groups;
    const float total = (float)u.rows * (float)cg;
    for (int g = threadIdx.x; g < a.groups; g += GN_NT) {
        const float2* p = a.part + (int64_t)u.first * a.groups + g;
        // (the units' means less the first one's: of equal values the mean is that value)
        const float m0 = p->x;
        float m = 0.f;
        for (int i = 1; i < u.count; ++i)
            m += (p[(int64_t)i * a.groups].x - m0) * ((float)min(a.per, u.rows - i * a.per) * (float)cg / total);
        m += m0;
        float q = 0.f;
        for (int i = 0; i < u.count; ++i) {
            const float2 t = p[(int64_t)i * a.groups];
            const float d = t.x - m;
            q += t.y + d * d * (float)min(a.per, u.rows - i * a.per) * (float)cg;
        }
        sMean[g] = m;
        sRstd[g] = 1.0f / sqrtf(q / total + a.eps);
    }
    __syncthreads();
}

template <int XDT, int ODT>
__global__ __launch_bounds__(GN_NT) void k_gn_apply(GnArgs a) {
    __shared__ float sMean[GN_MAX_GROUPS], sRstd[GN_MAX_GROUPS];
    const PackedUnit u = packed_unit(a.offsets, a.samples, (int)a.n, 1, a.per, blockIdx.x);
    if (u.sample < 0) return;
    join_units(a, u, sMean, sRstd);
    int64_t row;
    const int rows = unit_rows(u, blockIdx.x, a.per, row);
    const int cg = a.c / a.groups;
    const auto* x = reinterpret_cast<const typename Elem<XDT>::storage*>(a.x);
    auto* out = reinterpret_cast<typename Elem<ODT>::storage*>(a.out);
    for (int64_t e = threadIdx.x; e < (int64_t)rows * a.c; e += GN_NT) {
        const int ch = (int)(e % a.c), g = ch / cg;
        float y = (Elem<XDT>::load(x, row * a.c + e) - sMean[g]) * sRstd[g];
        if (a.gamma) y *= a.gamma[ch];
        if (a.beta) y += a.beta[ch];
        Elem<ODT>::store(out, row * a.c + e, act(y, a.silu));
    }
}

// Rows of a unit: about 512 units, of 16 rows at least.
int gn_per(int64_t n) { return (int)std::max<int64_t>(16, ceil_div(n, 512)); }
int64_t gn_units(int64_t n, int samples) { return ceil_div(n, gn_per(n)) + samples; }

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

extern "C" size_t tsp_group_norm_workspace_bytes(int64_t n, int c, int groups, int samples) {
    if (n <= 0 || n >= (1ll << 31) - (1ll << 24) || c <= 0 || groups <= 0 || samples <= 0) return 0;
    return (size_t)gn_units(n, samples) * groups * sizeof(float2);
}

extern "C" int tsp_group_norm(const void* d_x, int x_dtype, int64_t n, int c, int groups, const int32_t* d_offsets,
                              int samples, const float* d_gamma, const float* d_beta, float eps, int silu, void* d_out,
                              int out_dtype, void* d_workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    TSP_REQUIRE(n >= 0 && n < (1ll << 31) - (1ll << 24) && c > 0, TSP_ERR_INVALID, "tsp_group_norm: n=%lld c=%d out of range", (long long)n, c);
    TSP_REQUIRE(groups > 0 && c % groups == 0, TSP_ERR_INVALID, "tsp_group_norm: %d channels in %d groups", c, groups);
    TSP_REQUIRE(samples > 0 && (d_offsets || samples == 1), TSP_ERR_INVALID,
                "tsp_group_norm: samples=%d (without offsets: 1)", samples);
    TSP_REQUIRE(dtype_valid(x_dtype) && dtype_valid(out_dtype), TSP_ERR_INVALID, "tsp_group_norm: bad dtype");
    TSP_REQUIRE(eps >= 0.f, TSP_ERR_INVALID, "tsp_group_norm: negative eps");
    TSP_REQUIRE(groups <= GN_MAX_GROUPS, TSP_ERR_UNSUPPORTED, "tsp_group_norm: more than %d groups", GN_MAX_GROUPS);
    if (n == 0) return TSP_OK;
    TSP_REQUIRE(d_x && d_out && d_workspace, TSP_ERR_INVALID, "tsp_group_norm: null pointer");
    TSP_REQUIRE(d_out != d_x || x_dtype == out_dtype, TSP_ERR_INVALID, "tsp_group_norm: in place needs one dtype");
    TSP_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 8 == 0, TSP_ERR_INVALID, "tsp_group_norm: workspace not 8-byte aligned");
    TSP_REQUIRE(workspace_bytes >= tsp_group_norm_workspace_bytes(n, c, groups, samples), TSP_ERR_WORKSPACE,
                "tsp_group_norm: workspace of %zu bytes, needs %zu", workspace_bytes,
                tsp_group_norm_workspace_bytes(n, c, groups, samples));
    const int64_t units = gn_units(n, samples);
    TSP_REQUIRE(units * GN_NT < (1ll << 32), TSP_ERR_INVALID, "tsp_group_norm: too many samples");
    hipStream_t s = as_stream(stream);
    const GnArgs a{d_x, d_out, d_offsets, d_gamma, d_beta, static_cast<float2*>(d_workspace), n, c, groups, samples, gn_per(n), eps, silu};
    dt_switch(x_dtype, [&](auto xd) {
        constexpr int XD = decltype(xd)::value;
        hipLaunchKernelGGL((k_gn_stats<XD>), dim3((unsigned)units, (unsigned)groups), dim3(GN_NT), 0, s, a);
        dt_switch(out_dtype, [&](auto od) {
            hipLaunchKernelGGL((k_gn_apply<XD, decltype(od)::value>), dim3((unsigned)units), dim3(GN_NT), 0, s, a);
        });
    });
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
