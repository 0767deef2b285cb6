// Group norm over packed samples, channels last: for sample s and group g of C / G channels,
//   y = (x - mean) / sqrt(var + eps) * gamma[c] + beta[c], then y * sigmoid(y) where asked,
// mean and (biased) var over the sample's rows and the group's channels.
//
// Launches over the same units of rows: the first leaves each unit's mean and sum of squared deviations
// per group in the workspace, the last normalises the rows; between them a sample's units are joined (in
// the order of the units, whatever the order in which they ran), by a launch of its own where they are many.
// Small samples take one launch.
//
// Bound by memory: x is read twice and out written once. Eight channels a thread (16 bytes of a 16-bit row),
// four rows in flight; the last launch's first rows are on their way before its statistics. 599,577 x 128, f32 to
// bf16, 2 samples: 63 us (4.9 TB/s), 6 and 75 us (6.1 TB/s: the second read comes from the memory-side cache in
// part); 60,013 x 256, bf16, 6 samples: 10, 4 and 12 us.
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
    float2* stat;          // [sample][group]: mean, 1 / sqrt(var + eps); NULL: the last launch joins the units
    int64_t n;
    int c, groups, samples, per;
    float eps;
    int silu;
    int units;             // workgroups of the first and the last launch, units in part
    FastDiv by_cols, by_group, by_slots;      // 16-byte pieces of a row (or of a small sample's slab), channels of a group, its sums of a lane
};

__device__ __forceinline__ int unit_rows(const PackedUnit& u, int unit, int per, int64_t& row) {
    const int lo = (unit - u.first) * per;
    row = u.row0 + lo;
    return min(u.rows - lo, per);
}

// y * sigmoid(y): the hardware's exp2 and reciprocal (1 step each; the exponent's own rounding is |y| 2^-24
// of the result), an eighth of the instructions of expf and a division, which would bound the pass.
__device__ __forceinline__ float act(float y, int silu) {
    return silu ? y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * -1.44269504088896340736f)) : y;
}

// Eight consecutive values (16-byte accesses; the address is aligned).
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
    if constexpr (DT == TSP_F32) {
        const f32x4_t* x = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + i);
        const f32x4_t a = x[0], b = x[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
    } else {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint16_t lo = (uint16_t)(a[e] & 0xffffu), hi = (uint16_t)(a[e] >> 16);
            v[2 * e] = DT == TSP_BF16 ? bf16_bits_to_f32(lo) : f16_bits_to_f32(lo);
            v[2 * e + 1] = DT == TSP_BF16 ? bf16_bits_to_f32(hi) : f16_bits_to_f32(hi);
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
        for (int e = 0; e < 4; ++e)
            a[e] = DT == TSP_BF16 ? f32x2_to_bf16x2_bits(v[2 * e], v[2 * e + 1])
                                  : f32_to_f16_bits(v[2 * e]) | ((uint32_t)f32_to_f16_bits(v[2 * e + 1]) << 16);
        *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(p) + i) = a;
    }
}

// Lanes that share a group's sums, a power of two: all threads where there are few groups.
__device__ __forceinline__ int lanes_a_group(int groups) {
    int l = 64;
    while (l > 1 && l * groups > GN_NT) l >>= 1;
    return l;
}
__device__ __forceinline__ float sum_over(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Mean, sum of squared deviations and count of some values.
struct Stat {
    float mean, dev, n;
};
// ... from sums of x - shift and of its square. A shift among the values keeps a mean far from zero from
// swallowing the variance; of n values, one that is far from all others swallows log2 n bits of it.
__device__ __forceinline__ float2 stat_of(float s, float q, float shift, float n) {
    const float m = s / n;
    return float2{shift + m, fmaxf(q - s * m, 0.f)};
}
// `count` parts of `total` values joined by `lanes` lanes of which this is `sub`; all get the result. The sums go
// about the mean of the first parts' means, one a lane, so that a first part far from the others does no harm
// (parts that are all equal have their mean exactly).
template <class Part>
__device__ __forceinline__ float2 join_parts(int count, float total, int lanes, int sub, Part part) {
    const float first = part(0).mean;
    const float m0 = first + sum_over(part(min(sub, count - 1)).mean - first, lanes) / (float)lanes;
    float s = 0.f, q = 0.f;
#pragma unroll 8
    for (int i = sub; i < count; i += lanes) {
        const Stat t = part(i);
        const float d = t.mean - m0;
        s += t.n * d;
        q += t.dev + t.n * d * d;
    }
    return stat_of(sum_over(s, lanes), sum_over(q, lanes), m0, total);
}

// One group of one unit a workgroup, element by element: any width and alignment.
template <int XDT>
__global__ __launch_bounds__(GN_NT) void k_gn_stats(GnArgs a) {
    __shared__ float2 sPart[GN_NT];
    const PackedUnit u = packed_unit(a.offsets, a.samples, (int)a.n, 1, a.per, blockIdx.x);
    if (u.sample < 0) return;
    int64_t row;
    const int rows = unit_rows(u, blockIdx.x, a.per, row);
    const int cg = a.c / a.groups, g = blockIdx.y;
    const auto* x = reinterpret_cast<const typename Elem<XDT>::storage*>(a.x) + row * a.c + g * cg;
    const int64_t cnt = (int64_t)rows * cg;
    float s = 0.f, q = 0.f, shift = 0.f;
    for (int64_t e = threadIdx.x; e < cnt; e += GN_NT) {
        const int64_t r = e / cg;
        const float v = Elem<XDT>::load(x, r * a.c + (e - r * cg));
        if (e == threadIdx.x) shift = v;
        s += v - shift;
        q += (v - shift) * (v - shift);
    }
    auto held = [&](int t) { return (float)((cnt - t + GN_NT - 1) / GN_NT); };      // values of thread t
    if (threadIdx.x < cnt) sPart[threadIdx.x] = stat_of(s, q, shift, held(threadIdx.x));
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const float2 t = join_parts((int)min(cnt, (int64_t)GN_NT), (float)cnt, 64, threadIdx.x,
                                [&](int i) { return Stat{sPart[i].x, sPart[i].y, held(i)}; });
    if (threadIdx.x == 0) a.part[(int64_t)blockIdx.x * a.groups + g] = t;
}

// All groups of one unit a workgroup: a thread keeps the sums of eight channels (of one value, PER = 1,
// where they lie in one group, else of each) over every lanes-th row, about the mean of the first of them;
// they meet in LDS.
template <int XDT, int PER>
__global__ __launch_bounds__(GN_NT) void k_gn_stats_vec(GnArgs a) {
    __shared__ float2 sSum[GN_NT * PER];
    const PackedUnit u = packed_unit(a.offsets, a.samples, (int)a.n, 1, a.per, blockIdx.x);
    if (u.sample < 0) return;
    int64_t row;
    const int rows = unit_rows(u, blockIdx.x, a.per, row);
    const int cols = a.c / 8, lanes = GN_NT / cols, cg = a.c / a.groups;
    const int lane = (int)threadIdx.x / a.by_cols, col = threadIdx.x - lane * cols;
    const bool live = lane < lanes;
    constexpr int DEEP = 4, EACH = 8 / PER;      // rows in flight (past the last: the last again, not counted)
    const int whole = rows / lanes, more = rows - whole * lanes;
    auto held = [&](int l) { return (float)((whole + (l < more ? 1 : 0)) * EACH); };      // values of a sum of lane l
    if (live && lane < rows) {
        float s[PER] = {}, q[PER] = {}, shift[PER] = {};
        for (int r = lane; r < rows; r += DEEP * lanes) {
            float x[DEEP][8];
#pragma unroll
            for (int i = 0; i < DEEP; ++i) load8<XDT>(a.x, (row + min(r + i * lanes, rows - 1)) * a.c + col * 8, x[i]);
            if (r == lane) {
#pragma unroll
                for (int k = 0; k < PER; ++k) {
                    float d = 0.f;
#pragma unroll
                    for (int i = 0; i < DEEP; ++i)
#pragma unroll
                        for (int e = 0; e < EACH; ++e) d += x[i][k + e] - x[0][k];
                    shift[k] = x[0][k] + d * (1.f / (DEEP * EACH));
                }
            }
#pragma unroll
            for (int i = 0; i < DEEP; ++i) {
                if (r + i * lanes >= rows) break;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int k = PER == 1 ? 0 : e;
                    const float d = x[i][e] - shift[k];
                    s[k] += d;
                    q[k] += d * d;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) sSum[(lane * cols + col) * PER + k] = stat_of(s[k], q[k], shift[k], held(lane));
    }
    __syncthreads();
    const int lg = lanes_a_group(a.groups), sub = threadIdx.x & (lg - 1), slots = cg * PER / 8;
    const float total = (float)rows * (float)cg;
    for (int g0 = 0; g0 < a.groups; g0 += GN_NT / lg) {
        const int g = g0 + threadIdx.x / lg, at = min(g, a.groups - 1) * slots;
        const float2 t = join_parts(min(lanes, rows) * slots, total, lg, sub, [&](int e) {
            const int l = e / a.by_slots;
            const float2 v = sSum[l * cols * PER + at + (e - l * slots)];
            return Stat{v.x, v.y, held(l)};
        });
        if (g < a.groups && sub == 0) a.part[(int64_t)blockIdx.x * a.groups + g] = t;
    }
}

// Mean and 1 / sqrt(var + eps) of group g from the sample's units. (Offsets out of order can name more units
// than there are: those are not read.)
__device__ __forceinline__ float2 join_units(const GnArgs& a, const PackedUnit& u, int g, int lanes, int sub) {
    const float cg = (float)(a.c / a.groups), total = (float)u.rows * cg;
    const int first = max(u.first, 0), count = min(u.count, a.units - first);
    const float2* p = a.part + (int64_t)first * a.groups + g;
    const float2 t = join_parts(count, total, lanes, sub, [&](int i) {
        const float2 v = p[(int64_t)i * a.groups];
        return Stat{v.x, v.y, (float)min(a.per, u.rows - i * a.per) * cg};
    });
    return float2{t.x, 1.0f / sqrtf(t.y / total + a.eps)};
}

// A wave a sample and group: where there are more than GN_FEW units, every workgroup of the last launch
// joining them for itself would read them all some hundred times over (512 units of 32 groups: 15 us).
constexpr int GN_FEW = 256;
__global__ __launch_bounds__(256) void k_gn_join(GnArgs a) {
    const int g = blockIdx.y * 4 + (threadIdx.x >> 6), sample = blockIdx.x;
    if (g >= a.groups) return;
    const PackedUnit u = packed_sample(a.offsets, (int)a.n, 1, a.per, sample);
    if (u.rows == 0 || u.first >= a.units) return;
    const float2 t = join_units(a, u, g, 64, threadIdx.x & 63);
    if ((threadIdx.x & 63) == 0) a.stat[(int64_t)sample * a.groups + g] = t;
}

// The statistics of the unit's sample, into LDS.
__device__ __forceinline__ void sample_stats(const GnArgs& a, const PackedUnit& u, float* sMean, float* sRstd) {
    if (a.stat) {
        for (int g = threadIdx.x; g < a.groups; g += GN_NT) {
            const float2 t = a.stat[(int64_t)u.sample * a.groups + g];
            sMean[g] = t.x;
            sRstd[g] = t.y;
        }
    } else {
        const int lg = lanes_a_group(a.groups), sub = threadIdx.x & (lg - 1);
        for (int g0 = 0; g0 < a.groups; g0 += GN_NT / lg) {
            const int g = g0 + threadIdx.x / lg;
            const float2 t = join_units(a, u, min(g, a.groups - 1), lg, sub);
            if (g < a.groups && sub == 0) {
                sMean[g] = t.x;
                sRstd[g] = t.y;
            }
        }
    }
    __syncthreads();
}

template <int XDT, int ODT>
__global__ __launch_bounds__(GN_NT) void k_gn_apply(GnArgs a) {
    __shared__ float sMean[GN_MAX_GROUPS], sRstd[GN_MAX_GROUPS];
    const PackedUnit u = packed_unit(a.offsets, a.samples, (int)a.n, 1, a.per, blockIdx.x);
    if (u.sample < 0) return;
    sample_stats(a, u, sMean, sRstd);
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

// ... eight channels a thread, their factors in registers for all its rows. The units go in the reverse of
// the first launch's order: what it read last is still in the caches.
template <int XDT, int ODT>
__global__ __launch_bounds__(GN_NT) void k_gn_apply_vec(GnArgs a) {
    __shared__ float sMean[GN_MAX_GROUPS], sRstd[GN_MAX_GROUPS];
    const int unit = gridDim.x - 1 - blockIdx.x;
    const PackedUnit u = packed_unit(a.offsets, a.samples, (int)a.n, 1, a.per, unit);
    if (u.sample < 0) return;
    int64_t row;
    const int rows = unit_rows(u, unit, a.per, row);
    const int cols = a.c / 8, lanes = GN_NT / cols;
    const int lane = (int)threadIdx.x / a.by_cols, col = threadIdx.x - lane * cols;
    constexpr int DEEP = 4;
    float x[DEEP][8], f[8], b[8];
    auto load = [&](int r) {      // (past the last row: the last again, not stored)
#pragma unroll
        for (int i = 0; i < DEEP; ++i) load8<XDT>(a.x, (row + min(r + i * lanes, rows - 1)) * a.c + col * 8, x[i]);
    };
    // the first rows and the factors are on their way while the statistics are joined
    load(lane);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 1.f, b[e] = 0.f;
    if (a.gamma) load8<TSP_F32>(a.gamma, col * 8, f);
    if (a.beta) load8<TSP_F32>(a.beta, col * 8, b);
    sample_stats(a, u, sMean, sRstd);
    if (lane >= lanes) return;
    float mean[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int g = (col * 8 + e) / a.by_group;
        mean[e] = sMean[g];
        f[e] *= sRstd[g];
    }
    const int silu = a.silu;
    for (int r = lane; r < rows; r += DEEP * lanes) {
        if (r != lane) load(r);
#pragma unroll
        for (int i = 0; i < DEEP; ++i) {
            if (r + i * lanes >= rows) break;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = act((x[i][e] - mean[e]) * f[e] + b[e], silu);
            store8<ODT>(a.out, (row + r + i * lanes) * a.c + col * 8, y);
        }
    }
}

// Small samples in one launch: a workgroup takes one group of whole 16-byte pieces (or the groups of one
// piece, `PER` of them) of a whole sample, held in registers, so that x is read once and mean and deviations
// are formed one after the other. Where there is room, the workgroups of gridDim.z form the same sums, and each
// writes one row a thread only: SiLU and rounding are most of the work (2,606 x 64 f32: 9.4 us by one, 8.6 by three;
// not in place, where one would read what another has written).
constexpr int GS_NT = 1024, GS_ROWS = 4;          // threads, rows a thread holds at most
template <int XDT, int ODT, int PER>
__global__ __launch_bounds__(GS_NT) void k_gn_small(GnArgs a) {
    __shared__ float sSum[2][PER][GS_NT / 64];
    int row0, rows;
    packed_rows(a.offsets, blockIdx.y, (int)a.n, row0, rows);
    if (rows == 0) return;
    const int cg = a.c / a.groups, slab = cg < 8 ? 8 : cg, cols = slab / 8, lanes = GS_NT / cols;
    const int only = gridDim.z > 1 ? (int)blockIdx.z : -1;
    if (only * lanes >= rows) return;
    const int lane = (int)threadIdx.x / a.by_cols, col = threadIdx.x - lane * cols;
    const int ch = blockIdx.x * slab + col * 8;
    const int mine = lane < lanes ? (rows - lane + lanes - 1) / lanes : 0;       // rows of this thread
    const auto* first = reinterpret_cast<const typename Elem<XDT>::storage*>(a.x) + (int64_t)row0 * a.c + blockIdx.x * slab;
    float x[GS_ROWS][8], gamma[8], beta[8], shift[PER];
#pragma unroll
    for (int i = 0; i < GS_ROWS; ++i)
        if (i < mine) load8<XDT>(a.x, (int64_t)(row0 + lane + i * lanes) * a.c + ch, x[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) gamma[e] = 1.f, beta[e] = 0.f;
    if (a.gamma) load8<TSP_F32>(a.gamma, ch, gamma);
    if (a.beta) load8<TSP_F32>(a.beta, ch, beta);
    // the first sums go about one of the group's values, so that equal ones have their mean exactly: about the
    // median of three, as one far from all others would round the mean to its own precision
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        auto value = [&](int r) { return Elem<XDT>::load(first, (int64_t)r * a.c + k * (8 / PER)); };
        shift[k] = __builtin_amdgcn_fmed3f(value(0), value(rows / 2), value(rows - 1));
    }
    auto workgroup_sums = [&](float (&v)[PER], int buffer) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            v[k] = group_sum<64>(v[k]);
            if ((threadIdx.x & 63) == 0) sSum[buffer][k][threadIdx.x >> 6] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; ++k) v[k] = group_sum<16>(sSum[buffer][k][threadIdx.x & 15]);
    };
    const float count = (float)rows * (float)cg;
    float mean[PER] = {}, var[PER] = {};
#pragma unroll
    for (int i = 0; i < GS_ROWS; ++i)
        if (i < mine)
#pragma unroll
            for (int e = 0; e < 8; ++e) mean[e * PER / 8] += x[i][e] - shift[e * PER / 8];
    workgroup_sums(mean, 0);
#pragma unroll
    for (int k = 0; k < PER; ++k) mean[k] = shift[k] + mean[k] / count;
#pragma unroll
    for (int i = 0; i < GS_ROWS; ++i)
        if (i < mine)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = x[i][e] - mean[e * PER / 8];
                var[e * PER / 8] += d * d;
            }
    workgroup_sums(var, 1);
#pragma unroll
    for (int k = 0; k < PER; ++k) var[k] = 1.0f / sqrtf(var[k] / count + a.eps);
#pragma unroll
    for (int i = 0; i < GS_ROWS; ++i) {
        if (i >= mine) break;
        if (only >= 0 && i != only) continue;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = act((x[i][e] - mean[e * PER / 8]) * (var[e * PER / 8] * gamma[e]) + beta[e], a.silu);
        store8<ODT>(a.out, (int64_t)(row0 + lane + i * lanes) * a.c + ch, y);
    }
}

// Whether samples of up to n rows fit it. Eight rows a thread would still hold them, but lose to three
// launches (bf16: 8,192 x 64 in 32 groups 14.9 us and 10.5; four rows: 2,606 x 64 8.1 and 9.6).
bool gn_small(int64_t n, int c, int groups, int samples) {
    const int cg = c / groups;
    if ((cg % 8 && 8 % cg) || samples > 65535 || cg > 8 * GS_NT) return false;
    return n <= (int64_t)GS_ROWS * (GS_NT / (cg < 8 ? 1 : cg / 8));
}

// Rows of a unit. Four rows a thread at least (one batch of loads; eight channels a thread): 60,013 x 64 in
// bf16 takes 14.6 us so, 18.0 with two. About 512 units, which the device holds at once; 1024 where that is
// far more than the caches hold and only the loads in flight count (bf16 with SiLU: 300,000 x 512 takes
// 199 us with 512, 183 with 1024; 60,013 x 256 26 and 30).
int gn_per(int64_t n, int c) {
    return (int)std::max<int64_t>(4 * std::max(1, GN_NT * 8 / c), ceil_div(n, n * c > (1ll << 27) ? 1024 : 512));
}
int64_t gn_units(int64_t n, int c, int samples) { return ceil_div(n, gn_per(n, c)) + (samples > 1 ? samples : 0); }

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
    return (size_t)(gn_units(n, c, samples) + samples) * groups * sizeof(float2);
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
    // (in place a workgroup reads what it writes and no other's rows: only where both are the same values)
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(d_x), o0 = reinterpret_cast<uintptr_t>(d_out);
    auto bytes = [&](int dt) { return (uintptr_t)n * c * (dt == TSP_F32 ? 4 : 2); };
    TSP_REQUIRE(x0 == o0 || x0 + bytes(x_dtype) <= o0 || o0 + bytes(out_dtype) <= x0, TSP_ERR_INVALID,
                "tsp_group_norm: out overlaps x in part (it may be x, or apart)");
    const int64_t units = gn_units(n, c, samples);
    TSP_REQUIRE(units * GN_NT < (1ll << 32), TSP_ERR_INVALID, "tsp_group_norm: too many samples");
    hipStream_t s = as_stream(stream);
    float2* part = static_cast<float2*>(d_workspace);
    GnArgs a{d_x, d_out, d_offsets, d_gamma, d_beta, part, units > GN_FEW ? part + units * groups : nullptr, n, c, groups, samples, gn_per(n, c), eps, silu,
             (int)units, fast_div(std::max(1, c / 8)), fast_div(c / groups), fast_div(c / groups % 8 == 0 ? c / groups / 8 : c / groups)};
    // rows of whole 16-byte pieces, eight channels a thread; element by element otherwise
    const bool vec = c % 8 == 0 && c <= 8 * GN_NT && !(reinterpret_cast<uintptr_t>(d_x) % 16 || reinterpret_cast<uintptr_t>(d_out) % 16 ||
                       reinterpret_cast<uintptr_t>(d_gamma) % 16 || reinterpret_cast<uintptr_t>(d_beta) % 16);
    if (vec && gn_small(n, c, groups, samples)) {
        const int cg = c / groups;
        a.by_cols = fast_div(cg < 8 ? 1 : cg / 8);
        const int64_t slabs = c / (cg < 8 ? 8 : cg), rows = ceil_div(n, GS_NT / (cg < 8 ? 1 : cg / 8));      // (rows a thread)
        const bool share = d_out != d_x && slabs * samples * rows <= 256;
        const dim3 grid((unsigned)slabs, (unsigned)samples, share ? (unsigned)rows : 1), block(GS_NT);
        dt_switch(x_dtype, [&](auto xd) {
            dt_switch(out_dtype, [&](auto od) {
                constexpr int XD = decltype(xd)::value, OD = decltype(od)::value;
                if (cg >= 8) hipLaunchKernelGGL((k_gn_small<XD, OD, 1>), grid, block, 0, s, a);
                else if (cg == 4) hipLaunchKernelGGL((k_gn_small<XD, OD, 2>), grid, block, 0, s, a);
                else if (cg == 2) hipLaunchKernelGGL((k_gn_small<XD, OD, 4>), grid, block, 0, s, a);
                else hipLaunchKernelGGL((k_gn_small<XD, OD, 8>), grid, block, 0, s, a);
            });
        });
        TSP_CHECK_LAUNCH();
        return TSP_OK;
    }
    const dim3 grid((unsigned)units), block(GN_NT);
    dt_switch(x_dtype, [&](auto xd) {
        constexpr int XD = decltype(xd)::value;
        if (!vec) hipLaunchKernelGGL((k_gn_stats<XD>), dim3((unsigned)units, (unsigned)groups), block, 0, s, a);
        else if (c / groups % 8 == 0) hipLaunchKernelGGL((k_gn_stats_vec<XD, 1>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((k_gn_stats_vec<XD, 8>), grid, block, 0, s, a);
        if (a.stat) hipLaunchKernelGGL(k_gn_join, dim3((unsigned)samples, (unsigned)ceil_div(groups, 4)), dim3(256), 0, s, a);
        dt_switch(out_dtype, [&](auto od) {
            if (vec) hipLaunchKernelGGL((k_gn_apply_vec<XD, decltype(od)::value>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((k_gn_apply<XD, decltype(od)::value>), grid, block, 0, s, a);
        });
    });
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
