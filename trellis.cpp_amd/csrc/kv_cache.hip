// New keys and values into a paged cache, the queries and keys RMS-normalised (optional) and turned to their positions
// on the way; and the same rows out of it again.
//
// Row i of a sample that gets m rows becomes its key lengths[s] - m + i. A row's angles are formed once for all its
// heads, in turns and in 64 bits. Keys for 4 bits are normalised and turned in 64 bits too, so that a code is the
// right one of its value whatever the order of operations (32 bits would miss some two in a million); they come to
// the conversion with the bits that 32 lose kept as one that is odd. Queries, and keys for 16 bits, take 32.
//
// Bound by memory: one read and one write. 60,013 rows, 16 + 16 heads of 64 in f16 on three axes, take 156 us (738 MB, 4.7 TB/s,
// a large copy's rate); into 4 bits 155, where the 64-bit angles and turns weigh as much. 12,345 rows, 16 + 4 heads of 128 in
// bf16 with norms, into 4 bits take 38 us (134 MB moved, 3.5 TB/s; the vector units are 55 % busy) and
// 30.5 into 16; their gather 10 (37 MB). 16 rows take 6 us in a graph's replay (7.4 in a trace), the latency of offsets,
// length, table and sine one after the other, and their gather 2.9 (3.7).
// A group of lanes takes a row, so that its angles, place and page are formed once for all heads; where rows are few, heads
// are dealt to as many groups as fill the device. A loop over rows kept the sine's constants in registers for all of it
// (12,345 rows 46 us, 38 without).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "inverse_root.hpp"
#include "kv_cache.hpp"
#include "mx.hpp"
#include "overlap.hpp"
#include "packed.hpp"

namespace tsp {
namespace {

constexpr int KV_NT = 256;
constexpr int KV_MAX_AXES = 4, KV_MAX_PAIRS = KV_MAX_D / 2;

struct AppendArgs {
    KvArgs cache;
    const void *q, *k, *v;
    void* q_out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;     // strides in elements
    const float *q_gamma, *k_gamma;
    const int32_t *offsets, *pos;
    int64_t n, first;                // rows, the launch's first
    int samples, hq, d, axes, parts;
    double eps;
    double turns[KV_MAX_PAIRS];      // theta^(-j / P) / (2 pi) of each pair
    int8_t axis[KV_MAX_PAIRS];       // its axis, -1: not turned
};

// Four pairs of a head: elements 8 u .. 8 u + 7, or with halves 4 u .. 4 u + 3 of each half.
template <int DT, bool HALVES>
__device__ __forceinline__ void load_pairs(const void* p, int64_t at, int unit, int d, float (&u)[4], float (&v)[4]) {
    if constexpr (HALVES) {
        if constexpr (DT == TSP_F32) {
            const float* x = static_cast<const float*>(p) + at + 4 * unit;
            const f32x4_t a = *reinterpret_cast<const f32x4_t*>(x), b = *reinterpret_cast<const f32x4_t*>(x + d / 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = a[i], v[i] = b[i];
        } else {
            const uint16_t* x = static_cast<const uint16_t*>(p) + at + 4 * unit;
            const uint2 a = *reinterpret_cast<const uint2*>(x), b = *reinterpret_cast<const uint2*>(x + d / 2);
            auto f = [](uint32_t w) { return DT == TSP_BF16 ? bf16_bits_to_f32((uint16_t)w) : f16_bits_to_f32((uint16_t)w); };
            u[0] = f(a.x), u[1] = f(a.x >> 16), u[2] = f(a.y), u[3] = f(a.y >> 16);
            v[0] = f(b.x), v[1] = f(b.x >> 16), v[2] = f(b.y), v[3] = f(b.y >> 16);
        }
    } else {
        float x[8];
        load8<DT>(p, at + 8 * unit, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = x[2 * i], v[i] = x[2 * i + 1];
    }
}
template <int DT, bool HALVES>
__device__ __forceinline__ void store_pairs(void* p, int64_t at, int unit, int d, const float (&u)[4], const float (&v)[4]) {
    if constexpr (HALVES) {
        if constexpr (DT == TSP_F32) {
            float* y = static_cast<float*>(p) + at + 4 * unit;
            *reinterpret_cast<f32x4_t*>(y) = f32x4_t{u[0], u[1], u[2], u[3]};
            *reinterpret_cast<f32x4_t*>(y + d / 2) = f32x4_t{v[0], v[1], v[2], v[3]};
        } else {
            auto two = [](float a, float b) {
                return DT == TSP_BF16 ? f32x2_to_bf16x2_bits(a, b) : f32_to_f16_bits(a) | ((uint32_t)f32_to_f16_bits(b) << 16);
            };
            uint16_t* y = static_cast<uint16_t*>(p) + at + 4 * unit;
            *reinterpret_cast<uint2*>(y) = uint2{two(u[0], u[1]), two(u[2], u[3])};
            *reinterpret_cast<uint2*>(y + d / 2) = uint2{two(v[0], v[1]), two(v[2], v[3])};
        }
    } else {
        const float x[8] = {u[0], v[0], u[1], v[1], u[2], v[2], u[3], v[3]};
        store8<DT>(p, at + 8 * unit, x);
    }
}

template <int L>
__device__ __forceinline__ float sum_of(float v) { return group_sum<L>(v); }
template <int L>
__device__ __forceinline__ double sum_of(double v) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// v for a rounding to fewer bits that must be v's own: cut to 32 bits, the last of them 1 where that left any out.
__device__ __forceinline__ float to_odd(float v) { return v; }
__device__ __forceinline__ float to_odd(double v) {
    const float f = (float)v;
    if ((double)f == v || v != v || fabsf(f) == INFINITY) return f;
    const uint32_t b = __float_as_uint(f);
    // (towards zero where the rounding went away from it)
    return __uint_as_float((fabs((double)f) > fabs(v) ? b - 1 : b) | 1);
}

// Four pairs normalised and turned.
template <int L, class T>
__device__ __forceinline__ void turn(T (&u)[4], T (&v)[4], const float* gamma, bool halves, int unit, int d, bool live, double eps,
                                     const int (&axis)[4], const T (&cs)[4], const T (&sn)[4]) {
    if (gamma) {
        float gu[4] = {}, gv[4] = {};
        if (live) {
            if (halves) load_pairs<TSP_F32, true>(gamma, 0, unit, d, gu, gv);
            else load_pairs<TSP_F32, false>(gamma, 0, unit, d, gu, gv);
        }
        T q = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) q += u[i] * u[i] + v[i] * v[i];
        const T scale = inverse_root(sum_of<L>(q) / (T)d + (T)eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] *= scale * (T)gu[i];
            v[i] *= scale * (T)gv[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (axis[i] < 0) continue;      // (not 0 * Inf)
        const T p = u[i] * cs[i] - v[i] * sn[i], r = v[i] * cs[i] + u[i] * sn[i];
        u[i] = p;
        v[i] = r;
    }
}

// A group of L lanes takes one row and every `part`-th of its heads, eight channels a lane. HELD: TSP_KV_MX4, TSP_F16
// or TSP_BF16.
template <int XDT, int HELD, int L, bool HALVES>
__global__ __launch_bounds__(KV_NT) void k_kv_append(AppendArgs a) {
    using KT = std::conditional_t<HELD == TSP_KV_MX4, double, float>;      // what keys are turned in
    const int unit = threadIdx.x % L;
    const bool live = unit * 8 < a.d;
    int axis[4];
    double turns[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        axis[i] = live ? a.axis[4 * unit + i] : -1;
        turns[i] = axis[i] < 0 ? 0. : a.turns[4 * unit + i];
    }
    // (whole groups of lanes leave together. No loop: the sine's constants would be kept in registers for all of it)
    const unsigned item = (blockIdx.x * KV_NT + threadIdx.x) / L;
    const int64_t at = a.first + item / (unsigned)a.parts;
    if (at >= a.n) return;
    const int row = (int)at, part = (int)(item % (unsigned)a.parts);
    int sample, row0, rows;
    if (!row_sample<L>(a.offsets, a.samples, (int)a.n, row, sample, row0, rows)) return;
    KT cs[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        cs[i] = 1, sn[i] = 0;
        if (axis[i] >= 0) {
            const double t = (double)a.pos[(int64_t)row * a.axes + axis[i]] * turns[i];
            const KT f = 2 * (KT)(t - rint(t));
            if constexpr (HELD == TSP_KV_MX4) sincospi(f, &sn[i], &cs[i]);
            else sincospif(f, &sn[i], &cs[i]);
        }
        if constexpr (HELD == TSP_KV_MX4) __builtin_amdgcn_sched_barrier(0);      // (one after the other: registers)
    }
    const int64_t key = (int64_t)a.cache.lengths[sample] - rows + (row - row0);
    const int slot = (int)key & ((1 << a.cache.page_bits) - 1);
    uint8_t* page = key >= 0 && key < (int64_t)a.cache.max_pages << a.cache.page_bits ? kv_head(a.cache, sample, key, 0) : nullptr;
    // (keys first: their 64-bit angles are not kept for the queries)
    // In 16 bits two heads' loads go out at a time; in 4 their registers would cost more than that gains (12,345 rows: 38 us, and
    // 46 so).
    constexpr int KB = HELD == TSP_KV_MX4 ? 1 : 2;
    for (int h0 = part; page && h0 < a.cache.heads; h0 += KB * a.parts) {
        float kus[KB][4] = {}, kvs[KB][4] = {}, xs[KB][8] = {};
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int h = h0 + b * a.parts;
            if (!live || h >= a.cache.heads) continue;
            load_pairs<XDT, HALVES>(a.k, row * a.k_row + h * a.k_head, unit, a.d, kus[b], kvs[b]);
            load8<XDT>(a.v, row * a.v_row + h * a.v_head + 8 * unit, xs[b]);
        }
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int h = h0 + b * a.parts;
            if (h >= a.cache.heads) break;
            uint8_t* to = page + h * a.cache.head_bytes;
            float (&u)[4] = kus[b], (&v)[4] = kvs[b], (&x)[8] = xs[b];
            KT ku[4], kv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) ku[i] = u[i], kv[i] = v[i];
            turn<L, KT>(ku, kv, a.k_gamma ? a.k_gamma + h * a.d : nullptr, HALVES, unit, a.d, live, a.eps, axis, cs, sn);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = to_odd(ku[i]), v[i] = to_odd(kv[i]);
            if constexpr (HELD == TSP_KV_MX4) {
                float y[8];
                if constexpr (HALVES) {
                    // The lane's eight channels are two runs of four, which stand in the first half of some lane
                    // or the second of another.
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int run = 2 * unit + r, half = a.d / 8;
                        const bool second = run >= half;
                        const int from = second ? run - half : run;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float p = __shfl(u[i], from, L), q = __shfl(v[i], from, L);
                            y[4 * r + i] = !live ? 0.f : second ? q : p;
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[2 * i] = u[i], y[2 * i + 1] = v[i];
                }
                const uint32_t kp = mx_power_of<MX_E2M1>(y), vp = mx_power_of<MX_E2M1>(x);
                if (unit < 4 * a.cache.blocks) {        // (channels past d among them: zeros)
                    *reinterpret_cast<uint32_t*>(to + kv_codes_at(a.cache, 0, slot) + unit * 4) = mx_codes4(y, kp);
                    *reinterpret_cast<uint32_t*>(to + kv_codes_at(a.cache, 1, slot) + unit * 4) = mx_codes4(x, vp);
                    if ((unit & 3) == 0) {
                        to[kv_powers_at(a.cache, 0, slot) + unit / 4] = (uint8_t)kp;
                        to[kv_powers_at(a.cache, 1, slot) + unit / 4] = (uint8_t)vp;
                    }
                }
            } else if (live) {
                store_pairs<HELD, HALVES>(to, (int64_t)slot * a.d, unit, a.d, u, v);
                store8<HELD>(to, ((1ll << a.cache.page_bits) + slot) * a.d + 8 * unit, x);
            }
        }
    }
    float fc[4], fs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) fc[i] = (float)cs[i], fs[i] = (float)sn[i];
    // (heads' loads go out BATCH at a time)
    constexpr int BATCH = 4;
    for (int h0 = part; h0 < a.hq; h0 += BATCH * a.parts) {
        float u[BATCH][4] = {}, v[BATCH][4] = {};
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int h = h0 + b * a.parts;
            if (live && h < a.hq) load_pairs<XDT, HALVES>(a.q, row * a.q_row + h * a.q_head, unit, a.d, u[b], v[b]);
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int h = h0 + b * a.parts;
            if (h >= a.hq) break;
            turn<L, float>(u[b], v[b], a.q_gamma ? a.q_gamma + h * a.d : nullptr, HALVES, unit, a.d, live, a.eps, axis, fc, fs);
            if (live) store_pairs<XDT, HALVES>(a.q_out, row * a.o_row + h * a.o_head, unit, a.d, u[b], v[b]);
        }
    }
}

struct GatherArgs {
    KvArgs cache;
    void *k, *v;
    int64_t k_row, k_head, v_row, v_head;
    const int32_t* offsets;
    int64_t n;
    int samples;
};

// A group of L lanes takes a row and key head. A key that the cache does not hold reads as zeros.
template <int HELD, int ODT, int L>
__global__ __launch_bounds__(KV_NT) void k_kv_gather(GatherArgs a) {
    const int unit = threadIdx.x % L;
    const int64_t items = a.n * a.cache.heads;
    for (int64_t item = ((int64_t)blockIdx.x * KV_NT + threadIdx.x) / L; item < items; item += (int64_t)gridDim.x * (KV_NT / L)) {
        const int row = (int)(item / a.cache.heads), h = (int)(item - (int64_t)row * a.cache.heads);
        int sample, row0, rows;
        if (!row_sample<L>(a.offsets, a.samples, (int)a.n, row, sample, row0, rows)) continue;
        const int64_t key = (int64_t)a.cache.lengths[sample] - rows + (row - row0);
        const bool held = key >= 0 && key < (int64_t)a.cache.max_pages << a.cache.page_bits;
        const uint8_t* from = held ? kv_head(a.cache, sample, key, h) : nullptr;
        if (unit * 8 >= a.cache.d) continue;
        const int slot = (int)key & ((1 << a.cache.page_bits) - 1);
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            float x[8] = {};
            if (from) {
                if constexpr (HELD == TSP_KV_MX4) {
                    const uint32_t c = *reinterpret_cast<const uint32_t*>(from + kv_codes_at(a.cache, side, slot) + unit * 4);
                    const float s = mx_scale(from[kv_powers_at(a.cache, side, slot) + unit / 4]);
                    const f32x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
                    const f32x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
                    x[0] = p0[0], x[1] = p0[1], x[2] = p1[0], x[3] = p1[1], x[4] = p2[0], x[5] = p2[1], x[6] = p3[0], x[7] = p3[1];
                } else {
                    load8<HELD>(from, ((int64_t)(side << a.cache.page_bits) + slot) * a.cache.d + 8 * unit, x);
                }
            }
            if (side == 0) store8<ODT>(a.k, row * a.k_row + h * a.k_head + 8 * unit, x);
            else store8<ODT>(a.v, row * a.v_row + h * a.v_head + 8 * unit, x);
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
template <class F>
void held_switch(int format, F&& f) {
    switch (format) {
        case TSP_KV_MX4: f(std::integral_constant<int, TSP_KV_MX4>{}); break;
        case TSP_F16: f(std::integral_constant<int, TSP_F16>{}); break;
        default: f(std::integral_constant<int, TSP_BF16>{}); break;
    }
}

}  // namespace
}  // namespace tsp

using namespace tsp;

extern "C" size_t tsp_kv_page_bytes(int page, int heads, int d, int format) {
    const tsp_kv_cache c{nullptr, 0, page, heads, d, format};
    return kv_valid(c) ? (size_t)(kv_head_bytes(c) * heads) : 0;
}

extern "C" int tsp_kv_append(const tsp_kv_cache* cache, const tsp_heads* k, const tsp_heads* v, int dtype, int64_t n,
                             const int32_t* d_offsets, int samples, const int32_t* d_table, int max_pages, const int32_t* d_lengths,
                             const tsp_heads* q, int hq, const int32_t* d_pos, int axes, const int* pairs, double theta, int flags,
                             const float* d_q_gamma, const float* d_k_gamma, double eps, const tsp_heads* q_out, void* stream) {
    clear_error();
    TSP_REQUIRE(cache, TSP_ERR_INVALID, "tsp_kv_append: null cache");
    const tsp_kv_cache& c = *cache;
    TSP_REQUIRE(kv_valid(c), TSP_ERR_UNSUPPORTED, "tsp_kv_append: a cache of %lld pages of %d tokens, %d heads of %d, format %d", (long long)c.pages,
                c.page, c.heads, c.d, c.format);
    TSP_REQUIRE(n >= 0 && n < (1ll << 31), TSP_ERR_INVALID, "tsp_kv_append: n=%lld out of range", (long long)n);
    TSP_REQUIRE(dtype_valid(dtype), TSP_ERR_INVALID, "tsp_kv_append: bad dtype");
    TSP_REQUIRE(samples > 0 && (samples == 1 || d_offsets), TSP_ERR_INVALID, "tsp_kv_append: samples=%d (without offsets: 1)", samples);
    TSP_REQUIRE(max_pages > 0, TSP_ERR_INVALID, "tsp_kv_append: max_pages=%d", max_pages);
    TSP_REQUIRE(flags == 0 || flags == TSP_ROPE_HALVES, TSP_ERR_INVALID, "tsp_kv_append: bad flags %d", flags);
    TSP_REQUIRE(hq >= 0 && hq <= 4096 && (q != nullptr) == (hq > 0) && (q_out != nullptr) == (hq > 0), TSP_ERR_INVALID,
                "tsp_kv_append: hq=%d (q %s, q_out %s)", hq, q ? "given" : "NULL", q_out ? "given" : "NULL");
    TSP_REQUIRE(axes >= 0 && axes <= KV_MAX_AXES && (axes == 0 || pairs), TSP_ERR_INVALID, "tsp_kv_append: %d axes (up to %d)", axes, KV_MAX_AXES);
    TSP_REQUIRE(theta > 0 && std::isfinite(theta) && eps >= 0 && std::isfinite(eps), TSP_ERR_INVALID, "tsp_kv_append: theta=%g eps=%g", theta, eps);
    int64_t total = 0;
    for (int i = 0; i < axes; ++i) {
        TSP_REQUIRE(pairs[i] >= 0 && pairs[i] <= c.d / 2, TSP_ERR_INVALID, "tsp_kv_append: %d pairs on axis %d", pairs[i], i);
        total += pairs[i];
    }
    TSP_REQUIRE(total <= c.d / 2, TSP_ERR_INVALID, "tsp_kv_append: %lld pairs, a head of %d has %d", (long long)total, c.d, c.d / 2);
    if (n == 0) return TSP_OK;
    TSP_REQUIRE(k && v && k->data && v->data && d_table && d_lengths && (c.data || c.pages == 0) && (axes == 0 || d_pos) &&
                    (hq == 0 || (q->data && q_out->data)),
                TSP_ERR_INVALID, "tsp_kv_append: null pointer");
    TSP_REQUIRE(heads_aligned(*k) && heads_aligned(*v) && (hq == 0 || (heads_aligned(*q) && heads_aligned(*q_out))) &&
                    reinterpret_cast<uintptr_t>(c.data) % 16 == 0 && reinterpret_cast<uintptr_t>(d_q_gamma) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(d_k_gamma) % 16 == 0,
                TSP_ERR_INVALID, "tsp_kv_append: data must be 16-byte aligned, strides multiples of 8 (a row's up to 2^20)");
    const size_t size = dtype_size(dtype);
    const Runs held = runs_of(c.data, kv_head_bytes(c) * c.heads * c.pages), none = runs_of(nullptr, 0);
    const Runs q_runs = hq ? runs_of(*q, n, hq, c.d, size) : none, o_runs = hq ? runs_of(*q_out, n, hq, c.d, size) : none;
    const Runs read[8] = {runs_of(*k, n, c.heads, c.d, size), runs_of(*v, n, c.heads, c.d, size), runs_of(d_table, 4ll * samples * max_pages),
                          runs_of(d_lengths, 4ll * samples), runs_of(d_offsets, 4ll * (samples + 1ll)), runs_of(axes ? d_pos : nullptr, 4ll * n * axes),
                          runs_of(d_q_gamma, 4ll * hq * c.d), runs_of(d_k_gamma, 4ll * c.heads * c.d)};
    bool over = meet(held, q_runs);
    for (const Runs& r : read) over |= meet(held, r);
    TSP_REQUIRE(!over, TSP_ERR_INVALID, "tsp_kv_append: the cache overlaps another tensor of the call");
    if (hq) {
        const bool same = q->data == q_out->data && (n <= 1 || q->row_stride == q_out->row_stride) && (hq <= 1 || q->head_stride == q_out->head_stride);
        TSP_REQUIRE(heads_apart(*q_out, n, hq, c.d), TSP_ERR_INVALID, "tsp_kv_append: the output's heads overlap");
        // (a row may be shared by groups of lanes: one's q_out over what another has yet to read would be a race)
        over = meet(o_runs, held) || (!same && meet(o_runs, q_runs));
        for (const Runs& r : read) over |= meet(o_runs, r);
        TSP_REQUIRE(!over, TSP_ERR_INVALID, "tsp_kv_append: q_out may be q, with the same strides, and must overlap no other tensor of the call");
    }
    AppendArgs a{};
    a.cache = kv_args(c, d_table, max_pages, d_lengths);
    a.k = k->data, a.k_row = k->row_stride, a.k_head = k->head_stride;
    a.v = v->data, a.v_row = v->row_stride, a.v_head = v->head_stride;
    if (hq) {
        a.q = q->data, a.q_row = q->row_stride, a.q_head = q->head_stride;
        a.q_out = q_out->data, a.o_row = q_out->row_stride, a.o_head = q_out->head_stride;
    }
    a.q_gamma = d_q_gamma, a.k_gamma = d_k_gamma;
    a.offsets = d_offsets, a.pos = d_pos;
    a.n = n, a.samples = samples, a.hq = hq, a.d = c.d, a.axes = axes, a.eps = eps;
    for (int p = 0; p < c.d / 2; ++p) a.axis[p] = -1;
    int p = 0;
    for (int ax = 0; ax < axes; ++ax)
        for (int j = 0; j < pairs[ax]; ++j, ++p) {
            a.axis[p] = (int8_t)ax;
            a.turns[p] = std::pow(theta, -(double)j / pairs[ax]) / (2 * M_PI);
        }
    // A row is shared by as many groups as it takes to give the device some 2048 workgroups, at most one a head. (12,345 rows into 4
    // bits: 40 us with 1024, 37 so, 47 with 4096; into 16: 36, 31 and 35.)
    const int lanes = c.d <= 64 ? 8 : 16, groups = KV_NT / lanes;
    a.parts = (int)std::min<int64_t>(std::max(hq, c.heads), std::max<int64_t>(1, 2048ll * groups / n));
    constexpr int64_t kRows = 1 << 26;       // of a launch
    dt_switch(dtype, [&](auto xd) {
        held_switch(c.format, [&](auto held) {
            constexpr int XD = decltype(xd)::value, HELD = decltype(held)::value;
            const dim3 block(KV_NT);
            hipStream_t s = as_stream(stream);
            const bool halves = flags & TSP_ROPE_HALVES;
            for (a.first = 0; a.first < n; a.first += kRows) {
                const dim3 grid((unsigned)ceil_div(std::min(n - a.first, kRows) * a.parts, groups));
                if (lanes == 8 && halves) hipLaunchKernelGGL((k_kv_append<XD, HELD, 8, true>), grid, block, 0, s, a);
                else if (lanes == 8) hipLaunchKernelGGL((k_kv_append<XD, HELD, 8, false>), grid, block, 0, s, a);
                else if (halves) hipLaunchKernelGGL((k_kv_append<XD, HELD, 16, true>), grid, block, 0, s, a);
                else hipLaunchKernelGGL((k_kv_append<XD, HELD, 16, false>), grid, block, 0, s, a);
            }
        });
    });
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}

extern "C" int tsp_kv_gather(const tsp_kv_cache* cache, int64_t n, const int32_t* d_offsets, int samples, const int32_t* d_table,
                             int max_pages, const int32_t* d_lengths, const tsp_heads* k_out, const tsp_heads* v_out, int out_dtype,
                             void* stream) {
    clear_error();
    TSP_REQUIRE(cache, TSP_ERR_INVALID, "tsp_kv_gather: null cache");
    const tsp_kv_cache& c = *cache;
    TSP_REQUIRE(kv_valid(c), TSP_ERR_UNSUPPORTED, "tsp_kv_gather: a cache of %lld pages of %d tokens, %d heads of %d, format %d", (long long)c.pages,
                c.page, c.heads, c.d, c.format);
    TSP_REQUIRE(n >= 0 && n < (1ll << 31), TSP_ERR_INVALID, "tsp_kv_gather: n=%lld out of range", (long long)n);
    TSP_REQUIRE(dtype_valid(out_dtype), TSP_ERR_INVALID, "tsp_kv_gather: bad dtype");
    TSP_REQUIRE(samples > 0 && (samples == 1 || d_offsets), TSP_ERR_INVALID, "tsp_kv_gather: samples=%d (without offsets: 1)", samples);
    TSP_REQUIRE(max_pages > 0, TSP_ERR_INVALID, "tsp_kv_gather: max_pages=%d", max_pages);
    if (n == 0) return TSP_OK;
    TSP_REQUIRE(k_out && v_out && k_out->data && v_out->data && d_table && d_lengths && (c.data || c.pages == 0), TSP_ERR_INVALID,
                "tsp_kv_gather: null pointer");
    TSP_REQUIRE(heads_aligned(*k_out) && heads_aligned(*v_out) && reinterpret_cast<uintptr_t>(c.data) % 16 == 0, TSP_ERR_INVALID,
                "tsp_kv_gather: data must be 16-byte aligned, strides multiples of 8 (a row's up to 2^20)");
    TSP_REQUIRE(heads_apart(*k_out, n, c.heads, c.d) && heads_apart(*v_out, n, c.heads, c.d), TSP_ERR_INVALID,
                "tsp_kv_gather: the outputs' heads overlap");
    const Runs out[2] = {runs_of(*k_out, n, c.heads, c.d, dtype_size(out_dtype)), runs_of(*v_out, n, c.heads, c.d, dtype_size(out_dtype))};
    const Runs read[4] = {runs_of(c.data, kv_head_bytes(c) * c.heads * c.pages), runs_of(d_table, 4ll * samples * max_pages),
                          runs_of(d_lengths, 4ll * samples), runs_of(d_offsets, 4ll * (samples + 1ll))};
    bool over = meet(out[0], out[1]);
    for (const Runs& r : read) over |= meet(out[0], r) || meet(out[1], r);
    TSP_REQUIRE(!over, TSP_ERR_INVALID, "tsp_kv_gather: the outputs overlap each other, the cache, table, lengths or offsets");
    const GatherArgs a{kv_args(c, d_table, max_pages, d_lengths), k_out->data, v_out->data, k_out->row_stride, k_out->head_stride,
                       v_out->row_stride, v_out->head_stride, d_offsets, n, samples};
    const int lanes = c.d <= 64 ? 8 : 16;
    const dim3 grid((unsigned)std::min<int64_t>(ceil_div(n * c.heads, KV_NT / lanes), 16384)), block(KV_NT);
    held_switch(c.format, [&](auto held) {
        dt_switch(out_dtype, [&](auto od) {
            constexpr int HELD = decltype(held)::value, OD = decltype(od)::value;
            if (lanes == 8) hipLaunchKernelGGL((k_kv_gather<HELD, OD, 8>), grid, block, 0, as_stream(stream), a);
            else hipLaunchKernelGGL((k_kv_gather<HELD, OD, 16>), grid, block, 0, as_stream(stream), a);
        });
    });
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
