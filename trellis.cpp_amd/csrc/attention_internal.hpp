// What the 16-bit and the fp32 attention kernels share: the call's arguments, how a workgroup finds its rows.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "packed.hpp"

namespace tsp {

constexpr int AT_KEYS = 64, AT_KEYS_F32 = 32;   // keys of a tile
constexpr int AT_MAX_D = 128;

struct AttnArgs {
    const void *q, *k, *v;
    void* o;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;   // strides in elements
    const int32_t *q_off, *k_off;
    int64_t nq, nk;                           // below 2^31, nq * share too
    int samples, hkv, share, d, causal;
    int units;                                // of rows, a key head
    int whole, splits;                        // the first `whole` of units * hkv see their keys at once, the others in splits
    FastDiv by_share, by_heads, by_splits;
    float scale2;                             // scale * log2(e)
    float* part;                              // [unit past whole][split][row][d] sums of p v, and
    float2* stat;                             // [unit past whole][split][row] maximum and sum of p (-1: no key seen)
};

// A unit of `ROWS` rows (query, head of the group) of one key head.
struct AttnUnit {
    PackedUnit u;      // its sample (-1: none)
    int head, row0, rows;   // the key head, its first row, the sample's rows
};
// The key heads of one unit of rows follow each other (with 8 of them each XCD, which takes every eighth
// workgroup, has one head's keys in its L2), the longest samples come first, and with causal a sample's last
// rows, which see most.
template <int ROWS, class Args>
__device__ __forceinline__ AttnUnit attn_unit(const Args& a, int w) {
    AttnUnit t;
    const int unit = w / FastDiv{a.by_heads.mul, a.by_heads.shift};
    t.head = w - unit * a.hkv;
    t.u = packed_unit<true>(a.q_off, a.samples, (int)a.nq, a.share, ROWS, unit, a.k_off, (int)a.nk);
    t.row0 = (a.causal ? t.u.count - 1 - (unit - t.u.first) : unit - t.u.first) * ROWS;
    t.rows = t.u.rows * a.share;
    return t;
}

// The value of the other lane half (lane ^ 32), for both halves: {lower half's, upper half's}.
__device__ __forceinline__ float2 both_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return float2{__uint_as_float(r[0]), __uint_as_float(r[1])};
}

// Waits for this wave's loads into LDS (which the compiler's own waits do not always cover).
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// Keys of a tile that a row sees, for the rows of a wave's 32.
struct RowLimits {
    int lane, hi;      // this lane's row, the wave's last
};

// The fp32 kernel (attention_f32.hip) on `blocks` workgroups of nw waves.
void launch_attention_f32(const AttnArgs& a, int nw, unsigned blocks, hipStream_t s);

}  // namespace tsp
