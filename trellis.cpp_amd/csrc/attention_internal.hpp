// What the attention kernels share: the call's arguments, how a workgroup finds its rows, the 16-bit products'
// operands.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "packed.hpp"

namespace tsp {

constexpr int AT_KEYS = 64, AT_KEYS_F32 = 32;   // keys of a tile
constexpr int AT_MAX_D = 128;
constexpr int AT_MAX_SPLITS = 256;

struct AttnArgs {
    const void *q, *k, *v;
    void* o;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;   // strides in elements
    const int32_t *q_off, *k_off;
    int64_t nq, nk;                           // below 2^31, nq * share too
    int samples, hkv, share, d, causal;
    int whole, splits;                        // the first `whole` of units * hkv see their keys at once, the others in splits
    int extra;                                // several samples: as attn_item says (0: not), the share of its splits a key head
    int items;                                // workgroups there are for them
    FastDiv by_share, by_heads, by_splits;
    float scale2;                             // scale * log2(e)
    float* part;                              // [workgroup past whole][row][d] sums of p v, and
    float2* stat;                             // [workgroup past whole][row] maximum and sum of p (-1: no key seen)
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

// Up to 64 samples whose units do not fill the device. Where no sample has more than twice the tiles of the mean
// unit, each unit's keys are cut into `splits`; else by how many tiles its sample has, so that a long sample
// among short ones is shared by as many workgroups as its length asks for: with W = sum of units x tiles, a
// split has W / extra tiles or more, and all samples together have at most `extra` splits more than units. (One
// row each of 16 samples, 16 heads on 4 of 128: 48 us where one has 98,500 keys and the others 100, 166 all in equal
// numbers of splits. Of 14 unequal ones, 118,342 keys in all, 32 heads on 8 of 64: 50 us in equal numbers, 58 by
// length.)
// ITEMS: the w-th split of a unit and key head; else the w-th unit and key head, and `part` its first split.
struct AttnItem : AttnUnit {
    int part, split, splits;
};
template <int ROWS, int TILE, bool ITEMS, class Args>
__device__ __forceinline__ AttnItem attn_item(const Args& a, int w) {
    AttnItem t;
    const int lane = threadIdx.x & 63;
    t.u = PackedUnit{-1, 0, 0, 0, 0, 0, 0};
    t.head = t.row0 = t.rows = t.part = t.split = 0;
    t.splits = 1;
    int row0 = 0, rows = 0, other0 = 0, others = -1;
    if (lane < a.samples) {
        packed_rows(a.q_off, lane, (int)a.nq, row0, rows);
        packed_rows(a.k_off, lane, (int)a.nk, other0, others);
    }
    const int units = (int)((unsigned)(rows * a.share + ROWS - 1) / (unsigned)ROWS), tiles = (others + TILE - 1) / TILE;
    float work = (float)units * (float)tiles, all = (float)units, longest = units ? (float)tiles : 0.f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        work += __shfl_xor(work, o, 64);
        all += __shfl_xor(all, o, 64);
        longest = fmaxf(longest, __shfl_xor(longest, o, 64));
    }
    const float per = fmaxf(ceilf(work / (float)a.extra), 1.f);
    const int splits = longest * all <= 2.f * work ? a.splits : min(max((int)ceilf((float)tiles / per), 1), AT_MAX_SPLITS);
    const int items = units * a.hkv * splits, mine = ITEMS ? items : units * a.hkv;
    int end = mine, item_end = items;      // up to this sample's last
    if (a.samples <= kOrderedSamples) {    // (the longest first)
        for (int j = 0; j < a.samples; ++j) {
            const int v = __builtin_amdgcn_readlane(others, j), c = __builtin_amdgcn_readlane(mine, j), d = __builtin_amdgcn_readlane(items, j);
            if (v > others || (v == others && j < lane)) end += c, item_end += d;
        }
    } else {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int c = __shfl_up(end, o, 64), d = __shfl_up(item_end, o, 64);
            if (lane >= o) end += c, item_end += d;
        }
    }
    const uint64_t found = __ballot(w >= end - mine && w < end);
    if (!found) return t;
    const int l = __builtin_ctzll(found);
    t.u.sample = l;
    t.u.row0 = __builtin_amdgcn_readlane(row0, l);
    t.u.rows = __builtin_amdgcn_readlane(rows, l);
    t.u.other0 = __builtin_amdgcn_readlane(other0, l);
    t.u.others = __builtin_amdgcn_readlane(others, l);
    t.u.count = __builtin_amdgcn_readlane(units, l);
    t.splits = __builtin_amdgcn_readlane(splits, l);
    const int in = w - __builtin_amdgcn_readlane(end - mine, l);
    const int pair = ITEMS ? (int)((unsigned)in / (unsigned)t.splits) : in;      // (unit, key head)
    const int unit = pair / FastDiv{a.by_heads.mul, a.by_heads.shift};
    t.head = pair - unit * a.hkv;
    t.split = ITEMS ? in - pair * t.splits : 0;
    t.part = __builtin_amdgcn_readlane(item_end - items, l) + pair * t.splits;
    t.row0 = (a.causal ? t.u.count - 1 - unit : unit) * ROWS;
    t.rows = t.u.rows * a.share;
    return t;
}

template <bool BF16>
__device__ __forceinline__ f32x16_t mfma32(const u32x4_t& a, const u32x4_t& b, const f32x16_t& c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Two values rounded to nearest even into a packed pair.
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (BF16) return f32x2_to_bf16x2_bits(lo, hi);
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, f16x2_t));
}

// The sum of a packed pair and c, in fp32.
template <bool BF16>
__device__ __forceinline__ float add2(uint32_t p, float c) {
    if constexpr (BF16) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, p), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), c, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, p), __builtin_bit_cast(f16x2_t, 0x3c003c00u), c, false);
}

template <bool BF16>
__device__ __forceinline__ bool nonfinite16(uint32_t b) {
    constexpr uint32_t kExp = BF16 ? 0x7F80u : 0x7C00u;
    return (b & kExp) == kExp;
}

// Byte offsets in a staged tile of AT_KEYS rows of DP values, as 16-byte pieces. K is read 16 bytes of
// one d at 32 consecutive keys: the piece is xored with the key, so that 16 keys cover all banks. V is
// read 64 bytes of 4 consecutive keys: the 64-byte quarter is xored with the key. (Rows of 32 and 96 values
// begin in another quarter of the banks each by themselves.)
template <int DP>
__device__ __forceinline__ int k_piece(int key, int piece) {
    return key * (DP * 2) + (piece ^ (DP == 128 ? key & 15 : DP == 96 || DP == 32 ? (key >> 2) & 3 : (key >> 1) & 7)) * 16;
}
template <int DP>
__device__ __forceinline__ int v_piece(int key, int piece) {
    return key * (DP * 2) + (piece ^ (DP == 128 ? (key & 3) << 2 : DP == 96 || DP == 32 ? 0 : ((key >> 1) & 1) << 2)) * 16;
}

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4_ptr;

// V^T operand (32 d x 16 keys) of keys 16 ks + {4h..4h+3, 8+4h..8+4h+3}: each of the two transposing
// loads takes 4 keys x 16 d a group of 16 lanes.
template <int DP>
__device__ __forceinline__ u32x4_t v_operand(const char* sv, int ks, int db, int lane) {
    const int key = ks * 16 + 4 * (lane >> 5) + ((lane >> 2) & 3);
    const int piece = db * 4 + ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1), sub = (lane & 1) * 8;
    const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(sv + v_piece<DP>(key, piece) + sub));
    const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(sv + v_piece<DP>(key + 8, piece) + sub));
    const uint2 ua = __builtin_bit_cast(uint2, a), ub = __builtin_bit_cast(uint2, b);
    return u32x4_t{ua.x, ua.y, ub.x, ub.y};
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
