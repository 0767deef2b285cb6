// Softmax attention within packed samples: for query row i of sample s and head h (on key head
// h / (hq / hkv)),
//   out[i][h] = sum_j exp(scale q_i . k_j - max) v_j / sum_j exp(scale q_i . k_j - max)
// over the keys j that the row sees: all of its sample's, or with `causal` the first Lk - Lq + i + 1 of
// them. A row that sees no key gets zeros.
//
// One pass over the keys with the running maximum and sum of each row. Both products run on the matrix
// cores (v_mfma_f32_32x32x16) with their roles turned: S^T = K Q^T and O^T = V^T P^T. A lane then holds
// 16 of a tile's 32 scores of ONE query row (lane % 32; the other lane half holds the others), so a row's
// maximum and sum need no more than one exchange between the halves, and the probabilities are, after
// their rounding to 16 bits, the second product's operand where they stand: an operand lane wants eight
// keys, which eight does not matter as long as V's operand has the same, and V's lie in the order 4 of
// every 8 that S^T leaves.
//
// The rows of a workgroup are (query, head of the group) pairs: the heads that share a key head read its
// tiles once.
//
// Statistics and accumulators are fp32. P is rounded to the inputs' 16-bit type, as the matrix cores take
// it: half a step, 2^-8 of a probability in bf16 and 2^-11 in f16, there for those of 2^-25 of the row's largest and
// more; smaller ones are off by up to 2^-36 of the largest. A row's sum is of the rounded ones, so that rows of equal
// values have their mean exactly.
//
// Bound by the matrix cores and, at d <= 64, by the exponents beside them (a wave's tile of 64 keys is 16
// products of 32 cycles, and 33 exponents of 10 with some 140 other instructions of 2.7). A wave holds 32 rows'
// accumulators, its Q operands and two tiles' scores: where four share a workgroup in at most 256 registers, two waves a
// SIMD (three at d <= 64), so that the workgroups, two or three a CU, keep each other's barriers and loads covered;
// alone, at widths 96 and 128, in some 270 and 320 to 340, one a SIMD (at 64 KB of LDS each no more than two
// fit the four SIMDs of a CU). The scalar registers of bf16 at width 128 do not all fit: of its loop's
// instructions, two tiles long, 21 move them to and from a vector register (f16: none). 35,001 rows, 8 heads of
// 128, bf16: 4.25-4.4 ms, 1,140-1,180 TFLOP/s, 65 % of the matrix cores' cycles at the 1.6 GHz that power leaves (a
// library GEMM of 16,384^3: 1,391). 8 heads of 64, 10,000 rows and keys: 870. One row against 40,009 keys, 16
// heads on 2 of 128: 12 us and 6 for the join, 3.4 TB/s of keys and values.
// Tried and taken back: eight waves a workgroup (one a CU: as fast at 35,001 rows, 8-15 % slower at 1,029 to
// 12,345 keys); the loads spread between the products (7 % slower: a wave stops at each); values a tile later
// than exponents, so that both products run beside them (d 128: 8 % slower, d 64: 0-5 % faster); four waves a
// SIMD at d <= 64 (spills); sums by additions or by a product with ones (equal, or 3-7 % slower).
#include <algorithm>
#include <cmath>

#include "attention_internal.hpp"

namespace tsp {
namespace {

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

#ifdef __HIP_DEVICE_COMPILE__       // (the host pass knows neither the register constraint nor the argument segment)
// Keeps a value in scalar registers of its own from here on.
template <class T>
__device__ __forceinline__ void keep_scalar(T& x) {
    asm volatile("" : "+s"(x));
}

// The kernel's arguments read anew: kept in scalar registers from the start on they would push the main
// loop's own out of them.
typedef const __attribute__((address_space(4))) AttnArgs* AttnArgsPtr;
__device__ __forceinline__ AttnArgsPtr reread_args() {
    AttnArgsPtr p = (AttnArgsPtr)__builtin_amdgcn_kernarg_segment_ptr();
    keep_scalar(p);
    return p;
}
#endif

template <bool BF16, int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW == 1 && DP > 64 ? 1 : 2) void k_attention(AttnArgs) {
#ifdef __HIP_DEVICE_COMPILE__
    const auto& a = *reread_args();
    constexpr int KS = DP / 16, DB = DP / 32, P = DP / 8, ROWS = NW * 32;
    constexpr int TILE = AT_KEYS * DP * 2;
    __shared__ __attribute__((aligned(16))) char sK0[TILE], sK1[TILE], sV0[TILE], sV1[TILE];
    int split = 0, splits = 1;
    AttnUnit t;
    if (__builtin_expect(a.extra != 0, 0)) {      // (its code out of the way of the others')
        const AttnItem item = attn_item<ROWS, AT_KEYS, true>(a, blockIdx.x);
        t = item;
        split = item.split;
        splits = item.splits;
    } else {
        int work = blockIdx.x;
        if (work >= a.whole) {
            const int past = work - a.whole, at = past / FastDiv{a.by_splits.mul, a.by_splits.shift};
            splits = a.splits;
            work = a.whole + at;
            split = past - at * splits;
        }
        t = attn_unit<ROWS>(a, work);
    }
    const PackedUnit& u = t.u;
    const int head = t.head, rows = t.rows, tile0 = t.row0;
    if (u.sample < 0) return;
    const int krow0 = u.other0, lk = u.others;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;

    // rows past the sample's last are copies of it that are not stored
    auto limit = [&](int query) __attribute__((always_inline)) { return a.causal ? min(max(lk - u.rows + query + 1, 0), lk) : lk; };
    const FastDiv by_share{a.by_share.mul, a.by_share.shift};
    auto query = [&](int r) __attribute__((always_inline)) { return min(r, rows - 1) / by_share; };
    const int r = tile0 + wave * 32 + r32, qi = query(r);
    const RowLimits lim{limit(qi), limit(query(tile0 + wave * 32 + 31))};
    const int wg_end = limit(query(tile0 + ROWS - 1));
    const int hq = head * a.share + min(r, rows - 1) - qi * a.share;

    // Q^T operand: d = 16 ks + 8 h .. + 7 of the lane's row
    u32x4_t qf[KS];
    {
        const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (int64_t)(u.row0 + qi) * a.q_row + hq * a.q_head;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            qf[ks] = ks * 16 + h * 8 < a.d ? *reinterpret_cast<const u32x4_t*>(qp + ks * 16 + h * 8) : u32x4_t{0, 0, 0, 0};
    }
    const char* kp = static_cast<const char*>(a.k) + 2 * ((int64_t)krow0 * a.k_row + head * a.k_head);
    const char* vp = static_cast<const char*>(a.v) + 2 * ((int64_t)krow0 * a.v_row + head * a.v_head);
    int k_bytes = (int)a.k_row * 2, v_bytes = (int)a.v_row * 2;      // of a row
    float scale2 = a.scale2;
    keep_scalar(kp);
    keep_scalar(vp);
    keep_scalar(k_bytes);
    keep_scalar(v_bytes);
    keep_scalar(scale2);

    // A tile goes straight from memory to LDS, 1 KiB a wave and load: 16 bytes a lane, each from the piece
    // that belongs in its place. Rows past the sample's last key and pieces past d read as zeros (out of
    // the buffer's range).
    constexpr int LOADS = TILE / 1024 / NW;
    // A lane's byte offsets within the tile's rows; those of loads PERIOD apart differ by whole rows alone.
    constexpr int LOAD_PIECES = NW * 64, PERIOD = DP == 96 ? 3 : LOAD_PIECES / P >= 16 ? 1 : 16 * P / LOAD_PIECES;
    constexpr int PERIOD_ROWS = PERIOD * LOAD_PIECES / P;
    static_assert(PERIOD_ROWS % 16 == 0 && LOADS % PERIOD == 0, "the swizzles repeat every 16 keys");
    constexpr int NOWHERE = 1 << 30;         // past every tile's rows
    int k_at[PERIOD], v_at[PERIOD];
#pragma unroll
    for (int i = 0; i < PERIOD; ++i) {
        const int at = (i * NW + wave) * 64 + lane, key = at / P, slot = at % P;
        const int kp = k_piece<DP>(key, slot) / 16 % P, vp = v_piece<DP>(key, slot) / 16 % P;
        k_at[i] = kp * 8 < a.d ? key * k_bytes + kp * 16 : NOWHERE;
        v_at[i] = vp * 8 < a.d ? key * v_bytes + vp * 16 : NOWHERE;
        asm volatile("" : "+v"(k_at[i]), "+v"(v_at[i]));       // (computed here, not in every tile)
    }
    auto stage = [&](const char* p, int bytes, int base, const int (&at)[PERIOD], char* s) __attribute__((always_inline)) {
        const int n = min(AT_KEYS, lk - base);
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(p + (int64_t)base * bytes), (short)0, n * bytes, 0x00027000);
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(s + (i * NW + wave) * 1024), 16,
                                                     at[i % PERIOD] + i / PERIOD * PERIOD_ROWS * bytes, 0, 0, 0);
    };
    // K or V of the tile at key base
    auto stage_k = [&](int base, char* s) __attribute__((always_inline)) { stage(kp, k_bytes, base, k_at, s); };
    auto stage_v = [&](int base, char* s) __attribute__((always_inline)) { stage(vp, v_bytes, base, v_at, s); };

    f32x16_t o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16_t{};
    constexpr float LAG = BF16 ? 8.f : 4.f, LIFT = BF16 ? 0.f : 11.f;
    constexpr float FAR = 1024.f;
    float m = -INFINITY, l = 0.f, mc = -LIFT;      // maximum, sum, what the exponents are less by
    bool far = false;

    // this split's share of the workgroup's tiles
    const int tiles = (wg_end + AT_KEYS - 1) / AT_KEYS, per = (int)((unsigned)(tiles + splits - 1) / (unsigned)splits);
    const int begin = split * per * AT_KEYS, end = min(wg_end, begin + per * AT_KEYS);
    const bool causal = a.causal;

    // scores: s[kb][i] is key kb * 32 + 8 (i / 4) + 4 h + i % 4 of the tile
    auto scores = [&](const char* sK, f32x16_t (&s)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            s[kb] = f32x16_t{};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                s[kb] = mfma32<BF16>(*reinterpret_cast<const u32x4_t*>(sK + k_piece<DP>(kb * 32 + r32, ks * 2 + h)), qf[ks], s[kb]);
        }
    };
    // The maximum that the exponents are taken from moves only when a row's has grown by a factor of 2^LAG (p
    // and its sums have room for that), so that most tiles leave the sums as they are. In f16 p is 2^LIFT times
    // its value, in l and in o alike, so that it fills the type's range from the top, 2^15: a key of 2^-(14 + LIFT)
    // of the largest has all its bits, and one of up to 2^-(25 + LIFT) still counts.
    auto raise = [&](float mt) __attribute__((always_inline)) {
        const float2 mh = both_halves(mt);
        mt = fmaxf(mh.x, mh.y);
        if (__any((mt - m) * scale2 > LAG)) {
            const float mn = fmaxf(m, mt);
            const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * scale2);
            m = mn;
            far = __any(fabsf(mn) * scale2 > FAR && mn != -INFINITY);
            mc = (far || mn == -INFINITY ? 0.f : mn * scale2) - LIFT;       // (-inf: no key seen yet, or scores of -inf alone)
            l *= corr;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] *= corr;
        }
    };
    // m * scale2 is rounded, and half a step of it is off in every exponent: that does not cancel where the maximum
    // moves, and from 2^27 on takes p out of its type's range. So a wave with a maximum past FAR, where it is 2^-14,
    // takes the maximum from the scores themselves, after raise.
    auto near_top = [&](f32x16_t (&s)[2]) __attribute__((always_inline)) {
        if (__builtin_expect(!far, 1)) return;
        const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] -= from;
    };
    auto top = [&](const f32x16_t (&s)[2]) __attribute__((always_inline)) {
        float mt = s[0][0];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[kb][i]);
        return mt;
    };
    // s becomes p, pf the second product's operand
    auto exponents = [&](f32x16_t (&s)[2], u32x4_t (&pf)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], scale2, -mc));
        float sum = 0.f;      // (of the tile first: a sixteenth as many additions meet the row's whole sum)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pf[ks][e] = pack2<BF16>(s[ks / 2][8 * (ks % 2) + 2 * e], s[ks / 2][8 * (ks % 2) + 2 * e + 1]);
                sum = add2<BF16>(pf[ks][e], sum);
            }
        l += sum;
    };
    auto weigh = [&](const char* sV, const u32x4_t (&pf)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] = mfma32<BF16>(v_operand<DP>(sV, ks, db, lane), pf[ks], o[db]);
    };
    // A tile that not every row of the workgroup sees whole.
    auto attend_masked = [&](int base, const char* sK, const char* sV) __attribute__((always_inline)) {
        f32x16_t s[2];
        u32x4_t pf[4];
        scores(sK, s);
        const int left = lim.lane - base - 4 * h;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[kb][i] = kb * 32 + 8 * (i / 4) + i % 4 < left ? s[kb][i] : -INFINITY;
        raise(top(s));
        near_top(s);
        exponents(s, pf);
        // Rows of the tile that see different keys: a probability of zero must not meet an Inf or a NaN
        // of a key that its row does not see. Zero times V shows whether there is one.
        bool odd = false;
        if (causal) {
            f32x16_t z = f32x16_t{};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int db = 0; db < DB; ++db) z = mfma32<BF16>(v_operand<DP>(sV, ks, db, lane), u32x4_t{0, 0, 0, 0}, z);
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) t += z[i];
            odd = __any(t != t);
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                u32x4_t vf = v_operand<DP>(sV, ks, db, lane);
                if (odd) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (nonfinite16<BF16>(vf[e])) vf[e] &= 0xffff0000u;
                        if (nonfinite16<BF16>(vf[e] >> 16)) vf[e] &= 0xffffu;
                    }
                }
                o[db] = mfma32<BF16>(vf, pf[ks], o[db]);
            }
        if (odd) {      // the values left out, key by key, for the rows that see them
            for (int key = 0; key < AT_KEYS; ++key) {
                float p = 0.f;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if ((kb * 32 + 8 * (i / 4) + i % 4) == (key & ~4)) p = s[kb][i];
                const float2 ph = both_halves(p);
                p = key & 4 ? ph.y : ph.x;
                const bool sees = base + key < lim.lane;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int e = db * 32 + 8 * (i / 4) + 4 * h + i % 4;
                        const uint32_t b = *reinterpret_cast<const uint16_t*>(sV + v_piece<DP>(key, e >> 3) + (e & 7) * 2);
                        if (sees && nonfinite16<BF16>(b)) o[db][i] += p * (BF16 ? bf16_bits_to_f32((uint16_t)b) : f16_bits_to_f32((uint16_t)b));
                    }
            }
        }
    };
    // The wait is for this wave's own loads; the barrier then says that every wave's have landed, and that
    // no wave reads any more what was read before it.
    auto landed = []() __attribute__((always_inline)) {
        wait_loads();
        __syncthreads();
    };
    // Whole tiles: the scores of the next tile are formed while the exponents of this one are, and its
    // maximum while this one's values are weighed, so that the matrix cores and the vector units both have
    // work from one wave, in the order written here; operands are read four products ahead. Two buffers
    // each for K and V; K is a tile ahead of V.
    const int whole = min(end, limit(query(tile0)));
    auto k_operand = [&](const char* sK, int t) __attribute__((always_inline)) {
        return *reinterpret_cast<const u32x4_t*>(sK + k_piece<DP>((t & 1) * 32 + r32, (t >> 1) * 2 + h));
    };
    auto step = [&](int base, char* k_this, const char* k_next, const char* v_this, char* v_next, f32x16_t (&s)[2],
                    f32x16_t (&sn)[2]) __attribute__((always_inline)) {
        constexpr int AHEAD = 4, NK = 2 * KS, NV = 4 * DB;
        u32x4_t pf[4], ring[AHEAD];
        float sum = 0.f;
        landed();
        if (base + 2 * AT_KEYS < end) stage_k(base + 2 * AT_KEYS, k_this);
        if (base + AT_KEYS < end) stage_v(base + AT_KEYS, v_next);
#pragma unroll
        for (int t = 0; t < AHEAD; ++t) ring[t] = k_operand(k_next, t);
#pragma unroll
        for (int t = 0; t < NK; ++t) {
            sn[t & 1] = mfma32<BF16>(ring[t % AHEAD], qf[t >> 1], t < 2 ? f32x16_t{} : sn[t & 1]);
            if (t + AHEAD < NK) ring[t % AHEAD] = k_operand(k_next, t + AHEAD);
            else ring[t % AHEAD] = v_operand<DP>(v_this, (t + AHEAD - NK) / DB, (t + AHEAD - NK) % DB, lane);
#pragma unroll
            for (int e = t * 16 / NK; e < (t + 1) * 16 / NK; ++e) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[e / 8][2 * (e % 8)], scale2, -mc));
                const float y = __builtin_amdgcn_exp2f(fmaf(s[e / 8][2 * (e % 8) + 1], scale2, -mc));
                pf[e / 4][e % 4] = pack2<BF16>(x, y);
                sum = add2<BF16>(pf[e / 4][e % 4], sum);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l += sum;
        float mt = sn[0][0];
#pragma unroll
        for (int t = 0; t < NV; ++t) {
            o[t % DB] = mfma32<BF16>(ring[t % AHEAD], pf[t / DB], o[t % DB]);
            if (t + AHEAD < NV) ring[t % AHEAD] = v_operand<DP>(v_this, (t + AHEAD) / DB, (t + AHEAD) % DB, lane);
#pragma unroll
            for (int i = t * 32 / NV; i < (t + 1) * 32 / NV; ++i) mt = fmaxf(mt, sn[i / 16][i % 16]);
            __builtin_amdgcn_sched_barrier(0);
        }
        raise(mt);
        near_top(sn);
    };
    int base = begin;
    bool second = false;
    if (begin < end) {
        stage_k(begin, sK0);
        stage_v(begin, sV0);
        if (begin + AT_KEYS < end) stage_k(begin + AT_KEYS, sK1);
    }
    if (base + AT_KEYS <= whole) {
        f32x16_t s0[2], s1[2];
        landed();
        scores(sK0, s0);
        raise(top(s0));
        near_top(s0);
        for (; base + 3 * AT_KEYS <= whole; base += 2 * AT_KEYS) {
            step(base, sK0, sK1, sV0, sV1, s0, s1);
            step(base + AT_KEYS, sK1, sK0, sV1, sV0, s1, s0);
        }
        landed();
        if (base + 2 * AT_KEYS < end) stage_k(base + 2 * AT_KEYS, sK0);
        if (base + AT_KEYS < end) stage_v(base + AT_KEYS, sV1);
        u32x4_t pf[4];
        exponents(s0, pf);
        weigh(sV0, pf);
        base += AT_KEYS;
        second = true;
    }
    // the others, a whole one among them at times (K and V of the first are on their way, K of the second too)
    for (; base < end; base += AT_KEYS, second = !second) {
        landed();
        if (base < lim.hi) attend_masked(base, second ? sK1 : sK0, second ? sV1 : sV0);
        if (base + AT_KEYS < end) stage_v(base + AT_KEYS, second ? sV0 : sV1);
        if (base + 2 * AT_KEYS < end) {
            __syncthreads();
            stage_k(base + 2 * AT_KEYS, second ? sK1 : sK0);
        }
    }

    const float2 lh = both_halves(l);
    const float sum = lh.x + lh.y;
    const auto& b = *reread_args();
    if (splits > 1) {
        if (r >= rows) return;
        const int64_t item = (int64_t)((int)blockIdx.x - b.whole) * ROWS + (r - tile0);
        const bool seen = lim.lane > begin && begin < end;
        if (h == 0) b.stat[item] = float2{m, seen ? sum : -1.f};
        if (!seen) return;
        float* op = b.part + item * b.d;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int e = db * 32 + 8 * g + 4 * h;
                if (e < b.d) *reinterpret_cast<f32x4_t*>(op + e) = f32x4_t{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
            }
        return;
    }
    // Rows of out leave in 16-byte pieces, whole rows at a time: the wave's part of the tile goes through its own
    // piece of the K buffers (swizzled as K is), since a lane holds 8 bytes of every 16 of its row.
    const float inv = lim.lane == 0 ? 0.f : 1.0f / sum;      // (no key seen: zeros)
    char* sO = NW == 1 || wave < NW / 2 ? sK0 + wave * (32 * DP * 2) : sK1 + (wave - NW / 2) * (32 * DP * 2);
    static_assert(NW <= 4, "two waves' rows a buffer");
    __syncthreads();
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2*>(sO + k_piece<DP>(r32, db * 4 + g) + h * 8) =
                uint2{pack2<BF16>(o[db][4 * g] * inv, o[db][4 * g + 1] * inv), pack2<BF16>(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv)};
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
        const int row = (i * 64 + lane) / P, piece = (i * 64 + lane) % P, rr = tile0 + wave * 32 + row;
        const u32x4_t x = *reinterpret_cast<const u32x4_t*>(sO + k_piece<DP>(row, piece));
        if (rr >= rows || piece * 8 >= b.d) continue;
        const int qr = rr / FastDiv{b.by_share.mul, b.by_share.shift}, hr = head * b.share + rr - qr * b.share;
        *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(b.o) + (int64_t)(u.row0 + qr) * b.o_row + hr * b.o_head + piece * 8) = x;
    }
#endif
}

// The splits' sums joined: sum_s w_s (p v)_s / sum_s w_s (sum p)_s, w_s = exp(max_s - max). A row and head
// takes G groups of 16 lanes (8 elements each); the splits are dealt to the groups, whose sums are then
// added in a fixed order. A split whose scores were all -inf has sums of 0 (or NaN): its weight does
// not matter. G = 1 for up to 16 splits, 16 beyond; 4, a wave, for samples that are split by their lengths, where
// some have few (128 rows of 16 samples, 11 splits each: 15 us with 16 groups a row, 7 with 4), 16 beyond 32.
constexpr int AT_FEW_SPLITS = 16;
template <int DT, int G, int ROWS, bool BY_LENGTH>
__global__ __launch_bounds__(256) void k_attention_join(AttnArgs a) {
    constexpr int ITEMS = 16 / G, EACH = G == 4 ? AT_MAX_SPLITS / 64 : 1;      // rows a workgroup, splits a lane
    __shared__ float sW[ITEMS][G == 1 ? AT_FEW_SPLITS : AT_MAX_SPLITS];     // weights; -1: no key seen
    __shared__ float sAcc[G == 16 ? G : 1][AT_MAX_D], sSum[16];
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4, e = lane * 8;
    const int g = group % G, at = group / G, mine = threadIdx.x % (G * 16);
    const int past = blockIdx.y, first = blockIdx.x * ITEMS;
    AttnUnit w;
    int splits = a.splits;
    int64_t slot = (int64_t)past * a.splits;      // of the first of them in part
    if constexpr (BY_LENGTH) {
        const AttnItem t = attn_item<ROWS, DT == TSP_F32 ? AT_KEYS_F32 : AT_KEYS, false>(a, past);
        splits = t.splits;
        // (a unit of one split has been written; splits past the last are of offsets out of order)
        if (splits == 1 || t.part + splits > a.items) return;
        w = t;
        slot = t.part;
    } else {
        w = attn_unit<ROWS>(a, a.whole + past);
    }
    if (w.u.sample < 0) return;
    for (int row0 = first; row0 < ROWS && w.row0 + row0 < w.rows; row0 += gridDim.x * ITEMS) {
        const int row = row0 + at, r = w.row0 + row;
        const bool live = r < w.rows;
        const int64_t item = slot * ROWS + row;
        float2 t[EACH];
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            t[i] = float2{-INFINITY, -1.f};
            if (live && mine + i * 64 < splits) t[i] = a.stat[(int64_t)(mine + i * 64) * ROWS + item];
            m = fmaxf(m, t[i].x);
        }
#pragma unroll
        for (int o = G == 1 ? 8 : 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        if constexpr (G == 16) {
            if ((threadIdx.x & 63) == 0) sSum[threadIdx.x >> 6] = m;
            __syncthreads();
            m = fmaxf(fmaxf(sSum[0], sSum[1]), fmaxf(sSum[2], sSum[3]));
            __syncthreads();
        }
        // the sum of p over all splits, and whether any saw a key
        float sum = 0.f;
        bool seen = false;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const float w0 = t[i].y == -1.f ? -1.f : t[i].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((t[i].x - m) * a.scale2);
            if (mine + i * 64 < (G == 1 ? AT_FEW_SPLITS : AT_MAX_SPLITS)) sW[at][mine + i * 64] = w0;
            if (t[i].y != -1.f) {
                sum += w0 * t[i].y;
                seen = true;
            }
        }
#pragma unroll
        for (int o = G == 1 ? 8 : 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if constexpr (G == 16) {
            if ((threadIdx.x & 63) == 0) sSum[threadIdx.x >> 6] = sum;
            seen = __syncthreads_or(seen);
            sum = (sSum[0] + sSum[1]) + (sSum[2] + sSum[3]);
        } else {
            const uint64_t any = __ballot(seen);
            seen = G == 4 ? any != 0 : (any >> (threadIdx.x & 48) & 0xffff) != 0;
            __syncthreads();
        }
        float acc[8] = {};
        if (live && e < a.d) {
            constexpr int BATCH = 8;      // splits on their way at a time
            for (int s0 = g; s0 < splits; s0 += BATCH * G) {
                f32x4_t x[BATCH], y[BATCH];
                float c[BATCH];
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    const int s = s0 + b * G;
                    c[b] = s < splits ? sW[at][s] : -1.f;
                    x[b] = y[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                    if (c[b] == -1.f) continue;
                    const f32x4_t* p = reinterpret_cast<const f32x4_t*>(a.part + ((int64_t)s * ROWS + item) * a.d + e);
                    x[b] = p[0];
                    y[b] = p[1];
                }
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    if (c[b] == -1.f) continue;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        acc[i] += c[b] * x[b][i];
                        acc[4 + i] += c[b] * y[b][i];
                    }
                }
            }
        }
        if constexpr (G == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[i] += __shfl_xor(acc[i], 16, 64);
                acc[i] += __shfl_xor(acc[i], 32, 64);
            }
        } else if constexpr (G == 16) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sAcc[g][e + i] = acc[i];
            __syncthreads();
            if (g == 0) {
#pragma unroll
                for (int k = 1; k < G; ++k)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[i] += sAcc[k][e + i];
            }
        }
        if (live && e < a.d && g == 0) {
            const float inv = 1.0f / sum;
            const int qi = r / a.by_share, hq = w.head * a.share + r - qi * a.share;
            const int64_t to = (int64_t)(w.u.row0 + qi) * a.o_row + hq * a.o_head + e;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = seen ? acc[i] * inv : 0.f;
            if constexpr (DT == TSP_F32) {
                f32x4_t* y = reinterpret_cast<f32x4_t*>(static_cast<float*>(a.o) + to);
                y[0] = f32x4_t{acc[0], acc[1], acc[2], acc[3]};
                y[1] = f32x4_t{acc[4], acc[5], acc[6], acc[7]};
            } else {
                u32x4_t y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = pack2<DT == TSP_BF16>(acc[2 * i], acc[2 * i + 1]);
                *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.o) + to) = y;
            }
        }
        if constexpr (G > 1) __syncthreads();      // (the next rows' weights and sums go where these are read)
    }
}

constexpr float kLog2e = 1.44269504088896340736f;

// How a call is cut: waves of a workgroup (32 rows each), units of rows a key head, how many of them see
// their keys at once, splits of the others' keys.
struct AttnCut {
    int nw, splits, even;      // (even: of samples of nearly one length)
    int64_t units, whole;
    int64_t extra;        // or by the samples' lengths (attn_item), into this many items a key head beside one a unit
    int64_t blocks(int hkv) const { return extra ? (units * splits + 2) * hkv : whole + (units * hkv - whole) * splits; }      // (2: work's rounding)
};

AttnCut attn_cut(int64_t nq, int64_t nk, int samples, int hkv, int share, int d, bool causal, bool f32) {
    AttnCut c;
    // one wave where a sample has at most its 32 rows (by the mean: the host does not know the lengths)
    c.nw = ceil_div(nq, samples) * share <= 32 ? 1 : 4;
    const int64_t units = ceil_div(nq * share, c.nw * 32);
    c.units = units + (samples > 1 ? samples : 0);
    // The device holds `slots` workgroups at once (by registers and LDS), some on each of 256 CUs, and a round
    // of them on few slots a CU is shorter: alone on its CU a workgroup of width 64 takes 0.37 of the time
    // that it takes as one of three, of width 128 0.62 of that as one of two (measured: 0.75 and 2.0 us a
    // tile, 1.2 and 1.9); one-wave workgroups wait for memory, and half a round's take half and half a
    // round's time. Where there are not `slots` units, their keys are split; where one sample's units
    // leave a last round partly empty, that round's are. (Several samples, or causal ones, have units of
    // unequal length, which fill each other's gaps.) Time is counted in tiles: about three for a workgroup's
    // start and end, five or six for the join.
    // A sample leaves a partly filled unit, in the mean half of one. (A row each of 16, 65,536 keys, 32 heads on 8 of
    // 128: 55 us so, 89 with none counted, 52 with whole ones; with those, 64 samples of which one has nearly
    // all of 65,536 keys would fill the device by count and take 1,094 us, 66 so.)
    const int64_t busy = (units + (samples > 1 ? samples / 2 : 0)) * hkv;
    const int64_t slots = 256 * (c.nw == 4 ? (d > 64 ? 2 : 3) : d > 96 || (f32 && d > 64) ? 2 : d > 64 ? 3 : 5);
    const int64_t tiles = ceil_div(ceil_div(nk, samples), f32 ? AT_KEYS_F32 : AT_KEYS);
    c.whole = c.units * hkv;
    c.splits = c.even = 1;
    c.extra = 0;
    const int64_t full = busy / slots * slots;
    if (busy == full || (full > 0 && (samples > 1 || causal))) return c;
    auto rounds = [&](int64_t n, int64_t length) {
        const int64_t left = n % slots, used = ceil_div(left, 256);
        const double part = left == 0     ? 0.
                            : c.nw == 1   ? 0.5 + 0.5 * (double)left / (double)slots
                            : used == 1   ? (d > 64 ? 0.62 : 0.37)
                            : d > 64      ? 1.
                            : used == 2   ? 0.68
                                          : 1.;
        return ((double)(n / slots) + part) * (double)(length + 3);
    };
    double best = rounds(busy - full, tiles);
    for (int s = 2; s <= AT_MAX_SPLITS && (busy - full) * s <= 2 * slots; s += 1 + s / 32) {
        const double cost = rounds((busy - full) * s, ceil_div(tiles, s)) + (c.nw == 1 ? 6 : 5);
        if (cost < best) {
            best = cost;
            c.splits = s;
            c.whole = full;
        }
    }
    // Several samples may differ in length, which only the device knows. Those of few rows get a part in the join
    // even where their mean asks for none, if one of them can be long: a row each of 64 samples, 16 heads on 2 of
    // 128, 50,000 keys in all, takes 27 us, not 721, where one has nearly all of them (and 26, not 23, where all have 781).
    // From 16,384 keys on: 18.6 us and 271 where one has them, 15.4 and 12.2 where all have as many; of 8,192 keys 16
    // and 134, 15 and 12.
    // Two kinds of batch are not split by length: more than 64 samples (a wave holds them, one a lane) and those that
    // fill the device at their mean length, above. There a sample far longer than the mean is one workgroup's a unit
    // and key head: 827 us for 65 samples where 64 take 27, and 1,500 for one row on 100,000 keys beside
    // 4,000 causal rows (93 on 1,000 keys).
    c.even = c.splits;
    if (samples > 1 && samples <= 64 && (c.splits > 1 || (c.nw == 1 && tiles * samples >= 256))) {
        c.splits = std::max(c.splits, 2);
        c.whole = 0;
        // Whole rounds of equal splits, from 0.7 of one on: with the next whole number always, 4 samples of which one
        // has nearly all of 8,192 keys, 8 heads of 64, take 20 us (15 so); never, 5 of 100 rows and 100,000 keys, 16
        // heads on 2 of 128, 109 (103), though others gain up to 10 %.
        const int64_t items = busy * c.splits, n = items * 10 < slots * 7 ? items : std::max<int64_t>(1, (2 * items + slots) / (2 * slots)) * slots;
        c.extra = std::min(std::max(n / hkv - c.units, c.units), c.units * (c.splits - 1));
    }
    return c;
}

size_t attn_workspace(const AttnCut& c, int hkv, int d) {
    return c.splits == 1 ? 0 : (size_t)(c.blocks(hkv) - c.whole) * c.nw * 32 * (d * sizeof(float) + sizeof(float2));
}

}  // namespace
}  // namespace tsp

using namespace tsp;

extern "C" size_t tsp_attention_workspace_bytes(int64_t nq, int64_t nk, int samples, int hq, int hkv, int d) {
    if (nq <= 0 || nq >= (1ll << 31) || nk < 0 || nk >= (1ll << 31) - (1ll << 16) || samples <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || d <= 0) return 0;
    size_t most = 0;      // (of either mask and type)
    for (int i = 0; i < 4; ++i)
        most = std::max(most, attn_workspace(attn_cut(nq, nk, samples, hkv, hq / hkv, d, i & 1, i & 2), hkv, d));
    return most;
}

extern "C" int tsp_attention(const tsp_heads* q, const tsp_heads* k, const tsp_heads* v, int dtype, int64_t nq, int64_t nk, int hq,
                             int hkv, int d, const int32_t* d_q_offsets, const int32_t* d_k_offsets, int samples, float scale,
                             int causal, const tsp_heads* out, void* d_workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    TSP_REQUIRE(nq >= 0 && nq < (1ll << 31) && nk >= 0 && nk < (1ll << 31) - (1ll << 16), TSP_ERR_INVALID, "tsp_attention: nq=%lld nk=%lld out of range",
                (long long)nq, (long long)nk);
    TSP_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0 && hq <= 4096, TSP_ERR_INVALID, "tsp_attention: %d heads on %d", hq, hkv);
    TSP_REQUIRE(dtype_valid(dtype), TSP_ERR_INVALID, "tsp_attention: bad dtype");
    TSP_REQUIRE(samples > 0 && (samples == 1 || (d_q_offsets && d_k_offsets)), TSP_ERR_INVALID,
                "tsp_attention: samples=%d (without offsets: 1)", samples);
    TSP_REQUIRE(std::isfinite(scale * kLog2e) && scale > 0.f, TSP_ERR_INVALID, "tsp_attention: scale=%g", scale);
    TSP_REQUIRE(d > 0 && d % 8 == 0 && d <= AT_MAX_D, TSP_ERR_UNSUPPORTED, "tsp_attention: heads of %d (need a multiple of 8 up to %d)",
                d, AT_MAX_D);
    if (nq == 0) return TSP_OK;
    TSP_REQUIRE(q && out && q->data && out->data && (nk == 0 || (k && v && k->data && v->data)), TSP_ERR_INVALID,
                "tsp_attention: null pointer");
    const tsp_heads empty{nullptr, 0, 0};
    const tsp_heads kk = nk ? *k : empty, vv = nk ? *v : empty;
    TSP_REQUIRE(heads_aligned(*q) && heads_aligned(*out) && heads_aligned(kk) && heads_aligned(vv), TSP_ERR_INVALID,
                "tsp_attention: data must be 16-byte aligned, strides multiples of 8 (a row's up to 2^20)");
    TSP_REQUIRE(nk == 0 || (kk.row_stride >= d && vv.row_stride >= d), TSP_ERR_INVALID, "tsp_attention: k's and v's rows overlap");
    TSP_REQUIRE(heads_apart(*out, nq, hq, d), TSP_ERR_INVALID, "tsp_attention: the output's heads overlap");
    TSP_REQUIRE(out->data != kk.data && out->data != vv.data && out->data != q->data, TSP_ERR_INVALID, "tsp_attention: out must not alias q, k or v");
    const int share = hq / hkv;
    const AttnCut c = attn_cut(nq, nk, samples, hkv, share, d, causal != 0, dtype == TSP_F32);
    const int64_t past = c.units * hkv - c.whole, blocks = c.blocks(hkv);
    TSP_REQUIRE(blocks * c.nw * 64 < (1ll << 32) && nq * share < (1ll << 31) - 1024, TSP_ERR_INVALID, "tsp_attention: too many rows");
    const size_t need = attn_workspace(c, hkv, d);
    TSP_REQUIRE(need == 0 || d_workspace, TSP_ERR_INVALID, "tsp_attention: null workspace");
    TSP_REQUIRE(workspace_bytes >= need, TSP_ERR_WORKSPACE, "tsp_attention: workspace of %zu bytes, needs %zu", workspace_bytes, need);
    TSP_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0, TSP_ERR_INVALID, "tsp_attention: workspace not 16-byte aligned");
    float* part = need ? static_cast<float*>(d_workspace) : nullptr;
    float2* stat = need ? reinterpret_cast<float2*>(part + (blocks - c.whole) * c.nw * 32 * d) : nullptr;
    // workgroups of a unit's join, by the mean rows of a unit
    const bool many = c.splits > (c.extra ? 2 * AT_FEW_SPLITS : AT_FEW_SPLITS);
    const int rows = (int)std::min<int64_t>(ceil_div(nq * share, samples), c.nw * 32), spread = many ? rows : c.extra ? (rows + 3) / 4 : c.nw * 2;
    const AttnArgs a{q->data, kk.data, vv.data, out->data, q->row_stride, q->head_stride, kk.row_stride, kk.head_stride, vv.row_stride,
                     vv.head_stride, out->row_stride, out->head_stride, d_q_offsets, d_k_offsets, nq, nk, samples, hkv, share, d,
                     causal ? 1 : 0, (int)c.whole, c.extra ? c.even : c.splits, (int)c.extra, (int)blocks,
                     fast_div((uint32_t)share), fast_div((uint32_t)hkv), fast_div((uint32_t)c.splits), scale * kLog2e, part, stat};
    const dim3 grid((unsigned)blocks), block(c.nw * 64);
    hipStream_t s = as_stream(stream);
    using std::integral_constant;
    auto attend = [&](auto bf, auto dp, auto nw) {
        hipLaunchKernelGGL((k_attention<decltype(bf)::value, decltype(dp)::value, decltype(nw)::value>), grid, block, 0, s, a);
    };
    // Heads are widened to the next of four widths (zeros that cost products and LDS): 10,000 rows and keys, 8 heads
    // of 32 take 170-182 us at their own width and 238 at 64; of 80, 297-300 at 96 and 345 at 128.
    auto by_width = [&](auto bf, auto nw) {
        if (d <= 32) attend(bf, integral_constant<int, 32>{}, nw);
        else if (d <= 64) attend(bf, integral_constant<int, 64>{}, nw);
        else if (d <= 96) attend(bf, integral_constant<int, 96>{}, nw);
        else attend(bf, integral_constant<int, 128>{}, nw);
    };
    auto join = [&](auto dt, auto nw) {
        constexpr int DT = decltype(dt)::value, ROWS = decltype(nw)::value * 32;
        if (c.splits == 1) return;
        const dim3 joins((unsigned)spread, (unsigned)past);      // (a unit; there are few of them)
        if (c.extra && many) hipLaunchKernelGGL((k_attention_join<DT, 16, ROWS, true>), joins, dim3(256), 0, s, a);
        else if (c.extra) hipLaunchKernelGGL((k_attention_join<DT, 4, ROWS, true>), joins, dim3(256), 0, s, a);
        else if (many) hipLaunchKernelGGL((k_attention_join<DT, 16, ROWS, false>), joins, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_attention_join<DT, 1, ROWS, false>), joins, dim3(256), 0, s, a);
    };
    auto by_type = [&](auto nw) {
        if (dtype == TSP_BF16) {
            by_width(std::true_type{}, nw);
            join(integral_constant<int, TSP_BF16>{}, nw);
        } else if (dtype == TSP_F16) {
            by_width(std::false_type{}, nw);
            join(integral_constant<int, TSP_F16>{}, nw);
        } else {
            launch_attention_f32(a, c.nw, (unsigned)blocks, s);
            join(integral_constant<int, TSP_F32>{}, nw);
        }
    };
    if (c.nw == 1) by_type(integral_constant<int, 1>{});
    else by_type(integral_constant<int, 4>{});
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
