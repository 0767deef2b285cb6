// Attention of fp32 heads (the formula, the masks and the cut into units and splits are the 16-bit
// kernel's, attention.hip): both products on the fp32 matrix cores, v_mfma_f32_32x32x2, with the same roles,
// S^T = K Q^T and O^T = V^T P^T. Its operands hold one value a lane and two of the contracted index, one a
// lane half. So the scores that a lane has, key 8 (i / 4) + 4 h + i % 4 of a tile in element i for lane half
// h, are the second product's operand one by one, unrounded, beside V's values of those same two keys; in
// the first product a lane half takes d = 8 c + 4 h .. + 3 of K and Q as one 16-byte piece, four steps long.
//
// Bound by the matrix cores: 32x32x2 takes 64 cycles for an eighth of what 32x32x16 does in 32 (a sixteenth of the
// rate), so that a tile of 32 keys is (D / 2 + D / 2) * 64 cycles a wave and its 16 exponents, of 10 cycles, 2 to
// 4 % of that: nothing else is worth overlapping beyond the next tile's loads. 8,192 rows and keys, 8 heads of 128:
// 2.27 ms, 121 of the 157 TFLOP/s that the instruction has; of 64: 1.20 ms, 114. Heads of 32 and of 80 are widened to
// those and take as long. One row on 40,009 keys, 16 heads on 2 of 128: 44 us on a floor of 12.
#include "attention_internal.hpp"

namespace tsp {
namespace {

constexpr int KEYS = AT_KEYS_F32;

// Byte offsets in a staged tile of KEYS rows of DP floats, as 16-byte pieces: K's xored with the key (32 keys
// are read at one d), V's by half of 64 banks with the key's 4 (4 h is what tells the lane halves' keys apart).
template <int DP>
__device__ __forceinline__ int k_piece(int key, int piece) {
    return key * (DP * 4) + (piece ^ (key & 15)) * 16;
}
template <int DP>
__device__ __forceinline__ int v_piece(int key, int piece) {
    return key * (DP * 4) + (piece ^ ((key >> 2 & 1) << 3)) * 16;
}

template <int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW == 1 && DP > 64 ? 1 : 2) void k_attention_f32(AttnArgs a) {
    constexpr int C = DP / 8, DB = DP / 32, P = DP / 4, ROWS = NW * 32, TILE = KEYS * DP * 4;
    __shared__ __attribute__((aligned(16))) char sK[2][TILE], sV[2][TILE];
    int split = 0, splits = 1;
    AttnUnit t;
    if (__builtin_expect(a.extra != 0, 0)) {
        const AttnItem item = attn_item<ROWS, KEYS, true>(a, blockIdx.x);
        t = item;
        split = item.split;
        splits = item.splits;
    } else {
        int work = blockIdx.x;
        if (work >= a.whole) {
            const int past = work - a.whole, at = past / a.by_splits;
            splits = a.splits;
            work = a.whole + at;
            split = past - at * splits;
        }
        t = attn_unit<ROWS>(a, work);
    }
    const PackedUnit& u = t.u;
    if (u.sample < 0) return;
    const int krow0 = u.other0, lk = u.others, rows = t.rows, tile0 = t.row0;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;

    // rows past the sample's last are copies of it that are not stored
    auto limit = [&](int query) { return a.causal ? min(max(lk - u.rows + query + 1, 0), lk) : lk; };
    auto query = [&](int r) { return min(r, rows - 1) / a.by_share; };
    const int r = tile0 + wave * 32 + r32, qi = query(r), hq = t.head * a.share + min(r, rows - 1) - qi * a.share;
    const RowLimits lim{limit(qi), limit(query(tile0 + wave * 32 + 31))};
    const int first_end = limit(query(tile0 + wave * 32)), wg_end = limit(query(tile0 + ROWS - 1));

    f32x4_t qf[C];
    {
        const float* qp = static_cast<const float*>(a.q) + (int64_t)(u.row0 + qi) * a.q_row + hq * a.q_head;
#pragma unroll
        for (int c = 0; c < C; ++c)
            qf[c] = c * 8 < a.d ? *reinterpret_cast<const f32x4_t*>(qp + c * 8 + h * 4) : f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    const char* kp = static_cast<const char*>(a.k) + 4 * ((int64_t)krow0 * a.k_row + t.head * a.k_head);
    const char* vp = static_cast<const char*>(a.v) + 4 * ((int64_t)krow0 * a.v_row + t.head * a.v_head);
    const int k_bytes = (int)a.k_row * 4, v_bytes = (int)a.v_row * 4;

    // A tile straight into LDS, 1 KiB a wave and load; rows past the last key and pieces past d read as zeros
    // (out of the buffer's range).
    constexpr int LOADS = TILE / 1024 / NW, LOAD_ROWS = 1024 / (DP * 4), NOWHERE = 1 << 30;
    auto stage = [&](const char* p, int bytes, int base, char* s, bool is_v) {
        const int n = min(KEYS, lk - base);
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(p + (int64_t)base * bytes), (short)0, n * bytes, 0x00027000);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int key = (i * NW + wave) * LOAD_ROWS + lane / P;
            const int piece = (is_v ? v_piece<DP>(key, lane % P) : k_piece<DP>(key, lane % P)) / 16 % P;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(s + (i * NW + wave) * 1024), 16,
                                                     piece * 4 < a.d ? key * bytes + piece * 16 : NOWHERE, 0, 0, 0);
        }
    };

    f32x16_t o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16_t{};
    float m = -INFINITY, l = 0.f;
    const int tiles = (wg_end + KEYS - 1) / KEYS, per = (int)((unsigned)(tiles + splits - 1) / (unsigned)splits);
    const int begin = split * per * KEYS, end = min(wg_end, begin + per * KEYS);
    if (begin < end) {
        stage(kp, k_bytes, begin, sK[0], false);
        stage(vp, v_bytes, begin, sV[0], true);
    }
    for (int base = begin, at = 0; base < end; base += KEYS, at ^= 1) {
        wait_loads();
        __syncthreads();      // this tile has landed, and the other buffer is no longer read
        if (base + KEYS < end) {
            stage(kp, k_bytes, base + KEYS, sK[at ^ 1], false);
            stage(vp, v_bytes, base + KEYS, sV[at ^ 1], true);
        }
        if (base >= lim.hi) continue;
        const char *ks = sK[at], *vs = sV[at];
        f32x16_t s = f32x16_t{};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const f32x4_t kf = *reinterpret_cast<const f32x4_t*>(ks + k_piece<DP>(r32, 2 * c + h));
#pragma unroll
            for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j], qf[c][j], s, 0, 0, 0);
        }
        const bool masked = base + KEYS > first_end;
        if (masked) {
            const int left = lim.lane - base - 4 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 8 * (i / 4) + i % 4 < left ? s[i] : -INFINITY;
        }
        float mt = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mt = fmaxf(mt, s[i]);
        const float2 mh = both_halves(mt);
        mt = fmaxf(mh.x, mh.y);
        // (the maximum moves by factors of 2^8 only: most tiles leave the sums as they are)
        if (__any((mt - m) * a.scale2 > 8.f)) {
            const float mn = fmaxf(m, mt);
            const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * a.scale2);
            m = mn;
            l *= corr;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] *= corr;
        }
        const float top = m == -INFINITY ? 0.f : m;      // (taken from the scores: m * scale2 would be rounded)
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f((s[i] - top) * a.scale2);
            sum += s[i];
        }
        l += sum;
        // Rows of the tile that see different keys: a probability of zero must not meet an Inf or a NaN of a key
        // that its row does not see. Zero times V shows whether there is one.
        bool odd = false;
        if (masked && a.causal) {
            float z = 0.f;
            for (int i = lane; i < TILE / 16; i += 64) {
                const f32x4_t x = *reinterpret_cast<const f32x4_t*>(vs + i * 16);
                z += x[0] * 0.f + x[1] * 0.f + x[2] * 0.f + x[3] * 0.f;
            }
            odd = __any(z != z);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = 8 * (i / 4) + 4 * h + i % 4;
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                float x = *reinterpret_cast<const float*>(vs + v_piece<DP>(key, db * 8 + (r32 >> 2)) + (r32 & 3) * 4);
                if (odd && (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) x = 0.f;
                o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, s[i], o[db], 0, 0, 0);
            }
        }
        if (odd) {      // the values left out, key by key, for the rows that see them
            for (int key = 0; key < KEYS; ++key) {
                float p = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (8 * (i / 4) + i % 4 == (key & ~4)) p = s[i];
                const float2 ph = both_halves(p);
                p = key & 4 ? ph.y : ph.x;
                const bool sees = base + key < lim.lane;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int e = db * 32 + 8 * (i / 4) + 4 * h + i % 4;
                        const float x = *reinterpret_cast<const float*>(vs + v_piece<DP>(key, e >> 2) + (e & 3) * 4);
                        if (sees && (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) o[db][i] += p * x;
                    }
            }
        }
    }

    const float2 lh = both_halves(l);
    const float sum = lh.x + lh.y;
    if (r >= rows) return;
    const bool parts = splits > 1, seen = lim.lane > begin && begin < end;
    const int64_t item = (int64_t)((int)blockIdx.x - a.whole) * ROWS + (r - tile0);
    if (parts && h == 0) a.stat[item] = float2{m, seen ? sum : -1.f};
    if (parts && !seen) return;
    float* op = parts ? a.part + item * a.d : static_cast<float*>(a.o) + (int64_t)(u.row0 + qi) * a.o_row + hq * a.o_head;
    const float f = parts ? 1.f : lim.lane == 0 ? 0.f : 1.0f / sum;      // (no key seen: zeros)
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = db * 32 + 8 * g + 4 * h;
            if (e < a.d)
                *reinterpret_cast<f32x4_t*>(op + e) = f32x4_t{o[db][4 * g] * f, o[db][4 * g + 1] * f, o[db][4 * g + 2] * f, o[db][4 * g + 3] * f};
        }
}

}  // namespace

void launch_attention_f32(const AttnArgs& a, int nw, unsigned blocks, hipStream_t s) {
    const dim3 grid(blocks), block(nw * 64);
    if (a.d <= 64 && nw == 1) hipLaunchKernelGGL((k_attention_f32<64, 1>), grid, block, 0, s, a);
    else if (a.d <= 64) hipLaunchKernelGGL((k_attention_f32<64, 4>), grid, block, 0, s, a);
    else if (nw == 1) hipLaunchKernelGGL((k_attention_f32<128, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_attention_f32<128, 4>), grid, block, 0, s, a);
}

}  // namespace tsp
