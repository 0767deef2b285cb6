// Softmax attention of new queries to the keys and values of a paged cache (kv_cache.hpp), in 4 or 16 bits:
//   out[i][h] = sum_j exp(scale q_i . k_j - max) v_j / sum_j exp(scale q_i . k_j - max)
// over the keys j of i's sample that the row sees: all lengths[s] of them, or with `causal` those with
// j <= i + (lengths[s] - Lq). A row that sees none gets zeros.
//
// A row is a (query, head of the group) pair, a unit is up to ROWS rows of a sample and key head, its work the tiles of
// keys that they see. All units' tiles stand in one line, which is cut into as many equal parts as there are workgroups,
// whatever the samples' lengths: only the device knows those. A workgroup goes through its part unit by unit; a
// unit that a cut goes through leaves its rows' maxima, sums and sums of p v in the workspace, at most two a workgroup,
// and a second launch joins them, in their order. (The line's weights are a linear estimate of a unit's tiles,
// so that its sums have a closed form; where in a unit a cut falls goes by its true tiles.)
//
// 4-bit codes become 16-bit values with their power as they are read, two a conversion, exactly (in f16: for powers
// that fit it). Both products run on the matrix cores with their roles turned, S^T = K Q^T and O^T = V^T P^T, so that
// a lane holds scores of one row and P is the second product's operand where it stands. Statistics and accumulators are
// fp32; P is rounded to the heads' type, as the packed attention's (attention.hip) is, and formed as there.
//
// Two kernels. Few rows (k_cached_few): waves of their own, each with every fourth tile of 32 keys: K goes from memory to its
// operand, V through a piece of LDS that is the wave's alone, where it is turned. Many rows (k_cached_many): four waves of 32
// rows share a tile of 64 keys, widened into LDS by all of them.
//
// What bounds them, in bf16, heads of 128, 4 bits. One row of 16 heads on 2, 40,009 keys: 14.6 us, latency: the lengths, the table, the
// first tile and the next four one after the other on 500 workgroups, then the join's counts and pieces; 300 keys 9,
// 200,000 25. 16 samples' tokens, 16 heads on 4, 400,009 keys: 50 us, 46 of them at 4.6 TB/s of cache read, where widening keeps the
// vector units 40 % busy; in 16 bits 174-178 (4.7 TB/s). 64 samples' tokens of 512 keys, 16 heads on 8: 29; the line's parts are
// shorter than a unit there, so that nearly all are cut and joined. 5,003 rows on 35,001 keys, two samples: 807-838 us by the box,
// 960-1,000 TFLOP/s; the matrix cores are 42 % busy at 2.0 GHz, the vector units, which widen, form exponents and round, 45 %. In 16
// bits 945-960: a tile has one step to land. A causal prompt of 8,000 rows takes 411, 20,000 rows of 16 heads of 64 on 1,029
// keys 182: 8.0 us for 64 keys (3.7 of products; the exponents of short products) and some 46 whatever the keys, in which units start (the
// line, Q, a look at the pages, the first tiles) and end with nothing beside them. The packed attention takes 111 for the same.
// Tried and taken back: eight waves a workgroup of many rows (tiles wait for the slowest wave), four waves a SIMD in either kernel
// (registers spilled: a kernel with any scratch starts some 7 us later), one LDS array for both buffers (every
// load waited for), a launch of the join for each place where a cut can be (10 to 30 us).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_internal.hpp"
#include "kv_cache.hpp"
#include "mx.hpp"
#include "overlap.hpp"

namespace tsp {
namespace {

constexpr int CF_KEYS = 32, CF_NW = 4;                               // few rows: keys of a tile, waves
constexpr int CM_KEYS = 64, CM_NW = 4, CM_ROWS = CM_NW * 32;         // many

struct CachedArgs {
    const void* q;
    void* o;
    int64_t q_row, q_head, o_row, o_head;      // strides in elements
    KvArgs cache;
    const int32_t* q_off;
    int64_t nq;                                // below 2^31, nq * share too
    int samples, share, causal;
    int groups, least, finer, coarser;         // workgroups at most, what one has at least; weights are tiles << finer >> coarser
    FastDiv by_share, by_groups;
    float scale2;                              // scale * log2(e)
    float* part;                               // [2 * groups][row][d] sums of p v, and
    float2* stat;                              // [2 * groups][row] maximum and sum of p (-1: no key seen), and
    struct JoinItem* join;                     // [groups] the unit that is cut at the workgroup's end and began in it
};

// The unit's rows (0: there is none) and above them 256 times its last workgroup, its first row, the sample's, the key head.
struct JoinItem {
    int cut, first_row, row0, head;
};

#ifdef __HIP_DEVICE_COMPILE__       // (the host pass knows neither the register constraint nor the argument segment)
// The kernel's arguments read anew: kept in scalar registers from the start on they would push the loops' own out of them.
typedef const __attribute__((address_space(4))) CachedArgs* CachedArgsPtr;
__device__ __forceinline__ CachedArgsPtr reread_args() {
    CachedArgsPtr p = (CachedArgsPtr)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}
#endif

// A sample's units (one key head) and their weights, first + slope * j of the j-th. (All sums of weights are below 2^30.)
struct SampleWork {
    int row0, lq, lk, count;
    uint32_t first, slope;
    __device__ __forceinline__ uint32_t before(uint32_t j) const { return first * j + slope * j * (j - 1) / 2; }
};
// Keys that a row sees, by its query.
__device__ __forceinline__ int cached_limit(int causal, int lq, int lk, int query) { return causal ? min(max(lk - lq + query + 1, 0), lk) : lk; }
template <int ROWS, int TILE, class Args>
__device__ __forceinline__ int unit_tiles(const Args& a, int lq, int lk, int j) {
    const int last = min((j + 1) * ROWS, lq * a.share) - 1;
    return (cached_limit(a.causal, lq, lk, last / FastDiv{a.by_share.mul, a.by_share.shift}) + TILE - 1) / TILE;
}
template <int ROWS, int TILE, class Args>
__device__ __forceinline__ SampleWork sample_work(const Args& a, int s) {
    SampleWork w{0, 0, 0, 0, 1, 0};
    if (s >= a.samples) return w;
    packed_rows(a.q_off, s, (int)a.nq, w.row0, w.lq);
    w.lk = (int)min((int64_t)max(a.cache.lengths[s], 0), (int64_t)a.cache.max_pages << a.cache.page_bits);
    w.count = (int)((unsigned)(w.lq * a.share + ROWS - 1) / (unsigned)ROWS);
    if (w.count == 0) return w;
    auto weight = [&](int j) { return max(1, (unit_tiles<ROWS, TILE>(a, w.lq, w.lk, j) << a.finer) >> a.coarser); };
    w.first = weight(0);
    if (w.count > 1) w.slope = (uint32_t)max(0, weight(w.count - 1) - (int)w.first) / (uint32_t)(w.count - 1);
    return w;
}

// The line: its length, each workgroup's part, and where there are up to 64 samples, what a lane knows of its own (by whole waves).
struct Line {
    uint32_t length, per;
    SampleWork w;
    uint32_t end;      // of the sample's units
    __device__ __forceinline__ uint32_t cut(int group) const { return min(per * (uint32_t)group, length); }
    __device__ __forceinline__ int group(uint32_t at) const { return (int)(at / per); }
};
// The sum over a lane and those before it (moves along a row of 16 lanes, then rows' last lanes to the rows after them).
__device__ __forceinline__ uint32_t scan64(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);      // row_shr 1
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);      // 2
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);      // 4
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);      // 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);      // row_bcast 15, to rows 1 and 3
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);      // row_bcast 31, to rows 2 and 3
    return v;
}
template <int ROWS, int TILE, class Args>
__device__ __forceinline__ Line make_line(const Args& a) {
    Line l;
    l.length = 0;
    if (a.samples == 1) {
        l.w = sample_work<ROWS, TILE>(a, 0);
        l.length = l.end = __builtin_amdgcn_readfirstlane(l.w.before(l.w.count) * a.cache.heads);
    } else {
        bool falls = false;
        for (int s0 = 0; s0 < a.samples; s0 += 64) {
            const int s = s0 + (threadIdx.x & 63);
            l.w = sample_work<ROWS, TILE>(a, s);
            l.end = l.length + scan64(l.w.before(l.w.count) * a.cache.heads);
            l.length = __builtin_amdgcn_readlane(l.end, 63);
            if (s < a.samples) falls |= a.q_off[s] > a.q_off[s + 1];
        }
        if (__any(falls)) l.length = 0;      // (samples would overlap, and the line could be of any length: no row is anyone's)
    }
    l.length = __builtin_amdgcn_readfirstlane(l.length);
    // (two workgroups a CU until each has `least`: eight tiles of few rows, four of many. us with that many in each from the start,
    // and so: 1 row on 300 keys 13.1 and 8.9, on 40,009 15.7 and 15.2; 8 rows on 4,000 24 and 15.4; a prompt of 300 rows 34 and 24)
    const int least = max(min(a.least, (int)((l.length + 511) / 512)), max((1 << a.finer) >> a.coarser, 1));
    l.per = max(least, (int)(l.length + a.groups - 1) / FastDiv{a.by_groups.mul, a.by_groups.shift});
    return l;
}

// A unit and where it stands in the line.
struct CachedUnit {
    int sample, head, row0, lq, lk;
    int first_row;                       // of its rows among the sample's
    int tiles;
    uint32_t begin, end;
};
// The unit at a place in the line (by whole waves, all with one `at`).
template <int ROWS, int TILE, class Args>
__device__ __forceinline__ CachedUnit find_unit(const Args& a, const Line& line, uint32_t at) {
    CachedUnit u{0, 0, 0, 0, 0, 0, 0, 0, 0};
    auto first = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
    SampleWork k{(int)first(line.w.row0), (int)first(line.w.lq), (int)first(line.w.lk), (int)first(line.w.count), first(line.w.first), first(line.w.slope)};
    uint32_t base = 0;
    if (a.samples > 1) {
        SampleWork w = line.w;
        uint32_t end = line.end, mine = 0;
        uint64_t found = 0;
        for (int s0 = 0; s0 < a.samples; s0 += 64) {
            if (a.samples > 64) {
                w = sample_work<ROWS, TILE>(a, s0 + (threadIdx.x & 63));
                end = base + scan64(w.before(w.count) * a.cache.heads);
            }
            mine = w.before(w.count) * a.cache.heads;
            found = __ballot(at >= end - mine && at < end);
            u.sample = s0;
            if (found) break;
            base = __builtin_amdgcn_readlane(end, 63);
        }
        const int l = found ? __builtin_ctzll(found) : 0;      // (there is one: `at` is below the line's length)
        auto of = [&](uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane(x, l); };
        k = SampleWork{(int)of(w.row0), (int)of(w.lq), (int)of(w.lk), (int)of(w.count), of(w.first), of(w.slope)};
        base = of(end - mine);
        u.sample += l;
    }
    u.row0 = k.row0, u.lq = k.lq, u.lk = k.lk;
    const uint32_t per_head = k.before(k.count), in = at - base;
    const uint32_t head = first(in / per_head), x = in - head * per_head;
    u.head = (int)head;
    uint32_t j = 0;
    if (k.count > 1) {
        if (k.slope == 0) {
            j = x / k.first;
        } else {      // first j + slope j (j - 1) / 2 <= x
            const float b = (float)k.first - 0.5f * (float)k.slope;
            j = (uint32_t)max((int)((sqrtf(b * b + 2.f * (float)k.slope * (float)x) - b) / (float)k.slope), 0);
            j = min(j, (uint32_t)k.count - 1);
            while (j > 0 && k.before(j) > x) --j;
            while (j + 1 < (uint32_t)k.count && k.before(j + 1) <= x) ++j;
        }
        j = first(j);
    }
    u.first_row = (int)j * ROWS;
    u.begin = base + head * per_head + k.before(j);
    u.end = u.begin + k.first + k.slope * j;
    u.tiles = (int)first(unit_tiles<ROWS, TILE>(a, u.lq, u.lk, (int)j));
    return u;
}

// One workgroup's piece of a unit: tiles [t0, t1) of it, and its place in the workspace (-1: it has all of the unit).
struct CachedPiece {
    int t0, t1, slot;
};
__device__ __forceinline__ CachedPiece cut_unit(const CachedUnit& u, uint32_t from, uint32_t to, int w) {
    const uint32_t lo = max(from, u.begin) - u.begin, hi = min(to, u.end) - u.begin, weight = u.end - u.begin;
    // (a place of the line is one tile, whichever workgroup asks: the products are the same and grow with it)
    const float each = (float)u.tiles / (float)weight;
    auto tile = [&](uint32_t x) { return (uint32_t)u.tiles == weight ? (int)x : x == weight ? u.tiles : min((int)((float)x * each), u.tiles); };
    return CachedPiece{__builtin_amdgcn_readfirstlane(tile(lo)), __builtin_amdgcn_readfirstlane(tile(hi)), lo == 0 && hi == weight ? -1 : 2 * w + (lo == 0)};
}
// What the join has to know of a workgroup's last unit.
template <int ROWS, class Args>
__device__ __forceinline__ void tell_join(const Args& a, const CachedUnit& u, const Line& line, uint32_t to, int w, bool begins) {
    JoinItem j{};
    if (begins && u.end > to) j = JoinItem{min(u.lq * a.share - u.first_row, ROWS) | line.group(u.end - 1) << 8, u.first_row, u.row0, u.head};
    if (threadIdx.x == 0) a.join[w] = j;
}

// Four bytes of codes as eight 16-bit values.
template <bool BF16>
__device__ __forceinline__ u32x4_t widen4(uint32_t c, float s) {
    if constexpr (BF16)
        return u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
    else
        return u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 0)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 1)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 2)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 3))};
}

template <bool BF16>
__device__ __forceinline__ f32x4_t mfma16(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// The largest of a value over the four lanes 16 apart.
__device__ __forceinline__ float max_over_groups(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float2 h = both_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
    return fmaxf(h.x, h.y);
}

// Byte offset of a 16-byte piece of V in a staged tile: as v_piece, and the piece's lowest bit xored with the key's, so
// that the 16 pieces that two keys' lanes write at once (every fourth of each) lie in other banks.
template <int DP>
__device__ __forceinline__ int cv_piece(int key, int piece) { return v_piece<DP>(key, piece ^ (DP >= 64 ? key & 1 : 0)); }

template <bool BF16>
__device__ __forceinline__ bool any_nonfinite(const u32x4_t& v) {
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) odd |= nonfinite16<BF16>(v[i]) || nonfinite16<BF16>(v[i] >> 16);
    return odd;
}
template <bool BF16>
__device__ __forceinline__ u32x4_t finite_only(u32x4_t v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (nonfinite16<BF16>(v[e])) v[e] &= 0xffff0000u;
        if (nonfinite16<BF16>(v[e] >> 16)) v[e] &= 0xffffu;
    }
    return v;
}
template <bool BF16>
__device__ __forceinline__ float value16(uint32_t b) { return BF16 ? bf16_bits_to_f32((uint16_t)b) : f16_bits_to_f32((uint16_t)b); }

// ---- few rows ------------------------------------------------------------------------------------------------------
// NB: blocks of 32 channels a head; MX4: 4-bit pages; RT: tiles of 16 rows.
template <bool BF16, int NB, bool MX4, int RT>
__global__ __launch_bounds__(CF_NW * 64, 2) void k_cached_few(CachedArgs) {
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int DP = NB * 32, ROWS = RT * 16, DB = NB * 2;
    constexpr int VP = MX4 ? NB : NB * 4;                        // 16-byte pieces of a key's V in the page
    constexpr int VL = (16 * VP + 63) / 64;                      // loads of them a lane, for 16 keys
    constexpr int V_BYTES = CF_KEYS * DP * 2, O_BYTES = ROWS * DP * 4;
    __shared__ __attribute__((aligned(16))) char sBuf[CF_NW][V_BYTES > O_BYTES ? V_BYTES : O_BYTES];
    __shared__ float2 sStat[CF_NW][ROWS];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    char* sV = sBuf[wave];
    const Line line = make_line<ROWS, CF_KEYS>(*reread_args());
    const uint32_t to = line.cut(blockIdx.x + 1);
    if (line.cut(blockIdx.x) >= to) {
        if (threadIdx.x == 0) reread_args()->join[blockIdx.x].cut = 0;
        return;
    }
    constexpr float LAG = BF16 ? 8.f : 4.f, LIFT = BF16 ? 0.f : 11.f;

    for (uint32_t from = line.cut(blockIdx.x); from < to;) {
        const auto& a = *reread_args();
        const CachedUnit u = find_unit<ROWS, CF_KEYS>(a, line, from);
        const CachedPiece piece = cut_unit(u, from, to, blockIdx.x);
        if (u.end >= to) tell_join<ROWS>(a, u, line, to, blockIdx.x, from <= u.begin);
        from = u.end;
        const int rows = u.lq * a.share;
        const FastDiv by_share{a.by_share.mul, a.by_share.shift};
        // (what the loop needs)
        const int page_bits = a.cache.page_bits, page_mask = (1 << page_bits) - 1, pool = a.cache.pages, d = a.cache.d, lk = u.lk;
        const int64_t page_bytes = a.cache.page_bytes;
        const float scale2 = a.scale2;
        // rows past the sample's last are copies of it that are not stored
        int limit[RT];
        u32x4_t qf[RT][NB];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = min(u.first_row + rt * 16 + r16, rows - 1), qi = r / by_share, hq = u.head * a.share + r - qi * a.share;
            limit[rt] = cached_limit(a.causal, u.lq, u.lk, qi);
            const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (int64_t)(u.row0 + qi) * a.q_row + hq * a.q_head;
            // chunk c = NB g + i of eight channels
#pragma unroll
            for (int i = 0; i < NB; ++i) qf[rt][i] = (NB * g + i) * 8 < d ? *reinterpret_cast<const u32x4_t*>(qp + (NB * g + i) * 8) : u32x4_t{0, 0, 0, 0};
        }
        const int all_see = cached_limit(a.causal, u.lq, u.lk, u.first_row / by_share);      // (the first row sees least)
        f32x4_t o[RT][DB];
        float m[RT], l[RT];
        bool seen[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -INFINITY, l[rt] = 0.f, seen[rt] = false;
#pragma unroll
            for (int db = 0; db < DB; ++db) o[rt][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
        // What a tile's two runs of 16 keys are loaded into: K's chunks as they are read, V's pieces.
        struct Raw {
            u32x4_t k[2][MX4 ? 1 : NB], v[2][VL];
            uint32_t kp[2][MX4 && NB == 3 ? 2 : 1], vp[2];
        } w;
        // Their pages (-1: none), by scalar loads.
        const auto table = (const __attribute__((address_space(4))) int32_t*)(a.cache.table + (int64_t)u.sample * a.cache.max_pages);
        struct Pages {
            int p[2];
        };
        auto pages_of = [&](int tile) __attribute__((always_inline)) {
            Pages pages;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int key = __builtin_amdgcn_readfirstlane(tile * CF_KEYS + kb * 16);
                pages.p[kb] = key < lk && tile < piece.t1 ? table[key >> page_bits] : -1;
            }
            return pages;
        };
        auto held = [&](const Pages& pages, int kb) __attribute__((always_inline)) { return (unsigned)pages.p[kb] < (unsigned)pool; };
        // Within a head's bytes of a page: a lane's first byte of K and of V, and of their powers, at a run's slot 0.
        const uint8_t* const head = a.cache.data + u.head * a.cache.head_bytes;
        const int row_bytes = MX4 ? 16 * NB : d * 2;
        const int k_at = r16 * row_bytes + (MX4 ? 4 * NB : 16 * NB) * g, v_key = lane / VP, v_piece_of = lane % VP;
        const int v_at = v_key * row_bytes + v_piece_of * 16 + (row_bytes << page_bits);
        const int kp_at = (2 * row_bytes << page_bits) + r16 * NB + NB * g / 4, vp_at = ((2 * row_bytes + NB) << page_bits) + lane;
        auto load = [&](int tile, const Pages& pages) __attribute__((always_inline)) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                for (int i = 0; i < (MX4 ? 1 : NB); ++i) w.k[kb][i] = u32x4_t{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < VL; ++i) w.v[kb][i] = u32x4_t{0, 0, 0, 0};
                w.kp[kb][0] = w.vp[kb] = 0;
                if constexpr (MX4 && NB == 3) w.kp[kb][1] = 0;
                if (!held(pages, kb)) continue;
                const int key = tile * CF_KEYS + kb * 16, slot = key & page_mask;
                const uint8_t* const at = head + pages.p[kb] * page_bytes + slot * row_bytes;
                const int left = lk - key;        // (keys past the sample's last: V zeros, whatever the page holds)
                if constexpr (MX4) {
                    if constexpr (NB == 4) w.k[kb][0] = *reinterpret_cast<const u32x4_t*>(at + k_at);
                    else
#pragma unroll
                        for (int i = 0; i < NB; ++i) w.k[kb][0][i] = *reinterpret_cast<const uint32_t*>(at + k_at + 4 * i);
                    const uint8_t* const power = at - slot * (row_bytes - NB);
                    w.kp[kb][0] = power[kp_at];
                    if constexpr (NB == 3) w.kp[kb][1] = power[kp_at + (NB * g + 2) / 4 - NB * g / 4];
                    if (lane < 16 * VP && v_key < left) {
                        w.v[kb][0] = *reinterpret_cast<const u32x4_t*>(at + v_at);
                        w.vp[kb] = power[vp_at];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < NB; ++i)
                        if ((NB * g + i) * 8 < d) w.k[kb][i] = *reinterpret_cast<const u32x4_t*>(at + k_at + 16 * i);
#pragma unroll
                    for (int i = 0; i < VL; ++i) {
                        const int idx = i * 64 + lane, in = idx / VP, p = idx % VP;
                        if (in < 16 && in < left && p * 8 < d)
                            w.v[kb][i] = *reinterpret_cast<const u32x4_t*>(at + (row_bytes << page_bits) + in * row_bytes + p * 16);
                    }
                }
            }
        };
        // The tile whose keys have been loaded; the next one's loads go out once they have been used.
        auto attend = [&](int tile, const Pages& pages, const Pages& next) __attribute__((always_inline)) {
            const int base = tile * CF_KEYS;
            const bool held0 = held(pages, 0), held1 = held(pages, 1);
            // V to LDS, as 16-bit values. (Places that differ in a few bits are formed where they are used: kept from tile to
            // tile they would take the registers of two more waves.)
            bool odd = false;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                if constexpr (MX4) {
                    if (16 * VP < 64 && lane >= 16 * VP) continue;
                    const float s = mx_scale(w.vp[kb]);
                    odd |= w.vp[kb] >= (BF16 ? 253 : 141);      // (NaN, and powers with which the largest codes are past the range)
                    int to = cv_piece<DP>(v_key, v_piece_of * 4);
                    asm volatile("" : "+v"(to));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const u32x4_t x = widen4<BF16>(w.v[kb][0][j], s);
                        *reinterpret_cast<u32x4_t*>(sV + kb * 16 * DP * 2 + (to ^ (j * 16))) = x;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < VL; ++i) {
                        const int idx = i * 64 + lane, in = idx / VP, p = idx % VP;
                        if (16 * VP % 64 && in >= 16) continue;
                        odd |= any_nonfinite<BF16>(w.v[kb][i]);
                        *reinterpret_cast<u32x4_t*>(sV + kb * 16 * DP * 2 + cv_piece<DP>(in, p)) = w.v[kb][i];
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);      // (here and below: the registers of two more waves a SIMD)
            // scores: s[rt][kb][i] is key 16 kb + 4 g + i
            f32x4_t s[RT][2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) s[rt][kb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    u32x4_t k;
                    if constexpr (MX4) k = widen4<BF16>(w.k[kb][0][i], mx_scale(NB == 3 && (NB * g + i) / 4 != NB * g / 4 ? w.kp[kb][NB == 3 ? 1 : 0] : w.kp[kb][0]));
                    else k = w.k[kb][i];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) s[rt][kb] = mfma16<BF16>(k, qf[rt][i], s[rt][kb]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (tile + CF_NW < piece.t1) load(tile + CF_NW, next);
            const bool whole = base + CF_KEYS <= all_see && held0 && held1;
            u32x4_t pf[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (whole) {
                    seen[rt] = true;
                } else {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool sees = (kb ? held1 : held0) && kb * 16 + i < limit[rt] - base - 4 * g;
                            seen[rt] |= sees;
                            s[rt][kb][i] = sees ? s[rt][kb][i] : -INFINITY;
                        }
                }
                float mt = fmaxf(fmaxf(fmaxf(s[rt][0][0], s[rt][0][1]), fmaxf(s[rt][0][2], s[rt][0][3])),
                                 fmaxf(fmaxf(s[rt][1][0], s[rt][1][1]), fmaxf(s[rt][1][2], s[rt][1][3])));
                mt = max_over_groups(mt);
                // (the maximum moves where a row's has grown by a factor of 2^LAG alone; p has room for that)
                if (__any((mt - m[rt]) * scale2 > LAG)) {
                    const float mn = fmaxf(m[rt], mt), corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[rt] - mn) * scale2);
                    m[rt] = mn;
                    l[rt] *= corr;
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[rt][db][i] *= corr;
                }
                const float top = m[rt] == -INFINITY ? 0.f : m[rt];
                float sum = 0.f;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[rt][kb][i] = __builtin_amdgcn_exp2f(fmaf(s[rt][kb][i] - top, scale2, LIFT));
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        pf[rt][2 * kb + i] = pack2<BF16>(s[rt][kb][2 * i], s[rt][kb][2 * i + 1]);
                        sum = add2<BF16>(pf[rt][2 * kb + i], sum);
                    }
                }
                l[rt] += sum;
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            // A probability of zero must not meet an Inf or a NaN of a key that its row does not see.
            odd = !whole && __any(odd);
            int from_v = cv_piece<DP>(4 * g + ((lane >> 2) & 3), (lane >> 1) & 1) + (lane & 1) * 8;
            asm volatile("" : "+v"(from_v));
            auto values = [&](int db) __attribute__((always_inline)) {
                const char* const at = sV + (NB == 3 ? from_v + db * 32 : from_v ^ (db * 32));      // (rows of 96 are not swizzled so far)
                const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)at);
                const s16x4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(at + 16 * DP * 2));
                const uint2 ux = __builtin_bit_cast(uint2, x), uy = __builtin_bit_cast(uint2, y);
                return u32x4_t{ux.x, ux.y, uy.x, uy.y};
            };
            if (__builtin_expect(!odd, 1)) {
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    const u32x4_t v = values(db);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) o[rt][db] = mfma16<BF16>(v, pf[rt], o[rt][db]);
                    if (db % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
                return;
            }
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const u32x4_t v = finite_only<BF16>(values(db));
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) o[rt][db] = mfma16<BF16>(v, pf[rt], o[rt][db]);
                __builtin_amdgcn_sched_barrier(0);      // (one operand at a time: registers)
            }
            // the values left out, key by key, for the rows that see them
            {
                for (int key = 0; key < CF_KEYS; ++key) {
                    if (!(key < 16 ? held0 : held1)) continue;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        float p = 0.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if ((key & 19) == i) p = s[rt][0][i];
                            if ((key & 19) == 16 + i) p = s[rt][1][i];
                        }
                        p = __shfl(p, (key & 12) * 4 + r16, 64);
                        const bool sees = base + key < limit[rt];
                        int at = 4 * g;
                        asm volatile("" : "+v"(at));
#pragma unroll
                        for (int db = 0; db < DB; ++db)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int e = db * 16 + at + i;
                                const uint32_t b = *reinterpret_cast<const uint16_t*>(sV + cv_piece<DP>(key, e >> 3) + (e & 7) * 2);
                                if (sees && nonfinite16<BF16>(b)) o[rt][db][i] += p * value16<BF16>(b);
                                __builtin_amdgcn_sched_barrier(0);
                            }
                    }
                }
            }
        };
        int tile = piece.t0 + wave;
        if (tile < piece.t1) {
            Pages now = pages_of(tile), next = pages_of(tile + CF_NW);
            load(tile, now);
            for (; tile < piece.t1; tile += CF_NW) {
                const Pages after = pages_of(tile + 2 * CF_NW);
                attend(tile, now, next);
                now = next;
                next = after;
            }
        }
        // the waves' rows joined
        const auto& b = *reread_args();
        int tid = threadIdx.x;      // (as above: places of its own)
        asm volatile("" : "+v"(tid));
        const int row16 = tid & 15, group = tid >> 4 & 3;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            l[rt] += __shfl_xor(l[rt], 16, 64);
            l[rt] += __shfl_xor(l[rt], 32, 64);
            int any = seen[rt];
            any |= __shfl_xor(any, 16, 64);
            any |= __shfl_xor(any, 32, 64);
            if (group == 0) sStat[wave][rt * 16 + row16] = float2{m[rt], any ? l[rt] : -1.f};
#pragma unroll
            for (int db = 0; db < DB; ++db)
                *reinterpret_cast<f32x4_t*>(sV + ((rt * 16 + row16) * DP + ((db * 16 + 4 * group) ^ ((row16 & 7) * 4))) * 4) = o[rt][db];
        }
        __syncthreads();
        for (int item = tid; item < ROWS * (DP / 4); item += CF_NW * 64) {
            const int row = item / (DP / 4), e = item % (DP / 4) * 4, r = u.first_row + row;
            if (r >= rows || e >= b.cache.d) continue;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < CF_NW; ++w) top = fmaxf(top, sStat[w][row].y == -1.f ? -INFINITY : sStat[w][row].x);
            float sum = 0.f;
            bool any = false;
            f32x4_t acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < CF_NW; ++w) {
                const float2 st = sStat[w][row];
                if (st.y == -1.f) continue;
                any = true;
                const float c = st.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((st.x - top) * b.scale2);
                sum += c * st.y;
                const f32x4_t x = *reinterpret_cast<const f32x4_t*>(sBuf[w] + (row * DP + (e ^ ((row & 7) * 4))) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] += c * x[i];
            }
            if (piece.slot >= 0) {
                const int64_t at = (int64_t)piece.slot * ROWS + row;
                if (e == 0) b.stat[at] = float2{top, any ? sum : -1.f};
                *reinterpret_cast<f32x4_t*>(b.part + at * b.cache.d + e) = acc;
            } else {
                const float inv = any ? 1.f / sum : 0.f;
                const int qi = r / FastDiv{b.by_share.mul, b.by_share.shift}, hq = u.head * b.share + r - qi * b.share;
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(b.o) + (int64_t)(u.row0 + qi) * b.o_row + hq * b.o_head + e) =
                    uint2{pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv)};
            }
        }
        __syncthreads();
    }
#endif
}

// ---- many rows -----------------------------------------------------------------------------------------------------
template <bool BF16, int NB, bool MX4>
__global__ __launch_bounds__(CM_NW * 64, 2) void k_cached_many(CachedArgs) {
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int DP = NB * 32, KS = DP / 16, DB = NB, TILE = CM_KEYS * DP * 2, NT = CM_NW * 64;
    static_assert(CM_KEYS == 16 * CM_NW, "a wave loads 16 of a tile's keys");
    __shared__ __attribute__((aligned(16))) char sK0[TILE], sK1[TILE], sV0[TILE], sV1[TILE];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
    uint32_t from, to;
    {
        const Line line = make_line<CM_ROWS, CM_KEYS>(*reread_args());
        from = line.cut(blockIdx.x), to = line.cut(blockIdx.x + 1);
    }
    if (from >= to) {
        if (threadIdx.x == 0) reread_args()->join[blockIdx.x].cut = 0;
        return;
    }
    constexpr float LAG = BF16 ? 8.f : 4.f, LIFT = BF16 ? 0.f : 11.f, FAR = 1024.f;

    while (from < to) {
        const auto& a = *reread_args();
        const Line line = make_line<CM_ROWS, CM_KEYS>(a);      // (made anew: kept it would take seven registers of the loop's)
        const CachedUnit u = find_unit<CM_ROWS, CM_KEYS>(a, line, from);
        const CachedPiece piece = cut_unit(u, from, to, blockIdx.x);
        if (u.end >= to) tell_join<CM_ROWS>(a, u, line, to, blockIdx.x, from <= u.begin);
        from = u.end;
        const int rows = u.lq * a.share, lk = u.lk, causal = a.causal;
        const FastDiv by_share{a.by_share.mul, a.by_share.shift};
        const int t0 = piece.t0, t1 = piece.t1;
        // (what the loop needs)
        const int page_bits = a.cache.page_bits, page_mask = (1 << page_bits) - 1, pool = a.cache.pages, d = a.cache.d;
        const int64_t page_bytes = a.cache.page_bytes;
        const float scale2 = a.scale2;
        // rows past the sample's last are copies of it that are not stored
        auto query = [&](int r) __attribute__((always_inline)) { return min(r, rows - 1) / by_share; };
        auto limit = [&](int r) __attribute__((always_inline)) { return cached_limit(causal, u.lq, lk, query(r)); };
        const int lim = limit(u.first_row + wave * 32 + r32), wave_end = limit(u.first_row + wave * 32 + 31);
        // Q^T operand: d = 16 ks + 8 h .. + 7 of the lane's row
        u32x4_t qf[KS];
        {
            const int r = min(u.first_row + wave * 32 + r32, rows - 1), qi = r / by_share, hq = u.head * a.share + r - qi * a.share;
            const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (int64_t)(u.row0 + qi) * a.q_row + hq * a.q_head;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                qf[ks] = ks * 16 + h * 8 < d ? *reinterpret_cast<const u32x4_t*>(qp + ks * 16 + h * 8) : u32x4_t{0, 0, 0, 0};
        }
        // Whether all of the piece's pages are the pool's (else every tile is looked at key by key).
        const int32_t* const pages = a.cache.table + (int64_t)u.sample * a.cache.max_pages;
        bool sound = true;
        const int end_key = min(t1 * CM_KEYS, lk);
        for (int p = ((t0 * CM_KEYS) >> page_bits) + threadIdx.x; (int64_t)p << page_bits < end_key; p += NT) sound &= (unsigned)pages[p] < (unsigned)pool;
        sound = __syncthreads_and(sound);

        // A wave's 16 keys of a tile: their page (-1: none) by a scalar load, a lane's pieces of them. Keys past the sample's last,
        // and those of no page, are zeros.
        // 4-bit codes wait in registers, a tile more ahead than 16-bit values, which go straight into LDS (16 bytes a lane, each
        // from the piece that belongs in its place; what is out of the buffer's range reads as zeros).
        struct Raw {
            u32x4_t x;
            uint32_t p;
        };
        const auto table = (const __attribute__((address_space(4))) int32_t*)pages;
        const uint8_t* const head = a.cache.data + u.head * a.cache.head_bytes;
        const int row_bytes = MX4 ? 16 * NB : d * 2;
        const int in = lane / NB, at_piece = lane % NB;
        auto page_of = [&](int tile) __attribute__((always_inline)) {
            const int key = __builtin_amdgcn_readfirstlane(tile * CM_KEYS + wave * 16);
            return key < lk && tile < t1 ? table[key >> page_bits] : -1;
        };
        auto load = [&](int tile, int page, int side, Raw& w) __attribute__((always_inline)) {
            w.x = u32x4_t{0, 0, 0, 0};
            w.p = 0;
            if ((unsigned)page >= (unsigned)pool) return;
            const int key = tile * CM_KEYS + wave * 16, slot = key & page_mask;
            if (lane < 16 * NB && in < lk - key) {
                w.x = *reinterpret_cast<const u32x4_t*>(head + page * page_bytes + ((side << page_bits) + slot) * (16 * NB) + lane * 16);
                w.p = head[page * page_bytes + (32 * NB << page_bits) + ((side << page_bits) + slot) * NB + lane];
            }
        };
        // Into LDS, as 16-bit values. (Places that differ in a few bits are formed where they are used: registers.)
        auto put = [&](const Raw& w, int side, char* s) __attribute__((always_inline)) {
            int to = side ? cv_piece<DP>(in, at_piece * 4) : k_piece<DP>(in, at_piece * 4);
            asm volatile("" : "+v"(to));
            const float scale = mx_scale(w.p);
            if (NB == 4 || lane < 16 * NB) {
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x4_t*>(s + wave * 16 * DP * 2 + (to ^ (j * 16))) = widen4<BF16>(w.x[j], scale);
            }
        };
        auto stage = [&](int tile, int page, int side, char* s) __attribute__((always_inline)) {
            constexpr int P = DP / 8, NOWHERE = 1 << 30;
            const int key = tile * CM_KEYS + wave * 16, slot = key & page_mask, left = (unsigned)page < (unsigned)pool ? min(16, lk - key) : 0;
            const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(head + (left ? page : 0) * page_bytes + ((side << page_bits) + slot) * row_bytes), (short)0,
                                                                left * row_bytes, 0x00027000);
            int from_lane = lane;
            asm volatile("" : "+v"(from_lane));
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int at = i * 64 + from_lane, k = at / P, p = (side ? cv_piece<DP>(k, at % P) : k_piece<DP>(k, at % P)) / 16 % P;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(s + wave * 16 * DP * 2 + i * 1024), 16,
                                                         p * 8 < d ? k * row_bytes + p * 16 : NOWHERE, 0, 0, 0);
            }
        };
        f32x16_t o[DB];
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = f32x16_t{};
        float m = -INFINITY, l = 0.f, mc = -LIFT;      // maximum, sum, what the exponents are less by
        bool far = false, seen = false;

        // scores: s[kb][i] is key kb * 32 + 8 (i / 4) + 4 h + i % 4 of the tile
        // (operand places: of the first product, and what the others differ by)
        int k_from = k_piece<DP>(r32, h), v_from = cv_piece<DP>(4 * h + ((lane >> 2) & 3), ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1)) + (lane & 1) * 8;
        auto fresh = [&]() __attribute__((always_inline)) { asm volatile("" : "+v"(k_from), "+v"(v_from)); };
        auto k_operand = [&](const char* sK, int t) __attribute__((always_inline)) {
            const int q = t >> 1, at = DP == 96 ? (k_from ^ ((q & 1) * 32)) + (q >> 1) * 64 : k_from ^ (q * 32);
            return *reinterpret_cast<const u32x4_t*>(sK + at + (t & 1) * 32 * DP * 2);
        };
        auto scores = [&](const char* sK, f32x16_t (&s)[2]) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < 2 * KS; ++t) s[t & 1] = mfma32<BF16>(k_operand(sK, t), qf[t >> 1], t < 2 ? f32x16_t{} : s[t & 1]);
        };
        // (raise, near_top: as in the packed attention)
        auto raise = [&](float mt) __attribute__((always_inline)) {
            const float2 mh = both_halves(mt);
            mt = fmaxf(mh.x, mh.y);
            if (__any((mt - m) * scale2 > LAG)) {
                const float mn = fmaxf(m, mt);
                const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * scale2);
                m = mn;
                far = __any(fabsf(mn) * scale2 > FAR && mn != -INFINITY);
                mc = (far || mn == -INFINITY ? 0.f : mn * scale2) - LIFT;
                l *= corr;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[db][i] *= corr;
            }
        };
        auto near_top = [&](f32x16_t (&s)[2]) __attribute__((always_inline)) {
            if (__builtin_expect(!far, 1)) return;
            const float top = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[kb][i] -= top;
        };
        auto top_of = [&](const f32x16_t (&s)[2]) __attribute__((always_inline)) {
            float mt = s[0][0];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[kb][i]);
            return mt;
        };
        auto exponents = [&](f32x16_t (&s)[2], u32x4_t (&pf)[4]) __attribute__((always_inline)) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], scale2, -mc));
            float sum = 0.f;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    pf[ks][e] = pack2<BF16>(s[ks / 2][8 * (ks % 2) + 2 * e], s[ks / 2][8 * (ks % 2) + 2 * e + 1]);
                    sum = add2<BF16>(pf[ks][e], sum);
                }
            l += sum;
        };
        // V^T operand, as v_operand with this kernel's places
        auto values = [&](const char* sV, int ks, int db) __attribute__((always_inline)) {
            const char* const at = sV + (DP == 96 ? v_from + db * 64 : v_from ^ (db * 64)) + ks * 16 * DP * 2;
            const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)at);
            const s16x4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(at + 8 * DP * 2));
            const uint2 ux = __builtin_bit_cast(uint2, x), uy = __builtin_bit_cast(uint2, y);
            return u32x4_t{ux.x, ux.y, uy.x, uy.y};
        };
        // A tile that not every row of the workgroup sees whole.
        auto attend_masked = [&](int base, const char* sK, const char* sV) __attribute__((always_inline)) {
            f32x16_t s[2];
            u32x4_t pf[4];
            fresh();
            scores(sK, s);
            int held = 15;      // a bit for 16 keys
            if (!sound) {
                held = 0;
                for (int k = 0; k < 4; ++k) {
                    const int key = base + k * 16;
                    if (key < lk && (unsigned)pages[key >> page_bits] < (unsigned)pool) held |= 1 << k;
                }
            }
            const int left = lim - base - 4 * h;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const bool sees = kb * 32 + 8 * (i / 4) + i % 4 < left && (held >> (kb * 2 + i / 8) & 1);
                    seen |= sees;
                    s[kb][i] = sees ? s[kb][i] : -INFINITY;
                }
            raise(top_of(s));
            near_top(s);
            exponents(s, pf);
            // A probability of zero must not meet an Inf or a NaN of a key that its row does not see. Zero times V
            // shows whether there is one.
            bool odd = false;
            if (causal) {
                f32x16_t z = f32x16_t{};
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                    for (int db = 0; db < DB; ++db) z = mfma32<BF16>(values(sV, ks, db), u32x4_t{0, 0, 0, 0}, z);
                float t = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) t += z[i];
                odd = __any(t != t);
            }
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    u32x4_t vf = values(sV, ks, db);
                    if (odd) vf = finite_only<BF16>(vf);
                    o[db] = mfma32<BF16>(vf, pf[ks], o[db]);
                    if (db % 2 == 1 || DB == 1) __builtin_amdgcn_sched_barrier(0);      // (two operands at a time: registers)
                }
            if (odd) {      // the values left out, key by key, for the rows that see them
                for (int key = 0; key < CM_KEYS; ++key) {
                    float p = 0.f;
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if ((kb * 32 + 8 * (i / 4) + i % 4) == (key & ~4)) p = s[kb][i];
                    const float2 ph = both_halves(p);
                    p = key & 4 ? ph.y : ph.x;
                    const bool sees = base + key < lim;      // (a key of no page is zeros)
                    int from_e = 4 * h;
                    asm volatile("" : "+v"(from_e));
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int e = db * 32 + 8 * (i / 4) + from_e + i % 4;
                            const uint32_t b = *reinterpret_cast<const uint16_t*>(sV + cv_piece<DP>(key, e >> 3) + (e & 7) * 2);
                            if (sees && nonfinite16<BF16>(b)) o[db][i] += p * value16<BF16>(b);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                }
            }
        };
        // Whole tiles: the scores of the next tile are formed while the exponents of this one are, and its maximum while this one's
        // values are weighed; operands are read four products ahead. Two buffers each for K and V, K a tile ahead of V; in
        // registers both a tile further.
        const int all_see = sound ? limit(u.first_row) / CM_KEYS : 0;      // tiles that every row sees whole
        const int whole = min(t1, all_see);
        Raw wk, wv;
        int page1 = -1, page2 = -1, page3 = -1;      // of the tiles after the present one
        // Every wave's part of what has been on its way is in LDS, and none reads any more what was read before.
        auto landed = [&]() __attribute__((always_inline)) {
            if constexpr (!MX4) wait_loads();
            __syncthreads();
        };
        // K of the tile after next and V of the next into LDS; then the loads after them
        auto bring = [&](int tile, char* k_to, char* v_to) __attribute__((always_inline)) {
            if constexpr (MX4) {
                put(wk, 0, k_to);
                put(wv, 1, v_to);
                load(tile + 3, page3, 0, wk);
                load(tile + 2, page2, 1, wv);
                page2 = page3;
                page3 = page_of(tile + 4);
            } else {
                stage(tile + 2, page2, 0, k_to);
                stage(tile + 1, page1, 1, v_to);
                page1 = page2;
                page2 = page_of(tile + 3);
            }
        };
        auto step = [&](int tile, char* k_this, const char* k_next, const char* v_this, char* v_next, f32x16_t (&s)[2],
                        f32x16_t (&sn)[2]) __attribute__((always_inline)) {
            constexpr int AHEAD = NB == 4 ? 3 : 4, NK = 2 * KS, NV = 4 * DB;      // (four at width 128: registers spilled)
            u32x4_t pf[4], ring[AHEAD];
            float sum = 0.f;
            landed();
            bring(tile, k_this, v_next);
            fresh();
#pragma unroll
            for (int t = 0; t < AHEAD; ++t) ring[t] = k_operand(k_next, t);
#pragma unroll
            for (int t = 0; t < NK; ++t) {
                sn[t & 1] = mfma32<BF16>(ring[t % AHEAD], qf[t >> 1], t < 2 ? f32x16_t{} : sn[t & 1]);
                if (t + AHEAD < NK) ring[t % AHEAD] = k_operand(k_next, t + AHEAD);
                else ring[t % AHEAD] = values(v_this, (t + AHEAD - NK) / DB, (t + AHEAD - NK) % DB);
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
                o[t % DB] = mfma32<BF16>(ring[(NK + t) % AHEAD], pf[t / DB], o[t % DB]);
                if (t + AHEAD < NV) ring[(NK + t) % AHEAD] = values(v_this, (t + AHEAD) / DB, (t + AHEAD) % DB);
#pragma unroll
                for (int i = t * 32 / NV; i < (t + 1) * 32 / NV; ++i) mt = fmaxf(mt, sn[i / 16][i % 16]);
                __builtin_amdgcn_sched_barrier(0);
            }
            raise(mt);
            near_top(sn);
        };
        // on the way: K of the first two tiles and V of the first in LDS, and of 4 bits K of the third and V of the second in registers
        if (t0 < t1) {
            const int page0 = page_of(t0);
            page1 = page_of(t0 + 1);
            page2 = page_of(t0 + 2);
            if constexpr (MX4) {
                load(t0, page0, 0, wk);
                load(t0, page0, 1, wv);
                __syncthreads();        // (the last piece's rows have left LDS)
                put(wk, 0, sK0);
                put(wv, 1, sV0);
                load(t0 + 1, page1, 0, wk);
                put(wk, 0, sK1);
                load(t0 + 2, page2, 0, wk);
                load(t0 + 1, page1, 1, wv);
                page3 = page_of(t0 + 3);
            } else {
                __syncthreads();
                stage(t0, page0, 0, sK0);
                stage(t0, page0, 1, sV0);
                stage(t0 + 1, page1, 0, sK1);
            }
        }
        int tile = t0;
        bool second = false;
        if (tile < whole) {
            seen = true;
            f32x16_t s0[2], s1[2];
            landed();
            scores(sK0, s0);
            raise(top_of(s0));
            near_top(s0);
            for (; tile + 3 <= whole; tile += 2) {
                step(tile, sK0, sK1, sV0, sV1, s0, s1);
                step(tile + 1, sK1, sK0, sV1, sV0, s1, s0);
            }
            landed();
            bring(tile, sK0, sV1);
            u32x4_t pf[4];
            exponents(s0, pf);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int db = 0; db < DB; ++db) o[db] = mfma32<BF16>(values(sV0, ks, db), pf[ks], o[db]);
            ++tile;
            second = true;
        }
        // the others, a whole one among them at times
        for (; tile < t1; ++tile, second = !second) {
            landed();
            if (tile * CM_KEYS < wave_end) attend_masked(tile * CM_KEYS, second ? sK1 : sK0, second ? sV1 : sV0);
            __syncthreads();
            bring(tile, second ? sK1 : sK0, second ? sV0 : sV1);
        }
        if constexpr (!MX4) wait_loads();      // (none is on its way to LDS that the next piece uses)

        const auto& b = *reread_args();
        const int r = u.first_row + wave * 32 + r32;
        const float2 lh = both_halves(l);
        const float sum = lh.x + lh.y;
        const uint64_t some = __ballot(seen);
        const bool any = (some >> r32 & 1) || (some >> (r32 + 32) & 1);
        if (piece.slot >= 0) {
            if (r < rows) {
                const int64_t item = (int64_t)piece.slot * CM_ROWS + (r - u.first_row);
                if (h == 0) b.stat[item] = float2{m, any ? sum : -1.f};
                float* op = b.part + item * d;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int e = db * 32 + 8 * g + 4 * h;
                        if (any && e < d) *reinterpret_cast<f32x4_t*>(op + e) = f32x4_t{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
                    }
            }
            continue;
        }
        // Rows of out leave in 16-byte pieces, through the wave's piece of the K buffers.
        constexpr int P = DP / 8;
        const float inv = any ? 1.0f / sum : 0.f;
        char* sO = (wave < CM_NW / 2 ? sK0 : sK1) + wave % (CM_NW / 2) * (32 * DP * 2);
        __syncthreads();
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<uint2*>(sO + k_piece<DP>(r32, db * 4 + g) + h * 8) =
                    any ? uint2{pack2<BF16>(o[db][4 * g] * inv, o[db][4 * g + 1] * inv), pack2<BF16>(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv)} : uint2{0, 0};
#pragma unroll
        for (int i = 0; i < P / 2; ++i) {
            const int row = (i * 64 + lane) / P, p = (i * 64 + lane) % P, rr = u.first_row + wave * 32 + row;
            const u32x4_t x = *reinterpret_cast<const u32x4_t*>(sO + k_piece<DP>(row, p));
            if (rr >= rows || p * 8 >= d) continue;
            const int qr = rr / by_share, hr = u.head * b.share + rr - qr * b.share;
            *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(b.o) + (int64_t)(u.row0 + qr) * b.o_row + hr * b.o_head + p * 8) = x;
        }
    }
#endif
}

// ---- the pieces of units that were cut, joined -----------------------------------------------------------------------
// sum_s w_s (p v)_s / sum_s w_s (sum p)_s, w_s = exp(max_s - max), in an order that the pieces' number alone sets. Which units
// were cut only the device knows: every workgroup counts them, and takes its share of their rows (a launch of a workgroup
// for each place where one can be takes 10 to 30 us, nearly all of which leave at once).
constexpr int CJ_EACH = 3, CJ_MAX = CJ_EACH * 256;      // workgroups of the first launch, at most

template <bool BF16>
__device__ __forceinline__ void join_out(const CachedArgs& a, const JoinItem& j, int row, int e, bool seen, float sum, float (&acc)[8]) {
    const float inv = 1.f / sum;
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = seen ? acc[k] * inv : 0.f;
    const int r = j.first_row + row, qi = r / a.by_share, hq = j.head * a.share + r - qi * a.share;
    store8<BF16 ? TSP_BF16 : TSP_F16>(a.o, (int64_t)(j.row0 + qi) * a.o_row + hq * a.o_head + e, acc);
}

// Few pieces a unit: 16 / G rows at a time, G groups of 16 lanes a row (1, or 4: a wave), eight channels a lane.
template <bool BF16, int ROWS, int G>
__device__ __forceinline__ void join_rows(const CachedArgs& a, int g0, int cut, int first) {
    constexpr int BATCH = 8;
    const int group = threadIdx.x >> 4, g = group % G, e = (threadIdx.x & 15) * 8, mine = threadIdx.x % (G * 16);
    const JoinItem j = a.join[g0];
    const int row = first + group / G, pieces = (cut >> 8) - g0 + 1;
    const bool live = row < (cut & 255);
    auto at = [&](int i) { return (int64_t)(2 * (g0 + i) + (i == 0)) * ROWS + (live ? row : 0); };
    float2 st[BATCH];
    float x[BATCH][8];
    auto load = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int i = i0 + b * G;
            st[b] = i < pieces ? a.stat[at(i)] : float2{-INFINITY, -1.f};
            if (i < pieces && e < a.cache.d) load8<TSP_F32>(a.part, at(i) * a.cache.d + e, x[b]);
        }
    };
    load(g);      // (on their way while the largest maximum is found)
    float top = -INFINITY;
    for (int i = mine; i < pieces; i += G * 16) {
        const float2 one = a.stat[at(i)];
        if (one.y != -1.f) top = fmaxf(top, one.x);
    }
#pragma unroll
    for (int o = G == 1 ? 8 : 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    float sum = 0.f, acc[8] = {};
    bool any = false;
    for (int i0 = g; i0 < pieces; i0 += BATCH * G) {
        if (i0 >= BATCH * G) load(i0);
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            if (st[b].y == -1.f) continue;
            any = true;
            const float c = st[b].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((st[b].x - top) * a.scale2);
            sum += c * st[b].y;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += c * x[b][k];
        }
    }
    int seen = any;
    if constexpr (G == 4) {
        sum += __shfl_xor(sum, 16, 64), seen |= __shfl_xor(seen, 16, 64);
        sum += __shfl_xor(sum, 32, 64), seen |= __shfl_xor(seen, 32, 64);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            acc[k] += __shfl_xor(acc[k], 16, 64);
            acc[k] += __shfl_xor(acc[k], 32, 64);
        }
    }
    if (live && g == 0 && e < a.cache.d) join_out<BF16>(a, j, row, e, seen, sum, acc);
}

// Many pieces a unit: 32 channels of a row at a time, 64 groups of four lanes.
struct JoinShared {
    float weight[CJ_MAX], acc[4][32], top[4], sum[4];
};
template <bool BF16, int ROWS>
__device__ __forceinline__ void join_many(const CachedArgs& a, int g0, int cut, int row, int part, JoinShared& s) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, e = part * 32 + (lane & 3) * 8;
    const JoinItem j = a.join[g0];
    const int pieces = (cut >> 8) - g0 + 1;
    auto at = [&](int i) { return (int64_t)(2 * (g0 + i) + (i == 0)) * ROWS + row; };
    constexpr int BATCH = 4;
    float2 st[CJ_EACH];
    float x[BATCH][8];
    auto load = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
            if (i0 + b * 64 < pieces && e < a.cache.d) load8<TSP_F32>(a.part, at(i0 + b * 64) * a.cache.d + e, x[b]);
    };
    load(threadIdx.x >> 2);      // (on their way while the weights are formed)
    float top = -INFINITY, sum = 0.f;
    bool any = false;
#pragma unroll
    for (int i = 0; i < CJ_EACH; ++i) {
        const int p = i * 256 + threadIdx.x;
        st[i] = p < pieces ? a.stat[at(p)] : float2{-INFINITY, -1.f};
        if (st[i].y != -1.f) top = fmaxf(top, st[i].x), any = true;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (lane == 0) s.top[wave] = top;
    const bool seen = __syncthreads_or(any);
    top = fmaxf(fmaxf(s.top[0], s.top[1]), fmaxf(s.top[2], s.top[3]));
#pragma unroll
    for (int i = 0; i < CJ_EACH; ++i) {
        const int p = i * 256 + threadIdx.x;
        if (p >= pieces) break;
        const float c = st[i].y == -1.f ? -1.f : st[i].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((st[i].x - top) * a.scale2);
        s.weight[p] = c;
        if (c != -1.f) sum += c * st[i].y;
    }
    sum = group_sum<64>(sum);
    if (lane == 0) s.sum[wave] = sum;
    __syncthreads();
    sum = (s.sum[0] + s.sum[1]) + (s.sum[2] + s.sum[3]);
    float acc[8] = {};
    if (e < a.cache.d) {
        for (int i0 = threadIdx.x >> 2; i0 < pieces; i0 += BATCH * 64) {
            if (i0 >= BATCH * 64) load(i0);
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const float c = i0 + b * 64 < pieces ? s.weight[i0 + b * 64] : -1.f;
                if (c == -1.f) continue;
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[k] += c * x[b][k];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
        for (int o = 4; o < 64; o <<= 1) acc[k] += __shfl_xor(acc[k], o, 64);
        if (lane < 4) s.acc[wave][lane * 8 + k] = acc[k];
    }
    __syncthreads();
    if (threadIdx.x < 4 && e < a.cache.d) {
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = (s.acc[0][lane * 8 + k] + s.acc[1][lane * 8 + k]) + (s.acc[2][lane * 8 + k] + s.acc[3][lane * 8 + k]);
        join_out<BF16>(a, j, row, e, seen, sum, acc);
    }
}

// G: 1 or 4 groups of lanes a row, 64 of join_many.
template <bool BF16, int ROWS, int G>
__global__ __launch_bounds__(256) void k_cached_join(CachedArgs a) {
    __shared__ JoinShared s;
    __shared__ int sCount[CJ_EACH * 4], sFound[3];
    const int wave = threadIdx.x >> 6, blocks = a.cache.blocks;
    int cut[CJ_EACH], count[CJ_EACH], end[CJ_EACH];
#pragma unroll
    for (int i = 0; i < CJ_EACH; ++i) {
        const int w = i * 256 + threadIdx.x;
        cut[i] = w < a.groups ? a.join[w].cut : 0;
        const int rows = cut[i] & 255;
        count[i] = G == 64 ? rows * blocks : (rows + 16 / G - 1) / (16 / G);
    }
#pragma unroll
    for (int i = 0; i < CJ_EACH; ++i) {
        end[i] = (int)scan64((uint32_t)count[i]);
        if ((threadIdx.x & 63) == 63) sCount[i * 4 + wave] = end[i];
    }
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < CJ_EACH * 4; ++i) {
        const int c = sCount[i];
#pragma unroll
        for (int k = 0; k < CJ_EACH; ++k)
            if (i < k * 4 + wave) end[k] += c;
        total += c;
    }
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
#pragma unroll
        for (int i = 0; i < CJ_EACH; ++i)
            if (item < end[i] && item >= end[i] - count[i]) sFound[0] = i * 256 + threadIdx.x, sFound[1] = item - (end[i] - count[i]), sFound[2] = cut[i];
        __syncthreads();
        const int g0 = sFound[0], x = sFound[1];
        if constexpr (G == 64) join_many<BF16, ROWS>(a, g0, sFound[2], x / blocks, x % blocks, s);
        else join_rows<BF16, ROWS, G>(a, g0, sFound[2], x * (16 / G));
        __syncthreads();
    }
}

static_assert(CJ_MAX >= 768 && CM_ROWS < 256, "the join counts every workgroup, and its items hold a unit's rows");

constexpr float kLog2e = 1.44269504088896340736f;

// What a call may have: heads; keys a sample; (query, head of the group) pairs; units (cached_cut's numbers fit 64 bits up to it).
constexpr int kMostHeads = 4096;
constexpr int64_t kKeysEnd = (1ll << 31) - (1ll << 16), kRowsEnd = (1ll << 31) - 1024, kUnitsEnd = 1ll << 29;

// How a call is cut: the rows of a unit, the workgroups. Few rows are those that fit a unit of 32 in the mean (the host
// does not know the lengths). A batch of single tokens and a prompt is cut as its mean asks, and one of the two suffers: 255 tokens on
// 1,000 keys each with 2,000 rows on 2,000 keys, 8 heads on 8 of 128, take 1,578 us together (the prompt by 16 rows a unit) and 80 and 52
// as two calls; 16 heads on 4, 205 (the tokens by 128 rows a unit), 47 and 64; 63 tokens on 4,000, 2,000 rows on 20,000: 394, 37 and 337.
struct CachedCut {
    int rows, groups, least, finer, coarser;
    int64_t units;      // at most (kUnitsEnd and more: nothing else is known)
    int join;           // groups of lanes a row in the join
    unsigned joins;     // its workgroups
};
CachedCut cached_cut(int64_t nq, int samples, int hkv, int share, int64_t keys, int d, bool mx4) {
    CachedCut c{};
    const int64_t each = ceil_div(nq, samples) * share;
    c.rows = each <= 16 ? 16 : each <= 32 && mx4 ? 32 : CM_ROWS;      // (two tiles of rows beside 16-bit keys would spill registers)
    c.units = (ceil_div(nq * share, c.rows) + (samples > 1 ? samples : 0)) * hkv;
    if (c.units >= kUnitsEnd) return c;
    // The line is shorter than 2^30. Weights of many rows' units are in 64ths of a tile where that allows it: a causal
    // prompt's grow by less than a tile from one to the next (8,000 rows to themselves: 678 us in whole tiles).
    const int64_t tiles = ceil_div(keys, c.rows == CM_ROWS ? CM_KEYS : CF_KEYS);
    c.finer = c.rows == CM_ROWS ? 6 : 0;
    c.coarser = 0;
    auto longest = [&]() { return c.units * (((tiles << c.finer) >> c.coarser) + 1); };
    while (c.finer > 0 && (longest() >= 1ll << 30 || tiles << c.finer >= 1ll << 30)) --c.finer;
    while (c.coarser < 30 && longest() >= 1ll << 30) ++c.coarser;
    c.least = std::max(1, ((c.rows == CM_ROWS ? 4 : 2 * CF_NW) << c.finer) >> c.coarser);
    // two or three a CU, as registers and LDS allow, where the line can be that long
    c.groups = longest() <= c.least ? 1 : (int)std::min<int64_t>(c.rows == 16 ? 768 : 512, ceil_div(longest() << c.coarser, 1ll << c.finer));
    const int64_t cut = std::min<int64_t>(c.units, c.groups), pieces = c.groups / (std::max<int64_t>(ceil_div(nq * share, c.rows), std::min<int64_t>(samples, nq)) * hkv);
    const int64_t rows = std::min<int64_t>(each, c.rows);
    // (64 where its workgroups are few: 1 row on 200,000 keys 40 us by waves, 25 so; 256 rows of 4 heads on 20,000 45 and 55)
    const int64_t wide = cut * rows * ((d + 31) / 32);
    c.join = pieces > 32 && wide <= 2048 ? 64 : pieces > 2 ? 4 : 1;
    c.joins = (unsigned)std::min<int64_t>(c.join == 64 ? wide : cut * ceil_div(rows, 16 / c.join), 2048);
    return c;
}
size_t cached_workspace(const CachedCut& c, int d) {
    return (size_t)c.groups * (2 * c.rows * (d * sizeof(float) + sizeof(float2)) + sizeof(JoinItem));
}

}  // namespace
}  // namespace tsp

using namespace tsp;

extern "C" size_t tsp_attention_cached_workspace_bytes(int64_t nq, int samples, int hq, const tsp_kv_cache* cache, int max_pages) {
    if (!cache || !kv_valid(*cache) || nq <= 0 || nq >= (1ll << 31) || samples <= 0 || hq <= 0 || hq > kMostHeads || hq % cache->heads ||
        max_pages <= 0 || (int64_t)max_pages * cache->page >= kKeysEnd || nq * (hq / cache->heads) >= kRowsEnd)
        return 0;
    return cached_workspace(cached_cut(nq, samples, cache->heads, hq / cache->heads, (int64_t)max_pages * cache->page, cache->d,
                                       cache->format == TSP_KV_MX4), cache->d);
}

extern "C" int tsp_attention_cached(const tsp_heads* q, int dtype, int64_t nq, int hq, const tsp_kv_cache* cache, const int32_t* d_offsets,
                                    int samples, const int32_t* d_table, int max_pages, const int32_t* d_lengths, float scale, int causal,
                                    const tsp_heads* out, void* d_workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    TSP_REQUIRE(cache, TSP_ERR_INVALID, "tsp_attention_cached: null cache");
    const tsp_kv_cache& c = *cache;
    TSP_REQUIRE(kv_valid(c), TSP_ERR_UNSUPPORTED, "tsp_attention_cached: a cache of %lld pages of %d tokens, %d heads of %d, format %d",
                (long long)c.pages, c.page, c.heads, c.d, c.format);
    TSP_REQUIRE(dtype == TSP_F16 || dtype == TSP_BF16, dtype == TSP_F32 ? TSP_ERR_UNSUPPORTED : TSP_ERR_INVALID,
                "tsp_attention_cached: heads must be f16 or bf16");
    TSP_REQUIRE(c.format == TSP_KV_MX4 || c.format == dtype, TSP_ERR_UNSUPPORTED, "tsp_attention_cached: a 16-bit cache has the heads' dtype");
    TSP_REQUIRE(nq >= 0 && nq < (1ll << 31), TSP_ERR_INVALID, "tsp_attention_cached: nq=%lld out of range", (long long)nq);
    TSP_REQUIRE(hq > 0 && hq % c.heads == 0 && hq <= kMostHeads, TSP_ERR_INVALID, "tsp_attention_cached: %d heads on %d", hq, c.heads);
    TSP_REQUIRE(samples > 0 && (samples == 1 || d_offsets), TSP_ERR_INVALID, "tsp_attention_cached: samples=%d (without offsets: 1)", samples);
    TSP_REQUIRE(max_pages > 0 && (int64_t)max_pages * c.page < kKeysEnd, TSP_ERR_INVALID, "tsp_attention_cached: max_pages=%d", max_pages);
    TSP_REQUIRE(std::isfinite(scale * kLog2e) && scale > 0.f, TSP_ERR_INVALID, "tsp_attention_cached: scale=%g", scale);
    if (nq == 0) return TSP_OK;
    TSP_REQUIRE(q && out && q->data && out->data && d_table && d_lengths && (c.data || c.pages == 0), TSP_ERR_INVALID,
                "tsp_attention_cached: null pointer");
    TSP_REQUIRE(heads_aligned(*q) && heads_aligned(*out) && reinterpret_cast<uintptr_t>(c.data) % 16 == 0, TSP_ERR_INVALID,
                "tsp_attention_cached: data must be 16-byte aligned, strides multiples of 8 (a row's up to 2^20)");
    TSP_REQUIRE(heads_apart(*out, nq, hq, c.d), TSP_ERR_INVALID, "tsp_attention_cached: the output's heads overlap");
    // (an out that lies over q at an offset, for instance, would be written by one workgroup before another has read it)
    const Runs o_runs = runs_of(*out, nq, hq, c.d, 2), q_runs = runs_of(*q, nq, hq, c.d, 2);
    const Runs read[4] = {runs_of(c.data, kv_head_bytes(c) * c.heads * c.pages), runs_of(d_table, 4ll * samples * max_pages),
                          runs_of(d_lengths, 4ll * samples), runs_of(d_offsets, 4ll * (samples + 1ll))};
    bool alias = meet(o_runs, q_runs);
    for (const Runs& r : read) alias |= meet(o_runs, r);
    TSP_REQUIRE(!alias, TSP_ERR_INVALID, "tsp_attention_cached: out must not alias q, the cache, table, lengths or offsets");
    const int share = hq / c.heads;
    TSP_REQUIRE(nq * share < kRowsEnd, TSP_ERR_INVALID, "tsp_attention_cached: too many rows");
    const CachedCut cut = cached_cut(nq, samples, c.heads, share, (int64_t)max_pages * c.page, c.d, c.format == TSP_KV_MX4);
    TSP_REQUIRE(cut.units < kUnitsEnd, TSP_ERR_INVALID, "tsp_attention_cached: too many rows and heads");
    const size_t need = cached_workspace(cut, c.d);
    TSP_REQUIRE(d_workspace, TSP_ERR_INVALID, "tsp_attention_cached: null workspace");
    TSP_REQUIRE(workspace_bytes >= need, TSP_ERR_WORKSPACE, "tsp_attention_cached: workspace of %zu bytes, needs %zu", workspace_bytes, need);
    TSP_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0, TSP_ERR_INVALID, "tsp_attention_cached: workspace not 16-byte aligned");
    const Runs ws_runs = runs_of(d_workspace, (int64_t)need);
    alias = meet(ws_runs, o_runs) || meet(ws_runs, q_runs);
    for (const Runs& r : read) alias |= meet(ws_runs, r);
    TSP_REQUIRE(!alias, TSP_ERR_INVALID, "tsp_attention_cached: the workspace overlaps another tensor of the call");
    float* part = static_cast<float*>(d_workspace);
    float2* stat = reinterpret_cast<float2*>(part + (size_t)cut.groups * 2 * cut.rows * c.d);
    const CachedArgs a{q->data, out->data, q->row_stride, q->head_stride, out->row_stride, out->head_stride, kv_args(c, d_table, max_pages, d_lengths),
                       d_offsets, nq, samples, share, causal ? 1 : 0, cut.groups, cut.least, cut.finer, cut.coarser, fast_div((uint32_t)share),
                       fast_div((uint32_t)cut.groups), scale * kLog2e, part, stat,
                       reinterpret_cast<JoinItem*>(stat + (size_t)cut.groups * 2 * cut.rows)};
    hipStream_t s = as_stream(stream);
    auto go = [&](auto bf, auto nb, auto mx) {
        constexpr bool BF16 = decltype(bf)::value, MX4 = decltype(mx)::value;
        constexpr int NB = decltype(nb)::value;
        const dim3 grid((unsigned)cut.groups);
        if (cut.rows == 16) hipLaunchKernelGGL((k_cached_few<BF16, NB, MX4, 1>), grid, dim3(CF_NW * 64), 0, s, a);
        else if (MX4 && cut.rows == 32) hipLaunchKernelGGL((k_cached_few<BF16, NB, true, 2>), grid, dim3(CF_NW * 64), 0, s, a);
        else hipLaunchKernelGGL((k_cached_many<BF16, NB, MX4>), grid, dim3(CM_NW * 64), 0, s, a);
    };
    auto by_width = [&](auto bf, auto mx) {
        if (c.d <= 32) go(bf, std::integral_constant<int, 1>{}, mx);
        else if (c.d <= 64) go(bf, std::integral_constant<int, 2>{}, mx);
        else if (c.d <= 96) go(bf, std::integral_constant<int, 3>{}, mx);
        else go(bf, std::integral_constant<int, 4>{}, mx);
    };
    auto join = [&](auto bf, auto rows) {
        constexpr bool BF16 = decltype(bf)::value;
        constexpr int ROWS = decltype(rows)::value;
        if (cut.groups == 1) return;
        const dim3 grid(cut.joins), block(256);
        if (cut.join == 64) hipLaunchKernelGGL((k_cached_join<BF16, ROWS, 64>), grid, block, 0, s, a);
        else if (cut.join == 4) hipLaunchKernelGGL((k_cached_join<BF16, ROWS, 4>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((k_cached_join<BF16, ROWS, 1>), grid, block, 0, s, a);
    };
    auto by_type = [&](auto bf) {
        if (c.format == TSP_KV_MX4) by_width(bf, std::true_type{});
        else by_width(bf, std::false_type{});
        if (cut.rows == 16) join(bf, std::integral_constant<int, 16>{});
        else if (cut.rows == 32) join(bf, std::integral_constant<int, 32>{});
        else join(bf, std::integral_constant<int, CM_ROWS>{});
    };
    if (dtype == TSP_BF16) by_type(std::true_type{});
    else by_type(std::false_type{});
    TSP_CHECK_LAUNCH();
    return TSP_OK;
}
