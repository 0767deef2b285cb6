// The paged cache's layout and how a kernel finds a key in it.
//
// Pages are equal in size and hold `page` tokens of every key head, one head after another:
//   4 bits   K codes [page][16 B], V codes alike, K powers [page][B], V powers [page][B], B = ceil(d / 32)
//   16 bits  K [page][d], V [page][d]
// so that a head's keys of a page are whole runs of 16-byte pieces. Codes past d in a token's last block are zero.
// Key j of sample s lies in page table[s][j / page], slot j % page.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "mx.hpp"

namespace tsp {

constexpr int KV_MAX_D = 128;

struct KvArgs {
    uint8_t* data;
    const int32_t *table, *lengths;
    int64_t page_bytes, head_bytes;      // of a page, of a head in it
    int pages, max_pages;                // in the pool, columns of the table
    int page_bits, heads, d, blocks;     // page = 1 << page_bits tokens
};

// The bytes of key head `head` in the page that holds key j of sample s (0 <= j < max_pages * page), or NULL where
// the table names none of the pool's.
__device__ __forceinline__ uint8_t* kv_head(const KvArgs& a, int s, int64_t j, int head) {
    const int p = a.table[(int64_t)s * a.max_pages + (j >> a.page_bits)];
    return (unsigned)p < (unsigned)a.pages ? a.data + p * a.page_bytes + head * a.head_bytes : nullptr;
}

// Offsets in a head's bytes of a 4-bit cache: codes and power bytes of K (side 0) or V (side 1) at a slot.
__device__ __forceinline__ int kv_codes_at(const KvArgs& a, int side, int slot) { return ((side << a.page_bits) + slot) * 16 * a.blocks; }
__device__ __forceinline__ int kv_powers_at(const KvArgs& a, int side, int slot) {
    return (32 << a.page_bits) * a.blocks + ((side << a.page_bits) + slot) * a.blocks;
}

inline bool kv_valid(const tsp_kv_cache& c) {
    return c.pages >= 0 && c.pages < (1ll << 31) && c.page >= 16 && c.page <= 256 && (c.page & (c.page - 1)) == 0 && c.heads > 0 &&
           c.heads <= 4096 && c.d > 0 && c.d % 8 == 0 && c.d <= KV_MAX_D && (c.format == TSP_KV_MX4 || c.format == TSP_F16 || c.format == TSP_BF16);
}
inline int64_t kv_head_bytes(const tsp_kv_cache& c) {
    const int64_t blocks = (c.d + 31) / 32;
    return c.page * (c.format == TSP_KV_MX4 ? 34 * blocks : 4ll * c.d);
}
inline KvArgs kv_args(const tsp_kv_cache& c, const int32_t* table, int max_pages, const int32_t* lengths) {
    const int64_t head = kv_head_bytes(c);
    return KvArgs{static_cast<uint8_t*>(c.data), table, lengths, head * c.heads, head, (int)c.pages, max_pages, __builtin_ctz((unsigned)c.page),
                  c.heads, c.d, (c.d + 31) / 32};
}

// The sample of packed row `row` (offsets non-decreasing; n rows), its first row and rows: an L-ary search by the L
// lanes of a group, all of which get the same. False: the row is no sample's.
template <int L>
__device__ __forceinline__ bool row_sample(const int32_t* offsets, int samples, int n, int row, int& s, int& row0, int& rows) {
    s = 0;
    if (offsets) {
        const int lane = threadIdx.x % L, shift = (threadIdx.x & 63) / L * L;
        for (int span = samples; span > 0;) {       // the last sample that begins at row or before it
            const int step = (span - 1) / L + 1, i = lane * step;
            const bool before = i < span && offsets[s + i] <= row;
            const uint64_t mask = L == 64 ? ~0ull : (1ull << (L & 63)) - 1;
            const int c = __popcll((__ballot(before) >> shift) & mask);
            if (c == 0) return false;
            s += (c - 1) * step;
            span = step == 1 ? 0 : min(step, span - (c - 1) * step);
        }
    }
    row0 = offsets ? min(max(offsets[s], 0), n) : 0;
    rows = offsets ? max(min(offsets[s + 1], n), row0) - row0 : n;
    return row >= row0 && row < row0 + rows;
}

}  // namespace tsp
